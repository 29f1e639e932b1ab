// Rules on logits (repetition, frequency and presence penalties, biases,
// grammar masks), the greedy choice and its log-probability, in one pass.
//
// Every logit is read once, and written once where the adjusted row is wanted:
// HBM is the floor of a batch (64 rows of 256,206 f32 logits under every rule, the
// adjusted rows written too: 34.5 us, 3.8 TB/s, bound by barriers between the rules'
// phases and by issue slots), the launch and the merge of a single row (6.9 us). A row is cut over
// the CTAs of a cluster, which join their (maximum, sum of exponentials,
// index) through shared memory, so one launch needs no scratch and no atomics
// on global memory, and the merge order is fixed.
//
// The penalties and biases touch few tokens of a row. Each CTA marks those of
// its tile in a bitmap (one bit a token), whose running popcount gives each
// marked token a compact slot with its count and bias. The streaming pass
// leaves marked tokens out; a second, short pass goes over the slots.
#include <cooperative_groups.h>

#include "serving.cuh"
#include "sync.cuh"

namespace mgb {
namespace {

constexpr uint32_t kMaxTile = 32768;  // tokens of one bitmap
constexpr int kSlotBytes = 96 * 1024;  // shared memory for slots at most
constexpr uint32_t kNone = 0xffffffffu;

#define kPosInf __int_as_float(0x7f800000)
#define kLowest __int_as_float(0xff800000)
constexpr float kLog2e = 1.44269504088896341f, kLog2eRest = 1.92596299e-8f;  // their sum is log2 e to 48 bits

struct ChooseArgs {
    const void *x;
    long long stride;
    uint32_t vocab, tile, cap;  // cap: slots of a tile
    mgb_logit_rules rules;
    int32_t *ids;
    float *logp;
    void *y;
    long long y_stride;
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Running maximum m, its lowest index i, and the sum l of exp(y - m) over all
// logits but that one, whose own term is 1: the log-probability -log1p(l) keeps
// its relative precision where one token has nearly all of the weight.
struct Best {
    float m, l;
    uint32_t i;
};

// exp(m - top). It scales whole sums, so the rounding of its argument is made good:
// over a row of 250,000 logits that error (1e-6 of the sum) was what the result's was.
__device__ __forceinline__ float weight_of(float m, float top) {
    if (m == top) return 1.0f;
    const float d = m - top, h = d * kLog2e;
    if (!(h > -150.0f)) return 0.0f;
    const float rest = __fmaf_rn(d, kLog2e, -h) + d * kLog2eRest;
    return exp2_of(h) * __fmaf_rn(rest, 0.693147180559945f, 1.0f);
}

__device__ __forceinline__ Best merge(const Best &a, const Best &b) {
    const bool first = a.m > b.m || (a.m == b.m && a.i <= b.i);
    const float m = first ? a.m : b.m, w = weight_of(first ? b.m : a.m, m);
    // the loser's own term joins the sum, unless it has none
    const float own = (first ? b.i : a.i) == kNone ? 0.0f : 1.0f;
    return Best{m, first ? a.l + (own + b.l) * w : b.l + (own + a.l) * w, first ? a.i : b.i};
}

// All lanes' together: the maximum first, so that each sum is scaled once.
__device__ __forceinline__ Best join(const Best &a) {
    Best b = a;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b.m = fmaxf(b.m, __shfl_xor_sync(0xffffffffu, b.m, o));
    b.i = __reduce_min_sync(0xffffffffu, a.m == b.m ? a.i : kNone);
    // a lane's own term joins the sum, unless it has none or it is the maximum's
    b.l = ((a.i == kNone || a.i == b.i ? 0.0f : 1.0f) + a.l) * weight_of(a.m, b.m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b.l += __shfl_xor_sync(0xffffffffu, b.l, o);
    return b;
}

// N logits y (-inf where they do not count) at tokens `first` + place(e) into b.
template <int N, typename Place>
__device__ __forceinline__ void add(Best &b, const float (&y)[N], uint32_t first, Place place) {
    float top = y[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, y[e]);
    float own = 0.0f;  // the new maximum's own term, which the sum below would add
    if (top > b.m) {
        b.l = b.m == kLowest ? 0.0f : (1.0f + b.l) * weight_of(b.m, top);
        b.m = top;
#pragma unroll
        for (int e = N - 1; e >= 0; --e)
            if (y[e] == top) b.i = first + place(e);
        own = 1.0f;
    }
    if (b.m == kPosInf) {  // exp(inf - inf) counts as one
#pragma unroll
        for (int e = 0; e < N; ++e) b.l += y[e] == kPosInf ? 1.0f : 0.0f;
        b.l -= own;
    } else if (b.m > kLowest) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float w = exp2_of((y[e] - b.m) * kLog2e);
            s[e & 3] += own != 0.0f && b.i == first + place(e) ? 0.0f : w;
        }
        b.l += (s[0] + s[1]) + (s[2] + s[3]);
    }
}

template <int TYPE>
struct Num;  // logits of one type: 16-byte vectors of W numbers
template <>
struct Num<MGB_F32> {
    using T = float;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Num<MGB_F16> {
    using T = uint16_t;
    static __device__ __forceinline__ float get(uint16_t x) { return __half2float(__ushort_as_half(x)); }
    static __device__ __forceinline__ uint16_t put(float x) { return to_16(x, MGB_F16); }
};
template <>
struct Num<MGB_BF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ uint16_t put(float x) { return to_16(x, MGB_BF16); }
};

// Bits off .. off + 31 of a bit row of `words` words (off may be below 0).
__device__ __forceinline__ uint32_t bits_at(const uint32_t *row, uint32_t words, int64_t off) {
    const int64_t w = off >> 5;
    const uint32_t lo = w >= 0 && w < words ? row[w] : 0, hi = w + 1 >= 0 && w + 1 < words ? row[w + 1] : 0;
    return __funnelshift_r(lo, hi, (uint32_t)off & 31);
}

// THREADS of a CTA: 256, of which an SM holds four CTAs; 512 where all CTAs have
// an SM of their own, so that each has more in flight (one row of 256,206 tokens:
// 6.9 against 8.9 us).
template <int TYPE, bool RULES, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 4 : 1) choose_kernel(const ChooseArgs a) {
    constexpr int kThreads = THREADS, kWarps = kThreads / 32;
    constexpr int kPer = (kMaxTile / 32 + kThreads) / kThreads;  // words of a bit map a thread
    using N = Num<TYPE>;
    using T = typename N::T;
    constexpr int W = 16 / sizeof(T), UNROLL = 16 / W;
    extern __shared__ uint32_t smem[];
    __shared__ Best warp_best[kWarps];
    __shared__ Best cta_best[16];
    __shared__ uint32_t warp_sum[kWarps];
    const uint32_t parts = gridDim.x, part = blockIdx.x, row = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    begin();

    const mgb_logit_rules &r = a.rules;
    const T *x = reinterpret_cast<const T *>(a.x) + (size_t)row * a.stride;
    T *y = a.y ? reinterpret_cast<T *>(a.y) + (size_t)row * a.y_stride : nullptr;
    // the row's share of this CTA, in whole 64s
    const uint32_t share = ((a.vocab + parts - 1) / parts + 63) & ~63u;
    const uint32_t c0 = min(a.vocab, part * share), c1 = min(a.vocab, c0 + share);

    // Bit maps of the tile, bit i for the token at the tile's first 16-byte
    // boundary plus i, so that a vector's bits lie in one word.
    const uint32_t words = a.tile / 32 + 1;
    uint32_t *mark = smem, *off = mark + words, *rank = off + words;  // touched by a rule; ruled out by the grammar
    uint32_t *count = rank + words, *token = count + a.cap;
    float *bias = reinterpret_cast<float *>(token + a.cap);
    uint32_t nh = 0;
    const int32_t *hist = nullptr, *bias_ids = nullptr;
    const uint32_t *allow = nullptr;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if constexpr (RULES) {
        if (r.history) {
            hist = r.history + (size_t)row * r.history_stride;
            nh = r.history_len ? (uint32_t)min((long long)r.history_stride, (long long)max(0, r.history_len[row]))
                               : r.history_stride;
        }
        if (r.bias_count) bias_ids = r.bias_ids + (size_t)row * r.bias_count;
        if (r.repetition) rep = r.repetition[row];
        if (r.frequency) freq = r.frequency[row];
        if (r.presence) pres = r.presence[row];
        if (r.allow) {
            const int g = r.allow_row ? r.allow_row[row] : 0;
            if (g >= 0 && (uint32_t)g < r.allow_rows) allow = r.allow + (size_t)g * r.allow_stride;
        }
    }
    const bool slotted = nh || bias_ids;

    Best best{kLowest, 0.0f, kNone};
    for (uint32_t v0 = c0; v0 < c1; v0 += a.tile) {
        const uint32_t v1 = min(c1, v0 + a.tile), width = v1 - v0;
        const uint32_t shift = (uint32_t)(((uintptr_t)(x + v0) & 15) / sizeof(T));
        // vectors from the 16-byte boundary at or before v0; all but the first and last are whole
        const uint4 *vectors = reinterpret_cast<const uint4 *>(x + v0 - shift);
        const uint32_t nvec = (width + shift + W - 1) / W;
        const uint32_t whole0 = shift ? 1 : 0, whole1 = (width + shift) / W;
        uint4 raw[UNROLL];
        auto fetch = [&](uint32_t j0) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint32_t j = j0 + u * kThreads;
                if (j >= whole0 && j < whole1) raw[u] = __ldcs(vectors + j);
            }
        };
        fetch(tid);  // on their way while the bit maps are built
        uint32_t slots = 0;
        if constexpr (RULES) {
            for (uint32_t w = tid; w < words; w += kThreads) {
                mark[w] = 0;
                off[w] = allow ? ~bits_at(allow, r.allow_stride, (int64_t)v0 + 32 * w - shift) : 0u;
            }
            __syncthreads();
            if (slotted) {
                auto touch = [&](int32_t id) {
                    const uint32_t i = (uint32_t)id - v0;
                    if (i < width) atomicOr(&mark[(i + shift) >> 5], 1u << ((i + shift) & 31));
                };
                for (uint32_t i = tid; i < nh; i += kThreads) touch(hist[i]);
                for (uint32_t i = tid; i < r.bias_count; i += kThreads) touch(bias_ids[i]);
                __syncthreads();
                // rank[w]: touched tokens before word w; a thread has kPer words
                uint32_t pop[kPer], upto = 0;
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    pop[e] = kPer * tid + e < words ? __popc(mark[kPer * tid + e]) : 0;
                    upto += pop[e];
                }
                const uint32_t mine = upto;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += u;
                }
                if (lane == 31) warp_sum[warp] = upto;
                __syncthreads();
                uint32_t before = upto - mine;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    before += k < warp ? warp_sum[k] : 0;
                    slots += warp_sum[k];
                }
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    if (kPer * tid + e < words) rank[kPer * tid + e] = before;
                    before += pop[e];
                }
                for (uint32_t k = tid; k < slots; k += kThreads) {
                    count[k] = 0;
                    bias[k] = 0.0f;
                }
                __syncthreads();
                auto slot_of = [&](uint32_t i) {
                    const uint32_t bit = i + shift, k = rank[bit >> 5] + __popc(mark[bit >> 5] & ((1u << (bit & 31)) - 1));
                    token[k] = i;
                    return k;
                };
                for (uint32_t i = tid; i < nh; i += kThreads) {
                    const uint32_t at = (uint32_t)hist[i] - v0;
                    if (at < width) atomicAdd(&count[slot_of(at)], 1u);
                }
                // a warp an entry: the first entry of a token adds up all of them, in their order
                for (uint32_t i = warp; i < r.bias_count; i += kWarps) {
                    const int32_t id = bias_ids[i];
                    if ((uint32_t)id - v0 >= width) continue;
                    float sum = 0.0f;
                    bool first = true;
                    for (uint32_t j0 = 0; j0 < r.bias_count && first; j0 += 32) {
                        uint32_t same = __ballot_sync(0xffffffffu, j0 + lane < r.bias_count && bias_ids[j0 + lane] == id);
                        if (same && j0 + __ffs(same) - 1 < i) first = false;
                        for (; same && first; same &= same - 1) sum += r.bias[(size_t)row * r.bias_count + j0 + __ffs(same) - 1];
                    }
                    if (first && lane == 0) bias[slot_of((uint32_t)id - v0)] = sum;
                }
                __syncthreads();
            }
        }

        // streaming pass
        const bool y_vec = y && (((uintptr_t)(y + v0) & 15) / sizeof(T)) == shift;
        for (uint32_t j0 = tid; j0 < nvec; j0 += kThreads * UNROLL) {
            float f[UNROLL * W];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const uint32_t j = j0 + u * kThreads;
                uint32_t out_of = 0, touched = 0;  // bits of the vector
                if constexpr (RULES) {
                    const uint32_t w = (j * W) >> 5, s = (j * W) & 31;
                    if (j < nvec) {
                        touched = mark[w] >> s;
                        out_of = off[w] >> s;
                    }
                }
                T h[W];
                if (j >= whole0 && j < whole1) {
                    *reinterpret_cast<uint4 *>(h) = raw[u];
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const uint32_t o = j * W + e - shift;
                        h[e] = N::put(kLowest);
                        if (j < nvec && o < width) h[e] = x[v0 + o];
                    }
                }
                // touched tokens keep their logit until the second pass
                const uint32_t cut = out_of & ~touched;
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if ((cut >> e) & 1) h[e] = N::put(kLowest);
                if (y && j < nvec) {
                    if (y_vec && j >= whole0 && j < whole1) {
                        reinterpret_cast<uint4 *>(y + v0 - shift)[j] = *reinterpret_cast<const uint4 *>(h);
                    } else {
#pragma unroll
                        for (int e = 0; e < W; ++e)
                            if (j * W + e - shift < width) y[v0 + j * W + e - shift] = h[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    // fmax drops NaN
                    const float g = fmaxf(N::get(h[e]), kLowest);
                    f[u * W + e] = RULES && ((touched >> e) & 1) ? kLowest : g;
                }
            }
            fetch(j0 + kThreads * UNROLL);  // on its way during the sums
            add(best, f, v0 - shift + j0 * W, [](int e) { return (uint32_t)((e / W) * kThreads * W + e % W); });
        }
        if constexpr (RULES) {
            __syncthreads();
            for (uint32_t k = tid; k < slots; k += kThreads) {
                const uint32_t id = v0 + token[k], c = count[k];
                // a few numbers: in 64 bits and rounded once, since many occurrences make them large
                double d = N::get(x[id]);
                if (c) d = (d > 0.0 ? d / rep : d * rep) - ((double)freq * c + pres);
                if (bias_ids) d += bias[k];
                float f = (float)d;
                if (allow && !((allow[id >> 5] >> (id & 31)) & 1)) f = kLowest;
                if (y) y[id] = N::put(f);
                const Best one{fmaxf(f, kLowest), 0.0f, id};
                if (one.m > kLowest) best = merge(best, one);
            }
            __syncthreads();
        }
    }

    best = join(best);
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = join(lane < kWarps ? warp_best[lane] : Best{kLowest, 0.0f, kNone});
    }
    if (parts > 1) {
        namespace cg = cooperative_groups;
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the cluster runs
        if (tid == 0) *cg::this_cluster().map_shared_rank(&cta_best[part], 0) = best;
        cluster_sync();
        if (part != 0) return;
        if (warp == 0) {
            best = join(lane < parts ? cta_best[lane] : Best{kLowest, 0.0f, kNone});
        }
    }
    if (tid == 0) {
        const bool found = best.i != kNone;
        if (a.ids) a.ids[row] = found ? (int32_t)best.i : -1;
        // a sum below 2^-53 does not move 1 even in 64 bits
        if (a.logp) a.logp[row] = found ? (best.l < 1.1102230246251565e-16f ? 0.0f : -log1pf(best.l)) : kLowest;
    }
}

template <int TYPE, bool RULES, int THREADS>
cudaError_t launch(const ChooseArgs &a, uint32_t rows, uint32_t parts, int smem, cudaStream_t s) {
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = op_allow(choose_kernel<TYPE, RULES, THREADS>, kSlotBytes + (int)(kMaxTile / 32 + 1) * 12, true, done);
    if (e != cudaSuccess) return e;
    return op_launch(choose_kernel<TYPE, RULES, THREADS>, dim3(parts, rows), THREADS, smem, parts, a, s);
}

template <int TYPE>
cudaError_t launch(const ChooseArgs &a, bool ruled, bool wide, uint32_t rows, uint32_t parts, int smem, cudaStream_t s) {
    if (wide) return ruled ? launch<TYPE, true, 512>(a, rows, parts, smem, s) : launch<TYPE, false, 512>(a, rows, parts, smem, s);
    return ruled ? launch<TYPE, true, 256>(a, rows, parts, smem, s) : launch<TYPE, false, 256>(a, rows, parts, smem, s);
}

}  // namespace
}  // namespace mgb

extern "C" MGB_API mgb_status mgb_logits_choose(const void *logits, int type, int64_t row_stride, uint32_t rows,
                                                uint32_t vocab, const mgb_logit_rules *rules, int32_t *ids, float *logp,
                                                void *adjusted, int64_t adjusted_stride, void *stream) {
    using namespace mgb;
    static const char *op = "mgb_logits_choose";
    if (type < MGB_F32 || type > MGB_BF16) return op_fail(MGB_ERR_INVALID, op, "unknown number type");
    if (rows == 0) return MGB_OK;
    if (!logits) return op_fail(MGB_ERR_INVALID, op, "null logits");
    if (vocab == 0 || vocab > 0x7fffffffu) return op_fail(MGB_ERR_INVALID, op, "vocab out of range");
    if (rows > 65535) return op_fail(MGB_ERR_INVALID, op, "more than 65535 rows");
    const uintptr_t unit = type_size(type) - 1;
    if (((uintptr_t)logits | (uintptr_t)adjusted) & unit)
        return op_fail(MGB_ERR_INVALID, op, "logits are not aligned to their type");
    if (row_stride < 0 || (rows > 1 && row_stride < (int64_t)vocab) ||
        (adjusted && rows > 1 && adjusted_stride < (int64_t)vocab))
        return op_fail(MGB_ERR_INVALID, op, "rows overlap");
    ChooseArgs a{logits, row_stride, vocab, 0, 0, {}, ids, logp, adjusted, adjusted_stride};
    if (rules) a.rules = *rules;
    mgb_logit_rules &r = a.rules;
    if (r.bias_count && (!r.bias_ids || !r.bias)) return op_fail(MGB_ERR_INVALID, op, "null bias");
    if (r.allow && (uint64_t)r.allow_stride * 32 < vocab) return op_fail(MGB_ERR_INVALID, op, "grammar rows are too short");
    if (!r.repetition && !r.frequency && !r.presence) r.history = nullptr;
    if (!r.history) r.history_stride = 0;
    const bool ruled = r.history_stride || r.bias_count || r.allow;

    // A row is cut over 16 CTAs (the largest cluster), over fewer where they
    // would not all run at once (four an SM, 148 SMs), and never into shares
    // below 2048 tokens.
    uint32_t parts = 16;
    while (parts > 1 && ((uint64_t)rows * parts > 4 * 148 || (uint64_t)parts * 2048 > vocab + 2047ull)) parts /= 2;
    const uint32_t share = ((vocab + parts - 1) / parts + 63) & ~63u;
    a.tile = share < kMaxTile ? share : kMaxTile;
    const uint64_t entries = (uint64_t)r.history_stride + r.bias_count;
    auto cap = [&] { return (uint32_t)(entries < a.tile ? entries : a.tile); };
    while ((uint64_t)cap() * 12 > (uint64_t)kSlotBytes) a.tile = (a.tile / 2 + 63) & ~63u;
    a.cap = cap();
    const bool wide = (uint64_t)rows * parts <= 148;
    const int smem = ruled ? (int)((a.tile / 32 + 1) * 12 + a.cap * 12) : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    switch (type) {
        case MGB_F32: e = launch<MGB_F32>(a, ruled, wide, rows, parts, smem, s); break;
        case MGB_F16: e = launch<MGB_F16>(a, ruled, wide, rows, parts, smem, s); break;
        default: e = launch<MGB_BF16>(a, ruled, wide, rows, parts, smem, s); break;
    }
    return op_launch_status(e, op);
}
