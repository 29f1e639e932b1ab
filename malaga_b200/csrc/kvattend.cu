// Attention of new tokens over a paged K/V cache (f16, or 8-bit codes with a
// scale per row), from one token a sequence to long chunks.
//
// With K = c_k d_k and V = c_v d_v (codes and row scales; d = 1 for f16) a key
// j adds, to a row with running maximum m and sum l,
//     s_j = (q . c_k,j) * d_k,j * scale,  p_j = exp(s_j - m),
//     l += p_j,  o += (p_j d_v,j) c_v,j
// so the scales never touch the codes: both products run on the tensor cores in
// f16 (11 significant bits hold every code exactly) with f32 sums.
//
// Roundings to fewer than 32 bits, besides the output's:
//  * p d_v goes into its product as f16: 2^-11 relative, the size of one
//    rounding of a 16-bit output, and averaged over the keys. It is formed as
//    2^14 p (d_v 2^-E), E a running exponent of the largest d_v, so that f16's
//    narrow range costs nothing.
//  * q goes in as f16: exact for f16 q; bf16 q is first scaled by a power of
//    two per row, and then exact but for numbers 2^-38 of the row's largest.
//  * for f32 q both are split into a high and a low f16 part (SPLIT), two
//    products each, which keeps 22 bits.
#include <cooperative_groups.h>

#include "serving.cuh"
#include "sync.cuh"

namespace mgb {
namespace {

#define kLowest __int_as_float(0xff800000)
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kRaise = 14.0f;  // p is held as 2^14 p

struct AttendArgs {
    KvView kv;
    SeqView seq;
    const void *q;
    void *out;
    long long q_token, q_head, o_token, o_head;
    int q_type, o_type, causal;
    uint32_t group;  // query heads of a cache head
    float scale;     // times log2(e)
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float power_of_2(int e) { return e < -126 ? 0.0f : __int_as_float((e + 127) << 23); }

__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}

// Two codes (bytes sel of the word, each plus 128) as f16: 0x6400 + u is the
// f16 number 1024 + u.
__device__ __forceinline__ uint32_t codes2(uint32_t biased, uint32_t sel) {
    const uint32_t x = __byte_perm(biased, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&x), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// BYTES bytes at p (aligned to their size, at most 16) into words.
template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t *w) {
    if constexpr (BYTES == 16) {
        const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (BYTES == 8) {
        const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = x.x, w[1] = x.y;
    } else if constexpr (BYTES == 4) {
        w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    } else {
        w[0] = __ldg(reinterpret_cast<const uint16_t *>(p));
    }
}

// ---------------------------------------------------------------------------
// Few rows: 16 rows (token, head of the group) of one cache head a CTA.
//
// K and V go from global memory straight into the registers in which
// mma.m16n8k16 wants them, with 16-byte loads: the order of the head dimension
// inside q . k is free (Q is permuted the same way), and so is the order of the
// output's columns. For K, four lanes share a key and take every fourth vector
// of its row; for V, eight lanes share a key, and a byte permute pairs two keys.
// A warp takes blocks of BLOCK keys in turn and keeps its own maximum, sum and
// output; warps join in shared memory, the CTAs of a cluster (which cut the
// keys among them) through distributed shared memory, in a fixed order.

template <int D, bool Q8>
struct Frag {
    static constexpr int ESZ = Q8 ? 1 : 2;
    static constexpr int KB = D * ESZ / 4 < 16 ? D * ESZ / 4 : 16;  // bytes of a K load
    static constexpr int KN = D * ESZ / 4 / KB;                     // K loads of a key and lane
    static constexpr int VB = D * ESZ / 8 < 16 ? D * ESZ / 8 : 16;
    static constexpr int VN = D * ESZ / 8 / VB;
    static constexpr int KW = D * ESZ / 16, VW = D * ESZ / 32 ? D * ESZ / 32 : 1;  // words of a key and lane
    static constexpr int STEPS = D / 16, TILES = D / 8;
    // dim of element e of lane t's part of a K row, of lane g's part of a V row
    static __device__ __forceinline__ int k_dim(int t, int e) {
        constexpr int VE = KB / ESZ;
        return (t + 4 * (e / VE)) * VE + e % VE;
    }
    static __device__ __forceinline__ int v_dim(int g, int e) {
        constexpr int VE = VB / ESZ;
        return (g + 8 * (e / VE)) * VE + e % VE;
    }
};

template <int D, bool Q8>
struct Block {  // 16 keys of a warp in registers
    uint32_t k[2][Frag<D, Q8>::KW];
    uint32_t v[4][Frag<D, Q8>::VW];
    float ks[4], vs[4];  // scales of keys 2t, 2t+1, 2t+8, 2t+9
    bool hole;           // the table names no page of the cache
};

constexpr int kRowWarps = 8;

template <int D, bool Q8>
__device__ __forceinline__ void load_block(const AttendArgs &a, uint32_t head, uint32_t page, int key0, int end, int g,
                                           int t, Block<D, Q8> &blk) {
    using F = Frag<D, Q8>;
    const bool mapped = page < a.kv.pages;
    const size_t row = a.kv.row(mapped ? page : 0, head, (uint32_t)key0 & ((1u << a.kv.page_log2) - 1));
    const uint8_t *k = static_cast<const uint8_t *>(a.kv.k) + row * (D * F::ESZ);
    const uint8_t *v = static_cast<const uint8_t *>(a.kv.v) + row * (D * F::ESZ);
    const int left = mapped ? end - key0 : 0;  // keys of the block that exist; the others are read as zeros
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int key = g + 8 * u;
#pragma unroll
        for (int w = 0; w < F::KW; ++w) blk.k[u][w] = 0;
        if (key < left) {
#pragma unroll
            for (int c = 0; c < F::KN; ++c)
                load_words<F::KB>(k + (size_t)key * (D * F::ESZ) + (t + 4 * c) * F::KB, &blk.k[u][c * (F::KB / 4)]);
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int key = 2 * t + (u & 1) + 8 * (u >> 1);
#pragma unroll
        for (int w = 0; w < F::VW; ++w) blk.v[u][w] = 0;
        blk.ks[u] = blk.vs[u] = 0.0f;
        if (key < left) {
#pragma unroll
            for (int c = 0; c < F::VN; ++c)
                load_words<F::VB>(v + (size_t)key * (D * F::ESZ) + (g + 8 * c) * F::VB, &blk.v[u][c * (F::VB / 4)]);
            if constexpr (Q8) {
                blk.ks[u] = __ldg(a.kv.ks + row + key);
                blk.vs[u] = __ldg(a.kv.vs + row + key);
            }
        }
    }
    blk.hole = !mapped;
}

template <int D, bool Q8, bool SPLIT>
__global__ void __launch_bounds__(kRowWarps * 32) attend_rows_kernel(const AttendArgs a) {
    using F = Frag<D, Q8>;
    extern __shared__ __align__(16) uint8_t smem[];
    float *so = reinterpret_cast<float *>(smem);                 // [warps][16][D]
    __half *sq = reinterpret_cast<__half *>(smem);               // [SPLIT + 1][16][D], before so is used
    __shared__ float row_scale[16], wm[kRowWarps][16], wl[kRowWarps][16];
    __shared__ float cm[16], cl[16];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t parts = gridDim.x, part = blockIdx.x, heads = a.kv.heads;
    const uint32_t head = blockIdx.y % heads, b = blockIdx.z;
    int n;
    const int t0 = a.seq.first(b, n);
    const int len = a.seq.length(b, a.kv.page_log2), stand = a.seq.kv_len[b] - n;  // position of the first new token
    const int32_t *table = a.seq.table + (size_t)b * a.seq.table_stride;
    const long long rows = (long long)n * a.group;
    // keys that token i sees
    auto limit = [&](int i) { return a.causal ? max(0, min(len, stand + i + 1)) : len; };

    for (long long r0 = (long long)(blockIdx.y / heads) * 16; r0 < rows; r0 += (long long)(gridDim.y / heads) * 16) {
        // Q: 16 threads a row; the row's largest number to just below 2^14 (f16 q stays as it is)
        {
            const int r = tid >> 4, c = tid & 15;
            const long long rr = r0 + r;
            constexpr int E = D / 16;
            float x[E], m = 0.0f;
            const int i = (int)(rr / a.group), h = (int)(rr - (long long)i * a.group);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = rr < rows ? load1(a.q, (size_t)((t0 + i) * a.q_token + (long long)(head * a.group + h) * a.q_head) + c * E + e,
                                         a.q_type)
                                 : 0.0f;
                m = fmaxf(m, fabsf(x[e]));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            int shift = 0;
            if (a.q_type != MGB_F16 && m > 0.0f && m < __int_as_float(0x7f800000)) shift = 13 - ilogbf(m);
            // 2^shift in two factors, since either may leave the range of f32 alone
            const int s1 = max(-100, min(100, shift)), s2 = shift - s1;
            const float f1 = __int_as_float((127 + s1) << 23), f2 = __int_as_float((127 + s2) << 23);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float y = x[e] * f1 * f2;
                const __half hi = __float2half_rn(y);
                sq[r * D + c * E + e] = hi;
                if constexpr (SPLIT) sq[16 * D + r * D + c * E + e] = __float2half_rn(y - __half2float(hi));
            }
            if (c == 0) row_scale[r] = a.scale * __int_as_float((127 - s1) << 23) * __int_as_float((127 - s2) << 23);
        }
        __syncthreads();
        uint32_t q[SPLIT ? 2 : 1][F::STEPS][4];
#pragma unroll
        for (int z = 0; z < (SPLIT ? 2 : 1); ++z)
#pragma unroll
            for (int s = 0; s < F::STEPS; ++s) {
                const int d0 = F::k_dim(t, 4 * s);
                const uint2 lo = *reinterpret_cast<const uint2 *>(sq + (z * 16 + g) * D + d0);
                const uint2 hi = *reinterpret_cast<const uint2 *>(sq + (z * 16 + g + 8) * D + d0);
                q[z][s][0] = lo.x, q[z][s][1] = hi.x, q[z][s][2] = lo.y, q[z][s][3] = hi.y;
            }
        const float scale0 = row_scale[g], scale1 = row_scale[g + 8];
        const int lim0 = r0 + g < rows ? limit((int)((r0 + g) / a.group)) : 0;
        const int lim1 = r0 + g + 8 < rows ? limit((int)((r0 + g + 8) / a.group)) : 0;
        const long long last = r0 + 15 < rows ? r0 + 15 : rows - 1;
        const int end = limit((int)(last / a.group));  // no row of the tile sees further
        const int blocks = (end + 15) / 16;
        const int first = (int)((long long)blocks * part / parts), stop = (int)((long long)blocks * (part + 1) / parts);

        float o[F::TILES][4];
#pragma unroll
        for (int j = 0; j < F::TILES; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
        float m0 = kLowest, m1 = kLowest, l0 = 0.0f, l1 = 0.0f;
        int exp_v = -126;  // of the largest V scale so far

        auto page_of = [&](int blk) { return blk < stop ? (uint32_t)__ldg(table + ((uint32_t)(blk * 16) >> a.kv.page_log2)) : 0u; };
        auto step = [&](const Block<D, Q8> &x, int key0) {
            float s[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][e] = 0.0f;
#pragma unroll
                for (int st = 0; st < F::STEPS; ++st) {
                    uint32_t b0, b1;
                    if constexpr (Q8) {
                        const uint32_t w = x.k[u][st] ^ 0x80808080u;
                        b0 = codes2(w, 0x4140);
                        b1 = codes2(w, 0x4342);
                    } else {
                        b0 = x.k[u][2 * st];
                        b1 = x.k[u][2 * st + 1];
                    }
                    mma16(s[u], q[0][st], b0, b1);
                    if constexpr (SPLIT) mma16(s[u], q[1][st], b0, b1);
                }
            }
            float top0 = kLowest, top1 = kLowest;
            bool see0[4], see1[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int key = key0 + 2 * t + (u & 1) + 8 * (u >> 1);
                float &a0 = s[u >> 1][u & 1], &a1 = s[u >> 1][2 + (u & 1)];
                see0[u] = key < lim0 && !x.hole;
                see1[u] = key < lim1 && !x.hole;
                a0 = see0[u] ? a0 * (Q8 ? scale0 * x.ks[u] : scale0) : kLowest;
                a1 = see1[u] ? a1 * (Q8 ? scale1 * x.ks[u] : scale1) : kLowest;
                top0 = fmaxf(top0, a0);
                top1 = fmaxf(top1, a1);
            }
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 1));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 1));
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 2));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 2));
            int exp_new = exp_v;
            if constexpr (Q8) {
                float d = fmaxf(fmaxf(fabsf(x.vs[0]), fabsf(x.vs[1])), fmaxf(fabsf(x.vs[2]), fabsf(x.vs[3])));
                d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 1));
                d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 2));
                exp_new = max(exp_v, min(126, (__float_as_int(d) >> 23) - 126));  // d < 2^exp_new
            }
            const float n0 = fmaxf(m0, top0), n1 = fmaxf(m1, top1);
            if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1 || exp_new > exp_v)) {
                const float f = Q8 ? power_of_2(exp_v - exp_new) : 1.0f;
                const float a0 = m0 == kLowest ? 0.0f : exp2_of(m0 - n0), a1 = m1 == kLowest ? 0.0f : exp2_of(m1 - n1);
                l0 *= a0;
                l1 *= a1;
#pragma unroll
                for (int j = 0; j < F::TILES; ++j) {
                    o[j][0] *= a0 * f;
                    o[j][1] *= a0 * f;
                    o[j][2] *= a1 * f;
                    o[j][3] *= a1 * f;
                }
                m0 = n0;
                m1 = n1;
                exp_v = exp_new;
            }
            // rows that have seen nothing: s is -inf everywhere, any finite maximum gives p = 0
            const float z0 = (m0 == kLowest ? 0.0f : m0) - kRaise, z1 = (m1 == kLowest ? 0.0f : m1) - kRaise;
            float w0[4], w1[4];
            const float back = Q8 ? __int_as_float((127 - exp_v) << 23) : 1.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                w0[u] = exp2_of(s[u >> 1][u & 1] - z0);
                w1[u] = exp2_of(s[u >> 1][2 + (u & 1)] - z1);
                l0 += w0[u];
                l1 += w1[u];
                if constexpr (Q8) {
                    const float d = x.vs[u] * back;
                    w0[u] = see0[u] ? w0[u] * d : 0.0f;
                    w1[u] = see1[u] ? w1[u] * d : 0.0f;
                }
            }
            uint32_t p[SPLIT ? 2 : 1][4];
            p[0][0] = pack(w0[0], w0[1]);
            p[0][1] = pack(w1[0], w1[1]);
            p[0][2] = pack(w0[2], w0[3]);
            p[0][3] = pack(w1[2], w1[3]);
            if constexpr (SPLIT) {
                float2 h = unpack(p[0][0]);
                p[1][0] = pack(w0[0] - h.x, w0[1] - h.y);
                h = unpack(p[0][1]);
                p[1][1] = pack(w1[0] - h.x, w1[1] - h.y);
                h = unpack(p[0][2]);
                p[1][2] = pack(w0[2] - h.x, w0[3] - h.y);
                h = unpack(p[0][3]);
                p[1][3] = pack(w1[2] - h.x, w1[3] - h.y);
            }
            auto tile = [&](int j, uint32_t b0, uint32_t b1) {
                mma16(o[j], p[0], b0, b1);
                if constexpr (SPLIT) mma16(o[j], p[1], b0, b1);
            };
            if constexpr (Q8) {
                constexpr int PER = F::TILES < 4 ? F::TILES : 4;
#pragma unroll
                for (int w = 0; w < F::VW; ++w) {
                    const uint32_t x0 = x.v[0][w] ^ 0x80808080u, x1 = x.v[1][w] ^ 0x80808080u;
                    const uint32_t x2 = x.v[2][w] ^ 0x80808080u, x3 = x.v[3][w] ^ 0x80808080u;
                    const uint32_t lo0 = __byte_perm(x0, x1, 0x5140), hi0 = __byte_perm(x0, x1, 0x7362);
                    const uint32_t lo1 = __byte_perm(x2, x3, 0x5140), hi1 = __byte_perm(x2, x3, 0x7362);
                    tile(PER * w, codes2(lo0, 0x4140), codes2(lo1, 0x4140));
                    tile(PER * w + 1, codes2(lo0, 0x4342), codes2(lo1, 0x4342));
                    if constexpr (PER == 4) {
                        tile(PER * w + 2, codes2(hi0, 0x4140), codes2(hi1, 0x4140));
                        tile(PER * w + 3, codes2(hi0, 0x4342), codes2(hi1, 0x4342));
                    }
                }
            } else {
#pragma unroll
                for (int w = 0; w < F::VW; ++w) {
                    tile(2 * w, __byte_perm(x.v[0][w], x.v[1][w], 0x5410), __byte_perm(x.v[2][w], x.v[3][w], 0x5410));
                    tile(2 * w + 1, __byte_perm(x.v[0][w], x.v[1][w], 0x7632), __byte_perm(x.v[2][w], x.v[3][w], 0x7632));
                }
            }
        };

        // one block is computed while the next is on its way, and the page after that is looked up
        {
            int blk = first + warp;
            Block<D, Q8> x0, x1;
            uint32_t page = page_of(blk);
            if (blk < stop) load_block<D, Q8>(a, head, page, blk * 16, end, g, t, x0);
            page = page_of(blk + kRowWarps);
            while (blk < stop) {
                const int n1b = blk + kRowWarps, n2b = n1b + kRowWarps;
                if (n1b < stop) load_block<D, Q8>(a, head, page, n1b * 16, end, g, t, x1);
                page = page_of(n2b);
                step(x0, blk * 16);
                if (n1b >= stop) break;
                if (n2b < stop) load_block<D, Q8>(a, head, page, n2b * 16, end, g, t, x0);
                page = page_of(n2b + kRowWarps);
                step(x1, n1b * 16);
                blk = n2b;
            }
        }

        // the CTA's warps
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if (t == 0) {
            wm[warp][g] = m0, wm[warp][g + 8] = m1;
            wl[warp][g] = l0, wl[warp][g + 8] = l1;
        }
        __syncthreads();
        {
            float top0 = kLowest, top1 = kLowest;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                top0 = fmaxf(top0, wm[w][g]);
                top1 = fmaxf(top1, wm[w][g + 8]);
            }
            const float f = Q8 ? power_of_2(exp_v) : 1.0f;
            const float a0 = m0 == kLowest ? 0.0f : exp2_of(m0 - top0) * f, a1 = m1 == kLowest ? 0.0f : exp2_of(m1 - top1) * f;
            float *mine = so + warp * 16 * D;
#pragma unroll
            for (int j = 0; j < F::TILES; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int d = F::v_dim(2 * t + c, j);
                    mine[g * D + d] = o[j][c] * a0;
                    mine[(g + 8) * D + d] = o[j][2 + c] * a1;
                }
        }
        if (tid < 16) {
            float top = kLowest, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, wm[w][tid]);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w)
                if (wm[w][tid] != kLowest) sum += wl[w][tid] * exp2_of(wm[w][tid] - top);
            cm[tid] = top;
            cl[tid] = sum;
        }
        __syncthreads();
        namespace cg = cooperative_groups;
        auto cluster = cg::this_cluster();
        if (parts > 1) {
            for (int u = tid; u < 16 * D; u += kRowWarps * 32) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kRowWarps; ++w) sum += so[w * 16 * D + u];
                so[u] = sum;
            }
            cluster_sync();
        }
        // outputs; with several CTAs each takes its share of the tile
        for (int u = (int)part * (kRowWarps * 32) + tid; u < 16 * D; u += (int)parts * (kRowWarps * 32)) {
            const int r = u / D, d = u % D;
            const long long rr = r0 + r;
            float sum = 0.0f, l = 0.0f;
            if (parts == 1) {
                l = cl[r];
#pragma unroll
                for (int w = 0; w < kRowWarps; ++w) sum += so[w * 16 * D + u];
            } else {
                float top = kLowest;
                for (uint32_t c = 0; c < parts; ++c) top = fmaxf(top, *cluster.map_shared_rank(&cm[r], c));
                for (uint32_t c = 0; c < parts; ++c) {
                    const float m = *cluster.map_shared_rank(&cm[r], c);
                    const float f = m == kLowest ? 0.0f : exp2_of(m - top);
                    l += f * *cluster.map_shared_rank(&cl[r], c);
                    sum += f * *cluster.map_shared_rank(&so[u], c);
                }
            }
            if (rr < rows) {
                const int i = (int)(rr / a.group), h = (int)(rr - (long long)i * a.group);
                store1(a.out, (size_t)((t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head) + d, a.o_type,
                       l == 0.0f ? 0.0f : sum / l);
            }
        }
        if (parts > 1) cluster_sync();
        else __syncthreads();
    }
}

template <int D, bool Q8, bool SPLIT>
cudaError_t launch_rows(const AttendArgs &a, dim3 grid, cudaStream_t s) {
    constexpr int SMEM = kRowWarps * 16 * D * 4;
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = op_allow(attend_rows_kernel<D, Q8, SPLIT>, SMEM, true, done);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3(kRowWarps * 32);
    c.dynamicSmemBytes = SMEM;
    c.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = grid.x;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = grid.x > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&c, attend_rows_kernel<D, Q8, SPLIT>, a);
}

template <int D>
cudaError_t launch_rows(const AttendArgs &a, bool q8, dim3 grid, cudaStream_t s) {
    const bool split = a.q_type == MGB_F32;
    if (q8) return split ? launch_rows<D, true, true>(a, grid, s) : launch_rows<D, true, false>(a, grid, s);
    return split ? launch_rows<D, false, true>(a, grid, s) : launch_rows<D, false, false>(a, grid, s);
}

}  // namespace
}  // namespace mgb

extern "C" MGB_API mgb_status mgb_kv_attend(const mgb_kv *kv, const mgb_kv_seqs *seqs, const mgb_rows *q,
                                            const mgb_rows *out, float scale, int causal, void *stream) {
    using namespace mgb;
    static const char *op = "mgb_kv_attend";
    const char *bad = check_kv(kv);
    if (!bad) bad = check_seqs(seqs);
    if (!bad) bad = check_rows(q);
    if (!bad) bad = check_rows(out);
    if (!bad && (q->tokens != out->tokens || q->heads != out->heads)) bad = "q and out differ in shape";
    if (!bad && (q->heads == 0 || q->heads % kv->heads)) bad = "query heads are not a multiple of the cache's";
    if (bad) return op_fail(MGB_ERR_INVALID, op, bad);
    if (seqs->seqs == 0 || q->tokens == 0) return MGB_OK;
    AttendArgs a{view(*kv), view(*seqs, q->tokens), q->data, out->data, q->token_stride, q->head_stride,
                 out->token_stride, out->head_stride, q->type, out->type, causal != 0, q->heads / kv->heads,
                 scale * kLog2e};
    uint64_t tiles = ((uint64_t)bound_new(*seqs, q->tokens) * a.group + 15) / 16;
    if (tiles * kv->heads > 65535) tiles = 65535 / kv->heads;
    // Keys are cut over more CTAs while that adds parallelism (two CTAs an SM)
    // and leaves each at least a block a warp.
    const uint64_t base = tiles * kv->heads * seqs->seqs;
    uint32_t parts = 1;
    while (parts < 16 && base * parts * 2 <= 2 * 148 && bound_len(*seqs, kv->page) / (parts * 2) >= kRowWarps * 16) parts *= 2;
    const dim3 grid(parts, (unsigned)(tiles * kv->heads), seqs->seqs);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool q8 = kv->format == MGB_KV_Q8;
    cudaError_t e;
    switch (kv->dim) {
        case 16: e = launch_rows<16>(a, q8, grid, s); break;
        case 32: e = launch_rows<32>(a, q8, grid, s); break;
        case 64: e = launch_rows<64>(a, q8, grid, s); break;
        default: e = launch_rows<128>(a, q8, grid, s); break;
    }
    return op_launch_status(e, op);
}
