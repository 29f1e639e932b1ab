// Writing rows into a paged K/V cache, and reading them back.
//
// Both move each number once, so HBM is their floor. Measured, K and V of 16 heads
// of 128: writing 17,221 bf16 tokens as 8-bit codes takes 72 us (3.0 TB/s; the
// exact quotients keep 70 % of the issue slots busy and bound it), reading 45,789
// tokens of 8 heads back as f16 66 us (4.3 TB/s, waiting for loads). 64 tokens of 64
// take 2.7 us a launch.
// A CTA takes a run of the call's tokens: its threads first look up each
// token's place (a search for its sequence, then the page table), then move the
// rows of all heads, K and V. A row is spread over dim / 8 lanes of 8 numbers;
// the lanes' pieces are laid out so that a warp's 16-byte accesses to the packed
// rows are contiguous for 32-bit and for 16-bit numbers. Tokens are cut evenly over
// the CTAs whatever the sequences' lengths.
#include "serving.cuh"

namespace mgb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;  // tokens of a CTA, at most its threads: of 8 to 64, 8 to 16 write fastest (72 us where 32 take 77), all read alike

#define kInf __int_as_float(0x7f800000)
#define kNan __int_as_float(0x7fffffff)

struct Side {  // K or V: its packed rows and its half of the cache
    void *rows;
    long long token_stride, head_stride;  // in numbers
    uint8_t *data;
    float *scale;
};

struct MoveArgs {
    KvView kv;
    SeqView seq;
    Side side[2];
    uint32_t per_cta;  // tokens of a CTA
};

// Code bytes of x / d for eight numbers. x * (1 / d) is within 2^-15 of the f32
// quotient (|x / d| <= 127), so it rounds to the same whole number unless it
// lies that near a half; then the quotients themselves are taken. Adding
// 1.5 * 2^23 rounds to a whole number, halves to even, and leaves it in the low
// bits.
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float d) {
    constexpr float kWhole = 12582912.0f;
    const bool tiny = !(d > 1e-30f);  // 1 / d would leave f32's range, or there is no d
    const float inv = __frcp_rn(d);
    uint32_t r[8];
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = x[e] * inv, w = q + kWhole;
        r[e] = __float_as_uint(w);
        far = fmaxf(far, fabsf(q - (w - kWhole)));
    }
    if (tiny || far > 0.4999f) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            r[e] = d > 0.0f ? __float_as_uint(fminf(fmaxf(__fdiv_rn(x[e], d), -127.0f), 127.0f) + kWhole) : 0u;
    }
    return make_uint2(__byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410));
}

// Four code bytes as f32: the bytes 00 00 4b above u are the number 2^23 + u.
__device__ __forceinline__ void values_of(uint32_t codes, float d, float *x) {
    const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = d * (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + e)) - 8388736.0f);
}

// A lane's eight numbers of the row at `at`: two pieces of four, or one of eight.
template <int TYPE, bool VEC, bool APART>
__device__ __forceinline__ void load_pieces(const void *rows, int64_t at, int p0, int p1, float (&x)[8]) {
    if constexpr (VEC && TYPE != MGB_F32 && !APART) {
        const uint4 h = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(rows) + at + p0);
        const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = TYPE == MGB_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&w[e]))
                                             : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
            x[2 * e] = f.x, x[2 * e + 1] = f.y;
        }
    } else {
        load4(rows, at + p0, TYPE, VEC, &x[0]);
        load4(rows, at + p1, TYPE, VEC, &x[4]);
    }
}

template <int TYPE, bool VEC, bool APART>
__device__ __forceinline__ void store_pieces(void *rows, int64_t at, int p0, int p1, const float (&x)[8]) {
    if constexpr (VEC && TYPE != MGB_F32 && !APART) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = to_16(x[2 * e], TYPE) | (uint32_t)to_16(x[2 * e + 1], TYPE) << 16;
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(rows) + at + p0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        store4(rows, at + p0, TYPE, VEC, &x[0]);
        store4(rows, at + p1, TYPE, VEC, &x[4]);
    }
}

template <int DIM, bool Q8, bool WRITE, int TYPE, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_move_kernel(const MoveArgs a) {
    constexpr int LANES = DIM / 8, ROWS = kThreads / LANES;
    // rows of a thread in flight: more cost warps of an SM (reading, 1 / 2 / 4: 67 / 75 / 89 us; writing 87 / 77 / 77)
    constexpr int kBatch = WRITE ? 2 : 1;
    __shared__ int64_t place[kMaxTokens];  // row of head 0 in the cache, -1 where there is none
    begin();
    const uint32_t first = blockIdx.x * a.per_cta, tokens = min(a.per_cta, a.seq.tokens - first);
    if (threadIdx.x < tokens) {
        const int token = (int)(first + threadIdx.x);
        // the last sequence that starts at or before the token
        uint32_t lo = 0, hi = a.seq.seqs;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (a.seq.q_start[mid] <= token) lo = mid;
            else hi = mid;
        }
        int64_t row = -1;
        const int start = hi ? a.seq.q_start[lo] : 0, stop = hi ? a.seq.q_start[lo + 1] : 0;  // hi: there are sequences
        if (token >= start && token < stop) {
            const long long pos = (long long)a.seq.kv_len[lo] - (stop - token);
            if (pos >= 0 && (pos >> a.kv.page_log2) < a.seq.table_stride) {
                const uint32_t page = (uint32_t)a.seq.table[(size_t)lo * a.seq.table_stride + (pos >> a.kv.page_log2)];
                if (page < a.kv.pages) row = (int64_t)a.kv.row(page, 0, (uint32_t)pos & ((1u << a.kv.page_log2) - 1));
            }
        }
        place[threadIdx.x] = row;
    }
    __syncthreads();

    const Side &side = a.side[blockIdx.y];
    void *rows = side.rows;
    uint8_t *data = side.data;
    float *scale = side.scale;
    // a lane's two pieces of four numbers: apart for 32-bit rows, side by side for 16-bit ones
    constexpr bool APART = TYPE == MGB_F32;
    const int lane = threadIdx.x % LANES;
    const int p0 = APART ? 4 * lane : 8 * lane, p1 = APART ? DIM / 2 + 4 * lane : 8 * lane + 4;
    const uint32_t heads = a.kv.heads, total = tokens * heads;

    for (uint32_t r0 = 0; r0 < total; r0 += ROWS * kBatch) {
        float x[kBatch][8];
        int64_t at[kBatch], row[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t r = r0 + u * ROWS + threadIdx.x / LANES, i = r / heads, h = r - i * heads;
            row[u] = r < total ? place[i] : -2;  // -2: no such row
            if (row[u] >= 0) row[u] += (int64_t)h << a.kv.page_log2;
            at[u] = (int64_t)(first + i) * side.token_stride + (int64_t)h * side.head_stride;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[u][e] = 0.0f;
            if (row[u] < 0) continue;
            if constexpr (WRITE) {
                load_pieces<TYPE, VEC, APART>(rows, at[u], p0, p1, x[u]);
            } else if constexpr (Q8) {
                const uint8_t *c = data + row[u] * DIM;
                const float d = scale[row[u]];
                uint2 code;
                if constexpr (APART) code = make_uint2(*reinterpret_cast<const uint32_t *>(c + p0), *reinterpret_cast<const uint32_t *>(c + p1));
                else code = *reinterpret_cast<const uint2 *>(c + p0);
                values_of(code.x, d, &x[u][0]);
                values_of(code.y, d, &x[u][4]);
            } else {
                load_pieces<MGB_F16, true, APART>(data, row[u] * DIM, p0, p1, x[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if constexpr (!WRITE) {
                if (row[u] == -2) continue;
                store_pieces<TYPE, VEC, APART>(rows, at[u], p0, p1, x[u]);
            } else if constexpr (Q8) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fabsf(x[u][e]) < kInf ? fmaxf(m, fabsf(x[u][e])) : kInf;
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float d = m == kInf ? kNan : __fdiv_rn(m, 127.0f);
                const uint2 code = codes_of(x[u], d);
                if (row[u] >= 0) {
                    uint8_t *c = data + row[u] * DIM;
                    if constexpr (APART) {
                        *reinterpret_cast<uint32_t *>(c + p0) = code.x;
                        *reinterpret_cast<uint32_t *>(c + p1) = code.y;
                    } else {
                        *reinterpret_cast<uint2 *>(c + p0) = code;
                    }
                    if (lane == 0) scale[row[u]] = d;
                }
            } else if (row[u] >= 0) {
                store_pieces<MGB_F16, true, APART>(data, row[u] * DIM, p0, p1, x[u]);
            }
        }
    }
}

// Few tokens: as many a CTA as leave two CTAs an SM (148 SMs) on either side, so that
// all run at once. From 296 * kMaxTokens on kMaxTokens a CTA, and more CTAs.
template <int DIM, bool Q8, bool WRITE>
cudaError_t launch(MoveArgs a, int sides, int type, bool vec, cudaStream_t s) {
    const uint32_t n = a.seq.tokens / (2 * 148);
    a.per_cta = n < 1 ? 1 : n > kMaxTokens ? kMaxTokens : n;
    const dim3 grid((a.seq.tokens + a.per_cta - 1) / a.per_cta, sides);
    auto go = [&](auto kernel) { return op_launch(kernel, grid, kThreads, 0, 1, a, s); };
    if (type == MGB_F32) return vec ? go(kv_move_kernel<DIM, Q8, WRITE, MGB_F32, true>) : go(kv_move_kernel<DIM, Q8, WRITE, MGB_F32, false>);
    if (type == MGB_F16) return vec ? go(kv_move_kernel<DIM, Q8, WRITE, MGB_F16, true>) : go(kv_move_kernel<DIM, Q8, WRITE, MGB_F16, false>);
    return vec ? go(kv_move_kernel<DIM, Q8, WRITE, MGB_BF16, true>) : go(kv_move_kernel<DIM, Q8, WRITE, MGB_BF16, false>);
}

template <bool WRITE>
cudaError_t launch(const MoveArgs &a, int sides, bool q8, int type, bool vec, cudaStream_t s) {
    switch (a.kv.dim) {
        case 16: return q8 ? launch<16, true, WRITE>(a, sides, type, vec, s) : launch<16, false, WRITE>(a, sides, type, vec, s);
        case 32: return q8 ? launch<32, true, WRITE>(a, sides, type, vec, s) : launch<32, false, WRITE>(a, sides, type, vec, s);
        case 64: return q8 ? launch<64, true, WRITE>(a, sides, type, vec, s) : launch<64, false, WRITE>(a, sides, type, vec, s);
        default: return q8 ? launch<128, true, WRITE>(a, sides, type, vec, s) : launch<128, false, WRITE>(a, sides, type, vec, s);
    }
}

// Whether 16-byte accesses fit.
bool rows_wide(const mgb_rows &r) { return r.type == MGB_F32 ? rows_vec(r) : rows_vec16(r); }

template <bool WRITE>
mgb_status move(const mgb_kv *kv, const mgb_kv_seqs *seqs, const mgb_rows *k, const mgb_rows *v, void *stream,
                const char *op) {
    const char *bad = check_kv(kv);
    if (!bad) bad = check_seqs(seqs);
    if (!bad) bad = check_rows(k);
    if (!bad) bad = check_rows(v);
    if (!bad && !WRITE) bad = check_out(k);
    if (!bad && !WRITE) bad = check_out(v);
    if (!bad && (k->tokens != v->tokens)) bad = "K and V differ in their tokens";
    if (!bad && (k->heads != kv->heads || v->heads != kv->heads)) bad = "the rows' heads are not the cache's";
    if (bad) return op_fail(MGB_ERR_INVALID, op, bad);
    if (k->tokens == 0 || (WRITE && seqs->seqs == 0)) return MGB_OK;  // a read without sequences is of zeros
    MoveArgs a{view(*kv), view(*seqs, k->tokens),
               {{k->data, k->token_stride, k->head_stride, static_cast<uint8_t *>(kv->k), kv->k_scale},
                {v->data, v->token_stride, v->head_stride, static_cast<uint8_t *>(kv->v), kv->v_scale}},
               0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool q8 = kv->format == MGB_KV_Q8;
    if (k->type == v->type) return op_launch_status(launch<WRITE>(a, 2, q8, k->type, rows_wide(*k) && rows_wide(*v), s), op);
    // rows of two types: a launch each
    cudaError_t e = launch<WRITE>(a, 1, q8, k->type, rows_wide(*k), s);
    a.side[0] = a.side[1];
    if (e == cudaSuccess) e = launch<WRITE>(a, 1, q8, v->type, rows_wide(*v), s);
    return op_launch_status(e, op);
}

}  // namespace
}  // namespace mgb

extern "C" MGB_API mgb_status mgb_kv_write(const mgb_kv *kv, const mgb_kv_seqs *seqs, const mgb_rows *k,
                                           const mgb_rows *v, void *stream) {
    return mgb::move<true>(kv, seqs, k, v, stream, "mgb_kv_write");
}

extern "C" MGB_API mgb_status mgb_kv_read(const mgb_kv *kv, const mgb_kv_seqs *seqs, const mgb_rows *k,
                                          const mgb_rows *v, void *stream) {
    return mgb::move<false>(kv, seqs, k, v, stream, "mgb_kv_read");
}
