// Writing rows into a paged K/V cache, and reading them back.
//
// Both move each number once and compute next to nothing, so HBM bounds them.
// A row (one position of one head of K or V) is spread over dim / 8 lanes of 8
// numbers each: one 16-byte access of 16-bit numbers a lane, and the maximum
// over the row is a shuffle over at most 16 lanes. Rows run over heads first,
// as the packed rows lie; in the cache each row is its own contiguous run of
// dim to 2 * dim bytes. A row with an infinity or NaN has no 8-bit form: its
// scale is NaN, so all of it reads back as NaN.
#include "serving.cuh"

namespace mgb {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // rows of a thread in flight

#define kInf __int_as_float(0x7f800000)
#define kNan __int_as_float(0x7fffffff)

struct MoveArgs {
    KvView kv;
    SeqView seq;
    void *k, *v;
    long long k_token, k_head, v_token, v_head;  // strides in numbers
    int k_type, v_type;
    bool k_vec, v_vec;
};

// grid (row groups, sequences, K or V). A row group takes rows of its sequence
// in steps of the grid, so any number of new tokens is handled whatever the
// grid was sized for.
template <int DIM, bool Q8, bool WRITE>
__global__ void __launch_bounds__(kThreads) kv_move_kernel(const MoveArgs a) {
    constexpr int LANES = DIM / 8, ROWS = kThreads / LANES;
    const uint32_t b = blockIdx.y;
    const bool is_v = blockIdx.z;
    int n;
    const int t0 = a.seq.first(b, n);
    const int base = a.seq.length(b, a.kv.page_log2), len = a.seq.kv_len[b];
    const int32_t *table = a.seq.table + (size_t)b * a.seq.table_stride;
    void *rows = is_v ? a.v : a.k;
    const long long token = is_v ? a.v_token : a.k_token, head = is_v ? a.v_head : a.k_head;
    const int type = is_v ? a.v_type : a.k_type;
    const bool vec = is_v ? a.v_vec : a.k_vec;
    void *data = is_v ? a.kv.v : a.kv.k;
    float *scale = is_v ? a.kv.vs : a.kv.ks;
    const int lane = threadIdx.x % LANES, part = lane * 8;
    const uint32_t heads = a.kv.heads;
    const uint64_t total = (uint64_t)n * heads;

    for (uint64_t r0 = (uint64_t)blockIdx.x * (ROWS * kBatch); r0 < total; r0 += (uint64_t)gridDim.x * (ROWS * kBatch)) {
        const uint32_t i0 = (uint32_t)(r0 / heads), h0 = (uint32_t)(r0 - (uint64_t)i0 * heads) + threadIdx.x / LANES;
        float x[kBatch][8];
        size_t at[kBatch], row[kBatch];
        bool live[kBatch], placed[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t hu = h0 + u * ROWS, i = i0 + hu / heads, h = hu % heads;
            live[u] = i < (uint32_t)n;
            const long long pos = (long long)len - n + i;
            placed[u] = live[u] && pos >= 0 && pos < base;
            uint32_t page = 0;
            if (placed[u]) {
                page = (uint32_t)table[pos >> a.kv.page_log2];
                placed[u] = page < a.kv.pages;
            }
            at[u] = (size_t)((long long)(t0 + i) * token + h * head + part);
            row[u] = placed[u] ? a.kv.row(page, h, (uint32_t)pos & ((1u << a.kv.page_log2) - 1)) : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[u][e] = 0.0f;
            if constexpr (WRITE) {
                if (placed[u]) load8(rows, at[u], type, vec, x[u]);
            } else if (placed[u]) {
                if constexpr (Q8) {
                    const uint2 c = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(data) + row[u] * DIM + part);
                    const float d = scale[row[u]];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[u][e] = d * (float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
                } else {
                    load8(data, row[u] * DIM + part, MGB_F16, true, x[u]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if constexpr (!WRITE) {
                if (live[u]) store8(rows, at[u], type, vec, x[u]);
            } else if constexpr (Q8) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fabsf(x[u][e]) <= 3.402823466e38f ? fmaxf(m, fabsf(x[u][e])) : kInf;
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float d = m == kInf ? kNan : __fdiv_rn(m, 127.0f);
                uint32_t c[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // the quotient is at most 127 in magnitude but for the rounding of d in the subnormal range
                    const float q = d > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(x[u][e], d)), -127.0f), 127.0f) : 0.0f;
                    c[e >> 2] |= ((uint32_t)(int)q & 255u) << (8 * (e & 3));
                }
                if (placed[u]) {
                    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(data) + row[u] * DIM + part) = make_uint2(c[0], c[1]);
                    if (lane == 0) scale[row[u]] = d;
                }
            } else if (placed[u]) {
                store8(data, row[u] * DIM + part, MGB_F16, true, x[u]);
            }
        }
    }
}

template <int DIM, bool Q8, bool WRITE>
cudaError_t launch(const MoveArgs &a, uint32_t max_new, cudaStream_t s) {
    constexpr int ROWS = kThreads / (DIM / 8);
    const uint64_t rows = (uint64_t)max_new * a.kv.heads;
    uint64_t groups = (rows + ROWS * kBatch - 1) / (ROWS * kBatch);
    if (groups > 65536) groups = 65536;
    kv_move_kernel<DIM, Q8, WRITE><<<dim3((unsigned)groups, a.seq.seqs, 2), kThreads, 0, s>>>(a);
    return cudaGetLastError();
}

template <bool WRITE>
mgb_status move(const mgb_kv *kv, const mgb_kv_seqs *seqs, const mgb_rows *k, const mgb_rows *v, void *stream,
                const char *op) {
    const char *bad = check_kv(kv);
    if (!bad) bad = check_seqs(seqs);
    if (!bad) bad = check_rows(k);
    if (!bad) bad = check_rows(v);
    if (!bad && (k->tokens != v->tokens)) bad = "K and V differ in their tokens";
    if (!bad && (k->heads != kv->heads || v->heads != kv->heads)) bad = "the rows' heads are not the cache's";
    if (bad) return op_fail(MGB_ERR_INVALID, op, bad);
    if (seqs->seqs == 0 || k->tokens == 0) return MGB_OK;
    MoveArgs a{view(*kv), view(*seqs, k->tokens), k->data, v->data, k->token_stride, k->head_stride,
               v->token_stride, v->head_stride, k->type, v->type, rows_vec(*k), rows_vec(*v)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool q8 = kv->format == MGB_KV_Q8;
    const uint32_t most_new = bound_new(*seqs, k->tokens);
    cudaError_t e;
    switch (kv->dim) {
        case 16: e = q8 ? launch<16, true, WRITE>(a, most_new, s) : launch<16, false, WRITE>(a, most_new, s); break;
        case 32: e = q8 ? launch<32, true, WRITE>(a, most_new, s) : launch<32, false, WRITE>(a, most_new, s); break;
        case 64: e = q8 ? launch<64, true, WRITE>(a, most_new, s) : launch<64, false, WRITE>(a, most_new, s); break;
        default: e = q8 ? launch<128, true, WRITE>(a, most_new, s) : launch<128, false, WRITE>(a, most_new, s); break;
    }
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
