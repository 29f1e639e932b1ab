// What the serving-step operators share (kvcache.cu, kvattend.cu, logits.cu):
// the cache's addressing, conversions between number types, error reporting.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdio>

#include "../../include/malaga_b200.h"

// Sets the text mgb_last_error() returns (defined in engine.cu).
void mgb_internal_set_error(const char *msg);

namespace mgb {

constexpr int kMaxDevices = 64;

inline mgb_status op_fail(mgb_status s, const char *op, const char *what) {
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", op, what);
    try {
        mgb_internal_set_error(buf);
    } catch (...) {  // no memory for the text: the status alone goes back
    }
    return s;
}

inline mgb_status op_launch_status(cudaError_t e, const char *op) {
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e == cudaSuccess) return MGB_OK;
    cudaGetLastError();
    return op_fail(MGB_ERR_CUDA, op, cudaGetErrorString(e));
}

// Raises a kernel's shared-memory limit (and lets it run in clusters of 16)
// once per device; `done` is the caller's static flag array.
template <typename F>
cudaError_t op_allow(F *kernel, int smem, bool big_cluster, std::atomic<bool> (&done)[kMaxDevices]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && big_cluster)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
    return e;
}

// Every launch is a programmatic dependent one: its CTAs may be scheduled once
// those of the kernel before it (if that one, too, lets it) have all started, and
// wait in begin() until it has ended, before they touch memory. That takes the
// launch out of the way of short kernels (a decode step's attention 5.8 -> 3.7 us
// back to back).
template <typename Args>
cudaError_t op_launch(void (*kernel)(Args), dim3 grid, int threads, int smem, unsigned cluster, const Args &args, cudaStream_t s) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&c, kernel, args);
}

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// In this order: that the next kernel has started says that the one before this has ended.
__device__ __forceinline__ void begin() {
    wait_for_previous();
    let_next_start();
}

// The cache as the kernels see it. A position's row of one head starts
// row(page, head, slot) rows into k and v; products are 64-bit, since a cache
// of a 180 GB GPU has more than 2^31 numbers.
struct KvView {
    void *k, *v;
    float *ks, *vs;
    uint32_t pages, heads, page_log2, dim;
    __device__ __forceinline__ size_t row(uint32_t page, uint32_t head, uint32_t slot) const {
        return ((((size_t)page * heads + head) << page_log2) + slot);
    }
};

struct SeqView {
    const int32_t *table, *q_start, *kv_len;
    uint32_t seqs, table_stride, tokens;
    // First row and number of the new tokens of sequence b, kept inside the
    // call's rows, and the first one's position; `start` and `stop`, q_start as it
    // stands. Positions of the sequence, kept inside its table.
    __device__ __forceinline__ int first(uint32_t b, int &n, int &position, int &start, int &stop) const {
        start = q_start[b], stop = q_start[b + 1];
        const int t0 = max(0, start), t1 = stop;
        n = max(0, min((int)tokens, t1) - t0);
        // the last token's is kv_len - 1, whether or not its row is one of the call's
        position = (int)max(-0x7fffffffll, min(0x7fffffffll, (long long)kv_len[b] - ((long long)t1 - t0)));
        return t0;
    }
    __device__ __forceinline__ int length(uint32_t b, uint32_t page_log2) const {
        const long long room = (long long)table_stride << page_log2;
        return (int)min((long long)max(0, kv_len[b]), room);
    }
};

inline bool power_of_two(uint32_t x) { return x && !(x & (x - 1)); }

inline uint32_t log2_of(uint32_t x) {
    uint32_t n = 0;
    while ((1u << n) < x) ++n;
    return n;
}

inline const char *check_kv(const mgb_kv *kv) {
    if (!kv || !kv->k || !kv->v) return "null cache pointer";
    if (kv->format != MGB_KV_F16 && kv->format != MGB_KV_Q8) return "unknown cache format";
    if (kv->format == MGB_KV_Q8 && (!kv->k_scale || !kv->v_scale)) return "an 8-bit cache needs its scales";
    if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) return "the cache must be 16-byte aligned";
    if (kv->format == MGB_KV_Q8 && (((uintptr_t)kv->k_scale | (uintptr_t)kv->v_scale) & 15))
        return "the cache's scales must be 16-byte aligned";
    if (kv->dim != 16 && kv->dim != 32 && kv->dim != 64 && kv->dim != 128) return "head dim must be 16, 32, 64 or 128";
    if (!power_of_two(kv->page) || kv->page < 16 || kv->page > 1024) return "page must be a power of two from 16 to 1024";
    if (kv->heads == 0 || kv->heads > 65535 || kv->pages == 0 || kv->pages > 0x7fffffffu) return "heads or pages out of range";
    return nullptr;
}

inline const char *check_seqs(const mgb_kv_seqs *s) {
    if (!s || (s->seqs && (!s->q_start || !s->kv_len || (s->table_stride && !s->table)))) return "null sequence pointer";
    if (s->seqs > 65535) return "more than 65535 sequences";
    return nullptr;
}

inline const char *check_rows(const mgb_rows *r) {
    if (!r) return "null rows";
    if (r->type < MGB_F32 || r->type > MGB_BF16) return "unknown number type";
    if (r->tokens > 0x7fffffffu) return "too many tokens";
    if (r->tokens && !r->data) return "null rows";
    if ((uintptr_t)r->data & (r->type == MGB_F32 ? 3 : 1)) return "rows are not aligned to their type";
    return nullptr;
}

// Rows that are written: none of them is another's place.
inline const char *check_out(const mgb_rows *r) {
    if ((r->tokens > 1 && r->token_stride == 0) || (r->heads > 1 && r->head_stride == 0)) return "rows that are written overlap";
    return nullptr;
}

inline KvView view(const mgb_kv &kv) {
    return KvView{kv.k, kv.v, kv.k_scale, kv.v_scale, kv.pages, kv.heads, log2_of(kv.page), kv.dim};
}

inline SeqView view(const mgb_kv_seqs &s, uint32_t tokens) {
    return SeqView{s.table, s.q_start, s.kv_len, s.seqs, s.table_stride, tokens};
}

// The bounds that size a launch.
inline uint32_t bound_new(const mgb_kv_seqs &s, uint32_t tokens) { return s.max_new && s.max_new < tokens ? s.max_new : tokens; }
inline uint64_t bound_len(const mgb_kv_seqs &s, uint32_t page) {
    const uint64_t room = (uint64_t)s.table_stride * page;
    return s.max_len && s.max_len < room ? s.max_len : room;
}

// ---------------------------------------------------------------------------
// Numbers of a row as f32, and back

__device__ __forceinline__ uint16_t to_16(float x, int type) {
    return type == MGB_F16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

__device__ __forceinline__ float load1(const void *base, size_t at, int type) {
    if (type == MGB_F32) return reinterpret_cast<const float *>(base)[at];
    const uint16_t h = reinterpret_cast<const uint16_t *>(base)[at];
    return type == MGB_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float((uint32_t)h << 16);
}

__device__ __forceinline__ void store1(void *base, size_t at, int type, float x) {
    if (type == MGB_F32) reinterpret_cast<float *>(base)[at] = x;
    else reinterpret_cast<uint16_t *>(base)[at] = to_16(x, type);
}

// Four numbers; `vec`: their address is a multiple of their size.
__device__ __forceinline__ void load4(const void *base, int64_t at, int type, bool vec, float *x) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = load1(base, (size_t)(at + i), type);
    } else if (type == MGB_F32) {
        const float4 a = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + at);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
        const uint2 a = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(base) + at);
        const uint32_t w[2] = {a.x, a.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (type == MGB_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

__device__ __forceinline__ void store4(void *base, int64_t at, int type, bool vec, const float *x) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store1(base, (size_t)(at + i), type, x[i]);
    } else if (type == MGB_F32) {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(base) + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = to_16(x[i], type);
        *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(base) + at) =
            make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    }
}

inline size_t type_size(int type) { return type == MGB_F32 ? 4 : 2; }

// Whether every fourth number of the rows stands at a multiple of four numbers' size.
inline bool rows_vec(const mgb_rows &r) {
    return ((uintptr_t)r.data & (4 * type_size(r.type) - 1)) == 0 && r.token_stride % 4 == 0 && r.head_stride % 4 == 0;
}

// Whether they are 16-bit numbers, and every eighth stands at a multiple of 16 bytes.
inline bool rows_vec16(const mgb_rows &r) {
    return r.type != MGB_F32 && ((uintptr_t)r.data & 15) == 0 && r.token_stride % 8 == 0 && r.head_stride % 8 == 0;
}

}  // namespace mgb
