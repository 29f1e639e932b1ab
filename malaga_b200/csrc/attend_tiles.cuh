// Many rows: 256 rows (token, head of the group) of one cache head a CTA, on the
// 5th-generation tensor cores.
//
// Two row tiles of 128 share the keys, so that one's softmax runs under the
// other's products: while warps 0-3 (tile 0) or 4-7 (tile 1), a thread a row,
// turn S = Q K^T into P, the tensor core works for the other tile. S, P and O
// stay in tensor memory: P (f16) takes the place of the S it came from and is
// the A operand of O += P V, O is only rescaled when a row's maximum passes the
// one in use by 2^8. Warps 8-11 bring keys and values of the pages into shared
// memory as f16, two tiles of 128 keys ahead of the products; warp 12 issues
// them. Operands lie in the K-major layout without swizzle: 8 rows x 16 bytes
// are one 128-byte block, so a warp's 16-byte stores cover whole blocks; V is
// read from the same layout as the transposed operand.
//
// 8-bit caches: K's codes are exact in f16 and their scales multiply S; V's
// scales (over the running exponent) multiply its codes as they are unpacked,
// one rounding of the product to f16.
#pragma once

namespace tiles {

constexpr int kSoftWarps = 8, kLoadWarps = 4, kWarps = kSoftWarps + kLoadWarps + 1, kThreads = kWarps * 32;
constexpr int kKeys = 128;  // of a tile

template <int D>
struct Smem {
    static constexpr int TILE = kKeys * D * 2;  // bytes of 128 rows as f16
    static constexpr int Q = 0, K = 2 * TILE, V = K + 2 * TILE, BYTES = V + 2 * TILE;
    // tensor memory takes one CTA an SM, which the shared memory has to see to
    static constexpr int ASKED = BYTES > 120 * 1024 ? BYTES : 120 * 1024;
};

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operand without swizzle: lead and stride are the distances of
// neighbouring 128-byte blocks along K and along the rows (K-major), along the
// keys and along the rows of the transposed operand (MN-major).
__device__ __forceinline__ uint64_t operand(uint32_t smem, uint32_t lead, uint32_t stride) {
    return (uint64_t)((smem >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 |
           (uint64_t)((stride >> 4) & 0x3fff) << 32 | 1ull << 46;
}

// kind::f16, f32 sums, f16 operands, M = 128; B transposed or not.
__host__ __device__ constexpr uint32_t instruction(int n, bool b_mn) {
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t i, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(i),
                 "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t i, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(i),
                 "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

#define MGB_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define MGB_R16(r, i) MGB_R4(r, i), MGB_R4(r, i + 4), MGB_R4(r, i + 8), MGB_R4(r, i + 12)
#define MGB_W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : MGB_R16(r, 0)
                 : "r"(at));
}
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : MGB_R16(r, 0), MGB_R16(r, 16)
        : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        MGB_W4(r, 0), MGB_W4(r, 4), MGB_W4(r, 8), MGB_W4(r, 12)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bytes from a tile's start of 16-byte piece c of row r.
template <int D>
__device__ __forceinline__ uint32_t piece(int r, int c) {
    return (uint32_t)((r >> 3) * (D * 16) + c * 128 + (r & 7) * 16);
}

struct Shared {
    uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], o_full;
    // Of tile j at j & 3: the softmax of tile j may still read when the loading
    // of tile j + 2 begins (which waits for the scores of j), not when that of
    // j + 3 does (the scores of j + 1 follow the softmax of j).
    alignas(16) float k_scale[4][kKeys];
    int v_exp[4];       // V of the tile is over 2^v_exp
    uint32_t holes[4];  // bit i: keys 16 i .. 16 i + 15 of the tile have no page
    float row_scale[256];
    int row_limit[256];
    float m[256], l[256];
    uint32_t tmem;
    int lost;  // a wait ran out: every role stops, the rows become NaN
};

template <int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) attend_tiles_kernel(const AttendArgs a) {
    using SM = Smem<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t parts = gridDim.x, part = blockIdx.x, heads = a.kv.heads;
    const uint32_t head = blockIdx.y % heads, b = blockIdx.z;
    int n;
    const int t0 = a.seq.first(b, n);
    const long long rows = (long long)n * a.group;
    if (rows <= a.few) return;  // left to the kernel for few rows; the whole cluster leaves
    const int len = a.seq.length(b, a.kv.page_log2), stand = a.seq.kv_len[b] - n;
    const int32_t *table = a.seq.table + (size_t)b * a.seq.table_stride;
    auto limit = [&](int i) { return a.causal ? max(0, min(len, stand + i + 1)) : len; };

    if (warp == kWarps - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], kLoadWarps);
            mbar_init(&sh.v_full[i], kLoadWarps);
            mbar_init(&sh.k_free[i], 1);
            mbar_init(&sh.v_free[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], kSoftWarps / 2);
        }
        mbar_init(&sh.o_full, 1);
        sh.lost = 0;
    }
    __syncthreads();
    const uint32_t all_tiles = (uint32_t)((rows + 255) / 256);
    uint32_t ks = 0, ss[2] = {0, 0}, os = 0;  // tiles so far of the keys', the groups' and the outputs' pipes

    // the row tiles with the most keys first
    for (uint32_t rt = blockIdx.y / heads; rt < all_tiles; rt += gridDim.y / heads) {
        const long long r0 = (long long)(all_tiles - 1 - rt) * 256;
        const int live = (int)min(256ll, rows - r0), groups = live > 128 ? 2 : 1;
        const int end = limit((int)((r0 + live - 1) / a.group)), all = limit((int)(r0 / a.group));
        const int total = (end + kKeys - 1) / kKeys;
        const int first = (int)((long long)total * part / parts), stop = (int)((long long)total * (part + 1) / parts);
        // after a wait that ran out nothing is computed any more, but every barrier is still met
        const bool lost = *reinterpret_cast<volatile int *>(&sh.lost);
        const int count = lost ? 0 : stop - first;

        // Q: a warp a row; bf16 rows scaled by a power of two to just below 2^14
        for (int r = warp; r < 256; r += kWarps) {
            constexpr int E = D >= 32 ? D / 32 : 1;
            const long long rr = r0 + r;
            const int i = (int)(rr / a.group), h = (int)(rr - (long long)i * a.group);
            float x[E], m = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = rr < rows && lane * E + e < D
                           ? load1(a.q, (size_t)((t0 + i) * a.q_token + (long long)(head * a.group + h) * a.q_head) + lane * E + e, a.q_type)
                           : 0.0f;
                m = fmaxf(m, fabsf(x[e]));
            }
            int shift = 0;
            if (a.q_type != MGB_F16) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                if (m > 0.0f && m < __int_as_float(0x7f800000)) shift = 13 - ilogbf(m);
            }
            const int s1 = max(-100, min(100, shift)), s2 = shift - s1;
            const float f1 = __int_as_float((127 + s1) << 23), f2 = __int_as_float((127 + s2) << 23);
            if (lane * E < D) {
                __half *to = reinterpret_cast<__half *>(smem + SM::Q + (r >> 7) * SM::TILE + piece<D>(r & 127, lane * E / 8)) + lane * E % 8;
#pragma unroll
                for (int e = 0; e < E; ++e) to[e] = __float2half_rn(copysignf(1.0f, a.scale) * x[e] * f1 * f2);
            }
            if (lane == 0) {
                // above 0, so that -inf times it stays -inf
                sh.row_scale[r] = fmaxf(fabsf(a.scale) * __int_as_float((127 - s1) << 23) * __int_as_float((127 - s2) << 23), 1.2e-38f);
                sh.row_limit[r] = rr < rows ? limit(i) : 0;
            }
        }
        fence_smem();
        fence_before();
        __syncthreads();
        fence_after();
        const uint32_t tmem = sh.tmem;
        // every lane of a warp waits and sees the same outcome
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity & 1));
            if (!ok) sh.lost = 1;
            return ok && !*reinterpret_cast<volatile int *>(&sh.lost);
        };

        if (warp < kSoftWarps) {
            // ------------------------------------------------------ softmax
            const int group = warp >> 2, row = (warp << 5) + lane;
            const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // tensor-memory lanes of the warp
            const uint32_t s_at = tmem + lanes + group * 128, o_at = tmem + lanes + 256 + group * D;
            const float scale = sh.row_scale[row];
            const int lim = sh.row_limit[row];
            float m = kLowest, l = 0.0f;
            int exp_v = -126;
            bool ok = !lost;
            for (int j = 0; j < count && ok && group < groups; ++j) {
                const int key0 = (first + j) * kKeys;
                ok = wait(&sh.s_full[group], ss[group] + j);
                if (!ok) break;
                fence_after();
                const uint32_t slot = (ks + j) & 3, holes = sh.holes[slot];
                const float *kscale = sh.k_scale[slot];
                const bool whole = key0 + kKeys <= all && !holes;
                auto rescale_o = [&](float f) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t raw[16];
                        tmem_load16(o_at + c0, raw);
                        tmem_wait_load();
#pragma unroll
                        for (int c = 0; c < 16; ++c) raw[c] = __float_as_uint(__uint_as_float(raw[c]) * f);
                        tmem_store16(o_at + c0, raw);
                    }
                };
                if (Q8 && sh.v_exp[slot] != exp_v) {
                    if (j > 0) rescale_o(power_of_2(exp_v - sh.v_exp[slot]));
                    exp_v = sh.v_exp[slot];
                }
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c0 = 0; c0 < kKeys; c0 += 32) {
                    uint32_t raw[32], p[16];
                    tmem_load32(s_at + c0, raw);
                    tmem_wait_load();
                    float2 x[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) x[c] = make_float2(__uint_as_float(raw[2 * c]), __uint_as_float(raw[2 * c + 1]));
                    if constexpr (Q8) {
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            const float4 d = *reinterpret_cast<const float4 *>(kscale + c0 + 2 * c);
                            x[c] = mul2(x[c], make_float2(d.x, d.y));
                            x[c + 1] = mul2(x[c + 1], make_float2(d.z, d.w));
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            const int key = key0 + c0 + 2 * c;
                            const bool hole = (holes >> ((c0 + 2 * c) >> 4)) & 1;
                            if (key >= lim || hole) x[c].x = kLowest;
                            if (key + 1 >= lim || hole) x[c].y = kLowest;
                        }
                    }
                    float top[4] = {kLowest, kLowest, kLowest, kLowest};
#pragma unroll
                    for (int c = 0; c < 16; ++c) top[c & 3] = fmaxf(fmaxf(top[c & 3], x[c].x), x[c].y);
                    const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
                    if (__any_sync(0xffffffffu, best > m + kSlack)) {
                        const float now = fmaxf(m, best), w = m == kLowest ? 0.0f : exp2_of(m - now);
                        m = now;
                        l *= w;
                        sum[0] = mul2(sum[0], make_float2(w, w));
                        sum[1] = mul2(sum[1], make_float2(w, w));
                        if (j > 0) rescale_o(w);
                        if (c0 > 0) {  // what this tile has of P so far
                            const __half2 w2 = __float2half2_rn(w);
#pragma unroll 1
                            for (int k = 0; k < c0 / 2; k += 16) {
                                tmem_wait_store();
                                tmem_load16(s_at + k, p);
                                tmem_wait_load();
#pragma unroll
                                for (int c = 0; c < 16; ++c) {
                                    const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&p[c]), w2);
                                    p[c] = *reinterpret_cast<const uint32_t *>(&y);
                                }
                                tmem_store16(s_at + k, p);
                            }
                        }
                    }
                    const float z = kRaise - (m == kLowest ? 0.0f : m);
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        x[c] = fma2(x[c], make_float2(scale, scale), make_float2(z, z));
                        x[c].x = exp2_of(x[c].x);
                        x[c].y = exp2_of(x[c].y);
                        sum[c & 1] = add2(sum[c & 1], x[c]);
                        p[c] = pack(x[c].x, x[c].y);
                    }
                    tmem_store16(s_at + c0 / 2, p);  // over scores that are already read
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_store();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cta(&sh.p_full[group]);
            }
            if (count > 0 && ok) ok = wait(&sh.o_full, os);
            fence_after();
            if (!ok) l = __int_as_float(0x7fffffff);
            if (group >= groups) l = 0.0f;
            const float back = Q8 ? power_of_2(exp_v) : 1.0f;
            const long long rr = r0 + row;
            if (parts == 1) {
                if (group < groups && count > 0) {
                    const float f = l == 0.0f ? 0.0f : back / l;
                    const int i = (int)(rr / a.group), h = (int)(rr - (long long)i * a.group);
                    const int64_t to = (t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t raw[16];
                        tmem_load16(o_at + c0, raw);
                        tmem_wait_load();
                        float x[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) x[c] = l == 0.0f ? 0.0f : __uint_as_float(raw[c]) * f;
                        if (row < live) {
#pragma unroll
                            for (int c = 0; c < 16; c += 4) store4(a.out, to + c0 + c, a.o_type, a.o_vec, x + c);
                        }
                    }
                } else if (row < live) {
                    const int i = (int)(rr / a.group), h = (int)(rr - (long long)i * a.group);
                    const int64_t to = (t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head;
                    for (int c = 0; c < D; ++c) store1(a.out, (size_t)(to + c), a.o_type, ok ? 0.0f : l);
                }
            } else {
                // this CTA's part of the row where the keys stood, turned so that the warp's stores miss each other's banks
                float *mine = reinterpret_cast<float *>(smem + SM::K) + row * D;
                if (group < groups && count > 0) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t raw[16];
                        tmem_load16(o_at + c0, raw);
                        tmem_wait_load();
#pragma unroll
                        for (int c = 0; c < 16; ++c) mine[(c0 + c + row) % D] = __uint_as_float(raw[c]) * back;
                    }
                } else {
                    for (int c = 0; c < D; ++c) mine[(c + row) % D] = 0.0f;
                }
                sh.m[row] = m;
                sh.l[row] = l;
            }
        } else if (warp < kSoftWarps + kLoadWarps) {
            // ------------------------------------------------------ loading
            const int lw = warp - kSoftWarps;
            constexpr int ESZ = Q8 ? 1 : 2, PIECES = D * ESZ / 16;  // 16-byte pieces of a row in the cache
            constexpr int PER = kKeys * PIECES / (kLoadWarps * 32);  // pieces of a thread and tile
            bool ok = true;
            // page of 16-key group `lane` of tile j (lanes 0-7), of no page where there is none
            auto pages_of = [&](int j) {
                const int key = (first + j) * kKeys + 16 * lane;
                return lane < 8 && j < count && key < end ? (uint32_t)__ldg(table + ((uint32_t)key >> a.kv.page_log2)) : 0xffffffffu;
            };
            // a piece's row (one of the warp's 32) and place in it: eight rows and neighbouring pieces an access
            auto locate = [&](int u, int &r, int &c) {
                const int x = lane + 32 * u;
                r = 32 * lw + (x & 7) + 8 * (x / (8 * PIECES));
                c = (x >> 3) % PIECES;
            };
            // where row r of tile j lies, in rows of the cache; -1 where it does not exist
            auto row_of = [&](int j, uint32_t pages, int r) -> int64_t {
                const int key = (first + j) * kKeys + r;
                const uint32_t pg = __shfl_sync(0xffffffffu, pages, r >> 4);
                return key < end && pg < a.kv.pages ? (int64_t)a.kv.row(pg, head, (uint32_t)key & ((1u << a.kv.page_log2) - 1)) : -1;
            };
            auto publish = [&](uint64_t *bar) {
                fence_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cta(bar);
            };
            uint32_t pages = pages_of(0);
            if constexpr (Q8) {
                const uint8_t *kbase = static_cast<const uint8_t *>(a.kv.k), *vbase = static_cast<const uint8_t *>(a.kv.v);
                uint4 kraw[PER], vraw[PER];
                float kd, vd[kLoadWarps];  // scales of key 32 lw + lane, of keys lane, 32 + lane, ...
                auto fetch = [&](const uint8_t *base, int j, uint32_t pg, uint4 (&raw)[PER]) {
#pragma unroll
                    for (int u = 0; u < PER; ++u) {
                        int r, c;
                        locate(u, r, c);
                        const int64_t row = row_of(j, pg, r);
                        raw[u] = row >= 0 ? __ldg(reinterpret_cast<const uint4 *>(base + row * D) + c) : make_uint4(0, 0, 0, 0);
                    }
                };
                auto fetch_scales = [&](int j, uint32_t pg) {
                    kd = 0.0f;
#pragma unroll
                    for (int w = 0; w < kLoadWarps; ++w) {
                        const int64_t row = row_of(j, pg, 32 * w + lane);
                        vd[w] = row >= 0 ? __ldg(a.kv.vs + row) : 0.0f;
                        if (w == lw && row >= 0) kd = __ldg(a.kv.ks + row);
                    }
                };
                int exp_v = -126;
                if (count > 0) {
                    fetch(kbase, 0, pages, kraw);
                    fetch_scales(0, pages);
                }
                for (int j = 0; j < count && ok; ++j) {
                    const uint32_t stage = (ks + j) & 1, turn = (ks + j) >> 1, slot = (ks + j) & 3;
                    const uint32_t next = pages_of(j + 1);
                    fetch(vbase, j, pages, vraw);
                    const uint32_t holes = __ballot_sync(0xffffffffu, pages >= a.kv.pages) & 0xff;
                    float top = fabsf(vd[0]), mine = vd[0];
#pragma unroll
                    for (int w = 1; w < kLoadWarps; ++w) {
                        top = fmaxf(top, fabsf(vd[w]));
                        if (w == lw) mine = vd[w];
                    }
                    const int bits = (int)__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23;
                    exp_v = max(exp_v, min(126, bits - 126));
                    mine *= __int_as_float((127 - exp_v) << 23);
                    if (turn > 0) ok = wait(&sh.k_free[stage], turn - 1);
                    if (!ok) break;
                    sh.k_scale[slot][32 * lw + lane] = kd;
                    if (lw == 0 && lane == 0) {
                        sh.v_exp[slot] = exp_v;
                        sh.holes[slot] = holes;
                    }
                    uint8_t *tile = smem + SM::K + stage * SM::TILE;
#pragma unroll
                    for (int u = 0; u < PER; ++u) {
                        int r, c;
                        locate(u, r, c);
                        const uint32_t w[4] = {kraw[u].x, kraw[u].y, kraw[u].z, kraw[u].w};
                        uint32_t h[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            h[2 * i] = codes2(w[i] ^ 0x80808080u, 0x4140);
                            h[2 * i + 1] = codes2(w[i] ^ 0x80808080u, 0x4342);
                        }
                        *reinterpret_cast<uint4 *>(tile + piece<D>(r, 2 * c)) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4 *>(tile + piece<D>(r, 2 * c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                    publish(&sh.k_full[stage]);
                    if (j + 1 < count) {  // on their way while V is unpacked
                        fetch(kbase, j + 1, next, kraw);
                        fetch_scales(j + 1, next);
                    }
                    pages = next;
                    if (turn > 0) ok = wait(&sh.v_free[stage], turn - 1);
                    if (!ok) break;
                    tile = smem + SM::V + stage * SM::TILE;
                    // code * scale with one rounding: the scale as a high and a low f16 part
                    const __half hi = __float2half_rn(mine), lo = __float2half_rn(mine - __half2float(hi));
                    const __half2 both = __halves2half2(hi, lo);
#pragma unroll
                    for (int u = 0; u < PER; ++u) {
                        int r, c;
                        locate(u, r, c);
                        const uint32_t w[4] = {vraw[u].x, vraw[u].y, vraw[u].z, vraw[u].w};
                        const uint32_t d = __shfl_sync(0xffffffffu, *reinterpret_cast<const uint32_t *>(&both), r & 31);
                        const uint32_t d_hi = __byte_perm(d, 0, 0x1010), d_lo = __byte_perm(d, 0, 0x3232);
                        const __half2 hi2 = *reinterpret_cast<const __half2 *>(&d_hi), lo2 = *reinterpret_cast<const __half2 *>(&d_lo);
                        uint32_t h[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t x = codes2(w[i / 2] ^ 0x80808080u, i & 1 ? 0x4342 : 0x4140);
                            const __half2 q = *reinterpret_cast<const __half2 *>(&x);
                            const __half2 y = __hfma2(q, hi2, __hmul2(q, lo2));
                            h[i] = *reinterpret_cast<const uint32_t *>(&y);
                        }
                        *reinterpret_cast<uint4 *>(tile + piece<D>(r, 2 * c)) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4 *>(tile + piece<D>(r, 2 * c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                    publish(&sh.v_full[stage]);
                }
            } else {
                // copies of tile j's K or V into its stage, once the products with what was there are done
                auto copy = [&](const void *base, uint32_t part_at, uint64_t (&free)[2], int j, uint32_t pg) {
                    const uint32_t stage = (ks + j) & 1, turn = (ks + j) >> 1;
                    if (j < count && turn > 0) ok = ok && wait(&free[stage], turn - 1);
                    if (j < count && ok) {
#pragma unroll
                        for (int u = 0; u < PER; ++u) {
                            int r, c;
                            locate(u, r, c);
                            const int64_t row = row_of(j, pg, r);
                            const uint8_t *p = static_cast<const uint8_t *>(base) + max(row, (int64_t)0) * (D * 2) + 16 * c;
                            // what lies beyond the 0 or 16 bytes read becomes zeros
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                             smem_u32(smem + part_at + stage * SM::TILE + piece<D>(r, c))),
                                         "l"(p), "r"(row >= 0 ? 16 : 0)
                                         : "memory");
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                copy(a.kv.k, SM::K, sh.k_free, 0, pages);
                copy(a.kv.v, SM::V, sh.v_free, 0, pages);
                for (int j = 0; j < count && ok; ++j) {
                    const uint32_t stage = (ks + j) & 1, next = pages_of(j + 1);
                    const uint32_t holes = __ballot_sync(0xffffffffu, pages >= a.kv.pages) & 0xff;
                    copy(a.kv.k, SM::K, sh.k_free, j + 1, next);
                    if (!ok) break;
                    if (lw == 0 && lane == 0) sh.holes[(ks + j) & 3] = holes;
                    asm volatile("cp.async.wait_group 2;" ::: "memory");
                    publish(&sh.k_full[stage]);
                    copy(a.kv.v, SM::V, sh.v_free, j + 1, next);
                    if (!ok) break;
                    asm volatile("cp.async.wait_group 2;" ::: "memory");
                    publish(&sh.v_full[stage]);
                    pages = next;
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
        } else if (count > 0) {
            // ------------------------------------------------------ products
            constexpr uint32_t QK = instruction(kKeys, false), PV = instruction(D, true);
            const uint64_t q0 = operand(smem_u32(smem + SM::Q), 128, D * 16), k0 = operand(smem_u32(smem + SM::K), 128, D * 16);
            const uint64_t v0 = operand(smem_u32(smem + SM::V), D * 16, 128);
            auto scores = [&](int g, int j) {
                const uint64_t q = q0 + g * (SM::TILE >> 4), k = k0 + ((ks + j) & 1) * (SM::TILE >> 4);
#pragma unroll
                for (int s = 0; s < D / 16; ++s) mma_ss(tmem + g * 128, q + s * 16, k + s * 16, QK, s > 0);
                commit(&sh.s_full[g]);
            };
            bool ok = wait(&sh.k_full[ks & 1], ks >> 1);
            if (ok && lane == 0) {
                fence_after();
                for (int g = 0; g < groups; ++g) scores(g, 0);
                commit(&sh.k_free[ks & 1]);
            }
            for (int j = 0; j < count && ok; ++j) {
                const uint32_t stage = (ks + j) & 1;
                ok = wait(&sh.v_full[stage], (ks + j) >> 1);
                for (int g = 0; g < groups && ok; ++g) {
                    ok = wait(&sh.p_full[g], ss[g] + j);
                    if (ok && j + 1 < count && g == 0) ok = wait(&sh.k_full[(ks + j + 1) & 1], (ks + j + 1) >> 1);
                    if (!ok) break;
                    fence_after();
                    if (lane == 0) {
                        const uint64_t v = v0 + stage * (SM::TILE >> 4);
#pragma unroll
                        for (int s = 0; s < kKeys / 16; ++s)
                            mma_ts(tmem + 256 + g * D, tmem + g * 128 + s * 8, v + s * (2 * D), PV, j > 0 || s > 0);
                        if (j + 1 < count) scores(g, j + 1);
                    }
                    __syncwarp();
                }
                if (ok && lane == 0) {
                    commit(&sh.v_free[stage]);
                    if (j + 1 < count) commit(&sh.k_free[(ks + j + 1) & 1]);
                }
            }
            // also after a lost wait: nothing in flight when the CTA leaves
            if (lane == 0) commit(&sh.o_full);
            wait(&sh.o_full, os);
        }
        ks += count;
        os += count > 0;
        ss[0] += count;
        ss[1] += groups > 1 ? count : 0;
        fence_before();
        if (parts > 1) cluster_sync();
        else __syncthreads();
        fence_after();
        if (parts > 1) {
            namespace cg = cooperative_groups;
            auto cluster = cg::this_cluster();
            const float *o = reinterpret_cast<const float *>(smem + SM::K);
            for (int u = (int)part * kThreads + tid; u < live * (D / 4); u += (int)parts * kThreads) {
                const int row = u / (D / 4), c0 = u % (D / 4) * 4;
                float top = kLowest, l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (uint32_t c = 0; c < parts; ++c) top = fmaxf(top, *cluster.map_shared_rank(&sh.m[row], c));
                for (uint32_t c = 0; c < parts; ++c) {
                    const float m = *cluster.map_shared_rank(&sh.m[row], c), lc = *cluster.map_shared_rank(&sh.l[row], c);
                    const float f = m == kLowest ? 0.0f : exp2_of(m - top);
                    l += m == kLowest ? lc : f * lc;
                    const float *from = cluster.map_shared_rank(o + row * D, c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] += f * from[(c0 + e + row) % D];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = l == 0.0f ? 0.0f : x[e] / l;
                const long long rr = r0 + row;
                const int i = (int)(rr / a.group), h = (int)(rr - (long long)i * a.group);
                store4(a.out, (t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head + c0, a.o_type, a.o_vec, x);
            }
            cluster_sync();
        }
    }
    __syncthreads();
    if (warp == kWarps - 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem) : "memory");
}

}  // namespace tiles
