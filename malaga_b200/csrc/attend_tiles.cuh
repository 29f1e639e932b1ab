// Many rows: 256 rows (token, head of the group) of one cache head a CTA, on the
// 5th-generation tensor cores.
//
// Two row tiles of 128 share the keys, so that one's softmax runs under the
// other's products: while warps 0-3 (tile 0) or 4-7 (tile 1), a thread a row,
// turn S = Q K^T into P, the tensor core works for the other tile. S, P and O
// stay in tensor memory: P (f16) takes the place of the S it came from and is
// the A operand of O += P V, O is only rescaled when a row's maximum passes the
// one in use by 2^8. Warps 8-11 bring keys and values of the pages into shared
// memory as f16, up to two tiles of 128 keys ahead. Warp 12 issues the products,
// values and next scores of one row tile after those of the other. Warps 13-15 look
// over the values of the tiles that some rows do not see whole, before their product
// (done by the loading warps it cost 6 to 12 % on every tile, in registers).
// What bounds it: a step of 128 keys in f16 takes 4200 (dim 64) to 5600 cycles (dim 128) of
// which the tensor core computes 1024 and 2048 and the exponentials take 2048. No unit
// is full (4099 tokens over 20,011 positions, 8 bits: tensor pipe 32 % of the cycles,
// exponentials 25 %, issue slots 44 %); warps wait for scores, tensor memory and
// barriers, one row tile's chain of scores, softmax and product only partly under the
// other's. 8192 tokens over 16384 positions of 16 heads of dim 128, causal, take 1.05
// ms in f16 (790 TFLOP/s) and 1.22 ms in 8 bits, of dim 64 0.77 and 0.99 ms.
// Registers go where a whole row of scores is held (setmaxnreg). Operands lie
// in the K-major layout without swizzle: 8 rows x 16 bytes are one 128-byte
// block, so a warp's 16-byte stores cover whole blocks; V is read from the same
// layout as the transposed operand.
//
// 8-bit caches: K's codes are exact in f16 and their scales multiply S (folding
// them into K as it is unpacked was 4 % faster and made the error of f16
// outputs 3.2e-4 -> 6.8e-4); V's scales, over the running exponent, multiply its
// codes as they are unpacked, one rounding of the product to f16 (the scale
// enters as a high and a low part). In a tile that some rows do not see whole, and
// whose scales are far apart or no numbers, they multiply P instead, over a row's own
// exponent: that of a key which a row does not see must not move the row's numbers out
// of f16's range. (Done for all such tiles it took 700 tokens over 3000 positions, 16
// heads of 128, from 55.7 to 66.8 us.)
#pragma once

namespace tiles {

constexpr int kSoftWarps = 8, kLoadWarps = 4, kWarps = 16, kThreads = kWarps * 32;
constexpr int kMmaWarp = kSoftWarps + kLoadWarps;  // and three that look over values some rows do not see
// registers of a thread of the softmax, loading and product warpgroups; their sum is the launch's 128 a thread
constexpr int kSoftRegs = 184, kLoadRegs = 104, kMmaRegs = 40;
static_assert(2 * kSoftRegs + kLoadRegs + kMmaRegs == 4 * 128, "the split has to add up");
constexpr int kKeys = 128;  // of a tile
constexpr int kFolded = 1000;

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

// One lane of the warp. With lane == 0 in its place the compiler does not know that a
// single lane is left and passes the operands of each product through a loop over the
// warp's lanes: 60 to 100 cycles a product, where 32 to 64 are what it computes for.
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
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

template <int D>
struct Shared {
    uint64_t q_full, k_full[2], k_free[2], v_full[2], v_free[2], v_raw[2], s_full[2], p_full[2], o_full;
    // Of tile j at j & 3: the softmax of tile j may still read when the loading
    // of tile j + 2 begins (which waits for the scores of j), not when that of
    // j + 3 does (the scores of j + 1 follow the softmax of j).
    alignas(16) float k_scale[4][kKeys], v_scale[4][kKeys];
    int v_exp[4];       // V of the tile is over 2^v_exp, or without its scales (kFolded)
    uint32_t holes[4];  // bit i: keys 16 i .. 16 i + 15 of the tile have no page
    float m[256], l[256], weight[8][256];
    // Where some rows of the tile do not see a key, an infinity or NaN in its V is
    // taken out (0 times it would reach them) and noted: NaN (0), +inf (1) or -inf (2)
    // is added to dim d of rows that see key wild[.][d]. wild_any: whether there is one.
    int wild[3][D], wild_any;
    uint32_t tmem;
    int lost;  // a wait ran out: nothing more is computed, the rows become NaN, and the device's word says so
};

// Changes the warpgroup's registers a thread from the launch's 128 to N: .inc and
// .dec are only defined in their own direction.
template <int N>
__device__ __forceinline__ void set_registers() {
    if constexpr (N > 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    if constexpr (N < 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// All threads of the CTA, or of the cluster, from wherever their roles stand.
__device__ __forceinline__ void meet(bool cluster) {
    __syncwarp();
    if (cluster) cluster_sync();
    else asm volatile("barrier.sync 0;" ::: "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^y of both, by products alone (the exponentials' own unit has 16 a cycle): with n
// the integer next to y, 2^(y - n) is a polynomial of degree 4, fitted for the least
// relative error over [-1/2, 1/2]: 2.6e-6, where the rounding to f16 that follows has
// 2.4e-4. Below -126 it stays at 2^-126, which is 0 as f16; NaN stays NaN.
__device__ __forceinline__ float2 exp2_poly(float2 y) {
    auto both = [](float c) { return make_float2(c, c); };
    auto least = [](float v) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(-126.0f));
        return r;
    };
    y = make_float2(least(y.x), least(y.y));
    // 1.5 * 2^23 + 127: the sum's last bits are n + 127, an exponent
    const float2 big = both(12583039.0f), t = add2(y, big), r = add2(y, fma2(t, both(-1.0f), big));
    float2 p = fma2(both(0.009570101276f), r, both(0.055917859077f));
    p = fma2(p, r, both(0.240247443318f));
    p = fma2(p, r, both(0.693121790886f));
    p = fma2(p, r, both(0.999999284745f));
    return mul2(p, make_float2(__int_as_float(__float_as_int(t.x) << 23), __int_as_float(__float_as_int(t.y) << 23)));
}

// What all roles of a CTA know of its row tile.
struct Span {
    int r0, live, groups;  // its first row; rows of the tile; 128-row groups that have some
    int end, all;      // keys that its last row sees; keys that every row sees
    int first, count;  // its part's key tiles
    int clean;         // of them, those before the first that some row does not see all of
};

template <int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) attend_tiles_kernel(const AttendArgs a) {
    using SM = Smem<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Shared<D> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t parts = gridDim.x, part = blockIdx.x, heads = a.kv.heads;
    const uint32_t head = blockIdx.y % heads, b = blockIdx.z;
    wait_for_previous();
    if (a.turn && (part | blockIdx.y | b) == 0) {
        if (tid == 0) give_turn(a.turn);
        __syncthreads();
    }
    let_next_start();
    int n, stand, start, stop;
    const int t0 = a.seq.first(b, n, stand, start, stop);
    zero_outside(a, b, start, stop);
    const int rows = n * (int)a.group;  // the call has fewer than 2^31 query rows
    if ((uint32_t)rows <= a.few) return;  // left to the kernel for few rows; the whole cluster leaves
    const int len = a.seq.length(b, a.kv.page_log2);
    const int32_t *table = a.seq.table + (size_t)b * a.seq.table_stride;
    auto limit = [&](int i) { return a.causal ? max(0, min(len, stand + i + 1)) : len; };

    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        mbar_init(&sh.q_full, kSoftWarps);
        for (int i = 0; i < 2; ++i) {
            // the test hook has the first CTA wait for an arrival too many
            mbar_init(&sh.k_full[i], kLoadWarps + (a.withhold == i && (part | blockIdx.y | b) == 0));
            mbar_init(&sh.v_full[i], kLoadWarps);
            mbar_init(&sh.v_raw[i], kLoadWarps);
            mbar_init(&sh.k_free[i], 2);
            mbar_init(&sh.v_free[i], 2);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], kSoftWarps / 2);
        }
        mbar_init(&sh.o_full, 1);
        sh.lost = 0;
        sh.wild_any = 0;
    }
    for (int u = tid; u < 3 * D; u += kThreads) (&sh.wild[0][0])[u] = 0x7fffffff;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;

    const uint32_t row_tiles = (uint32_t)((rows + 255) / 256), tile0 = blockIdx.y / heads, tile_step = gridDim.y / heads;
    // the row tiles with the most keys first
    auto span_of = [&](uint32_t rt) {
        Span s;
        s.r0 = (int)(row_tiles - 1 - rt) * 256;
        s.live = min(256, rows - s.r0);
        s.groups = s.live > 128 ? 2 : 1;
        s.end = limit((s.r0 + s.live - 1) / (int)a.group);
        s.all = limit(s.r0 / (int)a.group);
        const int total = (s.end + kKeys - 1) / kKeys;
        // parts is at most 8 and a tile 128 keys, so the products stay below 2^31
        s.first = (int)((uint32_t)total * part / parts);
        s.count = (int)((uint32_t)total * (part + 1) / parts) - s.first;
        if (*reinterpret_cast<volatile int *>(&sh.lost)) s.count = 0;  // every barrier is still met
        s.clean = min(s.count, max(0, s.all / kKeys - s.first));
        return s;
    };
    // every lane of a warp waits and sees the same outcome
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity & 1));
        if (!ok) sh.lost = 1;
        return ok && !*reinterpret_cast<volatile int *>(&sh.lost);
    };
    // tiles so far, over all row tiles: stage and parity of the keys' and of the group's pipes; row tiles so far
    uint32_t ks = 0, ss[2] = {0, 0}, os = 0, turns = 0, cleaned = 0;
    auto next_tile = [&](const Span &s) {
        ks += s.count;
        os += s.count > 0;
        ss[0] += s.count;
        ss[1] += s.groups > 1 ? s.count : 0;
        cleaned += s.count - s.clean;
        ++turns;
    };
    // values that some rows do not see go by way of the warps that look them over (8-bit codes are finite)
    auto values_at = [&](const Span &s, int j) {
        return Q8 || j < s.clean ? &sh.v_full[(ks + j) & 1] : &sh.v_raw[(cleaned + j - s.clean) & 1];
    };

    if (warp < kSoftWarps) {
        // ---------------------------------------------------------- softmax
        set_registers<kSoftRegs>();
        const int group = warp >> 2, row = tid;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // tensor-memory lanes of the warp
        const uint32_t s_at = tmem + lanes + group * 128, o_at = tmem + lanes + 256 + group * D;
        uint8_t *mine = smem + SM::Q + group * SM::TILE + (warp & 3) * (32 * D * 2);  // the warp's 32 rows of Q
        for (uint32_t rt = tile0; rt < row_tiles; rt += tile_step) {
            const Span sp = span_of(rt);
            // Q of the warp's rows, eight at a time, four lanes a row; bf16 rows scaled by a power of two to just below 2^14
            float scale = 0.0f;
            {
                constexpr int PIECES = D / 8, PER = PIECES < 4 ? 1 : PIECES / 4;
                auto fetch = [&](int q, uint4 (&raw)[PER]) {
                    // rows past the last read it again; their scores are masked
                    const int rr = min(sp.r0 + 32 * warp + 8 * q + (lane & 7), rows - 1), i = rr / (int)a.group, h = rr - i * (int)a.group;
                    const uint16_t *from = static_cast<const uint16_t *>(a.q) + (t0 + i) * a.q_token + (long long)(head * a.group + h) * a.q_head;
                    if (a.q_vec16) {
#pragma unroll
                        for (int u = 0; u < PER; ++u) raw[u] = __ldg(reinterpret_cast<const uint4 *>(from) + min((lane >> 3) + 4 * u, PIECES - 1));
                    } else {
#pragma unroll
                        for (int u = 0; u < PER; ++u) {
                            const uint16_t *y = from + 8 * min((lane >> 3) + 4 * u, PIECES - 1);
                            raw[u] = make_uint4(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16, y[4] | (uint32_t)y[5] << 16, y[6] | (uint32_t)y[7] << 16);
                        }
                    }
                };
                // the loop is kept rolled: code that runs once costs its way into the instruction cache
                uint4 raw[PER], ahead[PER];
                fetch(0, ahead);
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int u = 0; u < PER; ++u) raw[u] = ahead[u];
                    if (q < 3) fetch(q + 1, ahead);
                    // the scale's sign goes into Q, and so does a scale of 0: the masked scores' -inf times it has to stay -inf
                    float mul = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
                    const float sign = a.scale == 0.0f ? 0.0f : copysignf(1.0f, a.scale);
                    if (a.q_type == MGB_F16) {
                        const __half2 s = __float2half2_rn(sign);
                        auto signed2 = [&](uint32_t w) {
                            const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&w), s);
                            return *reinterpret_cast<const uint32_t *>(&x);
                        };
#pragma unroll
                        for (int u = 0; u < PER; ++u) raw[u] = make_uint4(signed2(raw[u].x), signed2(raw[u].y), signed2(raw[u].z), signed2(raw[u].w));
                    } else {
                        uint32_t top = 0;  // of the magnitudes' bits
#pragma unroll
                        for (int u = 0; u < PER; ++u) {
                            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) top = max(top, max(w[e] << 16 & 0x7fff0000u, w[e] & 0x7fff0000u));
                        }
                        top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        // 2^shift in two factors, since either may leave the range of f32 alone
                        const int shift = top && top < 0x7f800000u ? 140 - (int)(top >> 23) : 0;
                        const int s1 = max(-100, min(100, shift)), s2 = shift - s1;
                        const float f1 = sign * __int_as_float((127 + s1) << 23), f2 = __int_as_float((127 + s2) << 23);
                        // above 0, so that -inf times it stays -inf
                        mul = fmaxf(mul * __int_as_float((127 - s1) << 23) * __int_as_float((127 - s2) << 23), 1.2e-38f);
                        auto half2_of = [&](uint32_t w) { return pack(__uint_as_float(w << 16) * f1 * f2, __uint_as_float(w & 0xffff0000u) * f1 * f2); };
#pragma unroll
                        for (int u = 0; u < PER; ++u) raw[u] = make_uint4(half2_of(raw[u].x), half2_of(raw[u].y), half2_of(raw[u].z), half2_of(raw[u].w));
                    }
                    const float its = __shfl_sync(0xffffffffu, mul, lane & 7);
                    if (lane >> 3 == q) scale = its;
#pragma unroll
                    for (int u = 0; u < PER; ++u)
                        if ((lane >> 3) + 4 * u < PIECES) *reinterpret_cast<uint4 *>(mine + piece<D>(8 * q + (lane & 7), (lane >> 3) + 4 * u)) = raw[u];
                }
            }
            fence_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cta(&sh.q_full);

            const int lim = row < sp.live ? limit((sp.r0 + row) / (int)a.group) : 0;
            float m = kLowest, l = 0.0f;
            int exp_v = -126;
            bool ok = !sh.lost;
            const int count = group < sp.groups ? sp.count : 0;
            for (int j = 0; j < count && ok; ++j) {
                const int key0 = (sp.first + j) * kKeys;
                ok = wait(&sh.s_full[group], ss[group] + j);
                if (!ok) break;
                fence_after();
                float2 x[kKeys / 2];
#pragma unroll
                for (int c0 = 0; c0 < kKeys; c0 += 32) tmem_load32(s_at + c0, reinterpret_cast<uint32_t *>(&x[c0 / 2]));
                const uint32_t slot = (ks + j) & 3, holes = sh.holes[slot];
                const float *kscale = sh.k_scale[slot];
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
                tmem_wait_load();
                if constexpr (Q8) {
#pragma unroll
                    for (int c = 0; c < kKeys / 2; c += 2) {
                        const float4 d = *reinterpret_cast<const float4 *>(kscale + 2 * c);
                        x[c] = mul2(x[c], make_float2(d.x, d.y));
                        x[c + 1] = mul2(x[c + 1], make_float2(d.z, d.w));
                    }
                }
                if (key0 + kKeys > sp.all || holes) {
#pragma unroll
                    for (int c = 0; c < kKeys / 2; ++c) {
                        const int key = key0 + 2 * c;
                        const bool hole = (holes >> ((2 * c) >> 4)) & 1;
                        if (key >= lim || hole) x[c].x = kLowest;
                        if (key + 1 >= lim || hole) x[c].y = kLowest;
                    }
                }
                float top[4] = {kLowest, kLowest, kLowest, kLowest};
#pragma unroll
                for (int c = 0; c < kKeys / 2; ++c) top[c & 3] = max3(top[c & 3], x[c].x, x[c].y);
                const float best = fmaxf(max3(top[0], top[1], top[2]), top[3]) * scale;
                const float *vscale = sh.v_scale[slot];
                int e = Q8 ? sh.v_exp[slot] : exp_v;
                if (Q8 && e == kFolded) {  // V's scales go into P
                    float most = 0.0f;
#pragma unroll 4
                    for (int key = 0; key < kKeys; key += 4) {
                        const float4 d = *reinterpret_cast<const float4 *>(vscale + key);
                        const float most4[4] = {fabsf(d.x), fabsf(d.y), fabsf(d.z), fabsf(d.w)};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (key0 + key + i < lim && !((holes >> (key >> 4)) & 1)) most = fmaxf(most, most4[i]);
                    }
                    e = max(exp_v, min(126, (__float_as_int(most) >> 23) - 126));
                }
                if (__any_sync(0xffffffffu, best > m + kSlack || e != exp_v)) {
                    const float now = fmaxf(m, best), w = m == kLowest ? 0.0f : exp2_of(m - now);
                    m = now;
                    l *= w;
                    if (j > 0) rescale_o(Q8 ? w * power_of_2(exp_v - e) : w);
                    exp_v = e;
                }
                const float z = kRaise - (m == kLowest ? 0.0f : m);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c0 = 0; c0 < kKeys / 2; c0 += 16) {
                    uint32_t p[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        float2 y = fma2(x[c0 + c], make_float2(scale, scale), make_float2(z, z));
                        // 8-bit: a quarter of them by products, 5 to 9 % faster; f16, whose softmax
                        // does less besides: 1 to 4 % slower
                        if (Q8 && (c & 3) == 3) {
                            y = exp2_poly(y);
                        } else {
                            y.x = exp2_of(y.x);
                            y.y = exp2_of(y.y);
                        }
                        sum[c & 1] = add2(sum[c & 1], y);
                        p[c] = pack(y.x, y.y);
                    }
                    tmem_store16(s_at + c0, p);  // over the scores
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_store();
                // In a pass of its own: within the loop above it cost 5 to 11 % on every tile, in registers; and so does
                // keeping the flag in one.
                if (Q8 && *reinterpret_cast<volatile int *>(&sh.v_exp[slot]) == kFolded) {
                    const float over_e = __int_as_float((127 - exp_v) << 23);
#pragma unroll 1
                    for (int c0 = 0; c0 < kKeys / 2; c0 += 16) {
                        uint32_t p[16];
                        tmem_load16(s_at + c0, p);
                        tmem_wait_load();
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            const int key = 2 * (c0 + c);
                            const float2 d = *reinterpret_cast<const float2 *>(vscale + key), y = unpack(p[c]);
                            // 0 where the key is not seen, whatever its scale
                            const bool hole = (holes >> (key >> 4)) & 1;
                            p[c] = pack(key0 + key < lim && !hole ? y.x * (d.x * over_e) : 0.0f,
                                        key0 + key + 1 < lim && !hole ? y.y * (d.y * over_e) : 0.0f);
                        }
                        tmem_store16(s_at + c0, p);
                    }
                    tmem_wait_store();
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cta(&sh.p_full[group]);
            }
            if (sp.count > 0 && ok) ok = wait(&sh.o_full, os);
            fence_after();
            if (!ok) l = __int_as_float(0x7fffffff);
            // a row that sees nothing has at most 128 times 2^-126 a tile
            const bool some = count > 0 && !(l < 1e-30f);
            const float f = some ? (Q8 ? power_of_2(exp_v) : 1.0f) / l : 0.0f;
            if (sh.wild_any) {
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 16) {
                    uint32_t raw[16];
                    tmem_load16(o_at + c0, raw);
                    tmem_wait_load();
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        for (int k = 0; k < 3; ++k)
                            if (sh.wild[k][c0 + c] < lim)
                                raw[c] = __float_as_uint(__uint_as_float(raw[c]) + __uint_as_float(k == 0 ? 0x7fffffffu : k == 1 ? 0x7f800000u : 0xff800000u));
                    tmem_store16(o_at + c0, raw);
                }
                tmem_wait_store();
            }
            if (parts == 1) {
                if (a.o_vec16) {
                    // through the warp's rows of Q, which no product reads any more, to whole rows of 16-bit numbers
                    constexpr int PIECES = D / 8;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t raw[16], w[8];
                        tmem_load16(o_at + c0, raw);
                        tmem_wait_load();
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const float u = some ? __uint_as_float(raw[2 * c]) * f : 0.0f;
                            const float v = some ? __uint_as_float(raw[2 * c + 1]) * f : 0.0f;
                            w[c] = to_16(ok ? u : l, a.o_type) | (uint32_t)to_16(ok ? v : l, a.o_type) << 16;
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            *reinterpret_cast<uint4 *>(mine + piece<D>(lane, c0 / 8 + c)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int u = lane; u < 32 * PIECES; u += 32) {
                        const int r = u / PIECES, c = u % PIECES;
                        const int rr = sp.r0 + 32 * warp + r;
                        if (32 * warp + r >= sp.live) break;
                        const int i = rr / (int)a.group, h = rr - i * (int)a.group;
                        const int64_t to = (t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head + 8 * c;
                        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + to) = *reinterpret_cast<const uint4 *>(mine + piece<D>(r, c));
                    }
                    __syncwarp();
                } else {
                    const int rr = sp.r0 + row;
                    const int i = rr / (int)a.group, h = rr - i * (int)a.group;
                    const int64_t to = (t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t raw[16];
                        tmem_load16(o_at + c0, raw);
                        tmem_wait_load();
                        if (row >= sp.live) continue;
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            store1(a.out, (size_t)(to + c0 + c), a.o_type, !ok ? l : some ? __uint_as_float(raw[c]) * f : 0.0f);
                    }
                }
            } else {
                // this CTA's part of the row where the keys stood, turned by 16 bytes a row so that stores miss each
                // other's banks
                float *o = reinterpret_cast<float *>(smem + SM::K) + row * D;
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 16) {
                    uint32_t raw[16];
                    tmem_load16(o_at + c0, raw);
                    tmem_wait_load();
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        float4 x = make_float4(__uint_as_float(raw[c]) * f, __uint_as_float(raw[c + 1]) * f,
                                               __uint_as_float(raw[c + 2]) * f, __uint_as_float(raw[c + 3]) * f);
                        if (!some) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        reinterpret_cast<float4 *>(o)[((c0 + c) / 4 + row) % (D / 4)] = x;
                    }
                }
                sh.m[row] = m;
                sh.l[row] = l;
            }
            asm volatile("barrier.sync 1, %0;" ::"n"(kSoftWarps * 32) : "memory");
            for (int u = tid; u < 3 * D; u += kSoftWarps * 32) (&sh.wild[0][0])[u] = 0x7fffffff;
            if (tid == 0) sh.wild_any = 0;
            fence_before();
            meet(parts > 1);
            if (parts > 1) {
                namespace cg = cooperative_groups;
                auto cluster = cg::this_cluster();
                // the parts' weights of a row
                if (row < sp.live) {
                    float its[8], sum = 0.0f, best = kLowest;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        its[c] = c < (int)parts ? *cluster.map_shared_rank(&sh.m[row], c) : kLowest;
                        best = fmaxf(best, its[c]);
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float lc = c < (int)parts ? *cluster.map_shared_rank(&sh.l[row], c) : 0.0f;
                        its[c] = lc != lc ? lc : its[c] == kLowest ? 0.0f : exp2_of(its[c] - best) * lc;
                        sum += its[c];
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) sh.weight[c][row] = sum < 1e-30f ? 0.0f : its[c] / sum;
                }
                asm volatile("barrier.sync 1, %0;" ::"n"(kSoftWarps * 32) : "memory");
                const float4 *o = reinterpret_cast<const float4 *>(smem + SM::K);
                for (int u = (int)part * (kSoftWarps * 32) + tid; u < sp.live * (D / 4); u += (int)parts * (kSoftWarps * 32)) {
                    const int r = u / (D / 4), c4 = u % (D / 4);
                    float4 from[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        from[c] = c < (int)parts ? *cluster.map_shared_rank(o + r * (D / 4) + (c4 + r) % (D / 4), c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float f = sh.weight[c][r];
                        x[0] += f * from[c].x, x[1] += f * from[c].y, x[2] += f * from[c].z, x[3] += f * from[c].w;
                    }
                    const int rr = sp.r0 + r;
                    const int i = rr / (int)a.group, h = rr - i * (int)a.group;
                    store4(a.out, (t0 + i) * a.o_token + (long long)(head * a.group + h) * a.o_head + 4 * c4, a.o_type, a.o_vec, x);
                }
                meet(true);
            }
            next_tile(sp);
        }
    } else if (warp < kMmaWarp) {
        // ---------------------------------------------------------- loading
        set_registers<kLoadRegs>();
        const int lw = warp - kSoftWarps;
        constexpr int ESZ = Q8 ? 1 : 2, PIECES = D * ESZ / 16;   // 16-byte pieces of a row in the cache
        constexpr int PER = kKeys * PIECES / (kLoadWarps * 32);  // pieces of a thread and tile
        constexpr int ROWS = PIECES < 4 ? PER : 4;               // and its rows
        // A warp has 32 rows of the tile; an access takes eight rows and neighbouring pieces.
        auto row_no = [&](int k) { return PIECES < 4 ? 32 * lw + (lane & 7) + 8 * ((lane + 32 * k) / (8 * PIECES)) : 32 * lw + (lane & 7) + 8 * k; };
        auto row_ix = [](int u) { return PIECES < 4 ? u : u / (PER / ROWS); };
        auto piece_no = [&](int u) { return PIECES < 4 ? ((lane + 32 * u) >> 3) % PIECES : (lane >> 3) + 4 * (u % (PER / ROWS)); };
        for (uint32_t rt = tile0; rt < row_tiles; rt += tile_step) {
            const Span sp = span_of(rt);
            bool ok = true;
            // page of 16-key group `lane` of tile j (lanes 0-7), of no page where there is none
            auto pages_of = [&](int j) {
                const int key = (sp.first + j) * kKeys + 16 * lane;
                return lane < 8 && j < sp.count && key < sp.end ? (uint32_t)__ldg(table + ((uint32_t)key >> a.kv.page_log2)) : 0xffffffffu;
            };
            // where row r of tile j lies, in rows of the cache; -1 where it does not exist
            auto row_of = [&](int j, uint32_t pages, int r) -> int64_t {
                const int key = (sp.first + j) * kKeys + r;
                const uint32_t pg = __shfl_sync(0xffffffffu, pages, r >> 4);
                return key < sp.end && pg < a.kv.pages ? (int64_t)a.kv.row(pg, head, (uint32_t)key & ((1u << a.kv.page_log2) - 1)) : -1;
            };
            auto publish = [&](uint64_t *bar) {
                fence_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cta(bar);
            };
            int64_t at[ROWS];
            auto rows_of = [&](int j, uint32_t pages) {
#pragma unroll
                for (int k = 0; k < ROWS; ++k) at[k] = row_of(j, pages, row_no(k));
            };
            uint32_t pages = pages_of(0), next = pages_of(1);
            rows_of(0, pages);
            if constexpr (Q8) {
                const uint8_t *kbase = static_cast<const uint8_t *>(a.kv.k), *vbase = static_cast<const uint8_t *>(a.kv.v);
                uint4 kraw[PER], vraw[PER];
                float kd, vd[kLoadWarps];  // scales of key 32 lw + lane, of keys lane, 32 + lane, ...
                auto fetch = [&](const uint8_t *base, uint4 (&raw)[PER]) {
#pragma unroll
                    for (int u = 0; u < PER; ++u)
                        raw[u] = at[row_ix(u)] >= 0 ? __ldg(reinterpret_cast<const uint4 *>(base + at[row_ix(u)] * D) + piece_no(u))
                                                    : make_uint4(0, 0, 0, 0);
                };
                auto fetch_scales = [&](int j, uint32_t pg) {
#pragma unroll
                    for (int w = 0; w < kLoadWarps; ++w) {
                        const int64_t row = row_of(j, pg, 32 * w + lane);
                        if (w == lw) kd = row >= 0 ? __ldg(a.kv.ks + row) : 0.0f;
                        vd[w] = row >= 0 ? __ldg(a.kv.vs + row) : 0.0f;
                    }
                };
                // bits of the largest of the tile's 128 scales (NaN above all), of the smallest but 0
                auto largest = [&](const float (&d)[kLoadWarps]) {
                    uint32_t top = 0;
#pragma unroll
                    for (int w = 0; w < kLoadWarps; ++w) top = max(top, __float_as_uint(fabsf(d[w])));
                    return __reduce_max_sync(0xffffffffu, top);
                };
                auto smallest = [&](const float (&d)[kLoadWarps]) {
                    uint32_t low = 0x7f7fffff;
#pragma unroll
                    for (int w = 0; w < kLoadWarps; ++w)
                        if (d[w] != 0.0f) low = min(low, __float_as_uint(fabsf(d[w])));
                    return __reduce_min_sync(0xffffffffu, low);
                };
                // the scale of the warp's key `lane`
                auto own_scale = [&](const float (&d)[kLoadWarps]) {
                    float x = d[0];
#pragma unroll
                    for (int w = 1; w < kLoadWarps; ++w)
                        if (w == lw) x = d[w];
                    return x;
                };
                // as a high and a low f16 part
                auto parts_of = [&](float x) {
                    const __half hi = __float2half_rn(x);
                    const __half2 both = __halves2half2(hi, __float2half_rn(x - __half2float(hi)));
                    return *reinterpret_cast<const uint32_t *>(&both);
                };
                // codes (times scales, one rounding) into a stage
                auto unpack_tile = [&](const uint4 (&raw)[PER], bool scaled, uint32_t scales, uint8_t *tile) {
#pragma unroll
                    for (int u = 0; u < PER; ++u) {
                        const int r = row_no(row_ix(u));
                        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                        const uint32_t d = __shfl_sync(0xffffffffu, scales, r & 31);
                        const uint32_t d_hi = __byte_perm(d, 0, 0x1010), d_lo = __byte_perm(d, 0, 0x3232);
                        const __half2 hi2 = *reinterpret_cast<const __half2 *>(&d_hi), lo2 = *reinterpret_cast<const __half2 *>(&d_lo);
                        uint32_t h[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            h[i] = codes2(w[i / 2] ^ 0x80808080u, i & 1 ? 0x4342 : 0x4140);
                            if (scaled) {
                                const __half2 q = *reinterpret_cast<const __half2 *>(&h[i]);
                                const __half2 v = __hfma2(q, hi2, __hmul2(q, lo2));
                                h[i] = *reinterpret_cast<const uint32_t *>(&v);
                            }
                        }
                        uint8_t *to = tile + piece<D>(r, 2 * piece_no(u));
                        *reinterpret_cast<uint4 *>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4 *>(to + 128) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                };
                int exp_v = -126;
                if (sp.count > 0) {
                    fetch(kbase, kraw);
                    fetch_scales(0, pages);
                }
                for (int j = 0; j < sp.count && ok; ++j) {
                    const uint32_t stage = (ks + j) & 1, turn = (ks + j) >> 1, slot = (ks + j) & 3;
                    fetch(vbase, vraw);
                    const uint32_t holes = __ballot_sync(0xffffffffu, pages >= a.kv.pages) & 0xff;
                    const float own = own_scale(vd);
                    const uint32_t top = largest(vd);
                    // scales less than 2^13 apart: even codes of 1 times the smallest are normal f16 numbers over the
                    // largest's exponent, which the scales stay below
                    const bool folded = j >= sp.clean && (top >= 0x7f800000u || (int)(top >> 23) - (int)(smallest(vd) >> 23) >= 13);
                    if (!folded) exp_v = max(exp_v, min(126, (int)(top >> 23) - 126));
                    const uint32_t v_own = parts_of(folded ? 1.0f : own * __int_as_float((127 - exp_v) << 23));
                    if (turn > 0) ok = wait(&sh.k_free[stage], turn - 1);
                    if (!ok) break;
                    sh.k_scale[slot][32 * lw + lane] = kd;
                    sh.v_scale[slot][32 * lw + lane] = own;
                    if (lw == 0 && lane == 0) {
                        sh.v_exp[slot] = folded ? kFolded : exp_v;
                        sh.holes[slot] = holes;
                    }
                    unpack_tile(kraw, false, 0, smem + SM::K + stage * SM::TILE);
                    publish(&sh.k_full[stage]);
                    if (j + 1 < sp.count) {  // on their way while V is unpacked
                        rows_of(j + 1, next);
                        fetch(kbase, kraw);
                        fetch_scales(j + 1, next);
                        pages = next;
                        next = pages_of(j + 2);
                    }
                    if (turn > 0) ok = wait(&sh.v_free[stage], turn - 1);
                    if (!ok) break;
                    unpack_tile(vraw, true, v_own, smem + SM::V + stage * SM::TILE);
                    publish(values_at(sp, j));
                }
            } else {
                // copies of tile j's K or V into its stage, once the products with what was there are done
                auto copy = [&](const void *base, uint32_t part_at, uint64_t (&free)[2], int j) {
                    const uint32_t stage = (ks + j) & 1, turn = (ks + j) >> 1;
                    if (j < sp.count && turn > 0) ok = ok && wait(&free[stage], turn - 1);
                    if (j < sp.count && ok) {
                        const uint32_t tile = smem_u32(smem + part_at + stage * SM::TILE);
#pragma unroll
                        for (int u = 0; u < PER; ++u) {
                            const int64_t row = at[row_ix(u)];
                            const uint8_t *p = static_cast<const uint8_t *>(base) + (row >= 0 ? row : 0) * (D * 2) + 16 * piece_no(u);
                            // what lies beyond the 0 or 16 bytes read becomes zeros
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tile + piece<D>(row_no(row_ix(u)), piece_no(u))),
                                         "l"(p), "r"(row >= 0 ? 16 : 0));
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                copy(a.kv.k, SM::K, sh.k_free, 0);
                copy(a.kv.v, SM::V, sh.v_free, 0);
                for (int j = 0; j < sp.count && ok; ++j) {
                    const uint32_t stage = (ks + j) & 1;
                    const uint32_t holes = __ballot_sync(0xffffffffu, pages >= a.kv.pages) & 0xff;
                    // what has arrived goes out before the next wait for room
                    if (lw == 0 && lane == 0) sh.holes[(ks + j) & 3] = holes;
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    publish(&sh.k_full[stage]);
                    pages = next;
                    rows_of(j + 1, pages);
                    next = pages_of(j + 2);
                    copy(a.kv.k, SM::K, sh.k_free, j + 1);
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    publish(values_at(sp, j));
                    copy(a.kv.v, SM::V, sh.v_free, j + 1);
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            meet(parts > 1);
            if (parts > 1) meet(true);
            next_tile(sp);
        }
    } else {
        // ---------------------------------------------------------- products
        set_registers<kMmaRegs>();
        constexpr uint32_t QK = instruction(kKeys, false), PV = instruction(D, true);
        for (uint32_t rt = tile0; rt < row_tiles; rt += tile_step) {
            const Span sp = span_of(rt);
            if (__shfl_sync(0xffffffffu, warp, 0) == kMmaWarp && elected()) {
                const uint64_t q0 = operand(smem_u32(smem + SM::Q), 128, D * 16), k0 = operand(smem_u32(smem + SM::K), 128, D * 16);
                const uint64_t v0 = operand(smem_u32(smem + SM::V), D * 16, 128);
                // an operand `by` 16-byte units on; computed where it is used: there are too many to keep in registers
                auto moved = [](uint64_t from, uint32_t by) {
                    uint32_t low = (uint32_t)from + by;
                    asm volatile("" : "+r"(low));
                    return (from >> 32 << 32) | low;
                };
                auto scores = [&](int g, int stage) {
                    const uint64_t q = moved(q0, g * (SM::TILE >> 4)), k = moved(k0, stage * (SM::TILE >> 4));
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) mma_ss(tmem + g * 128, q + s * 16, k + s * 16, QK, s > 0);
                    commit(&sh.s_full[g]);
                    commit(&sh.k_free[stage]);
                    if (sp.groups == 1) commit(&sh.k_free[stage]);
                };
                auto values = [&](int g, int stage, bool add) {
                    const uint64_t v = moved(v0, stage * (SM::TILE >> 4));
#pragma unroll
                    for (int s = 0; s < kKeys / 16; ++s)
                        mma_ts(tmem + 256 + g * D, tmem + g * 128 + s * 8, v + s * (2 * D), PV, add || s > 0);
                    commit(&sh.v_free[stage]);
                    if (sp.groups == 1) commit(&sh.v_free[stage]);
                };
                bool ok = mbar_wait(&sh.q_full, turns & 1);
                if (sp.count > 0) {
                    // the scores take the place of P, so a group's next follow its product with the values
                    for (int j = -1; j < sp.count && ok; ++j) {
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            if (g == 1 && sp.groups == 1) break;
                            if (j >= 0) {
                                ok = ok && mbar_wait(&sh.p_full[g], (ss[g] + j) & 1);
                                if (g == 0) ok = ok && mbar_wait(&sh.v_full[(ks + j) & 1], ((ks + j) >> 1) & 1);
                                fence_after();
                                if (ok) values(g, (ks + j) & 1, j > 0);
                            }
                            if (j + 1 < sp.count) {
                                if (g == 0) ok = ok && mbar_wait(&sh.k_full[(ks + j + 1) & 1], ((ks + j + 1) >> 1) & 1);
                                fence_after();
                                if (ok) scores(g, (ks + j + 1) & 1);
                            }
                        }
                        if (*reinterpret_cast<volatile int *>(&sh.lost)) ok = false;
                    }
                    // also after a lost wait: nothing in flight when the CTA leaves
                    commit(&sh.o_full);
                    ok = mbar_wait(&sh.o_full, os & 1) && ok;
                }
                if (!ok) sh.lost = 1;
            }
            if (warp > kMmaWarp) {
                // values that some rows do not see: 0 times an infinity or NaN would reach them
                const int me = tid - 32 * (kMmaWarp + 1);
                bool ok = true;
                for (int j = Q8 ? sp.count : sp.clean; j < sp.count && ok; ++j) {
                    const uint32_t stage = (ks + j) & 1;
                    ok = wait(&sh.v_raw[(cleaned + j - sp.clean) & 1], (cleaned + j - sp.clean) >> 1);
                    if (!ok) break;
                    uint8_t *tile = smem + SM::V + stage * SM::TILE;
#pragma unroll 1
                    for (int u = me; u < kKeys * (D / 8); u += 32 * (kWarps - kMmaWarp - 1)) {
                        const int r = u % kKeys, c = u / kKeys;
                        uint4 x = *reinterpret_cast<const uint4 *>(tile + piece<D>(r, c));
                        // an exponent of ones carries into its half's sign
                        auto hit = [](uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; };
                        if (!(hit(x.x) | hit(x.y) | hit(x.z) | hit(x.w))) continue;
#pragma unroll 1
                        for (int e = 0; e < 8; ++e) {
                            uint16_t *y = reinterpret_cast<uint16_t *>(tile + piece<D>(r, c)) + e;
                            if ((*y & 0x7c00) != 0x7c00) continue;
                            atomicMin(&sh.wild[*y & 0x3ff ? 0 : 1 + (*y >> 15)][8 * c + e], (sp.first + j) * kKeys + r);
                            *y = 0;
                            sh.wild_any = 1;
                        }
                    }
                    fence_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_cta(&sh.v_full[stage]);
                        if (me < kLoadWarps - (kWarps - kMmaWarp - 1)) mbar_arrive_cta(&sh.v_full[stage]);  // it counts the loaders
                    }
                }
            }
            __syncwarp();
            fence_before();
            meet(parts > 1);
            if (parts > 1) meet(true);
            next_tile(sp);
        }
        if (tid == kMmaWarp * 32 && *reinterpret_cast<volatile int *>(&sh.lost)) g_wait_lost = 1;
        if (warp == kMmaWarp) {
            fence_after();
            __syncwarp();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        }
    }
}

}  // namespace tiles
