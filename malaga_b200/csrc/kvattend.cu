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
//    2^7 p (d_v 2^-E), E a running exponent of the largest d_v, so that f16's
//    narrow range costs nothing.
//  * q goes in as f16: exact for f16 q; bf16 q is first scaled by a power of
//    two per row, and then exact but for numbers 2^-38 of the row's largest.
//  * for f32 q both are split into a high and a low f16 part (SPLIT), two
//    products each, which keeps 22 bits.
//  * Few rows over 8-bit caches: q is cut into 8-bit digits instead, so that
//    K's codes go into the integer mma as they are (mma.m16n8k32 measured the
//    rate of the f16 mma.m16n8k16, and unpacking K was a quarter of the
//    instructions). Two digits hold q to 2^-15 of the row's largest number, an
//    eighth of the error of P's rounding; three, for f32 q, to 2^-22. The sums
//    are exact.
#include <cooperative_groups.h>

#include <cstdlib>
#include <type_traits>

#include "numerics.cuh"
#include "serving.cuh"
#include "sync.cuh"

namespace mgb {
namespace {

#define kLowest __int_as_float(0xff800000)
constexpr float kLog2e = 1.44269504088896341f;

struct AttendArgs {
    KvView kv;
    SeqView seq;
    const void *q;
    void *out;
    long long q_token, q_head, o_token, o_head;
    int q_type, o_type, causal;
    bool o_vec, q_vec16, o_vec16;  // rows that allow accesses of four numbers, of eight 16-bit ones
    uint32_t group;  // query heads of a cache head
    bool overlap;    // the kernel for few rows runs beside the one for many
    uint32_t turn;   // the number of a call that launches both, else 0
    uint32_t few;    // sequences with at most this many rows a cache head go to the kernel for few rows
    float scale;     // times log2(e)
    uint32_t span;   // few rows: a sequence is cut into one part each `span` keys
    int withhold;    // test hook: the stage of keys that never fills in the tiles' first CTA, or -1
};

// Set by a kernel in which a wait ran out, until mgb_kv_status reads it.
__device__ uint32_t g_wait_lost;

// A call with both kernels: the second starts when every CTA of the first has, which
// is after all work before the call has ended. That the second sees that work's
// writes takes more than that: the first CTA of the tiles, for which they are visible,
// releases the call's number here, and whoever acquires it sees them, too. A CTA that
// does not find it (calls of several streams share the places) waits for the tiles.
// The last CTA to stay takes the number away, so that a replayed graph starts anew.
constexpr uint32_t kTurns = 256;
__device__ uint32_t g_turn[kTurns];

__device__ __forceinline__ void give_turn(uint32_t turn) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(&g_turn[turn % kTurns]), "r"(turn) : "memory");
}
__device__ __forceinline__ void take_turn(uint32_t turn) {
    uint32_t got;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(got) : "l"(&g_turn[turn % kTurns]) : "memory");
    if (got != turn) wait_for_previous();
}

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float power_of_2(int e) { return e < -126 ? 0.0f : __int_as_float((e + 127) << 23); }

// 1 / the power of two above d >= 0, kept between 2^-126 and 2^126; the inverse of such a number.
__device__ __forceinline__ float over(float d) { return __int_as_float((253 - min(252, __float_as_int(d) >> 23)) << 23); }
__device__ __forceinline__ float inverse(float power) { return __int_as_float((254 << 23) - __float_as_int(power)); }

__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8-bit integers, sums of 32 (or, with one word of a row, 16) products.
__device__ __forceinline__ void mma8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k16.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
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

// BYTES bytes of shared memory at p (aligned to their size, at most 16) into words.
template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t *w) {
    if constexpr (BYTES == 16) {
        const uint4 x = *reinterpret_cast<const uint4 *>(p);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (BYTES == 8) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x, w[1] = x.y;
    } else if constexpr (BYTES == 4) {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
        w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
}

// ---------------------------------------------------------------------------
// Few rows: tiles of 8 or 16 rows (token, head of the group) of one cache head.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that
// the rows are the 8-wide side of mma.m16n8k16 and a single query wastes as
// little as it can. A lane reads K and V from shared memory in 16-byte pieces
// that are its parts of the mma's A operand: the order of the head dimension
// inside q . k is free (Q is permuted the same way), and so is the order of the
// rows of O^T. For K, four lanes share a key and take every fourth vector of
// its row; for V, eight lanes share a key, and a byte permute pairs two keys.
// movmatrix turns P^T, as it leaves the first product, into the B operand of
// the second.
//
// A warp takes every fourth stage of keys and copies it itself, asynchronously,
// into its own ring of stages: each 16 keys of K, of V and of their scales are a
// contiguous run of a page, and what is in flight depends neither on registers
// nor on the page table's latency. (Bulk copies, one for each run, took a loop
// over the issuing lanes that was a third of all instructions.) The 16-byte
// pieces of a row stand turned by its key, so that the reads below meet in few
// banks. A warp keeps its own maximum, sum and output. The maximum only has to
// be near: it is raised when a score passes it
// by 2^8, so most blocks need one vote and no reduction across lanes. Warps
// join in shared memory, the CTAs of a cluster (which cut the keys among them)
// through distributed shared memory, in a fixed order.
//
// What bounds it: HBM with long f16 caches (6.3 TB/s at dim 128), the instructions a
// key with 8-bit ones (8 sequences, 233,369 positions, 8 heads of 128, four rows
// each: 116 us, 4.2 TB/s), latencies with short ones (one row of 33 positions, 16
// heads of 64: 4.1 us; 64 sequences of 272 positions on average and 1024 at most, 16
// heads of 64, 8 bits: 22 us, of which the longest sequence's loop is 12).

template <int D, bool Q8>
struct Frag {
    static constexpr int ESZ = Q8 ? 1 : 2;
    static constexpr int KB = D * ESZ / 4 < 16 ? D * ESZ / 4 : 16;  // bytes of a K load
    static constexpr int KN = D * ESZ / 4 / KB;                     // K loads of a key and lane
    static constexpr int VB = D * ESZ / 8 < 16 ? D * ESZ / 8 : 16;
    static constexpr int VN = D * ESZ / 8 / VB;
    static constexpr int KW = D * ESZ / 16, VW = D * ESZ / 32 ? D * ESZ / 32 : 1;  // words of a key and lane
    static constexpr int STEPS = D / 16;
    // Piece c (16 bytes) of key `key` stands at piece c ^ turn(key) of its row in a
    // stage. turn is linear over xor, and so are the places that a lane's reads and
    // copies derive from its first one.
    static constexpr int PIECES = D * ESZ / 16, ROW = D * ESZ;
    static __host__ __device__ constexpr int turn(int key) {
        return PIECES >= 8 ? ((key >> 1) & 3) << 1 ^ (key & 1) << 2 : PIECES == 4 ? key & 2 : 0;
    }
    // place of byte b of key `key`'s row
    static __device__ __forceinline__ int byte(int key, int b) { return key * ROW + ((b / 16 ^ turn(key)) * 16) + b % 16; }
    // CTAs of an SM that the registers have to leave room for
    static constexpr int ctas(int nt) { return D < 128 ? (nt == 1 ? 5 : 3) : nt == 2 && Q8 ? 2 : 3; }
    static constexpr int STATIC = 32 * D + 1536;  // static shared memory of a CTA a tile of 8 rows, at most
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

// Sequences of at most kFewRows rows a cache head go to the kernel for few rows;
// the others to the tensor-core tiles, but where that takes longer (launch()).
constexpr int kFewRows = 64;
constexpr int kRowWarps = 4, kRowThreads = kRowWarps * 32;
constexpr float kSlack = 8.0f;  // a score may pass the running maximum by 2^8
constexpr float kRaise = 7.0f;  // p is held as 2^7 p, up to 2^15

// A stage: BLOCKS times 16 keys of K, of V, then (8-bit caches) of their scales.
// 8-bit codes come 32 keys at a time, which halves what a stage costs beside its
// arithmetic; f16 ones, twice as large, 16.
template <int D, bool Q8>
struct Ring {
    static constexpr int BLOCKS = Q8 ? 2 : 1;
    static constexpr int ROWS = 16 * D * (Q8 ? 1 : 2), SCALES = Q8 ? 64 : 0;  // bytes of a block
    static constexpr int V = BLOCKS * ROWS, KS = 2 * V, VS = KS + BLOCKS * SCALES, STAGE = VS + BLOCKS * SCALES;
    // about 12 KB a warp, 2 to 4 stages: more would cost CTAs of an SM
    static constexpr int FIT = 12800 / STAGE;
    static constexpr int N = FIT < 2 ? 2 : FIT > 4 ? 4 : FIT;
    static constexpr int BYTES = kRowWarps * N * STAGE;
};

template <int D, bool Q8>
struct Block {  // a lane's share of 16 keys
    uint32_t k[2][Frag<D, Q8>::KW];  // keys g, g + 8
    uint32_t v[4][Frag<D, Q8>::VW];  // keys 2t, 2t + 1, 2t + 8, 2t + 9
    float ks[2], vs[2];              // scales of keys g, g + 8
    // left: keys that exist; the places of the others hold anything
    // k_at, v_at: F::byte(g, t * KB), F::byte(2 * t, g * VB)
    __device__ __forceinline__ void load_k(const uint8_t *stage, int blk, int g, int k_at) {
        using F = Frag<D, Q8>;
        using R = Ring<D, Q8>;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int c = 0; c < F::KN; ++c)
                load_words<F::KB>(stage + blk * R::ROWS + 8 * u * F::ROW + (k_at ^ 64 * c), &k[u][c * (F::KB / 4)]);
            if constexpr (Q8) ks[u] = reinterpret_cast<const float *>(stage + R::KS)[16 * blk + g + 8 * u];
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t *stage, int blk, int left, int g, int t, int v_at) {
        using F = Frag<D, Q8>;
        using R = Ring<D, Q8>;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int c = 0; c < F::VN; ++c)
                load_words<F::VB>(stage + R::V + blk * R::ROWS + ((u & 1) + 8 * (u >> 1)) * F::ROW + (v_at ^ F::turn(u & 1) * 16 ^ 128 * c), &v[u][c * (F::VB / 4)]);
        }
        if constexpr (Q8) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                vs[u] = reinterpret_cast<const float *>(stage + R::VS)[16 * blk + g + 8 * u];
        }
        if (left < 16) {  // 0 times what a stale place holds must stay 0
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (2 * t + (u & 1) + 8 * (u >> 1) >= left) {
#pragma unroll
                    for (int i = 0; i < F::VW; ++i) v[u][i] = 0;
                }
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (Q8 && g + 8 * u >= left) vs[u] = 0.0f;
        }
    }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Zeros into rows [from, to) of the call, by the CTAs of one sequence (all of them, in whatever shape of block). A
// call of its own: inlined into the kernels it moved their registers.
__device__ __noinline__ void zero_rows(void *out, int type, bool vec, long long o_token, long long o_head, uint32_t q_heads, uint32_t quads, int from, int to) {
    const size_t ctas = (size_t)gridDim.x * gridDim.y, cta = blockIdx.x + (size_t)gridDim.x * blockIdx.y;
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (size_t u = cta * blockDim.x + threadIdx.x; u < (size_t)(to - from) * q_heads * quads; u += ctas * blockDim.x) {
        const size_t r = u / quads;
        store4(out, (from + (long long)(r / q_heads)) * o_token + (long long)(r % q_heads) * o_head + 4 * (long long)(u % quads), type, vec, zero);
    }
}
__device__ __forceinline__ void zero_rows(const AttendArgs &a, int from, int to) {
    zero_rows(a.out, a.o_type, a.o_vec, a.o_token, a.o_head, a.kv.heads * a.group, a.kv.dim / 4, from, to);
}

// Rows before the first sequence's and behind the last one's see nothing: zeros. start, stop: sequence b's.
__device__ __forceinline__ void zero_outside(const AttendArgs &a, uint32_t b, int start, int stop) {
    const int tokens = (int)a.seq.tokens;
    if (b == 0 && start > 0) zero_rows(a, 0, min(tokens, start));
    if (b + 1 == a.seq.seqs && stop < tokens) zero_rows(a, max(0, stop), tokens);
}

// Over the eight lanes that share t (the keys of a block).
__device__ __forceinline__ float max_keys(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float sum_keys(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 4);
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

// A part's sum l of exponentials over its own maximum m, over `top`. Where it has seen nothing (-inf) l is 0, or NaN.
__device__ __forceinline__ float weighed(float m, float l, float top) { return m == kLowest ? l : l * exp2_of(m - top); }

// NT: tiles of 8 rows. State of a warp: per row (2t and 2t + 1 of each tile,
// the same in all lanes of equal t) the near maximum m; l is this lane's share.
template <int D, bool Q8, bool SPLIT, int NT>
struct Rows {
    using F = Frag<D, Q8>;
    static constexpr int DIGITS = SPLIT ? 3 : 2;  // of q, with 8-bit caches
    uint32_t q[Q8 ? DIGITS : SPLIT ? 2 : 1][NT][F::STEPS][Q8 ? 1 : 2];
    float scale[NT][2];
    int limit[NT][2];
    int all;  // keys below are seen by every row
    float o[NT][F::STEPS][4];
    float m[NT][2], l[NT][2];
    // 8-bit caches: of the V scales that the row has seen the largest is below 1 / back, a power of two. A row's
    // own: a scale in a place that it does not see must not push its weights out of f16's range.
    float back[NT][2];
    int k_at, v_at;  // where the lane's reads of a stage begin

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                m[n][r] = kLowest;
                l[n][r] = 0.0f;
                back[n][r] = over(0.0f);
            }
#pragma unroll
            for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][j][e] = 0.0f;
        }
    }

    // have: bit i, block i of the stage is in the cache; key0: the stage's first key; careful: look for infinities in
    // blocks that all rows see, too
    __device__ __forceinline__ void step(const uint8_t *stage, uint32_t have, int key0, int end, int g, int t, bool careful) {
        constexpr int B = Ring<D, Q8>::BLOCKS;
        Block<D, Q8> x[B];
        float s[B][NT][4];  // key g: rows 2t, 2t + 1; key g + 8: the same
#pragma unroll
        for (int i = 0; i < B; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][n][e] = 0.0f;
            if (B > 1 && !((have >> i) & 1)) continue;
            x[i].load_k(stage, i, g, k_at);
            if constexpr (Q8) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    int c[DIGITS][4];
#pragma unroll
                    for (int z = 0; z < DIGITS; ++z) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[z][e] = 0;
                        if constexpr (F::STEPS == 1) {
                            mma8(c[z], x[i].k[0][0], x[i].k[1][0], q[z][n][0][0]);
                        } else {
#pragma unroll
                            for (int st = 0; st < F::STEPS; st += 2)
                                mma8(c[z], x[i].k[0][st], x[i].k[1][st], x[i].k[0][st + 1], x[i].k[1][st + 1], q[z][n][st][0], q[z][n][st + 1][0]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[i][n][e] = SPLIT ? __fmaf_rn((float)c[0][e], 16384.0f, (float)(c[1][e] * 128 + c[DIGITS - 1][e]))
                                           : (float)(c[0][e] * 128 + c[1][e]);
                }
            } else {
#pragma unroll
                for (int st = 0; st < F::STEPS; ++st) {
                    const uint32_t a[4] = {x[i].k[0][2 * st], x[i].k[1][2 * st], x[i].k[0][2 * st + 1], x[i].k[1][2 * st + 1]};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16(s[i][n], a, q[0][n][st][0], q[0][n][st][1]);
                        if constexpr (SPLIT) mma16(s[i][n], a, q[SPLIT][n][st][0], q[SPLIT][n][st][1]);
                    }
                }
            }
        }
        const bool whole = key0 + 16 * B <= all && have == (1u << B) - 1;
        bool past = false;
        float d = 0.0f;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (B > 1 && !((have >> i) & 1)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][n][e] = kLowest;
                x[i].vs[0] = x[i].vs[1] = 0.0f;
                continue;
            }
            x[i].load_v(stage, i, end - key0 - 16 * i, g, t, v_at);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][n][e] *= Q8 ? scale[n][e & 1] * x[i].ks[e >> 1] : scale[n][e & 1];
            if (!whole) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (key0 + 16 * i + g + 8 * (e >> 1) >= limit[n][e & 1]) s[i][n][e] = kLowest;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) past |= s[i][n][e] > m[n][e & 1] + kSlack;
            if constexpr (Q8) {
                d = fmaxf(d, fmaxf(fabsf(x[i].vs[0]), fabsf(x[i].vs[1])));
                if (!whole) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) past |= key0 + 16 * i + g + 8 * (e >> 1) < limit[n][e & 1] && fabsf(x[i].vs[e >> 1]) * back[n][e & 1] >= 1.0f;
                }
            }
        }
        // a whole block follows keys that all rows have seen, so the first row's back is that of all
        if (Q8 && whole) past |= d * back[0][0] >= 1.0f;
        if (__any_sync(0xffffffffu, past)) {
            if constexpr (Q8) d = max_keys(d);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float top = fmaxf(s[0][n][r], s[0][n][2 + r]);
#pragma unroll
                    for (int i = 1; i < B; ++i) top = fmaxf(top, fmaxf(s[i][n][r], s[i][n][2 + r]));
                    top = fmaxf(m[n][r], max_keys(top));
                    const float w = m[n][r] == kLowest ? 0.0f : exp2_of(m[n][r] - top);
                    m[n][r] = top;
                    l[n][r] *= w;
                    float f = w;
                    if constexpr (Q8) {
                        float seen = d;
                        if (!whole) {
                            seen = 0.0f;
#pragma unroll
                            for (int i = 0; i < B; ++i)
#pragma unroll
                                for (int u = 0; u < 2; ++u)
                                    if (key0 + 16 * i + g + 8 * u < limit[n][r]) seen = fmaxf(seen, fabsf(x[i].vs[u]));
                            seen = max_keys(seen);
                        }
                        const float now = fminf(back[n][r], over(seen));
                        f *= now * inverse(back[n][r]);
                        back[n][r] = now;
                    }
#pragma unroll
                    for (int j = 0; j < F::STEPS; ++j) {
                        o[n][j][r] *= f;
                        o[n][j][2 + r] *= f;
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (B > 1 && !((have >> i) & 1)) continue;
            uint32_t p[SPLIT ? 2 : 1][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // where nothing was seen yet s is -inf, and any finite maximum gives p = 0
                const float z[2] = {(m[n][0] == kLowest ? 0.0f : m[n][0]) - kRaise, (m[n][1] == kLowest ? 0.0f : m[n][1]) - kRaise};
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = exp2_of(s[i][n][e] - z[e & 1]);
                    l[n][e & 1] += w[e];
                }
                if (Q8 && whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] *= x[i].vs[e >> 1] * back[0][0];
                } else if (Q8) {  // a masked key's scale may be NaN
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = s[i][n][e] == kLowest ? 0.0f : w[e] * (x[i].vs[e >> 1] * back[n][e & 1]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t hi = pack(w[2 * u], w[2 * u + 1]);
                    p[0][n][u] = transpose8(hi);
                    if constexpr (SPLIT) {
                        const float2 h = unpack(hi);
                        p[SPLIT][n][u] = transpose8(pack(w[2 * u] - h.x, w[2 * u + 1] - h.y));
                    }
                }
            }
            // O += the weights' high or low part times V^T's part
            auto part = [&](int low, int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                const uint32_t f[4] = {a0, a1, a2, a3};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16(o[n][j], f, p[low][n][0], p[low][n][1]);
            };
            auto products = [&](auto pair) {  // pair(step, its part of V^T)
#pragma unroll
                for (int c = 0; c < F::VW; ++c) {
                    if constexpr (Q8) {
                        const uint32_t x0 = x[i].v[0][c] ^ 0x80808080u, x1 = x[i].v[1][c] ^ 0x80808080u;
                        const uint32_t x2 = x[i].v[2][c] ^ 0x80808080u, x3 = x[i].v[3][c] ^ 0x80808080u;
                        const uint32_t lo0 = __byte_perm(x0, x1, 0x5140), lo1 = __byte_perm(x2, x3, 0x5140);
                        constexpr int PER = F::STEPS < 2 ? 1 : 2;
                        pair(PER * c, codes2(lo0, 0x4140), codes2(lo0, 0x4342), codes2(lo1, 0x4140), codes2(lo1, 0x4342));
                        if constexpr (PER == 2) {
                            const uint32_t hi0 = __byte_perm(x0, x1, 0x7362), hi1 = __byte_perm(x2, x3, 0x7362);
                            pair(PER * c + 1, codes2(hi0, 0x4140), codes2(hi0, 0x4342), codes2(hi1, 0x4140), codes2(hi1, 0x4342));
                        }
                    } else {
                        pair(c, __byte_perm(x[i].v[0][c], x[i].v[1][c], 0x5410), __byte_perm(x[i].v[0][c], x[i].v[1][c], 0x7632),
                             __byte_perm(x[i].v[2][c], x[i].v[3][c], 0x5410), __byte_perm(x[i].v[2][c], x[i].v[3][c], 0x7632));
                    }
                }
            };
            if constexpr (!Q8) {
                // 0 times an infinity or NaN would reach rows that do not see its key: such a block goes key by key,
                // and every row keeps what it had where the key is masked. The weights' low parts, which may be 0 or
                // below it, only meet finite values.
                bool wild = false;
                if (!whole || (SPLIT && careful)) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int c = 0; c < F::VW; ++c) {
                            const uint32_t e = x[i].v[u][c] & 0x7c007c00u;
                            wild |= (e & 0x7c00u) == 0x7c00u || (e >> 16) == 0x7c00u;
                        }
                    wild = __any_sync(0xffffffffu, wild);
                }
                if (wild) {
                    const Block<D, Q8> all_keys = x[i];
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int u = 0; u < 4; ++u)
#pragma unroll
                            for (int c = 0; c < F::VW; ++c) {
                                if ((x[i].v[u][c] & 0x7c00u) == 0x7c00u) x[i].v[u][c] &= 0xffff0000u;
                                if ((x[i].v[u][c] & 0x7c000000u) == 0x7c000000u) x[i].v[u][c] &= 0xffffu;
                            }
                        products([&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) { part(SPLIT, j, a0, a1, a2, a3); });
                    }
#pragma unroll 1
                    for (int key = 0; key < 16; ++key) {
                        float kept[NT][F::STEPS][4];
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e) kept[n][j][e] = o[n][j][e];
#pragma unroll
                        for (int u = 0; u < 4; ++u)
#pragma unroll
                            for (int c = 0; c < F::VW; ++c) x[i].v[u][c] = 2 * t + (u & 1) + 8 * (u >> 1) == key ? all_keys.v[u][c] : 0u;
                        products([&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) { part(0, j, a0, a1, a2, a3); });
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (key0 + 16 * i + key >= limit[n][e & 1]) o[n][j][e] = kept[n][j][e];
                    }
                    continue;
                }
            }
            products([&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                part(0, j, a0, a1, a2, a3);
                if constexpr (SPLIT) part(SPLIT, j, a0, a1, a2, a3);
            });
        }
    }
};

// 16 rows of dim 16 over f16 caches: a fourth CTA of an SM (f32 queries, 700 over 3000 positions: 51 against 55 us).
template <int D, bool Q8, bool SPLIT, int NT>
__global__ void __launch_bounds__(kRowThreads, Frag<D, Q8>::ctas(NT) + (D == 16 && !Q8 && NT == 2)) attend_rows_kernel(const AttendArgs a) {
    using F = Frag<D, Q8>;
    constexpr int R = 8 * NT, PER_ROW = kRowThreads / R, E = D / PER_ROW;
    static_assert(E >= 1, "at most one thread a number");
    using RG = Ring<D, Q8>;
    extern __shared__ __align__(128) uint8_t smem[];
    static_assert(RG::BYTES >= kRowWarps * R * D * 4, "the warps' outputs take the rings' place");
    float(*so)[R][D] = reinterpret_cast<float(*)[R][D]>(smem);
    constexpr int DIGITS = Rows<D, Q8, SPLIT, NT>::DIGITS;
    __shared__ __align__(16) __half sq[Q8 ? 1 : SPLIT ? 2 : 1][R][D];  // Q as f16 parts,
    __shared__ __align__(16) int8_t sd[Q8 ? DIGITS : 1][R][D];         // or as 8-bit digits
    __shared__ float row_scale[R], wm[kRowWarps][R], wl[kRowWarps][R], cm[R], cl[R], weight[16][R];
    __shared__ int row_limit[R];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t part = blockIdx.x, heads = a.kv.heads;
    const uint32_t head = blockIdx.y % heads, b = blockIdx.z;
    if (a.overlap) {  // beside the launch for many rows
        take_turn(a.turn);
        let_next_start();
    } else {
        begin();
    }
    int n, stand, start, after;  // stand: position of the first new token
    const int t0 = a.seq.first(b, n, stand, start, after);
    const int len = a.seq.length(b, a.kv.page_log2);
    const int32_t *table = a.seq.table + (size_t)b * a.seq.table_stride;
    const int rows = n * (int)a.group;  // the call has fewer than 2^31 query rows
    if (!a.overlap) zero_outside(a, b, start, after);
    // then one CTA sees to it that this kernel does not end first
    const bool keeper = a.overlap && blockIdx.x == 0 && blockIdx.y == gridDim.y - 1 && b == gridDim.z - 1;
    auto keep = [&] {
        if (!keeper) return;
        wait_for_previous();
        if (tid == 0) atomicCAS(&g_turn[a.turn % kTurns], a.turn, 0u);
    };
    if ((uint32_t)rows > a.few) {
        keep();
        return;
    }
    // a shorter sequence takes fewer of the cluster's CTAs; the others leave (its barriers count the threads that stay)
    const uint32_t parts = min(gridDim.x, ((uint32_t)max(len, 1) + a.span - 1) / a.span);
    if (part >= parts) return;
    uint8_t *ring = smem + warp * (RG::N * RG::STAGE);
    uint32_t put = 0, get = 0;  // next stage to fill and to read
    uint32_t have = 0;          // BLOCKS bits a stage: which of its blocks are in the cache
    const uint32_t page_mask = (1u << a.kv.page_log2) - 1;
    // keys that token i sees
    auto limit = [&](int i) { return a.causal ? max(0, min(len, stand + i + 1)) : len; };

    for (int r0 = (int)(blockIdx.y / heads) * R; r0 < rows; r0 += (int)(gridDim.y / heads) * R) {
        const int live = min(R, rows - r0);
        const int end = limit((r0 + live - 1) / (int)a.group);  // no row of the tile sees further
        // the CTA's part of the keys, in 16-key blocks; a warp takes every fourth stage
        const int blocks = (end + 15) / 16;
        const int first = (int)((uint64_t)blocks * part / parts), stop = (int)((uint64_t)blocks * (part + 1) / parts);
        const int stages = (stop - first + RG::BLOCKS - 1) / RG::BLOCKS;
        const int mine = warp < stages ? (stages - warp + kRowWarps - 1) / kRowWarps : 0;
        auto block_of = [&](int i) { return first + (warp + i * kRowWarps) * RG::BLOCKS; };
        uint32_t pages = 0;  // lane's: of block lane % BLOCKS of stage lane / BLOCKS of the group of stages in hand
        constexpr int GROUP = 32 / RG::BLOCKS;
        // 16 rows of K or V, 16 bytes a lane and access
        constexpr int KEYS = F::PIECES < 32 ? 32 / F::PIECES : 1;  // of an access
        const int copy_at = F::byte(lane / F::PIECES, lane % F::PIECES * 16);
        auto copy_rows = [&](uint32_t to, const void *base, size_t row) {
            const uint8_t *src = static_cast<const uint8_t *>(base) + row * F::ROW + 16 * lane;
#pragma unroll
            for (int u = 0; u < 16; u += KEYS)
                if (KEYS <= 16 || lane < 16 * F::PIECES)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * F::ROW + (copy_at ^ F::turn(u) * 16)), "l"(src + u * F::ROW));
        };
        auto issue = [&](int i) {  // one group of copies, empty past the last stage
            if (i < mine) {
                if (i % GROUP == 0) {
                    const int blk = block_of(i + lane / RG::BLOCKS) + lane % RG::BLOCKS;
                    pages = blk < stop ? (uint32_t)__ldg(table + ((uint32_t)(blk * 16) >> a.kv.page_log2)) : 0xffffffffu;
                }
                const uint32_t to = smem_u32(ring) + put * RG::STAGE;
                uint32_t got = 0;
#pragma unroll
                for (int blk = 0; blk < RG::BLOCKS; ++blk) {
                    const uint32_t page = __shfl_sync(0xffffffffu, pages, i % GROUP * RG::BLOCKS + blk);
                    if (page >= a.kv.pages) continue;
                    got |= 1u << blk;
                    const size_t row = a.kv.row(page, head, (uint32_t)((block_of(i) + blk) * 16) & page_mask);
                    copy_rows(to + blk * RG::ROWS, a.kv.k, row);
                    copy_rows(to + RG::V + blk * RG::ROWS, a.kv.v, row);
                    if (Q8 && lane < 8) {  // four pieces of either side's scales
                        const float *from = (lane < 4 ? a.kv.ks : a.kv.vs) + row + 4 * (lane & 3);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                         to + (lane < 4 ? RG::KS : RG::VS) + blk * RG::SCALES + 16 * (lane & 3)),
                                     "l"(from));
                    }
                }
                constexpr uint32_t ALL = (1u << RG::BLOCKS) - 1;
                have = (have & ~(ALL << (put * RG::BLOCKS))) | got << (put * RG::BLOCKS);
                put = put + 1 == RG::N ? 0 : put + 1;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < RG::N; ++i) issue(i);

        {
            const int r = tid / PER_ROW, c = tid % PER_ROW;
            const int rr = min(r0 + r, rows - 1), i = rr / (int)a.group, h = rr - i * (int)a.group;
            const int64_t at = (t0 + i) * a.q_token + (int64_t)(head * a.group + h) * a.q_head + c * E;
            constexpr float kHuge = 3.402823466e38f;
            float x[E], m = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = load1(a.q, (size_t)(at + e), a.q_type);
                m = fabsf(x[e]) <= kHuge ? fmaxf(m, fabsf(x[e])) : __int_as_float(0x7f800000);
            }
            float undo = a.scale;
            if (Q8 || a.q_type != MGB_F16) {
#pragma unroll
                for (int o = PER_ROW / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                // the row's largest number to just below 2^14 (f16 q over f16 caches stays as it is), by 2^shift in two
                // factors, since either may leave the range of f32 alone. Undone, a row below 2^-100 or so has lost bits
                // of its scale, which leaves f32's normal numbers.
                const int shift = m > 0.0f && m <= kHuge ? 140 - (__float_as_int(m) >> 23) : 0;
                const int s1 = max(-100, min(100, shift)), s2 = shift - s1;
                const float f1 = __int_as_float((127 + s1) << 23), f2 = __int_as_float((127 + s2) << 23);
                m = m * f1 * f2;
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = x[e] * f1 * f2;
                undo = undo * __int_as_float((127 - s1) << 23) * __int_as_float((127 - s2) << 23);
            }
            if constexpr (Q8) {
                // q as whole numbers over the row's largest; a row with an infinity or NaN gets an infinite scale, and
                // so scores of NaN
                constexpr float kMost = SPLIT ? 127 * 16384 + 8191 : 127 * 128 + 63;
                const float inv = m == 0.0f ? 0.0f : kMost / m;
                undo *= m / kMost;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    int v = __float2int_rn(x[e] * inv);
                    if constexpr (SPLIT) {
                        const int hi = (v + 8192) >> 14;
                        sd[0][r][c * E + e] = (int8_t)hi;
                        v -= hi << 14;
                    }
                    const int mid = (v + 64) >> 7;
                    sd[DIGITS - 2][r][c * E + e] = (int8_t)mid;
                    sd[DIGITS - 1][r][c * E + e] = (int8_t)(v - (mid << 7));
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const __half hi = __float2half_rn(x[e]);
                    sq[0][r][c * E + e] = hi;
                    if constexpr (SPLIT) sq[SPLIT][r][c * E + e] = __float2half_rn(x[e] - __half2float(hi));
                }
            }
            if (c == 0) {
                row_scale[r] = undo;
                row_limit[r] = r < live ? limit(i) : 0;
            }
        }
        __syncthreads();
        Rows<D, Q8, SPLIT, NT> st;
        st.k_at = F::byte(g, t * F::KB);
        st.v_at = F::byte(2 * t, g * F::VB);
        st.all = row_limit[0];  // what the rows past `live` see does not matter
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if constexpr (Q8) {
#pragma unroll
                for (int z = 0; z < DIGITS; ++z)
#pragma unroll
                    for (int s = 0; s < F::STEPS; ++s)
                        st.q[z][j][s][0] = *reinterpret_cast<const uint32_t *>(&sd[z][8 * j + g][F::k_dim(t, 4 * s)]);
            } else {
#pragma unroll
                for (int z = 0; z < (SPLIT ? 2 : 1); ++z)
#pragma unroll
                    for (int s = 0; s < F::STEPS; ++s) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(&sq[z][8 * j + g][F::k_dim(t, 4 * s)]);
                        st.q[z][j][s][0] = x.x, st.q[z][j][s][1] = x.y;
                    }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                st.scale[j][r] = row_scale[8 * j + 2 * t + r];
                st.limit[j][r] = row_limit[8 * j + 2 * t + r];
            }
        }

        // f32 queries over f16 caches: the weights' low parts times an infinity in V are NaN where the row has that
        // infinity. Looking for those in every block would cost a fifth of the instructions, so a warp whose
        // outputs have a NaN takes its keys again, looking.
        for (bool careful = false;; careful = true) {
            st.clear();
            for (int i = 0; i < mine; ++i) {
                asm volatile("cp.async.wait_group %0;" ::"n"(RG::N - 1) : "memory");
                __syncwarp();
                const uint32_t got = (have >> (get * RG::BLOCKS)) & ((1u << RG::BLOCKS) - 1);
                if (got) st.step(ring + get * RG::STAGE, got, block_of(i) * 16, end, g, t, careful);
                __syncwarp();  // every lane has read the stage
                issue(i + RG::N);
                get = get + 1 == RG::N ? 0 : get + 1;
            }
            if constexpr (SPLIT && !Q8) {
                bool nan = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int s = 0; s < F::STEPS; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) nan |= st.o[n][s][e] != st.o[n][s][e];
                if (careful || !__any_sync(0xffffffffu, nan)) break;
#pragma unroll
                for (int i = 0; i < RG::N; ++i) issue(i);  // the ring is empty, what is left in flight are empty groups
            } else {
                break;
            }
        }

        // the CTA's warps
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float l = sum_keys(st.l[j][r]);
                if (g == 0) {
                    wm[warp][8 * j + 2 * t + r] = st.m[j][r];
                    wl[warp][8 * j + 2 * t + r] = l;
                }
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 8 * j + 2 * t + r;
                if (row >= live) continue;
                float top = wm[0][row], unit = 1.0f;
#pragma unroll
                for (int w = 1; w < kRowWarps; ++w) top = fmaxf(top, wm[w][row]);
                float sum = 1.0f;
                if constexpr (Q8) {
                    // over the CTA's sum before V's power comes in: the outputs alone could pass f32's range
                    sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < kRowWarps; ++w) sum += weighed(wm[w][row], wl[w][row], top);
                    unit = inverse(st.back[j][r]);
                }
                const float f = st.m[j][r] == kLowest || sum == 0.0f ? 0.0f : exp2_of(st.m[j][r] - top) / sum;
#pragma unroll
                for (int s = 0; s < F::STEPS; ++s) {
                    so[warp][row][F::v_dim(g, 2 * s)] = st.o[j][s][r] * f * unit;
                    so[warp][row][F::v_dim(g, 2 * s + 1)] = st.o[j][s][2 + r] * f * unit;
                }
            }
        if ((!Q8 || parts > 1) && tid < live) {
            float top = kLowest, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, wm[w][tid]);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) sum += weighed(wm[w][tid], wl[w][tid], top);
            cm[tid] = top;
            cl[tid] = sum;
        }
        __syncthreads();
        namespace cg = cooperative_groups;
        auto cluster = cg::this_cluster();
        // W numbers at a time: with 16 rows of dim 64 or 128 four are 5 to 12 % of a short call faster (40 rows
        // over 500 positions, 16 heads of 128: 13.8 -> 12.2 us); with 8 rows (often one alone) or dim 16 one by
        // one keeps more threads busy, 0.2 to 0.7 us of 4 to 20
        constexpr bool WIDE = NT > 1 && D >= 64;
        constexpr int W = WIDE ? 4 : 1;
        using Numbers = typename std::conditional<W == 4, float4, float>::type;
        union Some {
            Numbers all;
            float at[W];
        };
        auto add = [](Some &x, float f, const float *from, int u) {
            Some y;
            y.all = reinterpret_cast<const Numbers *>(from)[u];
#pragma unroll
            for (int e = 0; e < W; ++e) x.at[e] += f * y.at[e];
        };
        auto of_warps = [&](int u) {
            Some sum{};
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) add(sum, 1.0f, &so[w][0][0], u);
            return sum;
        };
        if (parts > 1) {
            for (int u = tid; u < live * (D / W); u += kRowThreads) reinterpret_cast<Numbers *>(&so[0][0][0])[u] = of_warps(u).all;
            cluster_sync();
            // the CTAs' weights of a row and their sum; where WIDE, all of their maxima and sums are
            // fetched at once, into the place of the second warp's outputs
            float(*part_m)[R] = reinterpret_cast<float(*)[R]>(&so[1][0][0]), (*part_l)[R] = part_m + 16;
            static_assert(!WIDE || D >= 32, "two times sixteen parts' numbers fit in a warp's outputs");
            if constexpr (WIDE) {
                for (int u = tid; u < (int)parts * R; u += kRowThreads) {
                    part_m[u / R][u % R] = *cluster.map_shared_rank(&cm[u % R], u / R);
                    part_l[u / R][u % R] = *cluster.map_shared_rank(&cl[u % R], u / R);
                }
                __syncthreads();
            }
            if (tid < live) {
                auto m_of = [&](uint32_t c) { return WIDE ? part_m[c][tid] : *cluster.map_shared_rank(&cm[tid], c); };
                auto l_of = [&](uint32_t c) { return WIDE ? part_l[c][tid] : *cluster.map_shared_rank(&cl[tid], c); };
                float top = kLowest, sum = 0.0f;
                for (uint32_t c = 0; c < parts; ++c) top = fmaxf(top, m_of(c));
                for (uint32_t c = 0; c < parts; ++c) {
                    const float m = m_of(c), l = weighed(m, l_of(c), top);
                    weight[c][tid] = Q8 ? l : m == kLowest ? 0.0f : exp2_of(m - top);
                    sum += l;
                }
                row_scale[tid] = sum;
                if constexpr (Q8) {
                    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                    for (uint32_t c = 0; c < parts; ++c) weight[c][tid] *= f;
                }
            }
            __syncthreads();
        }
        // outputs; with several CTAs each takes its share of the tile
        for (int u = (int)part * kRowThreads + tid; u < live * (D / W); u += (int)parts * kRowThreads) {
            const int r = u / (D / W), d = u % (D / W) * W;
            Some sum{};
            if (parts == 1) {
                sum = of_warps(u);
            } else {
#pragma unroll 4
                for (uint32_t c = 0; c < parts; ++c) add(sum, weight[c][r], cluster.map_shared_rank(&so[0][0][0], c), u);
            }
            if constexpr (!Q8) {
                const float l = parts == 1 ? cl[r] : row_scale[r];
#pragma unroll
                for (int e = 0; e < W; ++e) sum.at[e] = l == 0.0f ? 0.0f : sum.at[e] / l;
            }
            const int rr = r0 + r, i = rr / (int)a.group, h = rr - i * (int)a.group;
            const int64_t to = (t0 + i) * a.o_token + (int64_t)(head * a.group + h) * a.o_head + d;
            if constexpr (W == 4) store4(a.out, to, a.o_type, a.o_vec, sum.at);
            else store1(a.out, (size_t)to, a.o_type, sum.at[0]);
        }
        if (parts > 1) cluster_sync();
        else __syncthreads();
    }
    keep();
}

template <int D, bool Q8, bool SPLIT, int NT>
cudaError_t launch_rows(const AttendArgs &a, dim3 grid, cudaStream_t s) {
    constexpr int SMEM = Ring<D, Q8>::BYTES;
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = op_allow(attend_rows_kernel<D, Q8, SPLIT, NT>, SMEM, true, done);
    if (e != cudaSuccess) return e;
    return op_launch(attend_rows_kernel<D, Q8, SPLIT, NT>, grid, kRowThreads, SMEM, grid.x, a, s);
}

// Keys are cut over the CTAs of a cluster (at most 16) while all CTAs still run
// at once and every warp keeps two blocks, and further, from 3 * 1024 positions on,
// while a CTA would have more than 1024 keys: sequences of unlike lengths then even
// out. A sequence that is shorter than the longest takes as few of the CTAs as keep
// the longest's share of keys, 512 at most. Against cuts at 2048 for all: 32 sequences
// of 200 to 6000 positions, 8 heads of 64, 8 bits 42 -> 30 us, 96 of 100 to 8000, dim
// 128, 107 -> 100; twice as many cuts cost sequences of like lengths up to 20 %.
template <int D, bool Q8, bool SPLIT, int NT>
cudaError_t launch_rows(AttendArgs a, uint64_t rows, uint64_t most_len, cudaStream_t s) {
    constexpr int SMEM = Ring<D, Q8>::BYTES + Frag<D, Q8>::STATIC * NT, FIT = 227 * 1024 / SMEM;
    constexpr int SLOTS = 148 * (FIT < Frag<D, Q8>::ctas(NT) ? FIT : Frag<D, Q8>::ctas(NT));
    uint64_t tiles = (rows + 8 * NT - 1) / (8 * NT);
    if (tiles * a.kv.heads > 65535) tiles = 65535 / a.kv.heads;
    const uint64_t base = tiles * a.kv.heads * a.seq.seqs;
    uint64_t parts = base < SLOTS ? SLOTS / base : 1;
    if (most_len >= 3 * 1024 && parts < most_len / 1024) parts = most_len / 1024;
    if (parts > most_len / (kRowWarps * 32)) parts = most_len / (kRowWarps * 32);
    // sizes that pack into the GPU's clusters of 16 or 18 SMs
    parts = parts >= 16 ? 16 : parts >= 8 ? 8 : parts >= 4 ? 4 : parts < 1 ? 1 : parts;
    a.span = (uint32_t)((most_len + parts - 1) / parts);
    a.span = a.span < 1 ? 1 : a.span > 512 ? 512 : a.span;
    return launch_rows<D, Q8, SPLIT, NT>(a, dim3((unsigned)parts, (unsigned)(tiles * a.kv.heads), a.seq.seqs), s);
}

// 8-row tiles where a call has no more rows a cache head than that, else 16.
template <int D, bool Q8, bool SPLIT>
cudaError_t launch_rows(const AttendArgs &a, uint64_t rows, uint64_t most_len, cudaStream_t s) {
    return rows <= 8 ? launch_rows<D, Q8, SPLIT, 1>(a, rows, most_len, s)
                     : launch_rows<D, Q8, SPLIT, 2>(a, rows, most_len, s);
}

template <int D>
cudaError_t launch_rows(const AttendArgs &a, bool q8, uint64_t rows, uint64_t most_len, cudaStream_t s) {
    if (a.q_type == MGB_F32)
        return q8 ? launch_rows<D, true, true>(a, rows, most_len, s) : launch_rows<D, false, true>(a, rows, most_len, s);
    return q8 ? launch_rows<D, true, false>(a, rows, most_len, s) : launch_rows<D, false, false>(a, rows, most_len, s);
}

#include "attend_tiles.cuh"

// A row tile's keys are cut over the CTAs of a cluster, in as many parts as make
// the shortest: rounds of CTAs (one an SM, 148 SMs) times the key tiles of a CTA,
// with four more for its beginning and end and two to join parts. The row tiles
// are estimated from all rows and half a tile a sequence, since lengths are only
// known on the device. Returns the key tiles one after another.
uint64_t tiles_cost(const AttendArgs &a, uint64_t most_new, uint64_t most_len, uint32_t &parts) {
    const uint64_t most = a.seq.seqs * ((most_new * a.group + 255) / 256);
    const uint64_t some = ((uint64_t)a.seq.tokens * a.group + 255) / 256 + a.seq.seqs / 2;
    const uint64_t base = a.kv.heads * (some < most ? some : most);
    const uint64_t key_tiles = (most_len + tiles::kKeys - 1) / tiles::kKeys;
    uint64_t best = ~0ull;
    parts = 1;
    for (uint32_t p = 1; p <= 8 && (p == 1 || key_tiles >= 4 * p); p *= 2) {
        const uint64_t cost = (base * p + 147) / 148 * ((key_tiles + p - 1) / p + 4 + (p > 1 ? 2 : 0));
        if (cost < best) best = cost, parts = p;
    }
    return best;
}

template <int D, bool Q8>
cudaError_t launch_tiles(const AttendArgs &a, uint64_t most_new, uint64_t most_len, cudaStream_t s) {
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = op_allow(tiles::attend_tiles_kernel<D, Q8>, tiles::Smem<D>::ASKED, false, done);
    if (e != cudaSuccess) return e;
    uint64_t row_tiles = (most_new * a.group + 255) / 256;
    if (row_tiles * a.kv.heads > 65535) row_tiles = 65535 / a.kv.heads;
    uint32_t parts;
    tiles_cost(a, most_new, most_len, parts);
    return op_launch(tiles::attend_tiles_kernel<D, Q8>, dim3(parts, (unsigned)(row_tiles * a.kv.heads), a.seq.seqs), tiles::kThreads,
                     tiles::Smem<D>::ASKED, parts, a, s);
}

// Numbers of calls with both kernels, of all dims alike; never 0.
uint32_t next_turn() {
    static std::atomic<uint32_t> calls{0};
    uint32_t turn = ++calls;
    while (!turn) turn = ++calls;
    return turn;
}

// Which kernel. f32 queries, whose two f16 parts only the kernel for few rows
// takes, and calls of at most kFewRows rows a cache head go there. So do calls of
// at most 256 rows where it is faster, which measurements at dims 16, 64 and 128
// (100 to 250 new tokens, 1500 to 16,000 positions, 8 and 16 heads, 1 to 16
// sequences) put as: it takes 6 us and 0.3 + dim / 95 us (8 bits: 0.6 + dim / 105)
// for every 28,500 pairs of a 16-row tile and a key, the tiles 30 us (8 bits: 34)
// and 0.3 + dim / 120 us for each of tiles_cost's key tiles (dim 32 follows from the
// others; causal calls have as little as half of these pairs, others all). Over 4000 positions,
// 16 heads of 64, f16: 100 rows 22 against 32 us, 200 rows 30 against 40; 100 rows
// over 1500 in 16 sequences 98 against 63.
template <int D>
cudaError_t launch(AttendArgs a, bool q8, uint64_t most_new, uint64_t most_len, cudaStream_t s) {
    const uint64_t rows = most_new * a.group;
    bool few = a.q_type == MGB_F32 || rows <= kFewRows;
    if (!few && rows <= 256) {
        uint32_t parts;
        const double pairs = (double)((rows + 15) / 16 * a.kv.heads * a.seq.seqs) * (double)most_len;
        few = 6.0 + pairs / 28500.0 * (q8 ? 0.6 + D / 105.0 : 0.3 + D / 95.0) <
              (q8 ? 34.0 : 30.0) + (double)tiles_cost(a, most_new, most_len, parts) * (0.3 + D / 120.0);
    }
    if (few) return launch_rows<D>(a, q8, rows, most_len, s);
    // Sequences of unlike lengths: there may be some of few rows, which go to the other
    // kernel. The host knows bounds, not lengths (the rows may be more than the sequences
    // have, a bound too small), so without the second launch the tiles take them all.
    const bool both = a.seq.tokens < most_new * a.seq.seqs;
    a.few = both ? kFewRows : 0;
    if (both) a.turn = next_turn();
    cudaError_t e = q8 ? launch_tiles<D, true>(a, most_new, most_len, s) : launch_tiles<D, false>(a, most_new, most_len, s);
    if (e == cudaSuccess && both) {
        a.overlap = true;
        e = launch_rows<D>(a, q8, kFewRows, most_len, s);
    }
    return e;
}

}  // namespace
}  // namespace mgb

extern "C" MGB_API mgb_status mgb_kv_status(void *stream) {
    using namespace mgb;
    static const char *op = "mgb_kv_status";
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint32_t lost = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&lost, g_wait_lost, sizeof lost, 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && lost) {
        const uint32_t none = 0;
        e = cudaMemcpyToSymbolAsync(g_wait_lost, &none, sizeof none, 0, cudaMemcpyHostToDevice, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
        if (e == cudaSuccess) return op_fail(MGB_ERR_CUDA, op, "a wait of the attention ran out of time: rows of NaN in its output");
    }
    return op_launch_status(e, op);
}

extern "C" MGB_API mgb_status mgb_kv_attend(const mgb_kv *kv, const mgb_kv_seqs *seqs, const mgb_rows *q,
                                            const mgb_rows *out, float scale, int causal, void *stream) {
    using namespace mgb;
    static const char *op = "mgb_kv_attend";
    const char *bad = check_kv(kv);
    if (!bad) bad = check_seqs(seqs);
    if (!bad) bad = check_rows(q);
    if (!bad) bad = check_rows(out);
    if (!bad) bad = check_out(out);
    if (!bad && (q->tokens != out->tokens || q->heads != out->heads)) bad = "q and out differ in shape";
    if (!bad && (q->heads == 0 || q->heads % kv->heads)) bad = "query heads are not a multiple of the cache's";
    if (!bad && (uint64_t)q->tokens * q->heads > 0x7fffffffu) bad = "more than 2^31 - 1 query rows";
    if (bad) return op_fail(MGB_ERR_INVALID, op, bad);
    if (seqs->seqs == 0 || q->tokens == 0) return MGB_OK;
    // Failure-path test hook, read once: a stage of keys (0 or 1) that never fills, so that a wait runs out. Off
    // unless the variable is set.
    static const int withhold = getenv("MGB_TEST_WITHHOLD_KEYS") ? atoi(getenv("MGB_TEST_WITHHOLD_KEYS")) : -1;
    AttendArgs a{view(*kv), view(*seqs, q->tokens), q->data, out->data, q->token_stride, q->head_stride,
                 out->token_stride, out->head_stride, q->type, out->type, causal != 0, rows_vec(*out), rows_vec16(*q), rows_vec16(*out),
                 q->heads / kv->heads,
                 false, 0, 0xffffffffu, scale * kLog2e, 1, withhold};
    const uint64_t most_new = bound_new(*seqs, q->tokens), most_len = bound_len(*seqs, kv->page);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool q8 = kv->format == MGB_KV_Q8;
    cudaError_t e;
    switch (kv->dim) {
        case 16: e = launch<16>(a, q8, most_new, most_len, s); break;
        case 32: e = launch<32>(a, q8, most_new, most_len, s); break;
        case 64: e = launch<64>(a, q8, most_new, most_len, s); break;
        default: e = launch<128>(a, q8, most_new, most_len, s); break;
    }
    return op_launch_status(e, op);
}
