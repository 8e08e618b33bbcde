/*
 * tria_attend_tile.cuh - attention of many query rows over a ragged cache on
 * the tcgen05 tensor cores.
 *
 * A block takes up to 256 query rows of a unit as two row tiles of 128 and
 * walks 128 cache rows a step, 64 at a time: S = Q K^T into tensor memory, one
 * thread per query row turns its row of S into weights P (written over S as
 * f16), and O += P V accumulates in tensor memory.  Each row tile has two S
 * buffers, so the next scores are made while the weights of the last ones are:
 * no role waits for the round trip through the others.
 */
#pragma once

#include "tria_attend.cuh"

namespace tria {

/* ------------------------------------------------------------------ */
/* tcgen05 and its descriptors                                          */
/* ------------------------------------------------------------------ */

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
/* Operand in shared memory as panels of 64 f16 columns: row r of a panel is the
 * 128 bytes at 128 r, its 16-byte chunks XORed with r mod 8 (128-byte swizzle);
 * eight rows are 1024 bytes on.  Where the columns are the operand's row
 * dimension (V), panels are `lead` bytes apart.  The low word of a descriptor
 * holds the address (in 16 bytes) and lead, the high word is the same for all. */
__device__ __forceinline__ uint32_t tile_desc(uint32_t addr, uint32_t lead) { return (addr & 0x3ffff) >> 4 | (lead >> 4) << 16; }
constexpr uint32_t TILE_DESC_HI = (1024 >> 4) | 1u << 14 | 2u << 29;
/* Instruction descriptor: fp32 sums, f16 operands, M = 128, B by rows (K) or by columns (V). */
__host__ __device__ constexpr uint32_t tile_idesc(int n, bool b_by_column) {
    return 1u << 4 | (b_by_column ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
/* Products are issued by the one lane whose `lead` is not 0, predicated within
 * the instruction: the warp stays converged and its operands uniform. */
__device__ __forceinline__ void tc_mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %6, 0;\n\t"
                 "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "n"(TILE_DESC_HI), "r"(lead) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %6, 0;\n\tmov.b64 b, {%2, %5};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "n"(TILE_DESC_HI), "r"(lead) : "memory");
}
/* The barrier completes when every product this thread issued so far has. */
__device__ __forceinline__ void tc_commit(uint32_t lead, uint64_t *bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(smem_u32(bar)), "r"(lead) : "memory");
}
#define TC_R8(x, o) "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7])
#define TC_I8(x, o) "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7])
/* 32 columns of the warp's 32 lanes: a thread gets (gives) its lane's. */
__device__ __forceinline__ void tc_ld32(uint32_t (&x)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : TC_R8(x, 0), TC_R8(x, 8), TC_R8(x, 16), TC_R8(x, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t (&x)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : TC_R8(x, 0), TC_R8(x, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_ld64(uint32_t (&x)[64], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
                 : TC_R8(x, 0), TC_R8(x, 8), TC_R8(x, 16), TC_R8(x, 24), 
                   TC_R8(x, 32), TC_R8(x, 40), TC_R8(x, 48), TC_R8(x, 56)
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&x)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 ::TC_I8(x, 0), TC_I8(x, 8), TC_I8(x, 16), TC_I8(x, 24), "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t (&x)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::TC_I8(x, 0), TC_I8(x, 8), "r"(addr) : "memory");
}

/* Two fp32 at a time (one instruction for both). */
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
/* tanh_small of both; SHORT: two terms less, the first omitted one is below
 * 2^-29 at |u| = 0.2. */
template <bool SHORT>
__device__ __forceinline__ uint64_t tanh_small2(uint64_t u) {
    const uint64_t z = mul2(u, u);
    uint64_t s = pair(62.0f / 2835.0f, 62.0f / 2835.0f);
    if (!SHORT) {
        s = pair(21844.0f / 6081075.0f, 21844.0f / 6081075.0f);
        s = fma2(s, z, pair(-1382.0f / 155925.0f, -1382.0f / 155925.0f));
        s = fma2(s, z, pair(62.0f / 2835.0f, 62.0f / 2835.0f));
    }
    s = fma2(s, z, pair(-17.0f / 315.0f, -17.0f / 315.0f));
    s = fma2(s, z, pair(2.0f / 15.0f, 2.0f / 15.0f));
    s = fma2(s, z, pair(-1.0f / 3.0f, -1.0f / 3.0f));
    return fma2(mul2(s, z), u, u);
}
/* Caps N scores u = s / c (as bits), the largest magnitude being `far`: c tanh u.
 * Scores large enough to need the exponential are rare; they take a rolled
 * loop through `scratch` (N columns of the warp's tensor memory), so that the
 * common paths stay short enough for the instruction cache. */
template <int N>
__device__ __forceinline__ void tile_cap(uint32_t (&v)[N], float c, float far, uint32_t scratch) {
    const uint64_t cc = pair(c, c);
    if (__any_sync(0xffffffffu, !(far < 0.4f))) {
#pragma unroll
        for (int e = 0; e < N / 32; e++) tc_st32(scratch + 32 * e, *reinterpret_cast<const uint32_t (*)[32]>(v + 32 * e));
        tc_wait_st();
#pragma unroll 1
        for (int x = 0; x < N / 16; x++) {
            uint32_t y[16];
            tc_ld16(y, scratch + 16 * x);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; e++) y[e] = __float_as_uint(c * tanh_both(__uint_as_float(y[e])));
            tc_st16(scratch + 16 * x, y);
        }
        tc_wait_st();
#pragma unroll
        for (int e = 0; e < N / 32; e++) tc_ld32(*reinterpret_cast<uint32_t (*)[32]>(v + 32 * e), scratch + 32 * e);
        tc_wait_ld();
    } else if (__any_sync(0xffffffffu, far > 0.2f)) {
#pragma unroll
        for (int e = 0; e < N / 2; e++) {
            const float2 z = unpair(mul2(cc, tanh_small2<false>(pair(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])))));
            v[2 * e] = __float_as_uint(z.x);
            v[2 * e + 1] = __float_as_uint(z.y);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N / 2; e++) {
            const float2 z = unpair(mul2(cc, tanh_small2<true>(pair(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])))));
            v[2 * e] = __float_as_uint(z.x);
            v[2 * e + 1] = __float_as_uint(z.y);
        }
    }
}
/* N scores x (as bits) to weights 2^(x mul - from) in f16 pairs; their fp32 sums go to `sum`. */
template <int N>
__device__ __forceinline__ void tile_weights(const uint32_t (&v)[N], uint64_t mul, uint64_t from, uint32_t (&p)[N / 2], uint64_t &sum) {
    uint64_t s[2] = {0ull, 0ull};
#pragma unroll
    for (int e = 0; e < N / 2; e++) {
        const float2 x = unpair(fma2(pair(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), mul, from));
        const float p0 = ex2(x.x), p1 = ex2(x.y);
        s[e & 1] = add2(s[e & 1], pair(p0, p1));
        p[e] = pack_half2(p0, p1);
    }
    sum = add2(sum, add2(s[0], s[1]));
}
template <int N>
__device__ __forceinline__ float tile_max(const uint32_t (&v)[N]) {
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < N; e += 8)
#pragma unroll
        for (int i = 0; i < 4; i++)
            m[i] = fmaxf(m[i], fmaxf(__uint_as_float(v[e + 2 * i]), __uint_as_float(v[e + 2 * i + 1])));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
/* Bits of the cache rows [e0, e0 + 32) that a query row sees by order: token t
 * of the last T rows of n, causal or by its row of the tree; t < 0: none. */
__device__ __forceinline__ uint32_t order_bits(const AttendArgs &a, int l, int t, int e0, int n) {
    if (t < 0 || e0 >= n) return 0u;
    const int own = e0 - (n - a.T);                       /* of the first row, among the tokens' own */
    if (own + 32 <= 0) return 0xffffffffu;
    const int live = a.tree ? n - e0 : t + 1 - own;       /* rows from e0 on that can be seen */
    uint32_t bits = live <= 0 ? 0u : live >= 32 ? 0xffffffffu : (1u << live) - 1u;
    if (a.tree && bits) {
        const uint32_t *row = a.tree + l * a.tree_stride + (int64_t)t * a.tree_words;
        const int w0 = own >> 5, sh = own & 31;            /* own >= -31: word -1 stands for rows before the tokens' */
        const uint32_t x = w0 < 0 ? 0xffffffffu : w0 < a.tree_words ? row[w0] : 0u;
        const uint32_t y = sh && w0 + 1 < a.tree_words ? row[w0 + 1] : 0u;
        bits &= __funnelshift_r(x, y, sh);
    }
    return bits;
}

/* ------------------------------------------------------------------ */
/* Layout                                                               */
/* ------------------------------------------------------------------ */

constexpr int TILE_Q = 128, TILE_ROWS = 2 * TILE_Q, TILE_K = 128;      /* cache rows a step */
static_assert(TILE_K == TILE_STEP, "plan");
/* Measured (blocks_used): 4000 f16 rows, 64 query rows: 66 us with every block, 75 at 0.2, 39 at 0.5, 44 at 1. */
constexpr float TILE_JOIN = 0.5f;
/* As FEW_LIFT and FEW_SLACK; a rescaled sum goes through tensor memory here.
 * Normal f16 weights down to 2^-24 of the maximum.  Slack 5, 6 and 8 measure the
 * same (2048 tokens over 8192 rows 290 us, tree of 48 over 30011 rows 165); 3
 * costs 2 % and 11 %. */
constexpr float TILE_LIFT = 10.0f, TILE_SLACK = 5.0f;
constexpr int TILE_SOFT = 2 * TILE_Q;                    /* threads of the two weight groups */

/* q8_0 rows become two f16 operands, the rounded value and what the rounding
 * left, so a product keeps the stored value's 19 bits. */
template <int KT, int HD>
struct TileLayout {
    static constexpr int PARTS = KT == KT_F16 ? 1 : 2;
    static constexpr int STAGES = KT == KT_F16 ? 2 : 1;
    static constexpr int LOADERS = KT == KT_F16 ? 96 : 224;
    static constexpr int THREADS = TILE_SOFT + 32 + LOADERS;
    static constexpr int PANEL = TILE_K * 128;           /* 128 rows of 64 f16 */
    static constexpr int SIDE = HD / 64 * PANEL;         /* one operand of one tile */
    static constexpr int Q = 0;
    static constexpr int K = Q + 2 * SIDE, V = K + STAGES * PARTS * SIDE;
    static constexpr int POS = V + STAGES * PARTS * SIDE;         /* int32 [STAGES][128] */
    static constexpr int BYTES = POS + STAGES * TILE_K * 4 + 1024;    /* 1024: the panels start on a multiple of it */
};

/* ------------------------------------------------------------------ */
/* Kernel                                                               */
/* ------------------------------------------------------------------ */

/* Where a block's walk stands: each role follows the same segments. */
struct TileWalk {
    int64_t at, end, base;
    int it, i0, i1;
    bool first;
};
__device__ __forceinline__ void tile_walk_start(TileWalk &w, const int32_t *steps, int items, int64_t total, int grid, int b) {
    w.at = b * total / grid;
    w.end = (b + 1) * total / grid;
    w.it = 0;
    w.first = true;
    int lo = 0, hi = items;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (steps[mid] <= w.at) lo = mid + 1;
        else hi = mid;
    }
    w.it = lo;
}
__device__ __forceinline__ bool tile_walk_segment(const AttendArgs &a, TileWalk &w, const int32_t *steps, int items, int64_t total) {
    if (w.at >= w.end || !bounds_ok(w.at >= 0 && w.end <= total, a.status)) return false;
    while (steps[w.it] <= w.at) w.it++;
    w.it = uniform(w.it);
    const int base = uniform(w.it ? steps[w.it - 1] : 0), last = uniform(steps[w.it]);
    w.base = base;
    w.i0 = (int)(w.at - base);
    w.i1 = (int)(min(w.end, (int64_t)last) - base);
    return walk_ok(a, items, w.it, w.at, total, a.span ? a.span[w.it] : make_int2(0, 0), TILE_STEP);
}
__device__ __forceinline__ void tile_walk_next(TileWalk &w) {
    w.at = w.base + w.i1;
    w.first = false;
}

/* One thread's wait on a pipeline barrier, bounded by the context's wait
 * limit: false when it gave up or another role did, with the status set. */
__device__ __forceinline__ bool tile_wait(uint64_t *bar, uint32_t parity, volatile int *s_abort, const AttendArgs &a) {
    if (mbar_test(bar, parity)) return true;
    if (*s_abort || !mbar_wait(bar, parity, a.wait_limit)) {
        *s_abort = 1;
        atomicOr(a.status, ST_TIMEOUT);
        return false;
    }
    return true;
}

/* Notes a query row (of `all`) for k_attend_redo. */
__device__ __forceinline__ void tile_redo(const AttendArgs &a, int row, int all) {
    const int i = atomicAdd(a.redo, 1);
    if (bounds_ok(i < all && row >= 0 && row < all, a.status)) a.redo[1 + i] = row;
}

/* A q8_0 block as nine words in registers (2-byte aligned in memory: a block
 * on a 4-byte boundary as it lies, others as the scale and the eight words
 * behind it), and its 32 values from them as f16 pairs: the value rounded (hi)
 * and its remainder (lo = q d - hi, exact in one f16 fma). */
__device__ __forceinline__ void block_words(const uint8_t *p, uint32_t (&x)[9]) {
    if (((uintptr_t)p & 2) == 0) {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __ldg(q + i);
        x[8] = __ldg(reinterpret_cast<const uint16_t *>(q + 8));
    } else {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p + 2);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __ldg(q + i);
        x[8] = __ldg(reinterpret_cast<const uint16_t *>(p));
    }
}
__device__ __forceinline__ void block_values(const uint32_t (&x)[9], bool even, uint32_t (&hi)[16], uint32_t (&lo)[16]) {
    const __half2 d = __half2half2(__ushort_as_half((unsigned short)(even ? x[0] : x[8])));
#pragma unroll
    for (int i = 0; i < 8; i++) {
        uint32_t y[2];
        int8x4_half(even ? __funnelshift_r(x[i], x[i + 1], 16) : x[i], y[0], y[1]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const __half2 q = *reinterpret_cast<const __half2 *>(&y[j]);
            const __half2 h = __hmul2(q, d), r = __hfma2(q, d, __hneg2(h));
            hi[2 * i + j] = *reinterpret_cast<const uint32_t *>(&h);
            lo[2 * i + j] = *reinterpret_cast<const uint32_t *>(&r);
        }
    }
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

/* Byte offset of 16-byte chunk c (of a row's HD / 8) of row r in an operand of PR rows. */
template <int PR = TILE_K>
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) { return (c >> 3) * (PR * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

/* f16: starts the copy of rows [r0, r0 + 128) of one side; rows at and behind
 * n become zeros. */
template <int HD, int LOADERS>
__device__ __forceinline__ void tile_copy(const AttendArgs &a, const uint8_t *p, int r0, int n, uint32_t st, int x) {
    constexpr int CH = HD / 8, RPW = 32 / CH, NW = LOADERS / 32;      /* rows a warp copies at a time */
    if (a.copy16) {
        const int w = x >> 5, r = (x & 31) / CH, c = x % CH;
        const uint8_t *s = p + (int64_t)(r0 + r + RPW * w) * a.cell_stride + 16 * c;
        const int64_t step = (int64_t)RPW * NW * a.cell_stride;
        if (r0 + TILE_K <= n) {
#pragma unroll 4
            for (int y = r + RPW * w; y < TILE_K; y += RPW * NW) {
                cp_async16(st + tile_chunk(y, c), s, 16u);
                s += step;
            }
        } else {
            for (int y = r + RPW * w; y < TILE_K; y += RPW * NW) {
                const bool in = r0 + y < n;
                cp_async16(st + tile_chunk(y, c), in ? s : p, in ? 16u : 0u);
                s += step;
            }
        }
    } else {
        for (int y = x; y < TILE_K * CH * 4; y += LOADERS) {
            const int r = y / (CH * 4), c = y / 4 % CH, q = y & 3;
            const bool in = r0 + r < n;
            cp_async4(st + tile_chunk(r, c) + 4 * q, p + (in ? (int64_t)(r0 + r) * a.cell_stride + 16 * c + 4 * q : 0), in ? 4u : 0u);
        }
    }
}

/* q8_0: one side's blocks on their way through registers, so that the reads of
 * a tile are out before its buffer is free.  A thread's blocks are the same
 * one of their rows (LOADERS is a multiple of the blocks in a row). */
template <int HD, int LOADERS>
struct TileBlocks {
    static constexpr int NB = HD / 32, PER = (TILE_K * NB + LOADERS - 1) / LOADERS;
    uint32_t x[PER][9];
    __device__ __forceinline__ void read(const AttendArgs &a, const uint8_t *p, int r0, int n, int tid) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int y = tid + i * LOADERS, r = y / NB;
            if (y < TILE_K * NB && r0 + r < n) {
                block_words(p + (int64_t)(r0 + r) * a.cell_stride + 34 * (y % NB), x[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 9; e++) x[i][e] = 0;      /* value 0, scale 0 */
            }
        }
    }
    __device__ __forceinline__ void write(uint32_t st, uint32_t part, int tid) const {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int y = tid + i * LOADERS, r = y / NB, b = y % NB;
            if (y >= TILE_K * NB) break;
            uint32_t hi[16], lo[16];
            block_values(x[i], (b & 1) == 0, hi, lo);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t d = st + tile_chunk(r, 4 * b + e);
                sts128(d, hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3]);
                sts128(d + part, lo[4 * e], lo[4 * e + 1], lo[4 * e + 2], lo[4 * e + 3]);
            }
        }
    }
};

/* Starts the copy of query rows [r0, r0 + ROWS) of kv head h of cache l as
 * operands of PR rows; rows at and behind R become zeros.  A warp copies 32 /
 * (HD / 8) rows at a time, token and head stepping along. */
template <int HD, int ROWS, int PR, int LOADERS>
__device__ __forceinline__ void tile_load_q(const AttendArgs &a, int l, int h, int r0, uint32_t st, int x) {
    constexpr int CH = HD / 8, RPW = 32 / CH, STEP = RPW * (LOADERS / 32), SIDE = HD / 64 * PR * 128;
    const int c = x % CH, first = (x >> 5) * RPW + (x & 31) / CH, R = a.T * a.G;
    int r = r0 + first, t = r / a.G, g = r - t * a.G;
    const int dt = STEP / a.G, dg = STEP - dt * a.G;
    const __half *base = a.q + l * a.q_cache + (int64_t)h * a.G * a.q_head + 8 * c;
    for (int q = first; q < ROWS; q += STEP, r += STEP) {
        const bool in = r < R;
        cp_async16(st + (q / PR) * SIDE + tile_chunk<PR>(q % PR, c), in ? base + t * a.q_tok + g * a.q_head : base, in ? 16u : 0u);
        t += dt;
        g += dg;
        if (g >= a.G) { g -= a.G; t++; }
    }
}

/* Warps 0-7 make weights (one thread a query row), warp 8 issues the products,
 * the others bring Q, K and V: f16 by 16-byte asynchronous copies, q8_0 through
 * registers.  Plain f16 calls use one score tile of 128 cache rows and hand
 * its weights over in halves; capped, biased and windowed calls, and q8_0
 * ones, hold fewer scores in registers and use two of 64 (whose products cost
 * nearly those of 128).
 *
 * 8 units of 8192 f16 rows, 2048 tokens of 4 heads each, head_dim 128: 255 us
 * with the rows in L2 (945 TFLOP/s), 295 us from DRAM (tensor pipe 42 % active);
 * 32768 rows: 1047 TFLOP/s.  Without the
 * weights a step of 128 cache rows takes 1.5 us, near cuBLAS's
 * rate, with them 2.4: bound by the chain scores - weights - values of a row
 * tile, for which the two 128-column sums leave no second score buffer.
 * Capped scores (tree of 48 over 2 caches of 8 units, 30011 rows): 157 us,
 * issue 41 % active; q8_0 rows cost 8 us a step, in conversion and twice the
 * products. */
template <int KT, int HD, bool EXTRA>
__global__ void __launch_bounds__(TileLayout<KT, HD>::THREADS, 1) k_attend_tile(const AttendArgs a) {
    using L = TileLayout<KT, HD>;
    constexpr int NB = EXTRA || KT == KT_Q8_0 ? 2 : 1, TILE_H = TILE_K / NB;      /* score buffers of a row tile, cache rows of each */
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t b_q_full, b_q_free, b_o_full, b_drain, b_pv[2], b_s_full[2][2], b_p_ready[2][2];
    __shared__ __align__(8) uint64_t b_k_full[L::STAGES], b_k_free[L::STAGES], b_v_full[L::STAGES], b_v_free[L::STAGES];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, w = uniform(tid >> 5);
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int32_t *s_pos = reinterpret_cast<const int32_t *>(smem_raw + (smem - smem_u32(smem_raw)) + L::POS);
    const int units = a.n_layer * a.n_head_kv, items = units * a.groups, R = a.T * a.G;
    const int32_t *steps = a.steps;
    const int64_t total = uniform(steps[items - 1]);
    const int b = blockIdx.x, grid = blocks_used(total, items, gridDim.x, TILE_JOIN);
    const bool want_pos = EXTRA && (a.window > 0 || a.slopes != nullptr);

    if (tid == 0) {
        mbar_init(&b_q_full, L::LOADERS / 32);
        mbar_init(&b_q_free, 1);
        mbar_init(&b_o_full, 1);
        mbar_init(&b_drain, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&b_pv[i], 1);
            for (int d = 0; d < 2; d++) {
                mbar_init(&b_s_full[i][d], 1);
                mbar_init(&b_p_ready[i][d], TILE_Q / 32);
            }
        }
        for (int i = 0; i < L::STAGES; i++) {
            mbar_init(&b_k_full[i], L::LOADERS / 32);
            mbar_init(&b_v_full[i], L::LOADERS / 32);
            mbar_init(&b_k_free[i], 1);
            mbar_init(&b_v_free[i], 1);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (w == TILE_SOFT / 32) {                                /* the product warp owns the tensor memory */
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    /* columns: S (and P) of row tile x, buffer d at 128 x + 64 d, O at 256 + 128 x */

    TileWalk wk;
    if (b < grid) tile_walk_start(wk, steps, items, total, grid, b);
    else wk.at = wk.end = 0;

    if (w > TILE_SOFT / 32) {
        /* ---------------- loaders ---------------- */
        const int x = tid - TILE_SOFT - 32;
        uint32_t kc = 0, vc = 0;
        uint64_t *pending = nullptr;                          /* the copy still to be announced */
        auto announce = [&]() {
            fence_async_smem();                               /* every lane's own writes, then one arrival a warp */
            __syncwarp();
            if (lane == 0) mbar_arrive(pending);
            pending = nullptr;
        };
        auto wait_free = [&](uint64_t *bar, uint32_t parity) -> bool {
            if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
            if (pending) {                                    /* nobody may wait for it while we wait */
                cp_async_wait<0>();
                announce();
            }
            return __all_sync(0xffffffffu, tile_wait(bar, parity, &s_abort, a));
        };
        auto issued = [&](uint64_t *bar) {
            cp_async_commit();
            if (KT != KT_F16) {                               /* the rows were converted, not copied */
                cp_async_wait<0>();
                if (pending) announce();
                pending = bar;
                announce();
            } else {
                if (pending) {
                    cp_async_wait<1>();
                    announce();
                }
                pending = bar;
            }
        };
        bool ok = true;
        for (uint32_t seg = 0; ok && tile_walk_segment(a, wk, steps, items, total); seg++, tile_walk_next(wk)) {
            const int u = wk.it / a.groups, grp = wk.it - u * a.groups, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
            const int n = attend_rows(a, u);
            const int2 span = a.span ? a.span[wk.it] : make_int2(0, 0);
            const int hs = (min(span.x, n) + TILE_K - 1) / TILE_K;
            const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride, *v = a.v[l] + (int64_t)h * a.head_stride;
            const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
            if (seg && !wait_free(&b_q_free, (seg - 1) & 1)) break;
            tile_load_q<HD, TILE_ROWS, TILE_Q, L::LOADERS>(a, l, h, grp * TILE_ROWS, smem + L::Q, x);
            issued(&b_q_full);
            for (int i = wk.i0; i < wk.i1; i++) {
                const int row0 = i < hs ? i * TILE_K : span.y + (i - hs) * TILE_K;
                const int ks = kc % L::STAGES, vs = vc % L::STAGES;
                const uint32_t k_at = smem + L::K + ks * L::PARTS * L::SIDE, v_at = smem + L::V + vs * L::PARTS * L::SIDE;
                TileBlocks<HD, L::LOADERS> kb, vb;            /* q8_0 only */
                if (KT == KT_Q8_0) {
                    kb.read(a, k, row0, n, x);
                    vb.read(a, v, row0, n, x);
                }
                if (kc >= L::STAGES && !wait_free(&b_k_free[ks], (kc / L::STAGES - 1) & 1)) { ok = false; break; }
                if (KT == KT_F16) tile_copy<HD, L::LOADERS>(a, k, row0, n, k_at, x);
                else kb.write(k_at, L::SIDE, x);
                issued(&b_k_full[ks]);
                kc++;
                if (vc >= L::STAGES && !wait_free(&b_v_free[vs], (vc / L::STAGES - 1) & 1)) { ok = false; break; }
                if (KT == KT_F16) tile_copy<HD, L::LOADERS>(a, v, row0, n, v_at, x);
                else vb.write(v_at, L::SIDE, x);
                for (int y = x; want_pos && y < TILE_K; y += L::LOADERS) {      /* with V: free once the weights are made */
                    const bool in = row0 + y < n;
                    cp_async4(smem + L::POS + (vs * TILE_K + y) * 4, pos + (in ? row0 + y : 0), in ? 4u : 0u);
                }
                issued(&b_v_full[vs]);
                vc++;
            }
        }
        cp_async_wait<0>();
        if (pending) announce();
    } else if (w == TILE_SOFT / 32) {
        /* ---------------- products ---------------- */
        /* Every other role waits for this warp, so a product has to cost few instructions: the warp stays converged
         * and one lane issues (operands then live in uniform registers), and the tensor-memory addresses are constants,
         * for all of it is this block's. */
        const uint32_t lead = lane == 0;
        {
            constexpr uint32_t qk = tile_idesc(TILE_H, false), pv = tile_idesc(HD, true);
            constexpr uint32_t STEP = L::PARTS * L::SIDE >> 4, PART = L::SIDE >> 4;      /* stage to stage, part to part */
            constexpr uint32_t HALF = 64 * 128 >> 4;                                     /* 64 rows of a panel */
            const uint32_t d_q = tile_desc(smem + L::Q, 16), d_k = tile_desc(smem + L::K, 16), d_v = tile_desc(smem + L::V, L::PANEL);
            uint32_t ks = 0, kp = 0, vs = 0, vp = 0, pp = 0;            /* stages and phases; pp: bit 2 x + d */
            auto wait = [&](uint64_t *bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, tile_wait(bar, parity, &s_abort, a)); };
            /* O += P V over cache rows 64 e .. 64 e + 63 of the step */
            auto values = [&](uint32_t x, uint32_t e, uint32_t vd, bool add) {
                const uint32_t o = 256 + 128 * x, p = 128 * x + (NB == 2 ? 64 : 32) * e;
                tc_mma_ts(lead, o, p, vd, pv, add);
#pragma unroll
                for (int s = 1; s < L::PARTS * (64 / 16); s++) {
                    constexpr int PER = 64 / 16;
                    tc_mma_ts(lead, o, p + 8 * (s % PER), vd + ((s / PER) * PART + (s % PER) * (2048 >> 4)), pv, true);
                }
                if (NB == 2) tc_commit(lead, &b_pv[x]);
            };
            auto scores = [&](uint32_t x, uint32_t d, uint32_t kd) {                     /* S = Q K^T */
#pragma unroll
                for (int s = 0; s < L::PARTS * (HD / 16); s++) {
                    constexpr int PER = HD / 16;
                    const int off = ((s % PER) / 4) * (L::PANEL >> 4) + (s % 4) * (32 >> 4);
                    tc_mma_ss(lead, 128 * x + 64 * d, d_q + x * PART + off, kd + ((s / PER) * PART + off), qk, s > 0);
                }
                tc_commit(lead, &b_s_full[x][d]);
            };
            if (tmem != 0) {
                s_abort = 1;
                atomicOr(a.status, ST_TIMEOUT);
            }
            bool ok = tmem == 0;
            for (uint32_t seg = 0; ok && tile_walk_segment(a, wk, steps, items, total); seg++, tile_walk_next(wk)) {
                const bool two = R - (wk.it % a.groups) * TILE_ROWS > TILE_Q;
                const int N = wk.i1 - wk.i0;
                if (!(ok = wait(&b_q_full, seg & 1) && wait(&b_k_full[ks], kp))) break;
                for (uint32_t d = 0; d < NB; d++) {
                    scores(0, d, d_k + ks * STEP + d * HALF);
                    if (two) scores(1, d, d_k + ks * STEP + d * HALF);
                }
                tc_commit(lead, &b_k_free[ks]);
                if (++ks == L::STAGES) { ks = 0; kp ^= 1; }
                if (N == 1) tc_commit(lead, &b_q_free);
                for (int i = 0; ok && i < N; i++) {
                    const uint32_t kd = d_k + ks * STEP, vd = d_v + vs * STEP;
                    const bool more = i + 1 < N;
                    if (!(ok = wait(&b_v_full[vs], vp))) break;
                    /* one row tile's weights of 64 cache rows, and the scores that take their place */
                    auto turn = [&](uint32_t x, uint32_t e) {
                        if (!(ok = wait(&b_p_ready[x][e], pp >> (2 * x + e) & 1))) return;
                        pp ^= 1u << (2 * x + e);
                        tc_fence_after();
                        values(x, e, vd + e * HALF, i > 0 || e > 0);
                        if (!more || (NB == 1 && e == 0)) return;
                        if (x == 0 && (NB == 1 || e == 0) && !(ok = wait(&b_k_full[ks], kp))) return;
                        scores(x, NB == 2 ? e : 0, kd + (NB == 2 ? e * HALF : 0));
                    };
                    if (NB == 2) {
                        for (uint32_t e = 0; ok && e < 2; e++) {
                            turn(0, e);
                            if (ok && two) turn(1, e);
                        }
                    } else {
                        for (uint32_t x = 0; ok && x < (two ? 2 : 1); x++) {
                            turn(x, 0);
                            if (ok) turn(x, 1);
                        }
                    }
                    if (!ok) break;
                    tc_commit(lead, &b_v_free[vs]);
                    if (++vs == L::STAGES) { vs = 0; vp ^= 1; }
                    if (more) {
                        tc_commit(lead, &b_k_free[ks]);
                        if (++ks == L::STAGES) { ks = 0; kp ^= 1; }
                        if (i + 2 == N) tc_commit(lead, &b_q_free);
                    }
                }
                if (!ok) break;
                tc_commit(lead, &b_o_full);
            }
        }
        __syncwarp();
    } else {
        /* ---------------- weights ---------------- */
        const int x = w >> 2, row = tid & (TILE_Q - 1);       /* row tile, query row in it */
        const uint32_t mine = tmem + ((uint32_t)(w & 3) << 21);      /* lanes 32 (w mod 4) on */
        const uint32_t S = mine + 128 * x, O = mine + 256 + 128 * x;
        const ScoreMap map(a);
        uint32_t sc = 0, tiles = 0;                           /* score tiles seen, steps of the segments before */
        bool ok = true;

        /* items without a row to see */
        for (int it = b; it < items; it += gridDim.x) {
            if (steps[it] != (it ? steps[it - 1] : 0)) continue;
            const int u = it / a.groups, grp = it - u * a.groups, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
            for (int y = tid; y < TILE_ROWS * HD / 8; y += TILE_SOFT) {
                const int r = grp * TILE_ROWS + y / (HD / 8);
                if (r >= R) break;
                *reinterpret_cast<uint4 *>(a.out + l * a.o_cache + (r / a.G) * a.o_tok + (h * a.G + r % a.G) * a.o_head +
                                           y % (HD / 8) * 8) = make_uint4(0, 0, 0, 0);
            }
            const int r = grp * TILE_ROWS + tid;
            if (r < R) {
                if (a.lse) a.lse[((int64_t)l * a.T + r / a.G) * a.n_head_kv * a.G + h * a.G + r % a.G] = -INFINITY;
                if (a.norm) a.norm[(int64_t)u * R + r] = make_float2(0.0f, 0.0f);
            }
        }

        for (uint32_t seg = 0; tile_walk_segment(a, wk, steps, items, total); seg++, tile_walk_next(wk)) {
            const int u = wk.it / a.groups, grp = wk.it - u * a.groups, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
            const int n = attend_rows(a, u);
            const int rows = min(TILE_ROWS, R - grp * TILE_ROWS);
            const bool active = x == 0 || rows > TILE_Q;
            const int2 span = a.span ? a.span[wk.it] : make_int2(0, 0);
            const int hs = (min(span.x, n) + TILE_K - 1) / TILE_K;
            const int r = grp * TILE_ROWS + x * TILE_Q + row;
            const bool in = r < R;
            const int t = in ? r / a.G : -1, head = h * a.G + r % a.G;
            const int tp = in && want_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
            const float slope2 = EXTRA && in && a.slopes ? a.slopes[head] * LOG2E : 0.0f;
            const int64_t lo = (int64_t)tp - a.window;
            float m = -INFINITY;
            uint64_t sum = 0ull;                              /* two partial sums */
            for (int y = 0; ok && active && y < NB * (wk.i1 - wk.i0); y++) {
                const int i = wk.i0 + y / NB;
                const uint32_t d = y % NB, tc = tiles + y / NB, T = S + 64 * d;
                const int j0 = (i < hs ? i * TILE_K : span.y + (i - hs) * TILE_K) + TILE_H * d;
                if (!tile_wait(&b_s_full[x][d], sc / NB & 1, &s_abort, a)) ok = false;
                if (want_pos && ok && !tile_wait(&b_v_full[tc % L::STAGES], (tc / L::STAGES) & 1, &s_abort, a)) ok = false;
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc_fence_after();
                const bool all = j0 + TILE_H <= n - a.T && (!EXTRA || a.window <= 0);    /* every token sees every row */
                uint32_t v[TILE_H];
                tc_ld64(*reinterpret_cast<uint32_t (*)[64]>(v), T);
                if (TILE_H > 64) tc_ld64(*reinterpret_cast<uint32_t (*)[64]>(v + TILE_H - 64), T + TILE_H - 64);
                tc_wait_ld();
                uint64_t mul = pair(map.scale, map.scale);
                if (EXTRA) {                                  /* the scores made final in place */
                    float far = 0.0f;
#pragma unroll
                    for (int e = 0; e < TILE_H / 2; e++) {
                        const float2 z = unpair(mul2(pair(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), mul));
                        v[2 * e] = __float_as_uint(z.x);
                        v[2 * e + 1] = __float_as_uint(z.y);
                        far = fmaxf(far, fmaxf(fabsf(z.x), fabsf(z.y)));
                    }
                    if (map.cap > 0.0f) tile_cap<TILE_H>(v, map.cap, far, T);
                    mul = pair(1.0f, 1.0f);
                }
                if (want_pos || !all || (!EXTRA && map.scale <= 0.0f)) {
                    uint32_t bits[TILE_H / 32];
#pragma unroll
                    for (int e = 0; e < TILE_H / 32; e++) bits[e] = order_bits(a, l, t, j0 + 32 * e, n);
                    if (want_pos) {
                        const int4 *ps = reinterpret_cast<const int4 *>(s_pos + (tc % L::STAGES) * TILE_K + TILE_H * d);
#pragma unroll
                        for (int e = 0; e < TILE_H / 4; e++) {
                            const int4 q = ps[e];
                            const int pj[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int f = 0; f < 4; f++) {
                                v[4 * e + f] = __float_as_uint(fmaf(-slope2, (float)(tp - pj[f]), __uint_as_float(v[4 * e + f])));
                                if (a.window > 0 && !(pj[f] >= lo || pj[f] < a.sink)) bits[e / 8] &= ~(1u << (4 * (e % 8) + f));
                            }
                        }
                    }
                    if (!EXTRA && map.scale <= 0.0f) {        /* a masked score below stays below only if final */
#pragma unroll
                        for (int e = 0; e < TILE_H; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * map.scale);
                        mul = pair(1.0f, 1.0f);
                    }
#pragma unroll
                    for (int e = 0; e < TILE_H; e++)
                        if (!(bits[e / 32] >> (e & 31) & 1u)) v[e] = 0xff800000u;
                }
                const float top = tile_max<TILE_H>(v) * unpair(mul).x;
                if (__any_sync(0xffffffffu, top > m + TILE_SLACK)) {
                    /* the maximum has outrun the sums: rescale them, once the products under way have landed */
                    const float to = fmaxf(m, top), f = to == m ? 1.0f : ex2(m - to);
                    m = to;
                    sum = mul2(sum, pair(f, f));
                    if (y > 0) {                              /* (with one buffer they have, or S would not be full) */
                        if (NB == 2 && !tile_wait(&b_pv[x], (sc - 1) & 1, &s_abort, a)) ok = false;
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD / 16; c++) {
                            uint32_t o[16];
                            tc_ld16(o, O + 16 * c);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tc_st16(O + 16 * c, o);
                        }
                    }
                }
                const float from = m == -INFINITY ? 0.0f : TILE_LIFT - m;
                const uint64_t off = pair(from, from);
#pragma unroll
                for (int e = 0; e < TILE_H / 32; e++) {       /* over the scores */
                    uint32_t p[16];
                    tile_weights<32>(*reinterpret_cast<const uint32_t (*)[32]>(v + 32 * e), mul, off, p, sum);
                    tc_st16(T + 16 * e, p);
                    if (e & 1) {                              /* 64 cache rows: the value product may start */
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&b_p_ready[x][NB == 2 ? d : e / 2]);
                    }
                }
                sc++;
            }
            /* a wait that gave up leaves the sums as they are (that call's output is undefined), but every thread still
             * comes to the barriers below, as often as the others */
            if (ok && !tile_wait(&b_o_full, seg & 1, &s_abort, a)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();

            const float2 halves = unpair(sum);
            const float total_w = halves.x + halves.y;
            const int64_t base = wk.base;
            const int c0 = (int)(((base + 1) * grid - 1) / total), c1 = (int)(((int64_t)steps[wk.it] * grid - 1) / total);
            if (!share_ok(a, c0, c1, b, grid)) {
                /* checked build: nothing is put out (the same for all threads) */
            } else if (c0 == c1) {
                const bool none = total_w == 0.0f;
                const float inv = none ? 0.0f : 1.0f / total_w;
                bool bad = false;
                if (active) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; c++) {
                        uint32_t v[32];
                        tc_ld32(v, O + 32 * c);
                        tc_wait_ld();
                        float fin = 0.0f;
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            const float y = none ? 0.0f : __uint_as_float(v[e]) * inv;
                            fin += y * 0.0f;
                            v[e] = __float_as_uint(y);
                        }
                        bad |= fin != 0.0f;                   /* NaN: some value is not finite */
                        if (in) {
                            uint4 *d = reinterpret_cast<uint4 *>(a.out + l * a.o_cache + t * a.o_tok + head * a.o_head + 32 * c);
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                d[e] = make_uint4(pack_half2(__uint_as_float(v[8 * e]), __uint_as_float(v[8 * e + 1])),
                                                  pack_half2(__uint_as_float(v[8 * e + 2]), __uint_as_float(v[8 * e + 3])),
                                                  pack_half2(__uint_as_float(v[8 * e + 4]), __uint_as_float(v[8 * e + 5])),
                                                  pack_half2(__uint_as_float(v[8 * e + 6]), __uint_as_float(v[8 * e + 7])));
                        }
                    }
                    if (in) {
                        if (a.lse) a.lse[((int64_t)l * a.T + t) * a.n_head_kv * a.G + head] = none ? -INFINITY : (m - TILE_LIFT + log2f(total_w)) * LN2;
                        if (a.norm) a.norm[(int64_t)u * R + r] = none ? make_float2(0.0f, 0.0f) : make_float2(m - TILE_LIFT, inv);
                        if (bad) tile_redo(a, u * R + r, units * R);
                    }
                }
            } else {
                const int slot = 2 * b + (wk.first ? 0 : 1);
                if (active) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; c++) {
                        uint32_t v[32];
                        tc_ld32(v, O + 32 * c);
                        tc_wait_ld();
                        if (in) {
                            /* [slot][dim / 4][row][4]: a warp's rows side by side */
                            uint4 *d = reinterpret_cast<uint4 *>(a.part_o) + ((int64_t)slot * (HD / 4) + 8 * c) * TILE_ROWS + x * TILE_Q + row;
#pragma unroll
                            for (int e = 0; e < 8; e++) d[e * TILE_ROWS] = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                        }
                    }
                    if (in) a.part_ml[(int64_t)slot * TILE_ROWS + x * TILE_Q + row] = make_float2(m, total_w);
                }
                __threadfence();
                asm volatile("bar.sync 1, %0;" ::"n"(TILE_SOFT) : "memory");
                if (tid == 0) s_last = atomicAdd(&a.arrived[c0], 1) == c1 - c0;
                asm volatile("bar.sync 1, %0;" ::"n"(TILE_SOFT) : "memory");
                if (s_last) {
                    __threadfence();
                    if (tid == 0) a.arrived[c0] = 0;
                    const int s0 = 2 * c0 + (c0 * total / grid >= base ? 0 : 1);
                    if (tid < rows) {                         /* a thread a row */
                        auto slot_of = [&](int s) { return (int64_t)(s == 0 ? s0 : 2 * (c0 + s)); };
                        const int rq = grp * TILE_ROWS + tid, tq = rq / a.G, hq = h * a.G + rq % a.G, nS = c1 - c0 + 1;
                        float mm = -INFINITY, ss = 0.0f;
#pragma unroll 4
                        for (int s = 0; s < nS; s++) mm = fmaxf(mm, __ldcg(&a.part_ml[slot_of(s) * TILE_ROWS + tid]).x);
#pragma unroll 4
                        for (int s = 0; s < nS; s++) {
                            const float2 y = __ldcg(&a.part_ml[slot_of(s) * TILE_ROWS + tid]);
                            ss = fmaf(y.y, y.x == -INFINITY ? 0.0f : ex2(y.x - mm), ss);
                        }
                        const bool none = ss == 0.0f;
                        const float inv = none ? 0.0f : 1.0f / ss;
                        float fin = 0.0f;
                        uint4 *dst = reinterpret_cast<uint4 *>(a.out + l * a.o_cache + tq * a.o_tok + hq * a.o_head);
#pragma unroll 1
                        for (int part = 0; part < HD / 32; part++) {     /* 32 dims at a time stay in registers */
                            float4 acc[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                            for (int s = 0; s < nS; s++) {
                                const float2 y = __ldcg(&a.part_ml[slot_of(s) * TILE_ROWS + tid]);
                                const float4 *src = reinterpret_cast<const float4 *>(a.part_o) + (slot_of(s) * (HD / 4) + 8 * part) * TILE_ROWS + tid;
                                float4 o[8];
#pragma unroll
                                for (int e = 0; e < 8; e++) o[e] = __ldcg(src + e * TILE_ROWS);
                                const float g = y.x == -INFINITY ? 0.0f : ex2(y.x - mm);
                                if (g != 0.0f) {
#pragma unroll
                                    for (int e = 0; e < 8; e++) {
                                        acc[e].x = fmaf(o[e].x, g, acc[e].x);
                                        acc[e].y = fmaf(o[e].y, g, acc[e].y);
                                        acc[e].z = fmaf(o[e].z, g, acc[e].z);
                                        acc[e].w = fmaf(o[e].w, g, acc[e].w);
                                    }
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                if (none) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                acc[e].x *= inv;
                                acc[e].y *= inv;
                                acc[e].z *= inv;
                                acc[e].w *= inv;
                                fin += acc[e].x * 0.0f + acc[e].y * 0.0f + acc[e].z * 0.0f + acc[e].w * 0.0f;
                            }
#pragma unroll
                            for (int e = 0; e < 8; e += 2)
                                dst[4 * part + e / 2] = make_uint4(pack_half2(acc[e].x, acc[e].y), pack_half2(acc[e].z, acc[e].w),
                                                                   pack_half2(acc[e + 1].x, acc[e + 1].y), pack_half2(acc[e + 1].z, acc[e + 1].w));
                        }
                        if (fin != 0.0f) tile_redo(a, u * R + rq, units * R);
                        if (a.lse) a.lse[((int64_t)l * a.T + tq) * a.n_head_kv * a.G + hq] = none ? -INFINITY : (mm - TILE_LIFT + log2f(ss)) * LN2;
                        if (a.norm) a.norm[(int64_t)u * R + rq] = none ? make_float2(0.0f, 0.0f) : make_float2(mm - TILE_LIFT, inv);
                    }
                }
            }
            tiles += wk.i1 - wk.i0;
            /* s_last is read before it is set again, and a group without rows stays with the other */
            asm volatile("bar.sync 1, %0;" ::"n"(TILE_SOFT) : "memory");
        }
        tc_fence_before();
    }

    __syncthreads();
    if (w == TILE_SOFT / 32) {
        tc_fence_after();
        if (s_abort) {                                        /* products may still run: wait for them, within a bound */
            tc_commit(lane == 0, &b_drain);
            mbar_wait(&b_drain, 0);
            __syncwarp();
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

/* ------------------------------------------------------------------ */
/* Masses                                                               */
/* ------------------------------------------------------------------ */

constexpr int MASS_TILE_THREADS = 256, MASS_Q = 64, MASS_C = MASS_Q / 2;      /* query rows a tile, a thread */
template <int KT, int HD>
struct MassTileLayout {
    using T = TileLayout<KT, HD>;
    static constexpr int QSIDE = HD / 64 * MASS_Q * 128;
    static constexpr int K = 0, Q = T::PARTS * T::SIDE;           /* two query tiles */
    static constexpr int COLS = Q + 2 * QSIDE;                   /* per query row: -log2 of its denominator, slope, position */
    static constexpr int SUM = COLS + 3 * 3 * MASS_Q * 4;         /* three tiles': the next is written while one is slow to read the last */
    static constexpr int BYTES = SUM + TILE_K * 4 + 1024;
};

/* The mass of q8_0 row j of unit u, whose position is pj, by one thread: where
 * a block of the key passes f16's range, else it is NaN for another reason. */
template <int KT, int HD>
__device__ __noinline__ float row_mass(const AttendArgs &a, int u, int j, int n, int pj) {
    const int l = u / a.n_head_kv, h = u - l * a.n_head_kv;
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride + (int64_t)j * a.cell_stride;
    bool past = false;
    for (int b = 0; b < HD / 32; b++) past |= fabsf(half_at(k + 34 * b)) >= TILE_SCALE;
    if (!past) return NAN;
    const ScoreMap map(a);
    float mass = 0.0f;
    for (int t = 0; t < a.T; t++) {
        const int tp = a.tok_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
        if (!attend_sees(a, l, t, j, n, pj, (int64_t)tp - a.window)) continue;
        for (int g = 0; g < a.G; g++) {
            const int head = h * a.G + g;
            const float2 nm = a.norm[((int64_t)u * a.T + t) * a.G + g];
            const float x = attend_score<KT, HD>(map, k, a.q + l * a.q_cache + t * a.q_tok + head * a.q_head,
                                                 a.slopes ? a.slopes[head] * LOG2E : 0.0f, tp, pj);
            mass = fmaf(ex2(x - nm.x), nm.y, mass);
        }
    }
    return mass;
}

/* The scores again, now with the denominators known: S^T = K Q^T with the 128
 * cache rows as the matrix rows, so a thread owns a cache row and adds up its
 * weights over the query rows as they come by, 64 a tile, in one order; no
 * weight leaves the thread.  Two threads share a cache row (32 columns each).
 * While a tile's weights are made, the next one's product runs; a block is
 * short (one tile of cache rows against a few of query rows), so two of them
 * share an SM and cover each other's start (32 units of 12289 q8_0 rows, 160
 * query rows, window 8192: 141 us with 128 query rows a tile and one block an
 * SM, 86 us so). */
template <int KT, int HD, bool EXTRA>
__global__ void __launch_bounds__(MASS_TILE_THREADS, 2) k_mass_tile(const __grid_constant__ AttendArgs a) {
    using L = TileLayout<KT, HD>;
    using M = MassTileLayout<KT, HD>;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t b_done[2], b_drain;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ int s_first[MASS_TILE_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, w = uniform(tid >> 5), row = tid & (TILE_K - 1), half = tid >> 7;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const base = smem_raw + (smem - smem_u32(smem_raw));
    float *const s_cols = reinterpret_cast<float *>(base + M::COLS);        /* [3][3][64] */
    float *const s_sum = reinterpret_cast<float *>(base + M::SUM);
    const int u = blockIdx.y, l = u / a.n_head_kv, h = u - l * a.n_head_kv, R = a.T * a.G;
    const int n = uniform(attend_rows(a, u));
    const bool want_pos = EXTRA && (a.window > 0 || a.slopes != nullptr);
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride;
    const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
    const ScoreMap map(a);
    if (blockIdx.x * TILE_K >= n) return;
    if (tid == 0) {
        mbar_init(&b_done[0], 1);
        mbar_init(&b_done[1], 1);
        mbar_init(&b_drain, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (w == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 128;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    /* the earliest position that some token's window reaches */
    int first = INT_MAX;
    if (EXTRA && a.window > 0) {
        for (int t = tid; t < a.T; t += MASS_TILE_THREADS) first = min(first, a.tok_pos[l * a.tok_pos_stride + t]);
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) s_first[w] = first;
    }
    __syncthreads();
    tc_fence_after();
    if (EXTRA && a.window > 0)
        for (int i = 0; i < MASS_TILE_THREADS / 32; i++) first = min(first, s_first[i]);
    const uint32_t tmem = uniform(s_tmem);
    uint32_t done = 0;                                        /* products issued so far, of the whole block */
    bool ok = true;
    for (int j0 = blockIdx.x * TILE_K; ok && j0 < n; j0 += gridDim.x * TILE_K) {
        const int j = j0 + row, pj = want_pos && j < n ? pos[j] : 0;
        const bool near = j < n && (!EXTRA || a.window <= 0 || pj >= (int64_t)first - a.window || pj < a.sink);
        uint64_t sum = 0ull;
        /* by order, token t sees row j only if j <= n - T + t: query rows before that see none of the tile */
        const int q_from = a.tree ? 0 : max(0, j0 - (n - a.T)) * a.G / MASS_Q * MASS_Q;
        const int tiles = R > q_from ? (R - q_from + MASS_Q - 1) / MASS_Q : 0;
        if (__syncthreads_or(near) && tiles > 0) {
            auto load = [&](int i) {                          /* query tile i and its columns' constants */
                const int r0 = q_from + i * MASS_Q;
                tile_load_q<HD, MASS_Q, MASS_Q, MASS_TILE_THREADS>(a, l, h, r0, smem + M::Q + (i & 1) * M::QSIDE, tid);
                if (tid < MASS_Q) {
                    const int r = r0 + tid;
                    const bool in = r < R;
                    const float2 nm = in ? a.norm[(int64_t)u * R + r] : make_float2(0.0f, 0.0f);
                    float *c = s_cols + (i % 3) * 3 * MASS_Q + tid;
                    c[0] = log2f(nm.y) - nm.x;
                    if (EXTRA) {
                        c[MASS_Q] = in && a.slopes ? -LOG2E * a.slopes[h * a.G + r % a.G] : 0.0f;
                        c[2 * MASS_Q] = __int_as_float(in && want_pos ? a.tok_pos[l * a.tok_pos_stride + r / a.G] : 0);
                    }
                }
            };
            const uint32_t lead = tid == 0;
            auto product = [&](int i) {
                if (w != 0) return;
                const uint32_t dk = tile_desc(smem + M::K, 16), dq = tile_desc(smem + M::Q + (i & 1) * M::QSIDE, 16);
                tc_fence_after();
#pragma unroll
                for (int s = 0; s < L::PARTS * (HD / 16); s++) {
                    constexpr int PER = HD / 16;
                    const int panel = (s % PER) / 4, in = (s % 4) * (32 >> 4);
                    tc_mma_ss(lead, tmem + MASS_Q * (i & 1), dk + (s / PER) * (L::SIDE >> 4) + panel * (L::PANEL >> 4) + in,
                              dq + panel * (MASS_Q * 128 >> 4) + in, tile_idesc(MASS_Q, false), s > 0);
                }
                tc_commit(lead, &b_done[(done + i) & 1]);
            };
            auto ready = [&]() {                              /* what was copied is there for all, and for the product */
                cp_async_commit();
                cp_async_wait<0>();
                fence_async_smem();
                tc_fence_before();
                __syncthreads();
            };
            if (KT == KT_F16) {
                tile_copy<HD, MASS_TILE_THREADS>(a, k, j0, n, smem + M::K, tid);
            } else {
                TileBlocks<HD, MASS_TILE_THREADS> kb;
                kb.read(a, k, j0, n, tid);
                kb.write(smem + M::K, L::SIDE, tid);
            }
            load(0);
            ready();
            product(0);
            for (int i = 0; i < tiles; i++) {
                if (i + 1 < tiles) load(i + 1);
                if (!tile_wait(&b_done[(done + i) & 1], ((done + i) >> 1) & 1, &s_abort, a)) ok = false;
                if (i + 1 < tiles) {
                    ready();                                  /* everyone is done with the product before this one, too */
                    product(i + 1);
                }
                if (!__all_sync(0xffffffffu, ok)) { ok = false; continue; }
                tc_fence_after();
                const int r0 = q_from + i * MASS_Q + MASS_C * half;
                uint32_t v[MASS_C];
                const uint32_t mine = tmem + ((uint32_t)(w & 3) << 21) + MASS_Q * (i & 1) + MASS_C * half;
                tc_ld32(v, mine);
                tc_wait_ld();
                const float *c = s_cols + (i % 3) * 3 * MASS_Q + MASS_C * half;
                uint64_t mul = pair(map.scale, map.scale);
                if (EXTRA) {
                    float far = 0.0f;
#pragma unroll
                    for (int e = 0; e < MASS_C / 2; e++) {
                        const float2 z = unpair(mul2(pair(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), mul));
                        v[2 * e] = __float_as_uint(z.x);
                        v[2 * e + 1] = __float_as_uint(z.y);
                        far = fmaxf(far, fmaxf(fabsf(z.x), fabsf(z.y)));
                    }
                    mul = pair(1.0f, 1.0f);
                    if (map.cap > 0.0f) tile_cap<MASS_C>(v, map.cap, far, mine);
                    if (want_pos) {
#pragma unroll
                        for (int e = 0; e < MASS_C; e++) {
                            const int tp = __float_as_int(c[2 * MASS_Q + e]);
                            float y = fmaf(c[MASS_Q + e], (float)(tp - pj), __uint_as_float(v[e]));
                            if (a.window > 0 && !(pj >= (int64_t)tp - a.window || pj < a.sink)) y = -INFINITY;
                            v[e] = __float_as_uint(y);
                        }
                    }
                }
                if (j0 + TILE_K > n - a.T || r0 + MASS_C > R) {   /* some query rows of these see the cache row, not all */
                    const int own = j - (n - a.T);
                    uint32_t bits = R - r0 >= 32 ? ~0u : R > r0 ? (1u << (R - r0)) - 1u : 0u;
                    if (j >= n) bits = 0u;
                    if (own > 0 && !a.tree) {
                        const int skip = own * a.G - r0;      /* tokens before `own` do not see it */
                        bits &= skip >= 32 ? 0u : skip > 0 ? ~0u << skip : ~0u;
                    }
                    if (own >= 0 && a.tree && j < n) {
                        int t = r0 / a.G, g = r0 - t * a.G;
                        bool see = false;
#pragma unroll 1
                        for (int e = 0; e < MASS_C && r0 + e < R; e++) {
                            if (e == 0 || g == 0)
                                see = a.tree[l * a.tree_stride + (int64_t)t * a.tree_words + (own >> 5)] >> (own & 31) & 1u;
                            if (!see) bits &= ~(1u << e);
                            if (++g == a.G) { g = 0; t++; }
                        }
                    }
                    if (!EXTRA) {                             /* a masked score stays masked only once it is final */
#pragma unroll
                        for (int e = 0; e < MASS_C; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * map.scale);
                        mul = pair(1.0f, 1.0f);
                    }
#pragma unroll
                    for (int e = 0; e < MASS_C; e++)
                        if (!(bits >> e & 1u)) v[e] = 0xff800000u;
                }
                uint64_t part[2] = {0ull, 0ull};
#pragma unroll
                for (int e = 0; e < MASS_C / 4; e++) {
                    const float4 nc = reinterpret_cast<const float4 *>(c)[e];
                    const float2 x = unpair(fma2(pair(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1])), mul, pair(nc.x, nc.y)));
                    const float2 y = unpair(fma2(pair(__uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3])), mul, pair(nc.z, nc.w)));
                    part[0] = add2(part[0], pair(ex2(x.x), ex2(x.y)));
                    part[1] = add2(part[1], pair(ex2(y.x), ex2(y.y)));
                }
                sum = add2(sum, add2(part[0], part[1]));
            }
            done += tiles;
        }
        const float2 s2 = unpair(sum);
        if (half) s_sum[row] = s2.x + s2.y;
        tc_fence_before();
        __syncthreads();
        if (!half && j < n) {
            float mass = s2.x + s2.y + s_sum[row];
            /* a key that f16 operands do not hold (TILE_SCALE): its weights from the definition */
            if (KT == KT_Q8_0 && mass != mass) mass = row_mass<KT, HD>(a, u, j, n, pj);
            const int64_t x = (int64_t)u * a.n_cells + j;
            a.mass_out[x] = a.mass_in ? fmaf(a.mass_decay, a.mass_in[x], mass) : mass;
        }
        ok = !__syncthreads_or(!ok);
    }
    tc_fence_before();
    __syncthreads();
    if (w == 0) {
        tc_fence_after();
        if (s_abort) {                                        /* a product may still run: wait for it, within a bound */
            tc_commit(lane == 0, &b_drain);
            mbar_wait(&b_drain, 0);
            __syncwarp();
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem) : "memory");
    }
}

/* Query rows whose result was not finite, one block each (see attend_row). */
template <int KT, int HD>
__global__ void __launch_bounds__(ROW_THREADS) k_attend_redo(const AttendArgs a) {
    __shared__ RowShared<HD> sm;
    const int R = a.T * a.G, all = a.n_layer * a.n_head_kv * R;
    int many = a.redo[0];
    if (!bounds_ok(many >= 0 && many <= all, threadIdx.x == 0 ? a.status : nullptr)) many = 0;
    int last = -1;
    bool bad = false;
    for (int i = blockIdx.x; i < many; i += gridDim.x) {
        const int q = a.redo[1 + i], u = q / R, r = q - u * R;
        if (!bounds_ok(q >= 0 && q < all, threadIdx.x == 0 ? a.status : nullptr)) continue;
        if (u != last) bad = result_in_doubt<KT, HD, true>(a, u);
        last = u;
        if (bad) attend_row<KT, HD>(a, u, r % a.G, r / a.G, sm);
    }
}

}  // namespace tria
