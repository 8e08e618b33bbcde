/*
 * tria_attend.cuh - attention over a ragged cache.
 *
 * For the query of token t and head h (kv head h / gqa) over the rows j that t
 * sees:
 *     s_j = scale q.k_j,  capped: c tanh(s_j / c),  biased: - slope_h (tok_pos_t - pos_j)
 *     p_j = exp(s_j - m) / sum_j exp(s_j - m),      out = sum_j p_j v_j
 * and the mass of row j gains the sum of p_j over the tokens and the heads of
 * its group.
 */
#pragma once

#include "tria_common.cuh"

namespace tria {

struct AttendArgs {
    const uint8_t *k[TRIA_MAX_LAYERS];
    const uint8_t *v[TRIA_MAX_LAYERS];
    int64_t cell_stride, head_stride;
    const int32_t *pos;
    int32_t pos_shared, n_cells;
    int32_t n_layer, n_head_kv, G, T;
    const int32_t *n_rows;
    const __half *q;
    __half *out;
    int64_t q_cache, q_tok, q_head, o_cache, o_tok, o_head;     /* elements */
    float *lse;                          /* [n_layer][T][n_head_kv * G], or NULL */
    const float *mass_in;
    float *mass_out;
    float mass_decay, scale, softcap;
    int32_t window, sink;
    const float *slopes;
    const int32_t *tok_pos;
    int64_t tok_pos_stride;
    const uint32_t *tree;
    int64_t tree_stride;
    int32_t tree_words;
    int32_t *status;
    /* plan and workspace (host-filled) */
    int32_t copy16;                      /* rows start on 16-byte boundaries (f16), 8-byte ones (q8_0) */
    int32_t groups;                      /* groups of query rows per unit */
    const int32_t *steps;                /* inclusive prefix of the items' steps, or NULL: scanned in the kernel */
    const int2 *span;                    /* windowed: (head, tail) of each item, else NULL */
    float *part_o;                       /* [2 * grid][rows][head_dim] */
    float2 *part_ml;                     /* [2 * grid][rows] */
    int32_t *arrived;                    /* [grid]: by the first block of an item (one such item a block); zero between calls */
    float2 *norm;                        /* [n_layer * n_head_kv][T * G]: (max, 1 / sum) of each query row, or NULL */
    float *scores;                       /* [n_layer * n_head_kv][T * G][score_stride], or NULL */
    int64_t score_stride;
};

/* Rows of unit u: a count outside the cache is clamped and reported. */
__device__ __forceinline__ int attend_rows(const AttendArgs &a, int u) {
    const int n = a.n_rows[u];
    if (n >= 0 && n <= a.n_cells) return n;
    atomicOr(a.status, ST_ROWS);
    return n < 0 ? 0 : a.n_cells;
}

/* Whether token t of cache l sees row j of a unit with n rows; pos: the row's
 * position, lo: tok_pos[t] - window (both read only with a window). */
__device__ __forceinline__ bool attend_sees(const AttendArgs &a, int l, int t, int j, int n, int pos, int64_t lo) {
    if (j >= n) return false;
    const int own = j - (n - a.T);
    if (own >= 0) {
        if (a.tree) {
            if (!(a.tree[l * a.tree_stride + (int64_t)t * a.tree_words + (own >> 5)] >> (own & 31) & 1u)) return false;
        } else if (own > t) {
            return false;
        }
    }
    return a.window <= 0 || pos >= lo || pos < a.sink;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

/* tanh(u).  1 - 2 / (1 + exp 2u) is right to an fp32 ulp of 1, which is what
 * large arguments need and too little where tanh u is small; there the series
 * u (1 - z/3 + 2 z^2/15 - ...), z = u^2, whose first omitted term is below
 * 2^-27 at |u| = 0.4. */
__device__ __forceinline__ float tanh_both(float u) {
    const float z = u * u;
    float s = 21844.0f / 6081075.0f;
    s = fmaf(s, z, -1382.0f / 155925.0f);
    s = fmaf(s, z, 62.0f / 2835.0f);
    s = fmaf(s, z, -17.0f / 315.0f);
    s = fmaf(s, z, 2.0f / 15.0f);
    s = fmaf(s, z, -1.0f / 3.0f);
    s = fmaf(s * z, u, u);
    const float b = fmaf(-2.0f, rcp(1.0f + ex2(2.0f * LOG2E * u)), 1.0f);
    return fabsf(u) < 0.4f ? s : b;
}

/* The call's score transform in the base-2 exponent: x = log2(e) s. */
struct ScoreMap {
    float scale;        /* of the product: log2(e) scale, or scale / softcap */
    float cap;          /* log2(e) softcap, 0: none */
    __device__ __forceinline__ explicit ScoreMap(const AttendArgs &a)
        : scale(a.softcap > 0.0f ? a.scale / a.softcap : a.scale * LOG2E), cap(a.softcap * LOG2E) {}
    __device__ __forceinline__ float operator()(float dot) const {
        const float x = dot * scale;
        return cap > 0.0f ? cap * tanh_both(x) : x;
    }
};

/* Element d of the cache row at p. */
template <int KT>
__device__ __forceinline__ float row_value(const uint8_t *p, int d) {
    if constexpr (KT == KT_F16) {
        return __half2float(reinterpret_cast<const __half *>(p)[d]);
    } else {
        const uint8_t *b = p + (d >> 5) * 34;
        return __half2float(*reinterpret_cast<const __half *>(b)) * (float)reinterpret_cast<const int8_t *>(b)[2 + (d & 31)];
    }
}

/* The base-2 score of a query against a cache row, in fp32 throughout;
 * slope2: log2(e) times the head's slope. */
template <int KT, int HD>
__device__ __forceinline__ float attend_score(const ScoreMap &f, const uint8_t *krow, const float *q, float slope2,
                                              int tok_pos, int pos) {
    float s = 0.0f;
    for (int d = 0; d < HD; d++) s = fmaf(q[d], row_value<KT>(krow, d), s);
    return fmaf(-slope2, (float)(tok_pos - pos), f(s));
}

constexpr int ROW_THREADS = 128;

template <int HD>
struct RowShared {
    float q[HD];
    float p[ROW_THREADS];
    float red[ROW_THREADS / 32];
};

__device__ __forceinline__ float block_max_128(float v, float *red) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    return v;
}

/* One query row by one block of ROW_THREADS threads, straight from the
 * definition: a thread scores a row of the cache, then owns an output element.
 * It is the way out of the tiled kernels for a query row whose result is not
 * finite (a product with another token's infinity or NaN, or its own).  Rows that
 * the token does not see are never multiplied, so what they hold is without
 * effect. */
template <int KT, int HD>
__device__ void attend_row(const AttendArgs &a, int u, int g, int t, RowShared<HD> &sm) {
    const int l = u / a.n_head_kv, h = u - l * a.n_head_kv, tid = threadIdx.x;
    const int n = attend_rows(a, u), head = h * a.G + g;
    const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
    const int tp = a.tok_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
    const int64_t lo = (int64_t)tp - a.window;
    const float slope2 = a.slopes ? a.slopes[head] * LOG2E : 0.0f;
    const ScoreMap map(a);
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride, *v = a.v[l] + (int64_t)h * a.head_stride;
    const __half *q = a.q + l * a.q_cache + t * a.q_tok + head * a.q_head;
    __syncthreads();
    for (int d = tid; d < HD; d += ROW_THREADS) sm.q[d] = __half2float(q[d]);
    __syncthreads();
    float m = -INFINITY, sum = 0.0f, acc = 0.0f;
    bool any = false;
    for (int j0 = 0; j0 < n; j0 += ROW_THREADS) {
        const int j = j0 + tid;
        const int pj = j < n ? pos[j] : 0;
        const bool see = attend_sees(a, l, t, j, n, pj, lo);
        float s = -INFINITY;
        if (see) s = attend_score<KT, HD>(map, k + (int64_t)j * a.cell_stride, sm.q, slope2, tp, pj);
        if (!__syncthreads_or(see)) continue;
        any = true;
        const float mt = fmaxf(m, block_max_128(s, sm.red));
        const float r = mt == m ? 1.0f : ex2(m - mt);
        sm.p[tid] = see ? ex2(s - (mt == -INFINITY ? 0.0f : mt)) : 0.0f;
        const unsigned bits = __ballot_sync(0xffffffffu, see);
        if ((tid & 31) == 0) reinterpret_cast<unsigned *>(sm.red)[tid >> 5] = bits;
        __syncthreads();
        sum *= r;
        acc *= r;
        m = mt;
        for (int i = 0; i < ROW_THREADS; i++) {
            if (!(reinterpret_cast<const unsigned *>(sm.red)[i >> 5] >> (i & 31) & 1u)) continue;
            sum += sm.p[i];
            if (tid < HD) acc = fmaf(sm.p[i], row_value<KT>(v + (int64_t)(j0 + i) * a.cell_stride, tid), acc);
        }
        __syncthreads();
    }
    if (tid < HD)
        a.out[l * a.o_cache + t * a.o_tok + head * a.o_head + tid] = __float2half_rn(any && sum != 0.0f ? acc / sum : 0.0f);
    if (a.lse && tid == 0)
        a.lse[((int64_t)l * a.T + t) * a.n_head_kv * a.G + head] = any && sum != 0.0f ? (m + log2f(sum)) * LN2 : -INFINITY;
}


/* ------------------------------------------------------------------ */
/* Plan: which rows of the cache each group of query rows walks         */
/* ------------------------------------------------------------------ */

/* Query rows r = t * G + g of a unit are taken in groups of `rows`; an item is
 * (unit, group).  An item walks steps of ATT_STEP cache rows: all rows up to
 * the last that its tokens see by order, or, with a window, the rows before
 * `head` (where the sink ends) and those from `tail` on (where the window
 * begins).  Positions need not ascend: head and tail enclose every row that
 * the window admits. */
constexpr int ATT_STEP = 64;

/* Rows of the unit that the group's last token can see by order. */
__device__ __forceinline__ int item_rows(const AttendArgs &a, int u, int grp, int rows) {
    const int n = attend_rows(a, u);
    const int r1 = min(a.T * a.G, (grp + 1) * rows) - 1;
    return max(0, a.tree ? n : min(n, n - a.T + r1 / a.G + 1));
}

__device__ __forceinline__ int span_steps(int n, int2 s) {
    const int hs = (s.x + ATT_STEP - 1) / ATT_STEP;
    return hs + (n > s.y ? (n - s.y + ATT_STEP - 1) / ATT_STEP : 0);
}

constexpr int PLAN_THREADS = 512;

/* Inclusive scan over a block of PLAN_THREADS; total in *sum. */
__device__ __forceinline__ int block_scan(int v, int *s_warp, int threads, int *sum) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, m);
        if (lane >= m) v += x;
    }
    __syncthreads();
    if (lane == 31) s_warp[w] = v;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < threads / 32; i++) {
        if (i < w) before += s_warp[i];
        all += s_warp[i];
    }
    *sum = all;
    return v + before;
}

/* With a window: block `it` finds its item's span.  The last block to finish
 * (the only one without a window) scans the items' steps. */
__global__ void __launch_bounds__(PLAN_THREADS) k_attend_plan(const AttendArgs a, int rows, int items, int2 *span,
                                                              int32_t *steps, int32_t *done) {
    __shared__ int s_min[PLAN_THREADS / 32], s_max[PLAN_THREADS / 32], s_last;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (span) {
        const int it = blockIdx.x, u = it / a.groups, grp = it - u * a.groups, l = u / a.n_head_kv;
        const int n = item_rows(a, u, grp, rows);
        const int t0 = grp * rows / a.G, t1 = (min(a.T * a.G, (grp + 1) * rows) - 1) / a.G;
        int first = INT_MAX;                                  /* the group's earliest position */
        for (int t = t0 + threadIdx.x; t <= t1; t += PLAN_THREADS) first = min(first, a.tok_pos[l * a.tok_pos_stride + t]);
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) s_min[w] = first;
        __syncthreads();
        for (int i = 0; i < PLAN_THREADS / 32; i++) first = min(first, s_min[i]);
        __syncthreads();
        const int64_t lo = (int64_t)first - a.window;
        const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
        int tail = n, head = 0;
        for (int j = threadIdx.x; j < n; j += PLAN_THREADS) {
            const int p = pos[j];
            if (p >= lo) tail = min(tail, j);
            if (p < a.sink) head = j + 1;
        }
        tail = __reduce_min_sync(0xffffffffu, tail);
        head = __reduce_max_sync(0xffffffffu, head);
        if (lane == 0) { s_min[w] = tail; s_max[w] = head; }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < PLAN_THREADS / 32; i++) { tail = min(tail, s_min[i]); head = max(head, s_max[i]); }
            tail = tail / ATT_STEP * ATT_STEP;
            if (head >= tail) { head = 0; tail = 0; }         /* one run of rows */
            span[it] = make_int2(head, tail);
            __threadfence();
            s_last = atomicAdd(done, 1) == (int)gridDim.x - 1;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (threadIdx.x == 0) *done = 0;
    }
    int base = 0;
    for (int i0 = 0; i0 < items; i0 += PLAN_THREADS) {
        const int it = i0 + threadIdx.x;
        int st = 0, sum;
        if (it < items) {
            const int u = it / a.groups, grp = it - u * a.groups, n = item_rows(a, u, grp, rows);
            const int2 s = span ? __ldcg(&span[it]) : make_int2(0, 0);
            st = span_steps(n, make_int2(min(s.x, n), s.y));
        }
        const int incl = block_scan(st, s_min, PLAN_THREADS, &sum);
        if (it < items) steps[it] = base + incl;
        base += sum;
    }
}

/* ------------------------------------------------------------------ */
/* Few query rows: warps on mma tiles, rows streamed once               */
/* ------------------------------------------------------------------ */

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
/* d += a b, 16 x 8 x 16, f16 operands, fp32 sums. */
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float lds_half(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
/* The int8 pairs (byte 0, byte 1) and (byte 2, byte 3) of w as f16 pairs,
 * exactly: with the sign bit flipped a byte is x + 128, the f16 0x6400 | (x + 128)
 * is 1024 + 128 + x, and 1152 comes off again. */
__device__ __forceinline__ void int8x4_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t u = w ^ 0x80808080u, bias = 0x64806480u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = *reinterpret_cast<const __half2 *>(&bias);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    lo = *reinterpret_cast<const uint32_t *>(&x);
    hi = *reinterpret_cast<const uint32_t *>(&y);
}

constexpr int FEW_WARPS = 4, FEW_THREADS = FEW_WARPS * 32;
constexpr int FEW_SLICE = ATT_STEP / FEW_WARPS;      /* cache rows a warp takes per step */
static_assert(FEW_SLICE == 16 && FEW_THREADS == ROW_THREADS, "warp tile");

/* Shared memory of a warp's stage: 16 K rows, 16 V rows, 16 positions.  f16
 * rows lie in 16-byte chunks XORed with the row (ldmatrix reads 8 rows of one
 * chunk without bank conflicts); q8_0 rows are padded so that the reads of a
 * block's bytes by 8 rows x 4 lanes (K, 8 bytes a lane) and 4 rows x 8 lanes
 * (V, 4 bytes a lane) fall in distinct banks. */
template <int KT, int HD>
struct FewStage {
    static constexpr int KS = KT == KT_F16 ? 2 * HD : (HD == 128 ? 160 : 96);
    static constexpr int VS = KT == KT_F16 ? 2 * HD : (HD == 128 ? 144 : 80);
    static constexpr int K = 0, V = 16 * KS, P = V + 16 * VS, BYTES = P + 64;
};

/* Stages a warp keeps in flight: as many as two blocks an SM leave room for. */
template <int KT, int HD>
__host__ __device__ constexpr int few_stages() { return KT == KT_F16 ? (HD == 128 ? 3 : 6) : (HD == 128 ? 5 : 8); }
template <int KT, int HD, int MT>
__host__ __device__ constexpr int few_smem() {
    const int ring = FEW_WARPS * few_stages<KT, HD>() * FewStage<KT, HD>::BYTES;
    const int merge = FEW_WARPS * 16 * MT * (HD + 8) * 4 + FEW_WARPS * 16 * MT * 8;
    return ring > merge ? ring : merge;
}

/* Scores are kept in units where a weight is 2^(x - m + FEW_LIFT): weights of
 * rows far below the maximum stay normal f16 numbers (2^-14 and up) down to
 * 2^-20 of it, and the maximum may fall FEW_SLACK behind before the sums are
 * rescaled: 2^(FEW_LIFT + FEW_SLACK) is still finite in f16. */
constexpr float FEW_LIFT = 6.0f, FEW_SLACK = 8.0f;

/* Copies the warp's slice: rows [r0, r0 + 16) below n; rows at and behind n
 * become zeros. */
template <int KT, int HD>
__device__ __forceinline__ void few_load(const AttendArgs &a, const uint8_t *k, const uint8_t *v, const int32_t *pos,
                                         bool want_pos, int r0, int n, uint32_t st, int lane) {
    using S = FewStage<KT, HD>;
    if constexpr (KT == KT_F16) {
        constexpr int CH = HD / 8, PER = 16 * CH / 32;
        if (a.copy16) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int x = lane + 32 * i, r = x / CH, c = x % CH;
                const bool in = r0 + r < n;
                const int64_t off = in ? (int64_t)(r0 + r) * a.cell_stride + 16 * c : 0;
                const uint32_t d = st + r * S::KS + 16 * (c ^ (r & 7));
                cp_async16(d + S::K, k + off, in ? 16u : 0u);
                cp_async16(d + S::V, v + off, in ? 16u : 0u);
            }
        } else {
            for (int x = lane; x < 16 * CH * 4; x += 32) {
                const int r = x / (CH * 4), c = x / 4 % CH, q = x & 3;
                const bool in = r0 + r < n;
                const int64_t off = in ? (int64_t)(r0 + r) * a.cell_stride + 16 * c + 4 * q : 0;
                const uint32_t d = st + r * S::KS + 16 * (c ^ (r & 7)) + 4 * q;
                cp_async4(d + S::K, k + off, in ? 4u : 0u);
                cp_async4(d + S::V, v + off, in ? 4u : 0u);
            }
        }
    } else {
        constexpr int RB = HD / 32 * 34;
        if (a.copy16 && RB % 8 == 0) {
            constexpr int CH = RB / 8;
            for (int x = lane; x < 16 * CH; x += 32) {
                const int r = x / CH, c = x - r * CH;
                const bool in = r0 + r < n;
                const int64_t off = in ? (int64_t)(r0 + r) * a.cell_stride + 8 * c : 0;
                cp_async8(st + S::K + r * S::KS + 8 * c, k + off, in ? 8u : 0u);
                cp_async8(st + S::V + r * S::VS + 8 * c, v + off, in ? 8u : 0u);
            }
        } else {
            constexpr int CH = RB / 4;
            for (int x = lane; x < 16 * CH; x += 32) {
                const int r = x / CH, c = x - r * CH;
                const bool in = r0 + r < n;
                const int64_t off = in ? (int64_t)(r0 + r) * a.cell_stride + 4 * c : 0;
                cp_async4(st + S::K + r * S::KS + 4 * c, k + off, in ? 4u : 0u);
                cp_async4(st + S::V + r * S::VS + 4 * c, v + off, in ? 4u : 0u);
            }
        }
    }
    if (want_pos && lane < 16) {
        const bool in = r0 + lane < n;
        cp_async4(st + S::P + 4 * lane, pos + (in ? r0 + lane : 0), in ? 4u : 0u);
    }
}

/* The dims of a row that k-step s takes, for lane column c: f16 16 s + 2 c,
 * +1 and those 8 on; q8_0 the bytes 8 c + 4 (s & 1) .. +3 of block s / 2, so that
 * a lane's share of a block is 8 bytes in a row. */
template <int KT>
__device__ __forceinline__ int few_qdim(int s, int c, int hi) {
    return KT == KT_F16 ? 16 * s + 2 * c + 8 * hi : 32 * (s >> 1) + 8 * c + 4 * (s & 1) + 2 * hi;
}
/* The dim of accumulator tile j, column n: q8_0 tiles stay within a block and
 * give lane row n the bytes 4 n .. 4 n + 3 of it over its four tiles. */
template <int KT>
__device__ __forceinline__ int few_odim(int j, int n) {
    return KT == KT_F16 ? 8 * j + n : 32 * (j >> 2) + 4 * n + (j & 3);
}

/* The products of the slice's 16 keys with MT x 16 query rows: s[m][t][.] in
 * the accumulator layout, tile t keys 8 t .. 8 t + 7. */
template <int KT, int HD, int MT>
__device__ __forceinline__ void few_qk(const uint32_t (&qf)[MT][HD / 16][4], uint32_t st, int lane, float (&s)[MT][2][4]) {
    using S = FewStage<KT, HD>;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[m][t][i] = 0.0f;
    if constexpr (KT == KT_F16) {
        const int row = (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
#pragma unroll
        for (int x = 0; x < HD / 16; x++) {
            uint32_t b[4];
            ldsm4(b, st + S::K + row * S::KS + 16 * ((2 * x + hi) ^ (row & 7)));
#pragma unroll
            for (int m = 0; m < MT; m++) {
                mma16816(s[m][0], qf[m][x], b[0], b[1]);
                mma16816(s[m][1], qf[m][x], b[2], b[3]);
            }
        }
    } else {
        const int r = lane >> 2, c = lane & 3;
#pragma unroll
        for (int blk = 0; blk < HD / 32; blk++) {
            constexpr int KS = S::KS;
            const int sh = (2 * blk + 2) & 7;                        /* bytes into the aligned 8-byte word */
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t at = st + S::K + (8 * t + r) * KS + 34 * blk + 2 + 8 * c - sh;
                const uint2 x = lds64(at);
                uint32_t w0, w1;
                if (sh == 0) {
                    w0 = x.x;
                    w1 = x.y;
                } else {
                    const uint2 y = lds64(at + 8);
                    w0 = sh == 2 ? __funnelshift_r(x.x, x.y, 16) : sh == 4 ? x.y : __funnelshift_r(x.y, y.x, 16);
                    w1 = sh == 2 ? __funnelshift_r(x.y, y.x, 16) : sh == 4 ? y.x : __funnelshift_r(y.x, y.y, 16);
                }
                uint32_t b0, b1, b2, b3;
                int8x4_half(w0, b0, b1);
                int8x4_half(w1, b2, b3);
                /* the block's scale belongs to the key, so it multiplies the block's sum: the f16 operands
                 * stay the stored integers and the scores keep fp32 */
                const float d0 = lds_half(st + S::K + (8 * t + 2 * c) * KS + 34 * blk);
                const float d1 = lds_half(st + S::K + (8 * t + 2 * c + 1) * KS + 34 * blk);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma16816(p, qf[m][2 * blk], b0, b1);
                    mma16816(p, qf[m][2 * blk + 1], b2, b3);
                    s[m][t][0] = fmaf(p[0], d0, s[m][t][0]);
                    s[m][t][1] = fmaf(p[1], d1, s[m][t][1]);
                    s[m][t][2] = fmaf(p[2], d0, s[m][t][2]);
                    s[m][t][3] = fmaf(p[3], d1, s[m][t][3]);
                }
            }
        }
    }
}

/* o += p v over the slice's 16 rows; keep0, keep1: 0xffff for each f16 of a V
 * pair whose row some query row sees (a row that none sees may hold NaN). */
template <int KT, int HD, int MT>
__device__ __forceinline__ void few_pv(const float (&p)[MT][2][4], uint32_t st, int lane, uint32_t keep0, uint32_t keep1,
                                       float (&o)[MT][HD / 8][4]) {
    using S = FewStage<KT, HD>;
    if constexpr (KT == KT_F16) {
        uint32_t pf[MT][4];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            pf[m][0] = pack_half2(p[m][0][0], p[m][0][1]);
            pf[m][1] = pack_half2(p[m][0][2], p[m][0][3]);
            pf[m][2] = pack_half2(p[m][1][0], p[m][1][1]);
            pf[m][3] = pack_half2(p[m][1][2], p[m][1][3]);
        }
        const int row = lane & 15, hi = lane >> 4;
#pragma unroll
        for (int j = 0; j < HD / 8; j += 2) {
            uint32_t b[4];
            ldsm4t(b, st + S::V + row * S::VS + 16 * ((j + hi) ^ (row & 7)));
            b[0] &= keep0;
            b[1] &= keep1;
            b[2] &= keep0;
            b[3] &= keep1;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                mma16816(o[m][j], pf[m], b[0], b[1]);
                mma16816(o[m][j + 1], pf[m], b[2], b[3]);
            }
        }
    } else {
        const int r = lane >> 2, c = lane & 3;
        constexpr int VS = S::VS;
        const uint32_t v0 = st + S::V + 2 * c * VS;                  /* rows 2c, 2c+1, 2c+8, 2c+9 */
#pragma unroll
        for (int blk = 0; blk < HD / 32; blk++) {
            const int sh = (2 * blk + 2) & 3;
            uint32_t w[4];
            float d[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t at = v0 + ((i & 1) + (i >> 1) * 8) * VS + 34 * blk;
                d[i] = lds_half(at);
                if (sh == 0) w[i] = lds32(at + 2 + 4 * r);
                else w[i] = __funnelshift_r(lds32(at + 4 * r), lds32(at + 4 + 4 * r), 16);
                /* a row that no query row sees: its scale may be anything */
                if (!((i >> 1 ? keep1 : keep0) >> (16 * (i & 1)) & 1u)) d[i] = 0.0f;
            }
            /* the scales go into the weights before their one rounding to f16; the V operands are the stored integers */
            uint32_t pf[MT][4];
#pragma unroll
            for (int m = 0; m < MT; m++) {
                pf[m][0] = pack_half2(p[m][0][0] * d[0], p[m][0][1] * d[1]);
                pf[m][1] = pack_half2(p[m][0][2] * d[0], p[m][0][3] * d[1]);
                pf[m][2] = pack_half2(p[m][1][0] * d[2], p[m][1][1] * d[3]);
                pf[m][3] = pack_half2(p[m][1][2] * d[2], p[m][1][3] * d[3]);
            }
            const uint32_t a01 = __byte_perm(w[0], w[1], 0x5140), a23 = __byte_perm(w[0], w[1], 0x7362);
            const uint32_t b01 = __byte_perm(w[2], w[3], 0x5140), b23 = __byte_perm(w[2], w[3], 0x7362);
            uint32_t x[4], y[4];
            int8x4_half(a01, x[0], x[1]);
            int8x4_half(a23, x[2], x[3]);
            int8x4_half(b01, y[0], y[1]);
            int8x4_half(b23, y[2], y[3]);
#pragma unroll
            for (int jj = 0; jj < 4; jj++)
#pragma unroll
                for (int m = 0; m < MT; m++) mma16816(o[m][4 * blk + jj], pf[m], x[jj], y[jj]);
        }
    }
}

/* Merges S partial results of query row r into val (thread d's dim) and (m, l). */
template <class Ml, class O>
__device__ __forceinline__ float merge_row(int S, Ml &&ml, O &&o, float &m, float &l) {
    m = -INFINITY;
    for (int s = 0; s < S; s++) m = fmaxf(m, ml(s).x);
    const float ms = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
    float v = 0.0f;
    for (int s = 0; s < S; s++) {
        const float2 x = ml(s);
        const float f = x.x == -INFINITY ? 0.0f : ex2(x.x - ms);
        l = fmaf(x.y, f, l);
        v = f == 0.0f ? v : fmaf(o(s), f, v);
    }
    return v;
}

/* Attention of the items' query rows (up to 16 * MT) over their steps.  The
 * steps of all items are shared out evenly: block b takes steps
 * [b * total / grid, (b + 1) * total / grid) (grid: at most `total`), whatever units they fall in, so
 * ragged counts read from the device keep every SM busy without the host
 * knowing them.  Within a step each warp takes 16 cache rows of its own and
 * keeps its own running maximum, sum and value sums: the loop has no block
 * barrier, and a warp's copies run `stages` slices ahead.  An item that ends
 * in several blocks leaves partial results; the block that arrives last
 * merges them in block order, so the result does not depend on timing.
 *
 * Bound by the cache's bytes up to a few tens of query rows: 16 rows cost 32
 * mma (f16, head_dim 128) for 8 KB. */
template <int KT, int HD, int MT>
__global__ void __launch_bounds__(FEW_THREADS, 2) k_attend_few(const AttendArgs a) {
    using S = FewStage<KT, HD>;
    constexpr int ROWS = 16 * MT, ST = few_stages<KT, HD>(), OS = HD + 8;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_steps[512];
    __shared__ int s_warp[FEW_WARPS];
    __shared__ int s_flag;
    __shared__ RowShared<HD> s_row;
    __shared__ int s_redo[ROWS];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, r8 = lane >> 2, c = lane & 3;
    const int units = a.n_layer * a.n_head_kv, items = units * a.groups, R = a.T * a.G;
    const int *steps = a.steps;
    if (!steps) {                                             /* few items, no window */
        int base = 0;
        for (int i0 = 0; i0 < items; i0 += FEW_THREADS) {
            const int it = i0 + tid;
            int st = 0, sum;
            if (it < items) st = (item_rows(a, it / a.groups, it % a.groups, ROWS) + ATT_STEP - 1) / ATT_STEP;
            const int incl = block_scan(st, s_warp, FEW_THREADS, &sum);
            if (it < items) s_steps[it] = base + incl;
            base += sum;
        }
        __syncthreads();
        steps = s_steps;
    }
    const int64_t total = steps[items - 1];
    const int b = blockIdx.x, grid = (int)min((int64_t)gridDim.x, total);     /* no block between an item's first and last is idle */
    const ScoreMap map(a);
    const bool want_pos = a.window > 0 || a.slopes != nullptr;
    const uint32_t ring = smem_u32(smem) + w * ST * S::BYTES;

    /* items without a row to see */
    for (int it = b; it < items; it += gridDim.x) {
        if (steps[it] != (it ? steps[it - 1] : 0)) continue;
        const int u = it / a.groups, grp = it - u * a.groups, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
        for (int x = tid; x < ROWS * HD / 8; x += FEW_THREADS) {
            const int r = grp * ROWS + x / (HD / 8);
            if (r >= R) break;
            *reinterpret_cast<uint4 *>(a.out + l * a.o_cache + (r / a.G) * a.o_tok + (h * a.G + r % a.G) * a.o_head +
                                       x % (HD / 8) * 8) = make_uint4(0, 0, 0, 0);
        }
        for (int x = tid; x < ROWS && grp * ROWS + x < R; x += FEW_THREADS) {
            const int r = grp * ROWS + x;
            if (a.lse) a.lse[((int64_t)l * a.T + r / a.G) * a.n_head_kv * a.G + h * a.G + r % a.G] = -INFINITY;
            if (a.norm) a.norm[(int64_t)u * R + r] = make_float2(0.0f, 0.0f);
        }
    }

    if (b >= grid) return;
    int64_t at = b * total / grid;
    const int64_t end = (b + 1) * total / grid;
    if (at >= end) return;
    int it = 0;                                               /* the item of step `at` */
    for (int lo = 0, hi = items; lo < hi;) {
        const int mid = (lo + hi) >> 1;
        if (steps[mid] <= at) lo = mid + 1;
        else hi = mid;
        it = lo;
    }
    for (bool first = true; at < end; first = false) {
        while (steps[it] <= at) it++;
        const int64_t base = it ? steps[it - 1] : 0;
        const int i0 = (int)(at - base), i1 = (int)(min(end, (int64_t)steps[it]) - base);
        const int u = it / a.groups, grp = it - u * a.groups, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
        const int n = attend_rows(a, u);
        const int2 span = a.span ? a.span[it] : make_int2(0, 0);
        const int head_steps = (min(span.x, n) + ATT_STEP - 1) / ATT_STEP;
        auto slice_row = [&](int i) { return (i < head_steps ? i * ATT_STEP : span.y + (i - head_steps) * ATT_STEP) + FEW_SLICE * w; };
        const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride, *v = a.v[l] + (int64_t)h * a.head_stride;
        const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);

        /* prologue: copies first, then the queries while they fly */
#pragma unroll
        for (int p = 0; p < ST - 1; p++) {
            if (i0 + p < i1) few_load<KT, HD>(a, k, v, pos, want_pos, slice_row(i0 + p), n, ring + p * S::BYTES, lane);
            cp_async_commit();
        }
        uint32_t qf[MT][HD / 16][4];
        int tok[MT][2], tp[MT][2];
        float slope2[MT][2];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
                const int r = grp * ROWS + 16 * m + r8 + 8 * hi, t = r / a.G, head = h * a.G + r % a.G;
                const bool in = r < R;
                tok[m][hi] = in ? t : -1;
                tp[m][hi] = in && want_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
                slope2[m][hi] = in && a.slopes ? a.slopes[head] * LOG2E : 0.0f;
                const __half *q = a.q + l * a.q_cache + (in ? t * a.q_tok + head * a.q_head : 0);
#pragma unroll
                for (int s = 0; s < HD / 16; s++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        qf[m][s][hi + 2 * e] = in ? *reinterpret_cast<const uint32_t *>(q + few_qdim<KT>(s, c, e)) : 0u;
            }
        float o[MT][HD / 8][4], mx[MT][2], sum[MT][2];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            mx[m][0] = mx[m][1] = -INFINITY;
            sum[m][0] = sum[m][1] = 0.0f;
#pragma unroll
            for (int j = 0; j < HD / 8; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[m][j][i] = 0.0f;
        }

        for (int i = i0; i < i1; i++) {
            const int nx = i + ST - 1;
            cp_async_wait<ST - 2>();
            __syncwarp();
            if (nx < i1) few_load<KT, HD>(a, k, v, pos, want_pos, slice_row(nx), n, ring + ((nx - i0) % ST) * S::BYTES, lane);
            cp_async_commit();
            const uint32_t st = ring + ((i - i0) % ST) * S::BYTES;
            const int row0 = slice_row(i);
            if (row0 >= n) continue;
            float s[MT][2][4];
            few_qk<KT, HD, MT>(qf, st, lane, s);
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
            const bool all = row0 + FEW_SLICE <= n - a.T && a.window <= 0;       /* every row is seen by every token */
            uint32_t seen = 0;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int hi = e >> 1, key = 8 * t + 2 * c + (e & 1);
                        float x = map(s[m][t][e]);
                        int pk = 0;
                        if (want_pos) {
                            pk = (int)lds32(st + S::P + 4 * key);
                            x = fmaf(-slope2[m][hi], (float)(tp[m][hi] - pk), x);
                        }
                        if (!all) {
                            const bool see = tok[m][hi] >= 0 &&
                                             attend_sees(a, l, tok[m][hi], row0 + key, n, pk, (int64_t)tp[m][hi] - a.window);
                            x = see ? x : -INFINITY;
                            seen |= see ? 1u << (2 * t + (e & 1)) : 0u;
                        }
                        s[m][t][e] = x;
                    }
            if (!all) {
                seen |= __shfl_xor_sync(0xffffffffu, seen, 4);
                seen |= __shfl_xor_sync(0xffffffffu, seen, 8);
                seen |= __shfl_xor_sync(0xffffffffu, seen, 16);
                keep0 = (seen & 1u ? 0xffffu : 0u) | (seen & 2u ? 0xffff0000u : 0u);
                keep1 = (seen & 4u ? 0xffffu : 0u) | (seen & 8u ? 0xffff0000u : 0u);
            }
            if (a.scores) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int hi = 0; hi < 2; hi++) {
                        const int r = grp * ROWS + 16 * m + r8 + 8 * hi;
                        if (r >= R) continue;
                        float *d = a.scores + ((int64_t)u * R + r) * a.score_stride + row0 + 2 * c;
                        *reinterpret_cast<float2 *>(d) = make_float2(s[m][0][2 * hi], s[m][0][2 * hi + 1]);
                        *reinterpret_cast<float2 *>(d + 8) = make_float2(s[m][1][2 * hi], s[m][1][2 * hi + 1]);
                    }
            }
            float top[MT][2];
            bool up = false;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int hi = 0; hi < 2; hi++) {
                    float x = fmaxf(fmaxf(s[m][0][2 * hi], s[m][0][2 * hi + 1]), fmaxf(s[m][1][2 * hi], s[m][1][2 * hi + 1]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    top[m][hi] = x;
                    up |= x > mx[m][hi] + FEW_SLACK;
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int hi = 0; hi < 2; hi++) {
                        const float to = fmaxf(mx[m][hi], top[m][hi]);
                        const float f = to == mx[m][hi] ? 1.0f : ex2(mx[m][hi] - to);
                        mx[m][hi] = to;
                        sum[m][hi] *= f;
#pragma unroll
                        for (int j = 0; j < HD / 8; j++) {
                            o[m][j][2 * hi] *= f;
                            o[m][j][2 * hi + 1] *= f;
                        }
                    }
            }
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int hi = 0; hi < 2; hi++) {
                    const float from = mx[m][hi] == -INFINITY ? 0.0f : mx[m][hi] - FEW_LIFT;
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float p = ex2(s[m][t][2 * hi + e] - from);
                            s[m][t][2 * hi + e] = p;
                            sum[m][hi] += p;
                        }
                }
            few_pv<KT, HD, MT>(s, st, lane, keep0, keep1, o);
        }
        cp_async_wait<0>();
        __syncthreads();                                      /* the ring becomes the merge buffer */

        float *mo = reinterpret_cast<float *>(smem);          /* [warp][ROWS][OS] */
        float2 *mml = reinterpret_cast<float2 *>(mo + FEW_WARPS * ROWS * OS);     /* [warp][ROWS] */
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
                const int r = 16 * m + r8 + 8 * hi;
                float x = sum[m][hi];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                if (c == 0) mml[w * ROWS + r] = make_float2(mx[m][hi], x);
                float *d = mo + (w * ROWS + r) * OS;
#pragma unroll
                for (int j = 0; j < HD / 8; j++) {
                    d[few_odim<KT>(j, 2 * c)] = o[m][j][2 * hi];
                    d[few_odim<KT>(j, 2 * c + 1)] = o[m][j][2 * hi + 1];
                }
            }
        __syncthreads();

        /* blocks that share the item: owner(s) = the block whose range holds step s */
        const int c0 = (int)(((base + 1) * grid - 1) / total), c1 = (int)(((int64_t)steps[it] * grid - 1) / total);
        const int rows = min(ROWS, R - grp * ROWS);
        constexpr int DPT = FEW_THREADS / HD;                 /* rows a pass covers */
        const int d = tid % HD, dr = tid / HD;
        bool last = true;
        if (c0 != c1) {
            const int slot = 2 * b + (first ? 0 : 1);
            for (int r = dr; r < rows; r += DPT) {
                float m, sm;
                const float val = merge_row(FEW_WARPS, [&](int s) { return mml[s * ROWS + r]; },
                                            [&](int s) { return mo[(s * ROWS + r) * OS + d]; }, m, sm);
                a.part_o[((int64_t)slot * ROWS + r) * HD + d] = val;
                if (d == 0) a.part_ml[(int64_t)slot * ROWS + r] = make_float2(m, sm);
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) s_flag = atomicAdd(&a.arrived[c0], 1) == c1 - c0;
            __syncthreads();
            last = s_flag != 0;
        }
        if (last) {
            if (c0 != c1) {
                __threadfence();
                if (tid == 0) a.arrived[c0] = 0;
            }
            const int s0 = 2 * c0 + (c0 * total / grid >= base ? 0 : 1);     /* block c0's slot; the others' first */
            auto slot_of = [&](int s) { return s == 0 ? s0 : 2 * (c0 + s); };
            int bad = 0;
            for (int r = dr; r < rows; r += DPT) {
                float m, sm, val;
                if (c0 == c1)
                    val = merge_row(FEW_WARPS, [&](int s) { return mml[s * ROWS + r]; },
                                    [&](int s) { return mo[(s * ROWS + r) * OS + d]; }, m, sm);
                else
                    val = merge_row(c1 - c0 + 1, [&](int s) { return __ldcg(&a.part_ml[(int64_t)slot_of(s) * ROWS + r]); },
                                    [&](int s) { return __ldcg(&a.part_o[((int64_t)slot_of(s) * ROWS + r) * HD + d]); }, m, sm);
                const int q = grp * ROWS + r, t = q / a.G, hq = h * a.G + q % a.G;
                const bool none = sm == 0.0f;
                val = none ? 0.0f : val / sm;
                a.out[l * a.o_cache + t * a.o_tok + hq * a.o_head + d] = __float2half_rn(val);
                if (!(fabsf(val) < INFINITY)) bad = 1;
                if (d == 0) {
                    if (a.lse) a.lse[((int64_t)l * a.T + t) * a.n_head_kv * a.G + hq] =
                        none ? -INFINITY : (m - FEW_LIFT + log2f(sm)) * LN2;
                    if (a.norm) a.norm[(int64_t)u * R + q] = none ? make_float2(0.0f, 0.0f) : make_float2(m - FEW_LIFT, 1.0f / sm);
                }
            }
            /* a value that is not finite may be 0 times another token's row: those query rows again, one by one */
            if (a.T > 1 && __syncthreads_or(bad)) {
                for (int r = tid; r < ROWS; r += FEW_THREADS) s_redo[r] = 0;
                __syncthreads();
                for (int r = dr; r < rows; r += DPT) {
                    const int q = grp * ROWS + r;
                    const float x = __half2float(a.out[l * a.o_cache + (q / a.G) * a.o_tok + (h * a.G + q % a.G) * a.o_head + d]);
                    if (!(fabsf(x) < INFINITY)) s_redo[r] = 1;
                }
                __syncthreads();
                for (int r = 0; r < rows; r++)
                    if (s_redo[r]) attend_row<KT, HD>(a, u, (grp * ROWS + r) % a.G, (grp * ROWS + r) / a.G, s_row);
            }
        }
        __syncthreads();
        at = base + i1;
    }
}

/* ------------------------------------------------------------------ */
/* Masses                                                               */
/* ------------------------------------------------------------------ */

/* From the scores that k_attend_few left: a thread per cache row, R weights
 * each; reads 4 R + 4 bytes a row. */
__global__ void __launch_bounds__(256) k_mass_scores(const AttendArgs a) {
    const int u = blockIdx.y, n = attend_rows(a, u), R = a.T * a.G;
    const int2 span = a.span ? a.span[u] : make_int2(0, 0);
    __shared__ float2 s_norm[16];
    if (threadIdx.x < R) s_norm[threadIdx.x] = a.norm[(int64_t)u * R + threadIdx.x];
    __syncthreads();
    for (int j = blockIdx.x * 256 + threadIdx.x; j < n; j += gridDim.x * 256) {
        float mass = 0.0f;
        /* whole steps of the head were walked, and everything from the tail on */
        if (j >= span.y || j < (span.x + ATT_STEP - 1) / ATT_STEP * ATT_STEP) {
            for (int r = 0; r < R; r++) {
                const float x = __ldcs(&a.scores[((int64_t)u * R + r) * a.score_stride + j]);
                mass = fmaf(ex2(x - s_norm[r].x), s_norm[r].y, mass);
            }
        }
        const int64_t i = (int64_t)u * a.n_cells + j;
        a.mass_out[i] = a.mass_in ? fmaf(a.mass_decay, a.mass_in[i], mass) : mass;
    }
}

constexpr int MASS_THREADS = 128, MASS_KEYS = 64;

/* Scores again, now with the denominators known: each warp holds 16 cache rows
 * of a unit and goes over all query rows, 16 at a time, so the weights of a
 * cache row are summed where they are made, in one order. */
template <int KT, int HD>
__global__ void __launch_bounds__(MASS_THREADS) k_mass_tiles(const AttendArgs a) {
    using S = FewStage<KT, HD>;
    __shared__ __align__(16) uint8_t s_keys[MASS_THREADS / 32][S::BYTES];
    const int u = blockIdx.y, l = u / a.n_head_kv, h = u - l * a.n_head_kv, R = a.T * a.G;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, r8 = lane >> 2, c = lane & 3;
    const int n = attend_rows(a, u);
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride;
    const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
    const bool want_pos = a.window > 0 || a.slopes != nullptr;
    const ScoreMap map(a);
    const uint32_t st = smem_u32(s_keys[w]);
    for (int row0 = (blockIdx.x * (MASS_THREADS / 32) + w) * 16; row0 < n; row0 += gridDim.x * MASS_KEYS) {
        __syncwarp();
        few_load<KT, HD>(a, k, k, pos, want_pos, row0, n, st, lane);
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        float mass[4] = {0.0f, 0.0f, 0.0f, 0.0f};               /* keys 2c, 2c+1, 2c+8, 2c+9 */
        /* by order, token t sees row j only if j <= n - T + t: query rows before that see none of these 16 */
        int q0 = 0;
        if (!a.tree) q0 = max(0, row0 - (n - a.T)) * a.G / 16 * 16;
        for (; q0 < R; q0 += 16) {
            uint32_t qf[1][HD / 16][4];
            int tok[2], tp[2];
            float slope2[2];
            float2 nm[2];
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
                const int r = q0 + r8 + 8 * hi, t = r / a.G, head = h * a.G + r % a.G;
                const bool in = r < R;
                tok[hi] = in ? t : -1;
                tp[hi] = in && want_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
                slope2[hi] = in && a.slopes ? a.slopes[head] * LOG2E : 0.0f;
                nm[hi] = in ? a.norm[(int64_t)u * R + r] : make_float2(0.0f, 0.0f);
                const __half *q = a.q + l * a.q_cache + (in ? t * a.q_tok + head * a.q_head : 0);
#pragma unroll
                for (int s = 0; s < HD / 16; s++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        qf[0][s][hi + 2 * e] = in ? *reinterpret_cast<const uint32_t *>(q + few_qdim<KT>(s, c, e)) : 0u;
            }
            float s[1][2][4];
            few_qk<KT, HD, 1>(qf, st, lane, s);
            const bool all = row0 + 16 <= n - a.T && a.window <= 0 && q0 + 16 <= R;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int hi = e >> 1, key = 8 * t + 2 * c + (e & 1);
                    float x = map(s[0][t][e]);
                    int pk = 0;
                    if (want_pos) {
                        pk = (int)lds32(st + S::P + 4 * key);
                        x = fmaf(-slope2[hi], (float)(tp[hi] - pk), x);
                    }
                    bool see = true;
                    if (!all) see = tok[hi] >= 0 && attend_sees(a, l, tok[hi], row0 + key, n, pk, (int64_t)tp[hi] - a.window);
                    if (see) mass[2 * t + (e & 1)] = fmaf(ex2(x - nm[hi].x), nm[hi].y, mass[2 * t + (e & 1)]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 4; m < 32; m <<= 1) mass[i] += __shfl_xor_sync(0xffffffffu, mass[i], m);
        if (r8 == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = row0 + 2 * c + (i & 1) + 8 * (i >> 1);
                if (j >= n) continue;
                const int64_t x = (int64_t)u * a.n_cells + j;
                a.mass_out[x] = a.mass_in ? fmaf(a.mass_decay, a.mass_in[x], mass[i]) : mass[i];
            }
        }
    }
}

}  // namespace tria
