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
    long long wait_limit;                /* cycles a pipeline wait may take before it gives up (ST_TIMEOUT) */
    /* plan and workspace (host-filled) */
    int32_t copy16;                      /* rows start on 16-byte boundaries (f16), 8-byte ones (q8_0) */
    int32_t groups;                      /* groups of query rows per unit */
    const int32_t *steps;                /* inclusive prefix of the items' steps, or NULL: scanned in the kernel */
    const int2 *span;                    /* windowed: (head, tail) of each item, else NULL */
    float *part_o;                       /* [2 * grid][rows][head_dim] */
    float2 *part_ml;                     /* [2 * grid][rows] */
    int32_t *arrived;                    /* [grid]: by the first block of an item (one such item a block); zero between calls */
    float2 *norm;                        /* [n_layer * n_head_kv][T * G]: (max, 1 / sum) of each query row, or NULL */
    int32_t *redo;                       /* [0] how many, then query rows (unit * T * G + r) to do again one by one */
    float *scores;                       /* [n_layer * n_head_kv][T * G][score_stride], or NULL */
    int64_t score_stride;
};

/* Lane 0's value for the whole warp, so that what depends on it is uniform. */
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

/* Rows of unit u: a count outside the cache is clamped and reported. */
__device__ __forceinline__ int attend_rows(const AttendArgs &a, int u) {
    const int n = a.n_rows[u];
    if (n >= 0 && n <= a.n_cells) return n;
    atomicOr(a.status, ST_ROWS);
    return n < 0 ? 0 : a.n_cells;
}

/* Checked build: a block's walk stands at step `at` of item `it`, whose rows
 * are shared by blocks c0 .. c1; span as the plan left it. */
__device__ __forceinline__ bool walk_ok(const AttendArgs &a, int items, int it, int64_t at, int64_t total, int2 span, int step) {
    return bounds_ok(it >= 0 && it < items && at >= 0 && at < total && span.x >= 0 && span.y >= 0 && span.x <= a.n_cells &&
                     span.y <= (a.n_cells + step - 1) / step * step && span.y % step == 0, a.status);
}
__device__ __forceinline__ bool share_ok(const AttendArgs &a, int c0, int c1, int b, int grid) {
    return bounds_ok(c0 >= 0 && c0 <= b && b <= c1 && c1 < grid && grid <= (int)gridDim.x, a.status);
}

/* Whether token t of cache l sees row j of a unit with n rows; pos: the row's
 * position, lo: tok_pos[t] - window (both read only with a window). */
__device__ __forceinline__ bool attend_sees(const AttendArgs &a, int l, int t, int j, int n, int pos, int64_t lo) {
    if (j >= n) return false;
    const int own = j - (n - a.T);
    if (own >= 0) {
        if (a.tree) {
            if (!bounds_ok(own < a.T && (own >> 5) < a.tree_words && t >= 0 && t < a.T, a.status)) return false;
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
__device__ __forceinline__ float tanh_small(float u) {
    const float z = u * u;
    float s = 21844.0f / 6081075.0f;
    s = fmaf(s, z, -1382.0f / 155925.0f);
    s = fmaf(s, z, 62.0f / 2835.0f);
    s = fmaf(s, z, -17.0f / 315.0f);
    s = fmaf(s, z, 2.0f / 15.0f);
    s = fmaf(s, z, -1.0f / 3.0f);
    return fmaf(s * z, u, u);
}
__device__ __forceinline__ float tanh_both(float u) {
    const float b = fmaf(-2.0f, rcp(1.0f + ex2(2.0f * LOG2E * u)), 1.0f);
    return fabsf(u) < 0.4f ? tanh_small(u) : b;
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

__device__ __forceinline__ float half_at(const uint8_t *p) { return __half2float(*reinterpret_cast<const __half *>(p)); }

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
template <int KT, int HD, class Q>
__device__ __forceinline__ float attend_score(const ScoreMap &f, const uint8_t *krow, const Q *q, float slope2,
                                              int tok_pos, int pos) {
    float s = 0.0f;
    for (int d = 0; d < HD; d++) s = fmaf((float)q[d], row_value<KT>(krow, d), s);
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
    const bool none = !any || sum == 0.0f;
    if (tid < HD) a.out[l * a.o_cache + t * a.o_tok + head * a.o_head + tid] = __float2half_rn(none ? 0.0f : acc / sum);
    if (tid == 0) {
        if (a.lse) a.lse[((int64_t)l * a.T + t) * a.n_head_kv * a.G + head] = none ? -INFINITY : (m + log2f(sum)) * LN2;
        if (a.norm) a.norm[((int64_t)u * a.T + t) * a.G + g] = none ? make_float2(0.0f, 0.0f) : make_float2(m, 1.0f / sum);
    }
}


/* Whether a result of unit u that is not finite can be wrong.  f16: if some
 * value that one token sees and another does not is not finite (0 times it), and
 * where weights are two parts, if any value is not (one part may be 0 or
 * negative).  q8_0: if a block's scale is not finite or, on the tiles, so large
 * that its values pass f16's 65504 and their remainders are lost.  For all
 * threads of a block of ROW_THREADS. */
constexpr float TILE_SCALE = 512.0f;     /* below it 128 times a scale is at most 65504 */
template <int KT, int HD, bool TILE>
__device__ bool result_in_doubt(const AttendArgs &a, int u) {
    const int l = u / a.n_head_kv, h = u - l * a.n_head_kv, n = attend_rows(a, u);
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride, *v = a.v[l] + (int64_t)h * a.head_stride;
    bool bad = false;
    if constexpr (KT == KT_F16) {
        const int from = !TILE || a.window > 0 ? 0 : max(0, n - a.T);
        for (int64_t x = threadIdx.x; x < (int64_t)(n - from) * HD; x += ROW_THREADS)
            bad |= !(fabsf(row_value<KT>(v + (from + x / HD) * a.cell_stride, (int)(x % HD))) < INFINITY);
    } else {
        constexpr int NB = HD / 32;
        for (int64_t x = threadIdx.x; x < (int64_t)n * NB; x += ROW_THREADS) {
            const int64_t at = x / NB * a.cell_stride + x % NB * 34;
            const float dk = fabsf(half_at(k + at)), dv = fabsf(half_at(v + at));
            bad |= TILE ? !(dk < TILE_SCALE && dv < TILE_SCALE) : !(dv < INFINITY);
        }
    }
    return __syncthreads_or(bad);
}

/* ------------------------------------------------------------------ */
/* Plan: which rows of the cache each group of query rows walks         */
/* ------------------------------------------------------------------ */

/* Query rows r = t * G + g of a unit are taken in groups of `rows`; an item is
 * (unit, group).  An item walks steps of `step` cache rows: all rows up to
 * the last that its tokens see by order, or, with a window, the rows before
 * `head` (where the sink ends) and those from `tail` on (where the window
 * begins).  Positions need not ascend: head and tail enclose every row that
 * the window admits. */
constexpr int ATT_STEP = 64;           /* few query rows */
constexpr int TILE_STEP = 128;         /* many */

/* Rows of the unit that the group's last token can see by order. */
__device__ __forceinline__ int item_rows(const AttendArgs &a, int u, int grp, int rows) {
    const int n = attend_rows(a, u);
    const int r1 = min(a.T * a.G, (grp + 1) * rows) - 1;
    return max(0, a.tree ? n : min(n, n - a.T + r1 / a.G + 1));
}

__device__ __forceinline__ int span_steps(int n, int2 s, int step) {
    const int hs = (s.x + step - 1) / step;
    return hs + (n > s.y ? (n - s.y + step - 1) / step : 0);
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
__global__ void __launch_bounds__(PLAN_THREADS) k_attend_plan(const AttendArgs a, int rows, int step, int items, int2 *span,
                                                              int32_t *steps, int32_t *done) {
    __shared__ int s_min[PLAN_THREADS / 32], s_max[PLAN_THREADS / 32], s_last;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (a.redo && blockIdx.x == 0 && threadIdx.x == 0) a.redo[0] = 0;
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
#pragma unroll 8
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
            tail = tail / step * step;
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
            st = span_steps(n, make_int2(min(s.x, n), s.y), step);
        }
        const int incl = block_scan(st, s_min, PLAN_THREADS, &sum);
        if (it < items) steps[it] = base + incl;
        base += sum;
    }
}

/* Blocks that share `total` steps of `items` items: at most the grid, and so
 * many that a block takes at least sqrt(join * steps of an item) steps.  A step
 * more in a row costs its time once; a partial result more costs `join` of that
 * in the one block that joins an item's results: their sum is least there. */
__device__ __forceinline__ int blocks_used(int64_t total, int items, int grid, float join) {
    const int64_t least = (int64_t)ceilf(sqrtf(join * (float)total / (float)items));
    return (int)min((int64_t)grid, (total + least - 1) / max(least, (int64_t)1));
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* d = a b. */
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t word_at(const uint8_t *p) { return *reinterpret_cast<const uint32_t *>(p); }
__device__ __forceinline__ uint2 two_words_at(const uint8_t *p) { return *reinterpret_cast<const uint2 *>(p); }
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

/* d += a b, 16 x 8 x 16, bf16 operands, fp32 sums. */
__device__ __forceinline__ void mma16816_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* x and y as f16 pairs, rounded (hi) and what the rounding left (lo). */
__device__ __forceinline__ void split_half(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pack_half2(x, y);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    lo = pack_half2(x - f.x, y - f.y);
}
/* x and y as bf16 pairs, rounded (hi) and what the rounding left (lo): 16 bits
 * of each over fp32's range. */
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t &hi, uint32_t &lo) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    const float rx = x - __uint_as_float(hi << 16), ry = y - __uint_as_float(hi & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(ry), "f"(rx));
}
/* The int8 pairs (byte 0, byte 1) and (byte 2, byte 3) of w as bf16 pairs,
 * exactly: 0x4300 | the low seven bits is 128 + them, 0x4300 | the sign bit is
 * 128 or, for a negative x = low bits - 128, 256; their difference is x. */
__device__ __forceinline__ void int8x4_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(a & 0xff7fff7fu), "r"(a & 0xff80ff80u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(b & 0xff7fff7fu), "r"(b & 0xff80ff80u));
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
    static constexpr int VS = KT == KT_F16 ? 2 * HD : (HD == 128 ? 144 : 80);      /* 8 + 136, 68 */
    static constexpr int K = 0, V = 16 * KS, P = V + 16 * VS, BYTES = P + 64;
};

/* Blocks an SM holds, by registers (value sums and queries are 48 of them per
 * 8 query rows), and the stages that their warps' rings leave room for. */
template <int KT, int NT>
__host__ __device__ constexpr int few_blocks() { return NT == 2 ? 2 : 3; }
template <int KT, int HD, int NT>
__host__ __device__ constexpr int few_stages() {
    const int fit = 200 * 1024 / few_blocks<KT, NT>() / FEW_WARPS / FewStage<KT, HD>::BYTES;
    return fit < 4 ? fit : 4;
}
template <int KT, int HD, int NT>
__host__ __device__ constexpr int few_smem() {
    const int ring = FEW_WARPS * few_stages<KT, HD, NT>() * FewStage<KT, HD>::BYTES;
    const int merge = FEW_WARPS * 8 * NT * (HD + 4) * 4 + FEW_WARPS * 8 * NT * 8;
    return ring > merge ? ring : merge;
}

/* Scores are kept in units where a weight is 2^(x - m + FEW_LIFT): weights of
 * rows far below the maximum stay normal f16 numbers (2^-14 and up) down to
 * 2^-26 of it, and the maximum may fall FEW_SLACK behind before the sums are
 * rescaled: 2^(FEW_LIFT + FEW_SLACK) is still finite in f16.  (q8_0 weights take
 * no part in this: see few_pv.)  Sums rescaled sooner cost 32 multiplications a
 * thread and 8 query rows: with slack 8, the same for one token (8 units of
 * 65521 rows, 74 us) and 73 us instead of 75 for 32 query rows over 32000. */
constexpr float FEW_LIFT = 12.0f, FEW_SLACK = 3.0f;
/* Measured (blocks_used): 4000 rows, 12 query rows: 30 us at 0.05, 27 at 0.2, 23 at
 * 0.6; 500 rows: 16, 16 and 27 us. */
constexpr float FEW_JOIN = 0.2f;

/* Copies one side of the warp's slice: rows [r0, r0 + 16) from p to `st`, row
 * stride RS; rows at and behind n become zeros.  A full slice of aligned rows
 * takes 16-byte copies with addresses stepped from one to the next: f16 a row
 * by HD / 8 lanes, q8_0 rows of 136 bytes (8 bytes off a 16-byte boundary in
 * every other head) by eight lanes and one 8-byte piece, on the side `lead`. */
template <int KT, int HD, int RS>
__device__ __forceinline__ void few_load(const AttendArgs &a, const uint8_t *p, int lead, int r0, int n, uint32_t st, int lane) {
    const bool full = r0 + 16 <= n;
    if (KT == KT_F16 && full && a.copy16) {
        constexpr int CH = HD / 8, RPI = 32 / CH;
        const int r = lane / CH, c = lane % CH;
        const int64_t step = RPI * a.cell_stride;
        p += (int64_t)(r0 + r) * a.cell_stride + 16 * c;
        const uint32_t d = st + r * RS, cx = 16 * (c ^ r);
#pragma unroll
        for (int i = 0; i < 16 / RPI; i++) {
            cp_async16(d + RPI * i * RS + (cx ^ (16 * ((RPI * i) & 7))), p, 16u);
            p += step;
        }
    } else if (KT == KT_Q8_0 && HD == 128 && full && a.copy16) {
        const int r = lane >> 3, c = lane & 7;
        const int64_t step = 4 * a.cell_stride;
        const uint8_t *q = p + (int64_t)(r0 + r) * a.cell_stride + lead + 16 * c;
        const uint32_t d = st + r * RS + 2 * lead + 16 * c;     /* a row starts lead bytes in, its chunks on 16 */
#pragma unroll
        for (int i = 0; i < 4; i++) {
            cp_async16(d + 4 * i * RS, q, 16u);
            q += step;
        }
        if (lane < 16)
            cp_async8(st + lane * RS + (lead ? lead : 128), p + (int64_t)(r0 + lane) * a.cell_stride + (lead ? 0 : 128), 8u);
    } else {
        constexpr int W = KT == KT_F16 ? HD / 2 : HD / 32 * 34 / 4;
        for (int x = lane; x < 16 * W; x += 32) {
            const int r = x / W, c = x - r * W;
            const bool in = r0 + r < n;
            const uint32_t at = KT == KT_F16 ? 16 * ((c >> 2) ^ (r & 7)) + 4 * (c & 3) : lead + 4 * c;
            cp_async4(st + r * RS + at, p + (in ? (int64_t)(r0 + r) * a.cell_stride + 4 * c : 0), in ? 4u : 0u);
        }
    }
}
__device__ __forceinline__ void few_load_pos(const int32_t *pos, int r0, int n, uint32_t st, int lane) {
    if (lane < 16) {
        const bool in = r0 + lane < n;
        cp_async4(st + 4 * lane, pos + (in ? r0 + lane : 0), in ? 4u : 0u);
    }
}

/* The dims that k-step s takes of a row, for lane column c: f16 16 s + 2 c, +1
 * and those 8 on; q8_0 the bytes 8 c + 4 (s & 1) .. +3 of block s / 2, so that a
 * lane's share of a block is 8 bytes in a row. */
template <int KT>
__device__ __forceinline__ int few_qdim(int s, int c, int hi) {
    return KT == KT_F16 ? 16 * s + 2 * c + 8 * hi : 32 * (s >> 1) + 8 * c + 4 * (s & 1) + 2 * hi;
}
/* The dim of row r8 (+ 8 hi) of value tile j: q8_0 tiles stay within a block and
 * give a lane row the bytes 4 r8 .. 4 r8 + 3 of it over the block's two tiles. */
template <int KT>
__device__ __forceinline__ int few_odim(int j, int r8, int hi) {
    return KT == KT_F16 ? 16 * j + r8 + 8 * hi : 32 * (j >> 1) + 4 * r8 + 2 * (j & 1) + hi;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

/* The products of 16 cache rows with 8 NT query rows, rows of the cache as the
 * matrix rows: s[t][e] is cache row r8 + 8 (e >> 1) with query row 8 t + 2 c + (e & 1). */
template <int KT, int HD, int NT>
__device__ __forceinline__ void few_qk(const uint32_t (&qf)[NT][HD / 16][2], const uint8_t *st, int lead, int lane, float (&s)[NT][4]) {
    constexpr int KS = FewStage<KT, HD>::KS;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = 0.0f;
    if constexpr (KT == KT_F16) {
        const int row = lane & 15, hi = lane >> 4;
        const uint32_t at = smem_u32(st) + row * KS;
#pragma unroll
        for (int x = 0; x < HD / 16; x++) {
            uint32_t k[4];
            ldsm4(k, at + 16 * ((2 * x + hi) ^ (row & 7)));
#pragma unroll
            for (int t = 0; t < NT; t++) mma16816(s[t], k, qf[t][x][0], qf[t][x][1]);
        }
    } else {
        const int r8 = lane >> 2, c = lane & 3;
        st += lead + r8 * KS;
#pragma unroll
        for (int blk = 0; blk < HD / 32; blk++) {
            const int sh = (2 * blk + 2) & 7;                        /* bytes into the aligned 8-byte word */
            uint32_t k[2][4];
            float d[2];
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
                const uint8_t *at = st + 8 * c + (8 * hi * KS + 34 * blk + 2 - sh);
                const uint2 x = two_words_at(at);
                uint32_t w0, w1;
                if (sh == 0) {
                    w0 = x.x;
                    w1 = x.y;
                } else {
                    const uint2 y = two_words_at(at + 8);
                    w0 = sh == 2 ? __funnelshift_r(x.x, x.y, 16) : sh == 4 ? x.y : __funnelshift_r(x.y, y.x, 16);
                    w1 = sh == 2 ? __funnelshift_r(x.y, y.x, 16) : sh == 4 ? y.x : __funnelshift_r(y.x, y.y, 16);
                }
                int8x4_half(w0, k[0][hi], k[0][hi + 2]);
                int8x4_half(w1, k[1][hi], k[1][hi + 2]);
                d[hi] = half_at(st + 8 * hi * KS + 34 * blk);
            }
            /* the block's scale belongs to the cache row, so it multiplies the block's sum: the f16 operands stay the
             * stored integers and the scores keep fp32 */
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float p[4];
                mma16816_first(p, k[0], qf[t][2 * blk][0], qf[t][2 * blk][1]);
                mma16816(p, k[1], qf[t][2 * blk + 1][0], qf[t][2 * blk + 1][1]);
                s[t][0] = fmaf(p[0], d[0], s[t][0]);
                s[t][1] = fmaf(p[1], d[0], s[t][1]);
                s[t][2] = fmaf(p[2], d[1], s[t][2]);
                s[t][3] = fmaf(p[3], d[1], s[t][3]);
            }
        }
    }
}

/* o += v^T p over the slice's 16 rows, the weights in two parts (rounded value
 * and remainder), for which the tensor pipe has room.  FULL: every query row sees them all.
 * Otherwise a weight of 0 meets 0: keep0, keep1 (f16) have the bits of a V pair
 * whose row some query row sees, and a q8_0 scale only enters where p is not 0
 * (a row that is not seen may hold NaN).
 *
 * f16: one token over 8 units of 65521 rows takes 75 us with two parts and 74
 * with one, whose rounding (2^-11 of each weight) showed in the results.
 *
 * q8_0: the V operands are the stored integers, so the scales go into the
 * weights: products whose size follows the values', not the weights' alone,
 * and for which f16 has no range.  bf16 has it, and its two parts keep 16 bits
 * (128 units of 8197 to 32768 rows: 236 us, with one f16 operand 242). */
template <int KT, int HD, int NT, bool FULL>
__device__ __forceinline__ void few_pv(const float (&p)[NT][4], const uint8_t *st, int lead, int lane, uint32_t keep0, uint32_t keep1,
                                       float (&o)[NT][HD / 16][4]) {
    constexpr int VS = FewStage<KT, HD>::VS;
    if constexpr (KT == KT_F16) {
        uint32_t h[NT][2], r[NT][2];                           /* weights rounded, and what the rounding left */
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                split_half(p[t][2 * i], p[t][2 * i + 1], h[t][i], r[t][i]);
                h[t][i] = transpose8(h[t][i]);
                r[t][i] = transpose8(r[t][i]);
            }
        const int row = (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
        const uint32_t at = smem_u32(st) + row * VS;
#pragma unroll
        for (int j = 0; j < HD / 16; j++) {
            uint32_t v[4];
            ldsm4t(v, at + 16 * ((2 * j + hi) ^ (row & 7)));
            if (!FULL) {
                v[0] &= keep0;
                v[1] &= keep0;
                v[2] &= keep1;
                v[3] &= keep1;
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                mma16816(o[t][j], v, h[t][0], h[t][1]);
                mma16816(o[t][j], v, r[t][0], r[t][1]);
            }
        }
    } else {
        const int r8 = lane >> 2, c = lane & 3;
        st += lead;
        const uint8_t *v0 = st + 2 * c * VS + 4 * r8, *d0 = st + r8 * VS;      /* rows 2c, 2c+1, 2c+8, 2c+9; scales of r8, r8+8 */
#pragma unroll
        for (int blk = 0; blk < HD / 32; blk++) {
            const int sh = (2 * blk + 2) & 3;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint8_t *at = v0 + ((i & 1) + (i >> 1) * 8) * VS + 34 * blk;
                if (sh == 0) w[i] = word_at(at + 2);
                else w[i] = __funnelshift_r(word_at(at), word_at(at + 4), 16);
            }
            uint32_t lo[4], hi[4];
            int8x4_bf16(__byte_perm(w[0], w[1], 0x5140), lo[0], lo[1]);
            int8x4_bf16(__byte_perm(w[0], w[1], 0x7362), hi[0], hi[1]);
            int8x4_bf16(__byte_perm(w[2], w[3], 0x5140), lo[2], lo[3]);
            int8x4_bf16(__byte_perm(w[2], w[3], 0x7362), hi[2], hi[3]);
            const float da = half_at(d0 + 34 * blk), db = half_at(d0 + 8 * VS + 34 * blk);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float x[4] = {p[t][0] * da, p[t][1] * da, p[t][2] * db, p[t][3] * db};
                if (!FULL) {
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = p[t][i] == 0.0f ? 0.0f : x[i];
                }
                uint32_t h[2], r[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    split_bf16(x[2 * i], x[2 * i + 1], h[i], r[i]);
                    h[i] = transpose8(h[i]);
                    r[i] = transpose8(r[i]);
                }
                mma16816_bf16(o[t][2 * blk], lo, h[0], h[1]);
                mma16816_bf16(o[t][2 * blk + 1], hi, h[0], h[1]);
                mma16816_bf16(o[t][2 * blk], lo, r[0], r[1]);
                mma16816_bf16(o[t][2 * blk + 1], hi, r[0], r[1]);
            }
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

/* Attention of the items' query rows (8 NT a group) over their steps.  The
 * steps of all items are shared out evenly: block b takes steps
 * [b * total / grid, (b + 1) * total / grid) (grid: blocks_used), whatever
 * units they fall in, so ragged counts read from the device keep every SM busy
 * without the host knowing them.  Within a step each warp takes 16 cache rows
 * of its own and keeps its own running maximum, sum and value sums: the loop
 * has no block barrier.  A warp's ring is refilled side by side, K as soon as
 * the scores are made and V after the sums, so a stage is in flight but for the
 * half being read.  An item that ends in several blocks leaves partial
 * results; the block that arrives last merges them in block order, so the
 * result does not depend on timing.
 *
 * Cache rows are the matrix rows and query rows its columns, so few query rows
 * waste little: 16 cache rows cost 16 mma per 8 query rows (head_dim 128), and
 * the weights turn around in registers (movmatrix) for the value product.
 * EXTRA: the call caps, biases or windows its scores.
 *
 * Bound by memory: 8 units of 65521 f16 rows (268 MB), 4 query rows each, take
 * 64 us (4.2 TB/s; 42 at copy rate) with start and join 12 of them; 128 units of
 * 8197 to 32768 q8_0 rows (710 MB) take 236 us a call, because a 136-byte row
 * costs the 64-byte pieces that it touches.  Three blocks an SM: f16 stages of
 * 8 KB fill shared memory, and q8_0 bytes need registers (that case in 279 us
 * with four, which spill). */
template <int KT, int HD, int NT, bool EXTRA>
__global__ void __launch_bounds__(FEW_THREADS, few_blocks<KT, NT>()) k_attend_few(const AttendArgs a) {
    using S = FewStage<KT, HD>;
    constexpr int ROWS = 8 * NT, ST = few_stages<KT, HD, NT>(), OS = HD + 4;
    static_assert(ST >= 2, "ring");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_steps[512];
    __shared__ int s_warp[FEW_WARPS];
    __shared__ int s_flag;
    __shared__ RowShared<HD> s_row;
    __shared__ int s_redo[ROWS];
    __shared__ float s_inv[ROWS];
    const int tid = threadIdx.x, lane = tid & 31, w = uniform(tid >> 5), r8 = lane >> 2, c = lane & 3;
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
    const int64_t total = uniform(steps[items - 1]);
    const int b = blockIdx.x, grid = blocks_used(total, items, gridDim.x, FEW_JOIN);     /* none idle between an item's first and last */
    const ScoreMap map(a);
    const bool want_pos = EXTRA && (a.window > 0 || a.slopes != nullptr);
    uint8_t *const ring = smem + w * ST * S::BYTES;

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
        it = uniform(it);
        const int64_t base = uniform(it ? steps[it - 1] : 0), upto = uniform(steps[it]);
        const int i0 = (int)(at - base), i1 = (int)(min(end, upto) - base);
        const int u = it / a.groups, grp = it - u * a.groups, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
        const int n = uniform(attend_rows(a, u));
        int2 span = a.span ? a.span[it] : make_int2(0, 0);
        span = make_int2(uniform(span.x), uniform(span.y));
        if (!walk_ok(a, items, it, at, total, span, ATT_STEP)) break;
        const int head_steps = (min(span.x, n) + ATT_STEP - 1) / ATT_STEP;
        auto slice_row = [&](int i) { return (i < head_steps ? i * ATT_STEP : span.y + (i - head_steps) * ATT_STEP) + FEW_SLICE * w; };
        const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride, *v = a.v[l] + (int64_t)h * a.head_stride;
        const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);

        const int lead = KT == KT_Q8_0 && HD == 128 ? (int)((h * a.head_stride) & 8) : 0;

        auto load_k = [&](int i) {
            if (i < i1) {
                const int row = slice_row(i);
                const uint32_t st = smem_u32(ring + (i - i0) % ST * S::BYTES);
                few_load<KT, HD, S::KS>(a, k, lead, row, n, st + S::K, lane);
                if (want_pos) few_load_pos(pos, row, n, st + S::P, lane);
            }
            cp_async_commit();
        };
        auto load_v = [&](int i) {
            if (i < i1) few_load<KT, HD, S::VS>(a, v, lead, slice_row(i), n, smem_u32(ring + (i - i0) % ST * S::BYTES + S::V), lane);
            cp_async_commit();
        };
        /* prologue: copies first, then the queries while they fly */
#pragma unroll
        for (int p = 0; p < ST; p++) {
            load_k(i0 + p);
            load_v(i0 + p);
        }
        uint32_t qf[NT][HD / 16][2];
        int tok[NT][2], tp[NT][2];
        float slope2[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            {
                const int r = grp * ROWS + 8 * t + r8;
                const bool in = r < R;
                const __half *q = a.q + l * a.q_cache + (in ? (r / a.G) * a.q_tok + (h * a.G + r % a.G) * a.q_head : 0);
#pragma unroll
                for (int s = 0; s < HD / 16; s++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        qf[t][s][e] = in ? *reinterpret_cast<const uint32_t *>(q + few_qdim<KT>(s, c, e)) : 0u;
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = grp * ROWS + 8 * t + 2 * c + e;
                const bool in = r < R;
                tok[t][e] = in ? r / a.G : -1;
                tp[t][e] = in && want_pos ? a.tok_pos[l * a.tok_pos_stride + r / a.G] : 0;
                slope2[t][e] = EXTRA && in && a.slopes ? a.slopes[h * a.G + r % a.G] * LOG2E : 0.0f;
            }
        }
        float o[NT][HD / 16][4], mx[NT][2], sum[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            mx[t][0] = mx[t][1] = -INFINITY;
            sum[t][0] = sum[t][1] = 0.0f;
#pragma unroll
            for (int x = 0; x < HD / 16; x++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[t][x][i] = 0.0f;
        }

        for (int i = i0; i < i1; i++) {
            const uint8_t *const st = ring + (i - i0) % ST * S::BYTES;
            const int row0 = slice_row(i);
            const bool live = row0 < n;
            float s[NT][4];
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
            const bool all = row0 + FEW_SLICE <= n - a.T && (!EXTRA || a.window <= 0);   /* every token sees every row */
            cp_async_wait<2 * ST - 1>();
            __syncwarp();
            if (live) {
                few_qk<KT, HD, NT>(qf, st + S::K, lead, lane, s);
                if (EXTRA && map.cap > 0.0f) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[t][e] = map.cap * tanh_both(s[t][e] * map.scale);
                } else {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[t][e] *= map.scale;
                }
                int pk[2] = {0, 0};
                if (want_pos) {
                    pk[0] = (int)word_at(st + S::P + 4 * r8);
                    pk[1] = (int)word_at(st + S::P + 4 * (r8 + 8));
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            s[t][e] = fmaf(-slope2[t][e & 1], (float)(tp[t][e & 1] - pk[e >> 1]), s[t][e]);
                }
                if (!all) {
                    bool seen[2] = {false, false};
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const bool see = tok[t][e & 1] >= 0 &&
                                             attend_sees(a, l, tok[t][e & 1], row0 + r8 + 8 * (e >> 1), n, pk[e >> 1],
                                                         (int64_t)tp[t][e & 1] - a.window);
                            s[t][e] = see ? s[t][e] : -INFINITY;
                            seen[e >> 1] |= see;
                        }
                    /* rows 2c, 2c+1 (+ 8): four lanes each */
                    const uint32_t b0 = __ballot_sync(0xffffffffu, seen[0]) >> (8 * c), b1 = __ballot_sync(0xffffffffu, seen[1]) >> (8 * c);
                    keep0 = (b0 & 0xfu ? 0xffffu : 0u) | (b0 & 0xf0u ? 0xffff0000u : 0u);
                    keep1 = (b1 & 0xfu ? 0xffffu : 0u) | (b1 & 0xf0u ? 0xffff0000u : 0u);
                }
                if (a.scores) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int r = grp * ROWS + 8 * t + 2 * c + e;
                            if (r >= R) continue;
                            if (!bounds_ok(row0 >= 0 && row0 + FEW_SLICE <= a.score_stride, a.status)) continue;
                            float *d = a.scores + ((int64_t)u * R + r) * a.score_stride + row0 + r8;
                            d[0] = s[t][e];
                            d[8] = s[t][e + 2];
                        }
                }
            }
            __syncwarp();
            load_k(i + ST);
            if (live) {
                float top[NT][2];
                bool up = false;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = fmaxf(s[t][e], s[t][e + 2]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        top[t][e] = x;
                        up |= x > mx[t][e] + FEW_SLACK;
                    }
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float to = fmaxf(mx[t][e], top[t][e]);
                            const float f = to == mx[t][e] ? 1.0f : ex2(mx[t][e] - to);
                            mx[t][e] = to;
                            sum[t][e] *= f;
#pragma unroll
                            for (int x = 0; x < HD / 16; x++) {
                                o[t][x][e] *= f;
                                o[t][x][e + 2] *= f;
                            }
                        }
                }
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float from = mx[t][e & 1] == -INFINITY ? 0.0f : mx[t][e & 1] - FEW_LIFT;
                        s[t][e] = ex2(s[t][e] - from);
                        sum[t][e & 1] += s[t][e];
                    }
            }
            cp_async_wait<2 * ST - 1>();
            __syncwarp();
            if (live) {
                if (all) few_pv<KT, HD, NT, true>(s, st + S::V, lead, lane, keep0, keep1, o);
                else few_pv<KT, HD, NT, false>(s, st + S::V, lead, lane, keep0, keep1, o);
            }
            __syncwarp();
            load_v(i + ST);
        }
        cp_async_wait<0>();
        __syncthreads();                                      /* the ring becomes the merge buffer */

        float *mo = reinterpret_cast<float *>(smem);          /* [warp][ROWS][OS] */
        float2 *mml = reinterpret_cast<float2 *>(mo + FEW_WARPS * ROWS * OS);     /* [warp][ROWS] */
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = 8 * t + 2 * c + e;
                float x = sum[t][e];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (r8 == 0) mml[w * ROWS + r] = make_float2(mx[t][e], x);
                float *d = mo + (w * ROWS + r) * OS;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    d[few_odim<KT>(j, r8, 0)] = o[t][j][e];
                    d[few_odim<KT>(j, r8, 1)] = o[t][j][e + 2];
                }
            }
        __syncthreads();

        /* blocks that share the item: owner(s) = the block whose range holds step s */
        const int c0 = (int)(((base + 1) * grid - 1) / total), c1 = (int)((upto * grid - 1) / total);
        const int rows = min(ROWS, R - grp * ROWS);
        if (!share_ok(a, c0, c1, b, grid) ||
            !bounds_ok((int64_t)(c1 - c0 + 1) * rows * 8 <= (int64_t)dynamic_smem_bytes(), a.status)) break;
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
            for (int r = tid; r < ROWS; r += FEW_THREADS) s_redo[r] = 0;
            if (c0 != c1) {
                __threadfence();
                if (tid == 0) a.arrived[c0] = 0;
            }
            auto put = [&](int r, int dim, float x) {
                const int q = grp * ROWS + r;
                if (!(fabsf(x) < INFINITY)) s_redo[r] = 1;
                return a.out + l * a.o_cache + (q / a.G) * a.o_tok + (h * a.G + q % a.G) * a.o_head + dim;
            };
            auto put_sums = [&](int r, float m, float sm) {
                const int q = grp * ROWS + r;
                const bool none = sm == 0.0f;
                if (a.lse) a.lse[((int64_t)l * a.T + q / a.G) * a.n_head_kv * a.G + h * a.G + q % a.G] =
                    none ? -INFINITY : (m - FEW_LIFT + log2f(sm)) * LN2;
                if (a.norm) a.norm[(int64_t)u * R + q] = none ? make_float2(0.0f, 0.0f) : make_float2(m - FEW_LIFT, 1.0f / sm);
            };
            __syncthreads();
            if (c0 == c1) {
                for (int r = dr; r < rows; r += DPT) {
                    float m, sm;
                    float val = merge_row(FEW_WARPS, [&](int s) { return mml[s * ROWS + r]; },
                                          [&](int s) { return mo[(s * ROWS + r) * OS + d]; }, m, sm);
                    val = sm == 0.0f ? 0.0f : val / sm;
                    *put(r, d, val) = __float2half_rn(val);
                    if (d == 0) put_sums(r, m, sm);
                }
            } else {
                /* the factor of every partial result first (a warp per row), then the value sums, four dims a thread and
                 * several results in flight */
                const int nS = c1 - c0 + 1, s0 = 2 * c0 + (c0 * total / grid >= base ? 0 : 1);   /* c0's slot; the others' first */
                float2 *f = reinterpret_cast<float2 *>(smem);                /* [nS][rows] */
                for (int x = tid; x < nS * rows; x += FEW_THREADS) {
                    const int s = x / rows, r = x - s * rows;
                    f[x] = __ldcg(&a.part_ml[(int64_t)(s == 0 ? s0 : 2 * (c0 + s)) * ROWS + r]);
                }
                __syncthreads();
                for (int r = w; r < rows; r += FEW_WARPS) {
                    float m = -INFINITY, sm = 0.0f;
                    for (int s = lane; s < nS; s += 32) m = fmaxf(m, f[s * rows + r].x);
#pragma unroll
                    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                    for (int s = lane; s < nS; s += 32) {
                        const float2 y = f[s * rows + r];
                        const float g = y.x == -INFINITY ? 0.0f : ex2(y.x - m);
                        sm = fmaf(y.y, g, sm);
                        f[s * rows + r].x = g;
                    }
#pragma unroll
                    for (int x = 16; x; x >>= 1) sm += __shfl_xor_sync(0xffffffffu, sm, x);
                    if (lane == 0) {
                        put_sums(r, m, sm);
                        s_inv[r] = sm == 0.0f ? 0.0f : 1.0f / sm;
                    }
                }
                __syncthreads();
                constexpr int RPP = FEW_THREADS / (HD / 4);
                const int dim = tid % (HD / 4) * 4;
                for (int r = tid / (HD / 4); r < rows; r += RPP) {
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int sb = 0; sb < nS; sb += 8) {
                        float4 x[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int s = sb + i;
                            if (s < nS)
                                x[i] = __ldcg(reinterpret_cast<const float4 *>(
                                    a.part_o + ((int64_t)(s == 0 ? s0 : 2 * (c0 + s)) * ROWS + r) * HD + dim));
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float g = sb + i < nS ? f[(sb + i) * rows + r].x : 0.0f;
                            if (g != 0.0f) {             /* not 0 times what may be infinite */
                                acc.x = fmaf(x[i].x, g, acc.x);
                                acc.y = fmaf(x[i].y, g, acc.y);
                                acc.z = fmaf(x[i].z, g, acc.z);
                                acc.w = fmaf(x[i].w, g, acc.w);
                            }
                        }
                    }
                    const float inv = s_inv[r];
                    if (inv == 0.0f) acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    acc.x *= inv;
                    acc.y *= inv;
                    acc.z *= inv;
                    acc.w *= inv;
                    __half *dst = put(r, dim, acc.x + acc.y + acc.z + acc.w);
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_half2(acc.x, acc.y), pack_half2(acc.z, acc.w));
                }
            }
            /* a value that is not finite may be 0 times another token's row: those query rows again, one by one */
            int any = 0;
            __syncthreads();
            for (int r = tid; r < rows; r += FEW_THREADS) any |= s_redo[r];
            if (__syncthreads_or(any) && result_in_doubt<KT, HD, false>(a, u)) {
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
 * each; reads 4 R + 4 bytes a row and writes 4 (8 units of 65521 rows, R = 4:
 * 8 us, a launch and two rounds of memory latency). */
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
                if (!bounds_ok(j < a.score_stride, a.status)) continue;
                const float x = __ldcs(&a.scores[((int64_t)u * R + r) * a.score_stride + j]);
                mass = fmaf(ex2(x - s_norm[r].x), s_norm[r].y, mass);
            }
        }
        const int64_t i = (int64_t)u * a.n_cells + j;
        a.mass_out[i] = a.mass_in ? fmaf(a.mass_decay, a.mass_in[i], mass) : mass;
    }
}

constexpr int MASS_THREADS = 128, MASS_KEYS = 64;

/* Scores again, now with the denominators known, for at most 16 query rows a
 * unit whose scores were too many to keep (and for no query row at all): each
 * warp holds 16 cache rows of a unit, so the weights of a cache row are summed
 * where they are made, in one order. */
template <int KT, int HD>
__global__ void __launch_bounds__(MASS_THREADS) k_mass_tiles(const AttendArgs a) {
    using S = FewStage<KT, HD>;
    constexpr int NT = 2;
    __shared__ __align__(16) uint8_t s_keys[MASS_THREADS / 32][16 * S::KS + 64];
    const int u = blockIdx.y, l = u / a.n_head_kv, h = u - l * a.n_head_kv, R = a.T * a.G;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, r8 = lane >> 2, c = lane & 3;
    const int n = attend_rows(a, u);
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride;
    const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
    const bool want_pos = a.window > 0 || a.slopes != nullptr;
    const ScoreMap map(a);
    const uint8_t *const st = s_keys[w];
    const int lead = KT == KT_Q8_0 && HD == 128 ? (int)((h * a.head_stride) & 8) : 0;
    for (int row0 = (blockIdx.x * (MASS_THREADS / 32) + w) * 16; row0 < n; row0 += gridDim.x * MASS_KEYS) {
        __syncwarp();
        few_load<KT, HD, S::KS>(a, k, lead, row0, n, smem_u32(st), lane);
        if (want_pos) few_load_pos(pos, row0, n, smem_u32(st) + 16 * S::KS, lane);
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        int pk[2] = {0, 0};
        if (want_pos) {
            pk[0] = (int)word_at(st + 16 * S::KS + 4 * r8);
            pk[1] = (int)word_at(st + 16 * S::KS + 4 * (r8 + 8));
        }
        float mass[2] = {0.0f, 0.0f};                           /* cache rows r8, r8 + 8 */
        if (R > 0) {
            uint32_t qf[NT][HD / 16][2];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int r = 8 * t + r8;
                const bool in = r < R;
                const __half *q = a.q + l * a.q_cache + (in ? (r / a.G) * a.q_tok + (h * a.G + r % a.G) * a.q_head : 0);
#pragma unroll
                for (int s = 0; s < HD / 16; s++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        qf[t][s][e] = in ? *reinterpret_cast<const uint32_t *>(q + few_qdim<KT>(s, c, e)) : 0u;
            }
            float s[NT][4];
            few_qk<KT, HD, NT>(qf, st, lead, lane, s);
            const bool all = row0 + 16 <= n - a.T && a.window <= 0 && R == 8 * NT;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = 8 * t + 2 * c + e, tk = r / a.G;
                    const bool in = r < R;
                    const float2 nm = in ? a.norm[(int64_t)u * R + r] : make_float2(0.0f, 0.0f);
                    const int tp = in && want_pos ? a.tok_pos[l * a.tok_pos_stride + tk] : 0;
                    const float slope2 = in && a.slopes ? a.slopes[h * a.G + r % a.G] * LOG2E : 0.0f;
#pragma unroll
                    for (int hi = 0; hi < 2; hi++) {
                        float x = map(s[t][e + 2 * hi]);
                        if (want_pos) x = fmaf(-slope2, (float)(tp - pk[hi]), x);
                        bool see = in;
                        if (!all) see = in && attend_sees(a, l, tk, row0 + r8 + 8 * hi, n, pk[hi], (int64_t)tp - a.window);
                        if (see) mass[hi] = fmaf(ex2(x - nm.x), nm.y, mass[hi]);
                    }
                }
        }
#pragma unroll
        for (int hi = 0; hi < 2; hi++) {
            mass[hi] += __shfl_xor_sync(0xffffffffu, mass[hi], 1);
            mass[hi] += __shfl_xor_sync(0xffffffffu, mass[hi], 2);
            const int j = row0 + r8 + 8 * hi;
            if (c == 0 && j < n) {
                const int64_t x = (int64_t)u * a.n_cells + j;
                a.mass_out[x] = a.mass_in ? fmaf(a.mass_decay, a.mass_in[x], mass[hi]) : mass[hi];
            }
        }
    }
}

}  // namespace tria
