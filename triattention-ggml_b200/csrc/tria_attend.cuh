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

/* c tanh(s / c) = c (1 - 2 / (1 + exp(2 s / c))): right to a few fp32 ulps of
 * c, and exactly +-c where the exponential over- or underflows. */
__device__ __forceinline__ float soft_cap(float s, float c, float inv_c) {
    return c * (1.0f - 2.0f / (1.0f + __expf(2.0f * s * inv_c)));
}

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

/* The score of (t, head h * G + g) against row j, in fp32 throughout. */
template <int KT, int HD>
__device__ __forceinline__ float attend_score(const AttendArgs &a, const uint8_t *krow, const float *q, float slope,
                                              int tok_pos, int pos) {
    float s = 0.0f;
    for (int d = 0; d < HD; d++) s = fmaf(q[d], row_value<KT>(krow, d), s);
    s *= a.scale;
    if (a.softcap > 0.0f) s = soft_cap(s, a.softcap, 1.0f / a.softcap);
    if (a.slopes) s -= slope * (float)(tok_pos - pos);
    return s;
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

/* One query row by one block of ROW_THREADS threads, from the definition: a
 * thread scores a row of the cache, then owns an output element.  Rows that
 * the token does not see are never multiplied, so what they hold is without
 * effect. */
template <int KT, int HD>
__device__ void attend_row(const AttendArgs &a, int u, int g, int t, RowShared<HD> &sm) {
    const int l = u / a.n_head_kv, h = u - l * a.n_head_kv, tid = threadIdx.x;
    const int n = attend_rows(a, u), head = h * a.G + g;
    const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
    const int tp = a.tok_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
    const int64_t lo = (int64_t)tp - a.window;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
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
        if (see) s = attend_score<KT, HD>(a, k + (int64_t)j * a.cell_stride, sm.q, slope, tp, pj);
        if (!__syncthreads_or(see)) continue;
        any = true;
        const float mt = fmaxf(m, block_max_128(s, sm.red));
        const float r = mt == m ? 1.0f : __expf(m - mt);
        sm.p[tid] = see ? __expf(s - (mt == -INFINITY ? 0.0f : mt)) : 0.0f;
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
        a.lse[((int64_t)l * a.T + t) * a.n_head_kv * a.G + head] = any && sum != 0.0f ? m + logf(sum) : -INFINITY;
}

template <int KT, int HD>
__global__ void __launch_bounds__(ROW_THREADS) k_attend_rows(const AttendArgs a) {
    __shared__ RowShared<HD> sm;
    const int64_t r = blockIdx.x;
    const int t = (int)(r % a.T), ug = (int)(r / a.T);
    attend_row<KT, HD>(a, ug / a.G, ug % a.G, t, sm);
}

/* Masses from the scores once the denominators are known: a thread per row of
 * a unit, all its tokens and heads in turn. */
template <int KT, int HD>
__global__ void __launch_bounds__(128) k_mass_rows(const AttendArgs a) {
    const int u = blockIdx.y, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
    const int n = attend_rows(a, u), H = a.n_head_kv * a.G;
    __shared__ float q[HD];
    const int32_t *pos = a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells);
    const uint8_t *k = a.k[l] + (int64_t)h * a.head_stride;
    for (int j0 = blockIdx.x * 128; j0 < n; j0 += gridDim.x * 128) {
        const int j = j0 + threadIdx.x;
        const int pj = j < n ? pos[j] : 0;
        float mass = 0.0f;
        for (int r = 0; r < a.T * a.G; r++) {
            const int t = r / a.G, head = h * a.G + r % a.G;
            const __half *qr = a.q + l * a.q_cache + t * a.q_tok + head * a.q_head;
            __syncthreads();
            for (int d = threadIdx.x; d < HD; d += 128) q[d] = __half2float(qr[d]);
            __syncthreads();
            const int tp = a.tok_pos ? a.tok_pos[l * a.tok_pos_stride + t] : 0;
            const float lse = a.lse[((int64_t)l * a.T + t) * H + head];
            if (lse != -INFINITY && attend_sees(a, l, t, j, n, pj, (int64_t)tp - a.window))
                mass += __expf(attend_score<KT, HD>(a, k + (int64_t)j * a.cell_stride, q, a.slopes ? a.slopes[head] : 0.0f,
                                                    tp, pj) - lse);
        }
        if (j < n) {
            const int64_t i = (int64_t)u * a.n_cells + j;
            a.mass_out[i] = a.mass_in ? fmaf(a.mass_decay, a.mass_in[i], mass) : mass;
        }
    }
}

}  // namespace tria
