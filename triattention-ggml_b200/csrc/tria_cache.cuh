/*
 * tria_cache.cuh - kernels that write and trim a ragged cache: tokens appended
 * behind each unit's rows, the accepted path of drafted tokens moved up, and
 * the masses of the rows an eviction kept.
 *
 * All three only move (or round) bytes, so their floor is the bytes at copy
 * bandwidth; at one token a layer they are a launch long.
 */
#pragma once

#include "tria_common.cuh"

namespace tria {

/* ------------------------------------------------------------------ */
/* Append                                                               */
/* ------------------------------------------------------------------ */

struct AppendArgs {
    uint8_t *k[TRIA_MAX_LAYERS];
    uint8_t *v[TRIA_MAX_LAYERS];
    int64_t cell_stride, head_stride;
    int32_t *pos;
    int32_t pos_shared, n_cells;
    int32_t n_head_kv, n_tok;
    int32_t first;                       /* this launch holds unit 0 of the view (shared positions) */
    const int32_t *n_rows;
    int32_t *n_rows_out;                 /* NULL when a later launch writes the counts */
    const uint8_t *src_k, *src_v;
    int64_t src_cache, src_tok, src_head;   /* bytes */
    const int32_t *tok_pos;
    int64_t tok_pos_stride;
    float *mass;
    int32_t *status;
};

constexpr int APPEND_THREADS = 256;

/* Eight consecutive source values as fp32. */
template <bool F32>
__device__ __forceinline__ void load8(const uint8_t *p, float (&x)[8]) {
    if constexpr (F32) {
        const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

/* HD / 8 lanes take one row (8 values a lane, four lanes a q8_0 block), so a
 * warp converts 256 / HD rows at a time.  A converted row is put together in
 * shared memory and leaves as 4-byte words in order: a q8_0 row is 2-byte
 * data at a 4-byte alignment, and storing each lane's bytes directly would
 * send every 32-byte sector four times.  blockIdx.x is the unit, so the heads
 * of a cell, whose rows share sectors, are written side by side in time.
 * Bound by DRAM: 512 fp32 tokens of 36 layers of 8 heads to q8_0, 192 MB, take
 * 40 us from a warm L2 and 57 us from a cold one, against 29 us at copy rate. */
template <int KT, int HD, bool F32>
__global__ void __launch_bounds__(APPEND_THREADS) k_append(const AppendArgs a) {
    constexpr int LPR = HD / 8, RPW = 32 / LPR;
    constexpr int RB = KT == KT_F16 ? 2 * HD : HD / 32 * 34, WORDS = RB / 4;
    __shared__ __align__(16) uint8_t s_row[APPEND_THREADS / 32][RPW][RB];
    const int u = blockIdx.x, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = lane % LPR, sub = lane / LPR;
    const int n = a.n_rows[u];
    const bool fits = n >= 0 && n <= a.n_cells && a.n_tok <= a.n_cells - n;
    if (!fits) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.status, ST_ROWS);
    } else {
        const int wg = blockIdx.y * (APPEND_THREADS / 32) + w, nw = gridDim.y * (APPEND_THREADS / 32);
        const uint8_t *sk = a.src_k + l * a.src_cache + h * a.src_head;
        const uint8_t *sv = a.src_v + l * a.src_cache + h * a.src_head;
        uint8_t *dk = a.k[l] + (int64_t)h * a.head_stride, *dv = a.v[l] + (int64_t)h * a.head_stride;
        for (int t0 = wg * RPW; t0 < a.n_tok; t0 += nw * RPW) {
            const int t = t0 + sub;
            const bool live = t < a.n_tok;
            float x[2][8];
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[kv][i] = 0.0f;
                if (live) load8<F32>((kv ? sv : sk) + (int64_t)t * a.src_tok + c * (F32 ? 32 : 16), x[kv]);
            }
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                if constexpr (KT == KT_F16) {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const __half2 p = __floats2half2_rn(x[kv][2 * i], x[kv][2 * i + 1]);
                        o[i] = *reinterpret_cast<const uint32_t *>(&p);
                    }
                    *reinterpret_cast<uint4 *>(&s_row[w][sub][16 * c]) = make_uint4(o[0], o[1], o[2], o[3]);
                } else {
                    float m = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[kv][i]));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    const float d = __fmul_rn(m, 1.0f / 127.0f);
                    const float inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
                    uint8_t *blk = &s_row[w][sub][(c >> 2) * 34];
                    if ((c & 3) == 0) *reinterpret_cast<__half *>(blk) = __float2half_rn(d);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int q0 = __float2int_rn(fminf(fmaxf(__fmul_rn(x[kv][2 * i], inv), -127.0f), 127.0f));
                        const int q1 = __float2int_rn(fminf(fmaxf(__fmul_rn(x[kv][2 * i + 1], inv), -127.0f), 127.0f));
                        *reinterpret_cast<uint16_t *>(blk + 2 + (c & 3) * 8 + 2 * i) =
                            (uint16_t)((q0 & 0xff) | ((q1 & 0xff) << 8));
                    }
                }
                __syncwarp();
                for (int i = lane; i < RPW * WORDS; i += 32) {
                    const int rr = i / WORDS, ww = i - rr * WORDS;
                    if (t0 + rr < a.n_tok && bounds_ok(n + t0 + rr < a.n_cells, a.status))
                        *reinterpret_cast<uint32_t *>((kv ? dv : dk) + (int64_t)(n + t0 + rr) * a.cell_stride + 4 * ww) =
                            *reinterpret_cast<const uint32_t *>(&s_row[w][rr][4 * ww]);
                }
                __syncwarp();
            }
        }
        const int tid = blockIdx.y * APPEND_THREADS + threadIdx.x, nt = gridDim.y * APPEND_THREADS;
        const int64_t row0 = (int64_t)u * a.n_cells + n;
        for (int t = tid; t < a.n_tok; t += nt) {
            if (!bounds_ok(n + t < a.n_cells, a.status)) continue;
            const int32_t p = a.tok_pos[l * a.tok_pos_stride + t];
            if (!a.pos_shared) a.pos[row0 + t] = p;
            else if (a.first && u == 0) a.pos[n + t] = p;
            if (a.mass) a.mass[row0 + t] = 0.0f;
        }
    }
    /* the host gives n_rows_out only where this block is the unit's one reader
     * of n_rows, or the two are different arrays */
    if (a.n_rows_out && blockIdx.y == 0) {
        __syncthreads();
        if (threadIdx.x == 0) a.n_rows_out[u] = fits ? n + a.n_tok : n;
    }
}

/* Counts after an append whose units were shared by several blocks. */
__global__ void k_append_counts(const int32_t *n_rows, int32_t *out, int32_t units, int32_t n_tok, int32_t n_cells) {
    const int u = blockIdx.x * blockDim.x + threadIdx.x;
    if (u >= units) return;
    const int n = n_rows[u];
    out[u] = n >= 0 && n <= n_cells && n_tok <= n_cells - n ? n + n_tok : n;
}

/* ------------------------------------------------------------------ */
/* Accept                                                               */
/* ------------------------------------------------------------------ */

struct AcceptArgs {
    uint8_t *k[TRIA_MAX_LAYERS];
    uint8_t *v[TRIA_MAX_LAYERS];
    int64_t cell_stride, head_stride;
    int32_t *pos;
    int32_t pos_shared, n_cells;
    int32_t n_head_kv, row_words, n_tok;
    int32_t first;
    const int32_t *n_rows;
    int32_t *n_rows_out;
    const int32_t *path, *n_path;
    int64_t path_stride;
    float *mass;
    int32_t *status;
};

constexpr int ACCEPT_THREADS = 160;     /* 64 words of K, 64 of V, a position and a mass */

/* One block per unit; a thread owns one 4-byte column (of K, V, the positions
 * or the masses) and walks the path in order.  A destination i is never above
 * its source path[i], and both ascend, so the sources still to come lie above
 * every destination written: four loads go out before their four stores.
 * 288 units, 3 rows each: 2.7 us, a launch and two rounds of memory latency. */
__global__ void __launch_bounds__(ACCEPT_THREADS) k_accept(const AcceptArgs a) {
    const int u = blockIdx.x, l = u / a.n_head_kv, h = u - l * a.n_head_kv;
    const int n = a.n_rows[u], li = a.path_stride ? l : 0;
    const int m = a.n_path[li];
    const int32_t *path = a.path + (int64_t)li * a.path_stride;
    const bool fits = n >= a.n_tok && n <= a.n_cells && m >= 0 && m <= a.n_tok;
    int ok = fits;
    for (int i = threadIdx.x; fits && i < m; i += ACCEPT_THREADS) {
        const int p = path[i];
        ok &= p >= 0 && p < a.n_tok && (i == 0 || p > path[i - 1]);
    }
    ok = __syncthreads_and(ok);
    if (threadIdx.x == 0) {
        if (!ok) atomicOr(a.status, ST_ROWS);
        a.n_rows_out[u] = ok ? n - a.n_tok + m : n;
    }
    if (!ok) return;
    const int base = n - a.n_tok, W = a.row_words;
    for (int col = threadIdx.x; col < 2 * W + 2; col += ACCEPT_THREADS) {
        uint8_t *p;
        int64_t stride;
        if (col < 2 * W) {
            p = (col < W ? a.k[l] : a.v[l]) + (int64_t)h * a.head_stride + 4 * (col < W ? col : col - W);
            stride = a.cell_stride;
        } else if (col == 2 * W) {
            if (a.pos_shared && !(a.first && u == 0)) continue;
            p = reinterpret_cast<uint8_t *>(a.pos + (a.pos_shared ? 0 : (int64_t)u * a.n_cells));
            stride = 4;
        } else {
            if (!a.mass) continue;
            p = reinterpret_cast<uint8_t *>(a.mass + (int64_t)u * a.n_cells);
            stride = 4;
        }
        p += base * stride;
        for (int i = 0; i < m; i += 4) {
            uint32_t x[4];
            int from[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                from[q] = i + q < m ? path[i + q] : i + q;
                if (!bounds_ok(i + q >= m || (from[q] >= i + q && base + from[q] < a.n_cells), a.status)) from[q] = i + q;
                if (from[q] != i + q) x[q] = *reinterpret_cast<const uint32_t *>(p + from[q] * stride);
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (from[q] != i + q) *reinterpret_cast<uint32_t *>(p + (i + q) * stride) = x[q];
        }
    }
}

/* ------------------------------------------------------------------ */
/* Masses of the kept rows                                              */
/* ------------------------------------------------------------------ */

/* mass_dst[u][j] = mass[u][kept[u][j]], j < n_kept[u]: blockIdx.y a unit,
 * grid-stride over its kept rows. */
__global__ void __launch_bounds__(256) k_carry_mass(const float *mass, int64_t src_cells, float *out, int64_t dst_cells,
                                                    const int32_t *kept_idx, int64_t kept_stride,
                                                    const int32_t *n_kept, int32_t *status) {
    const int64_t u = blockIdx.y;
    int nk = n_kept[u];
    if (!bounds_ok(nk >= 0 && nk <= dst_cells && nk <= kept_stride, threadIdx.x == 0 ? status : nullptr)) nk = 0;
    for (int j = blockIdx.x * 256 + threadIdx.x; j < nk; j += gridDim.x * 256) {
        const int r = kept_idx[u * kept_stride + j];
        if (bounds_ok(r >= j && r < src_cells, status)) out[u * dst_cells + j] = mass[u * src_cells + r];
    }
}

}  // namespace tria
