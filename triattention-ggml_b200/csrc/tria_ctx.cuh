/*
 * tria_ctx.cuh - the context behind the C ABI and the host helpers that its
 * translation units share.
 */
#pragma once

#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <cstdint>
#include <mutex>
#include <vector>

#include "tria_common.cuh"

/* The step's completion event.  Inside a stream capture a plain record only
 * orders work within the capture; recorded as an external event node it is
 * recorded again at every replay of the graph, so tria_get_n_kv waits for the
 * replayed step. */
static inline cudaError_t record_done(cudaEvent_t ev, cudaStream_t st) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(st, &cs);
    if (e != cudaSuccess) return e;
    return cs == cudaStreamCaptureStatusActive ? cudaEventRecordWithFlags(ev, st, cudaEventRecordExternal)
                                               : cudaEventRecord(ev, st);
}

/* NVTX ranges on the host timeline (a profiler shows them beside the
 * kernels; ncu --nvtx filters launches by them): a call, and the stages of an
 * eviction step.  With no tool attached a push or pop is a branch. */
struct NvtxRange {
    explicit NvtxRange(const char *name) { nvtxRangePushA(name); }
    ~NvtxRange() { nvtxRangePop(); }
    NvtxRange(const NvtxRange &) = delete;
    NvtxRange &operator=(const NvtxRange &) = delete;
};
struct NvtxStages {
    bool open = false;
    void next(const char *name) {
        close();
        nvtxRangePushA(name);
        open = true;
    }
    void close() {
        if (open) nvtxRangePop();
        open = false;
    }
    ~NvtxStages() { close(); }
};

#define FAIL(code, ...) do { tria_set_error(__VA_ARGS__); return (code); } while (0)
#define CUDA_TRY(call) do { cudaError_t e_ = (call); if (e_ != cudaSuccess) \
    FAIL(e_ == cudaErrorMemoryAllocation ? TRIA_ERR_NOMEM : TRIA_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); } while (0)

/* Restores the caller's current device on scope exit. */
struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

struct tria_ctx {
    int device = 0;
    uint32_t L = 0, H = 0, KV = 0, hd = 0, fc = 0, G = 0;
    std::vector<float> scales;           /* layer budget scales (host) */
    float attn_scale = 1.0f;             /* rope attention scaling of the stats (post-RoPE keys) */
    /* position table for post-RoPE views: rows p in [0, ptab_cur] of trigger ptab_cur */
    float2 *d_ptab = nullptr;
    int64_t ptab_cap = 0, ptab_cur = -1;
    int64_t ptab_t_lo = 0, ptab_t_len = 0;
    float *d_q = nullptr;                /* [L][H][3][fc] */
    float *d_omega = nullptr;            /* [fc] */
    /* delta table: entries for d in [t_lo, t_lo + t_len), capacity t_cap rows */
    float2 *d_table = nullptr;
    int64_t t_lo = 0, t_len = 0, t_cap = 0;
    /* scratch */
    uint8_t *d_scratch = nullptr;
    size_t scratch_cap = 0;
    float *raw = nullptr;
    float2 *ms = nullptr;
    uint32_t *keys = nullptr;
    int32_t *kept = nullptr;
    int32_t *cnt = nullptr;
    int64_t raw_stride = 0, cell_stride = 0;
    int sm_count = 148;
    /* host-API staging */
    uint8_t *d_io = nullptr;
    size_t io_cap = 0;
    cudaStream_t own_stream = nullptr;
    /* status / counts read-back */
    int32_t *d_status = nullptr;         /* [0] ST_* bits the kernels set, cleared when read back; [1] units of the last step */
    long long wait_limit = tria::WAIT_LIMIT_DEFAULT;   /* bound of the scoring kernel's pipeline waits */
    int select_split = 0;                        /* CTAs per unit in selection: 0 automatic, 1 one block */
    /* [0] status, [1] units, [2..] counts: room for every unit of the stats, so that it never moves (captured steps
     * write it), and its unit count from the device, so that a replayed step brings its own */
    int32_t *h_pinned = nullptr;
    cudaEvent_t ev_done = nullptr;
    bool have_step = false;
    /* stage timing (tria_ctx_set_timing) */
    bool timing = false, have_timing = false;
    cudaEvent_t ev_stage[6] = {};
    int64_t launches = 0;
    std::mutex mu;
    /* tria_evict_host: double-buffered device staging of K (and positions) */
    cudaStream_t copy_stream = nullptr;
    uint8_t *hs_k[2] = {nullptr, nullptr};
    int32_t *hs_pos[2] = {nullptr, nullptr};
    size_t hs_k_cap = 0, hs_pos_cap = 0;
    cudaEvent_t hs_copied[2] = {nullptr, nullptr}, hs_freed[2] = {nullptr, nullptr};
    bool hs_used[2] = {false, false};
    int32_t *d_cnt_all = nullptr;
    int64_t cnt_all_cap = 0;
    /* tria_attend's workspace.  Once a call was captured, graphs may hold the
     * scratch of this context: blocks that are outgrown afterwards are kept
     * in `outgrown` until the context goes. */
    uint8_t *d_attend = nullptr;
    size_t attend_cap = 0;
    bool captured = false;
    std::vector<void *> outgrown;
};

/* Whether `st` is being captured (noted in the context), 0 or 1; negative on error. */
int note_capture(tria_ctx *c, cudaStream_t st);
/* Frees a scratch block, or keeps it if a graph may hold it. */
void drop_scratch(tria_ctx *c, void *p);

static inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

cudaError_t raise_smem_limit(const void *fn, int bytes);
int ensure_scratch(tria_ctx *c, int64_t units, int64_t cells, cudaStream_t st);
int64_t view_row_bytes(int type, int hd);
int validate_view(const tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows, const char *what, bool need_v);
int check_pair(const tria_kv_view *s, const tria_kv_view *d);
void keep_requests(const tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows, const tria_evict_params *p,
                   std::vector<int32_t> &keep);
int launch_select(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows, const std::vector<int32_t> &keep,
                  const tria_evict_params *p, bool fused, const float *scores, int32_t *kept_idx,
                  int64_t kept_stride, int32_t *n_kept, cudaStream_t st, int64_t step_units = 0);
/* Queues the read-back of a step's status, unit count (launch_select's step_units) and kept counts, and records its end. */
int read_back_step(tria_ctx *c, const int32_t *cnt, int64_t units, cudaStream_t st);
int launch_compact(tria_ctx *c, const tria_kv_view *s, const tria_kv_view *d, const int32_t *n_rows,
                   const int32_t *kept_idx, int64_t kept_stride, const int32_t *n_kept, cudaStream_t st,
                   int rows_hint = -1);
