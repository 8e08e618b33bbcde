/*
 * tria_serve.cu - host side of the calls that write, read and evict a ragged
 * cache by attention: tria_append, tria_attend, tria_accept, tria_evict_mass.
 */
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "tria_attend.cuh"
#include "tria_attend_tile.cuh"
#include "tria_cache.cuh"
#include "tria_ctx.cuh"

using namespace tria;

/* The host side may allocate: what it throws stops at the C boundary. */
template <class F>
static int no_throw(const char *what, F &&f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        FAIL(TRIA_ERR_NOMEM, "%s: host allocation failed", what);
    } catch (...) {
        FAIL(TRIA_ERR_CUDA, "%s: unexpected exception", what);
    }
}

/* A view whose rows attention reads or the serving calls write: any number of
 * caches (no stats are read), post-RoPE keys, K and V. */
static int validate_cache(const tria_kv_view *v, const char *what) {
    if (!v) FAIL(TRIA_ERR_INVALID, "%s: null view", what);
    if (v->type != TRIA_TYPE_F16 && v->type != TRIA_TYPE_Q8_0)
        FAIL(TRIA_ERR_UNSUPPORTED, "%s: cache type %d unsupported", what, v->type);
    if (v->n_layer < 1 || v->n_head_kv < 1 || v->n_head_kv > TRIA_MAX_UNITS)
        FAIL(TRIA_ERR_INVALID, "%s: %d caches of %d kv heads", what, v->n_layer, v->n_head_kv);
    if ((int64_t)v->n_layer * v->n_head_kv > INT32_MAX)
        FAIL(TRIA_ERR_INVALID, "%s: more than 2^31 units", what);
    if (v->n_cells < 0) FAIL(TRIA_ERR_INVALID, "%s: negative n_cells", what);
    if (v->flags & ~TRIA_VIEW_POST_ROPE) FAIL(TRIA_ERR_INVALID, "%s: unknown view flags 0x%x", what, v->flags);
    if (!(v->flags & TRIA_VIEW_POST_ROPE))
        FAIL(TRIA_ERR_UNSUPPORTED, "%s: the cache must hold keys as attention reads them (TRIA_VIEW_POST_ROPE)", what);
    if (!v->k || !v->v || !v->pos) FAIL(TRIA_ERR_INVALID, "%s: null k, v or pos", what);
    if ((v->cell_stride & 3) || (v->head_stride & 3) || v->cell_stride <= 0 || v->head_stride < 0)
        FAIL(TRIA_ERR_INVALID, "%s: strides must be positive multiples of 4", what);
    if ((uintptr_t)v->pos & 3) FAIL(TRIA_ERR_INVALID, "%s: pos misaligned", what);
    for (int l = 0; l < v->n_layer; l++)
        if (!v->k[l] || ((uintptr_t)v->k[l] & 15) || !v->v[l] || ((uintptr_t)v->v[l] & 15))
            FAIL(TRIA_ERR_INVALID, "%s: k[%d] or v[%d] null or not 16-byte aligned", what, l, l);
    return TRIA_OK;
}

/* Whether rows of `rb` bytes of one cache of a view share bytes.  Heads may lie
 * within cells, cells within heads, or neither: for each distance of heads the
 * two cells around it are the ones that come near enough. */
static bool rows_overlap(const tria_kv_view *v, int64_t rb) {
    using wide = __int128;               /* strides are the caller's: nothing here may overflow */
    if (v->cell_stride >= rb && v->head_stride >= rb &&
        (v->cell_stride >= (wide)(v->n_head_kv - 1) * v->head_stride + rb || v->head_stride >= (wide)(v->n_cells - 1) * v->cell_stride + rb))
        return false;                    /* one within the other */
    if (v->n_cells > 1 && v->cell_stride < rb) return true;
    for (int dh = 1; v->n_cells > 0 && dh < v->n_head_kv; dh++) {
        const wide off = (wide)dh * v->head_stride;
        const wide at = std::min<wide>(off / v->cell_stride, v->n_cells - 1);
        const wide rest = off - at * v->cell_stride;         /* to the cell before, >= 0 */
        if (rest < rb) return true;
        if (at + 1 < v->n_cells && v->cell_stride - rest < rb) return true;
    }
    return false;
}

/* What a call writes to: no row twice (without a context, rows of the smallest head_dim). */
static int check_written(const tria_kv_view *v, const char *what, const tria_ctx *c) {
    if (rows_overlap(v, view_row_bytes(v->type, c ? (int)c->hd : 64)))
        FAIL(TRIA_ERR_INVALID, "%s: the view's strides let rows of %d kv heads overlap", what, v->n_head_kv);
    return TRIA_OK;
}

/* Caches of a view that is written: each k and v is memory of its own. */
static int check_apart(const tria_kv_view *v, const char *what) {
    const int L = v->n_layer;
    auto addr = [](const void *p) { return (uintptr_t)p; };
    /* K and V each by rising address, one behind the other: nothing to sort */
    bool rising = !v->v || addr(v->k[L - 1]) < addr(v->v[0]) || addr(v->v[L - 1]) < addr(v->k[0]);
    for (int l = 1; rising && l < L; l++)
        rising = addr(v->k[l - 1]) < addr(v->k[l]) && (!v->v || addr(v->v[l - 1]) < addr(v->v[l]));
    if (rising) return TRIA_OK;
    std::vector<uintptr_t> at;
    at.reserve(2 * (size_t)L);
    for (int l = 0; l < L; l++) {
        at.push_back(addr(v->k[l]));
        if (v->v) at.push_back(addr(v->v[l]));
    }
    std::sort(at.begin(), at.end());
    if (std::adjacent_find(at.begin(), at.end()) != at.end())
        FAIL(TRIA_ERR_INVALID, "%s: the view lists one cache twice", what);
    return TRIA_OK;
}

/* The context's part of the checks, after all that needs none. */
static int check_ctx(const tria_ctx *c, const char *what) {
    if (!c) FAIL(TRIA_ERR_INVALID, "%s: null context", what);
    if (c->hd != 64 && c->hd != 128)
        FAIL(TRIA_ERR_UNSUPPORTED, "%s: head_dim %u unsupported (64 or 128)", what, c->hd);
    return TRIA_OK;
}

static int check_ints(const char *what, const char *name, const void *p) {
    if (!p || ((uintptr_t)p & 3)) FAIL(TRIA_ERR_INVALID, "%s: %s null or misaligned", what, name);
    return TRIA_OK;
}

/* Whether arrays of na and nb four-byte entries share some. */
static bool arrays_meet(const void *a, int64_t na, const void *b, int64_t nb) {
    const __int128 d = (__int128)(uintptr_t)b - (__int128)(uintptr_t)a;
    return d < (__int128)na * 4 && -d < (__int128)nb * 4;
}
static int64_t view_cells(const tria_kv_view *v) { return (int64_t)v->n_layer * v->n_head_kv * std::max(v->n_cells, 0); }

/* Whether the counts are updated in place; arrays that overlap in part are refused. */
static int counts_alias(const char *what, const int32_t *in, const int32_t *out, int64_t units, bool *alias) {
    *alias = arrays_meet(in, units, out, units);
    if (*alias && in != out) FAIL(TRIA_ERR_INVALID, "%s: n_rows and n_rows_out overlap in part", what);
    return TRIA_OK;
}

/* Launches of at most TRIA_MAX_LAYERS caches and TRIA_MAX_UNITS units. */
template <class F>
static int for_cache_chunks(const tria_kv_view *v, F &&fn) {
    const int per = std::max(1, std::min(TRIA_MAX_LAYERS, TRIA_MAX_UNITS / v->n_head_kv));
    for (int l0 = 0; l0 < v->n_layer; l0 += per) {
        const int rc = fn(l0, std::min(per, v->n_layer - l0));
        if (rc) return rc;
    }
    return TRIA_OK;
}

/* ------------------------------------------------------------------ */
/* Append                                                               */
/* ------------------------------------------------------------------ */

template <int KT, int HD>
static void launch_append(const AppendArgs &a, bool f32, dim3 grid, cudaStream_t st) {
    if (f32) k_append<KT, HD, true><<<grid, APPEND_THREADS, 0, st>>>(a);
    else k_append<KT, HD, false><<<grid, APPEND_THREADS, 0, st>>>(a);
}

static int do_append(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows,
                     const tria_append_params *p, const void *k, const void *vv, float *mass,
                     int32_t *n_rows_out, void *stream) {
    NvtxRange range("tria_append");
    const char *fn = "tria_append";
    if (!p) FAIL(TRIA_ERR_INVALID, "%s: null parameters", fn);
    int rc = validate_cache(v, fn);
    if (!rc) rc = check_ints(fn, "n_rows", n_rows);
    if (!rc) rc = check_ints(fn, "n_rows_out", n_rows_out);
    if (rc) return rc;
    if (p->n_tok < 0) FAIL(TRIA_ERR_INVALID, "%s: n_tok %d < 0", fn, p->n_tok);
    if (p->src_type != TRIA_SRC_F16 && p->src_type != TRIA_SRC_F32)
        FAIL(TRIA_ERR_UNSUPPORTED, "%s: source type %d unsupported", fn, p->src_type);
    if (p->tok_pos_stride < 0) FAIL(TRIA_ERR_INVALID, "%s: negative tok_pos_stride", fn);
    if (v->pos_shared && p->tok_pos_stride) FAIL(TRIA_ERR_INVALID, "%s: shared positions take one tok_pos for all caches", fn);
    const bool f32 = p->src_type == TRIA_SRC_F32;
    const int esz = f32 ? 4 : 2, unit16 = 16 / esz;
    if (p->n_tok > 0) {
        if ((rc = check_ints(fn, "tok_pos", p->tok_pos))) return rc;
        if (!k || !vv || ((uintptr_t)k & 15) || ((uintptr_t)vv & 15))
            FAIL(TRIA_ERR_INVALID, "%s: k or v null or not 16-byte aligned", fn);
        if (p->cache_stride % unit16 || p->tok_stride % unit16 || p->head_stride % unit16)
            FAIL(TRIA_ERR_INVALID, "%s: source strides must be multiples of 16 bytes", fn);
        if (mass && ((uintptr_t)mass & 3)) FAIL(TRIA_ERR_INVALID, "%s: mass misaligned", fn);
    }
    /* a unit's count may be overwritten only once all its blocks have read it */
    const int units_all = v->n_layer * v->n_head_kv;
    bool alias = false;
    if ((rc = counts_alias(fn, n_rows, n_rows_out, units_all, &alias))) return rc;
    if ((rc = check_written(v, fn, c)) || (rc = check_ctx(c, fn)) || (rc = check_apart(v, fn))) return rc;
    DeviceGuard g(c->device);
    cudaStream_t st = (cudaStream_t)stream;
    if ((rc = note_capture(c, st)) < 0) return rc;
    /* enough blocks per unit to fill the GPU; one when the rows are few */
    const int rows_per_block = APPEND_THREADS / 32 * (256 / (int)c->hd);
    const int want = std::max(1, 16 * c->sm_count / std::max(1, std::min(units_all, TRIA_MAX_UNITS)));
    const int bx = std::max(1, std::min((p->n_tok + rows_per_block - 1) / rows_per_block, want));
    const bool later = alias && bx > 1;
    rc = for_cache_chunks(v, [&](int l0, int nl) -> int {
        AppendArgs a;
        memset(&a, 0, sizeof a);
        const int64_t u0 = (int64_t)l0 * v->n_head_kv;
        for (int l = 0; l < nl; l++) { a.k[l] = (uint8_t *)v->k[l0 + l]; a.v[l] = (uint8_t *)v->v[l0 + l]; }
        a.cell_stride = v->cell_stride;
        a.head_stride = v->head_stride;
        a.pos = v->pos_shared ? v->pos : v->pos + u0 * v->n_cells;
        a.pos_shared = v->pos_shared ? 1 : 0;
        a.n_cells = v->n_cells;
        a.n_head_kv = v->n_head_kv;
        a.n_tok = p->n_tok;
        a.first = l0 == 0;
        a.n_rows = n_rows + u0;
        a.n_rows_out = later ? nullptr : n_rows_out + u0;
        a.src_cache = p->cache_stride * esz;
        a.src_tok = p->tok_stride * esz;
        a.src_head = p->head_stride * esz;
        a.src_k = (const uint8_t *)k + l0 * a.src_cache;
        a.src_v = (const uint8_t *)vv + l0 * a.src_cache;
        a.tok_pos = p->tok_pos + l0 * p->tok_pos_stride;
        a.tok_pos_stride = p->tok_pos_stride;
        a.mass = mass ? mass + u0 * v->n_cells : nullptr;
        a.status = c->d_status;
        const dim3 grid((unsigned)(nl * v->n_head_kv), (unsigned)bx);
        if (v->type == TRIA_TYPE_F16) {
            if (c->hd == 128) launch_append<KT_F16, 128>(a, f32, grid, st);
            else launch_append<KT_F16, 64>(a, f32, grid, st);
        } else {
            if (c->hd == 128) launch_append<KT_Q8_0, 128>(a, f32, grid, st);
            else launch_append<KT_Q8_0, 64>(a, f32, grid, st);
        }
        CUDA_TRY(cudaGetLastError());
        c->launches++;
        return TRIA_OK;
    });
    if (rc) return rc;
    if (later) {
        k_append_counts<<<(units_all + 255) / 256, 256, 0, st>>>(n_rows, n_rows_out, units_all, p->n_tok, v->n_cells);
        CUDA_TRY(cudaGetLastError());
        c->launches++;
    }
    return TRIA_OK;
}

/* ------------------------------------------------------------------ */
/* Accept                                                               */
/* ------------------------------------------------------------------ */

static int do_accept(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows, int32_t n_tok,
                     const int32_t *path, int64_t path_stride, const int32_t *n_path, float *mass,
                     int32_t *n_rows_out, void *stream) {
    NvtxRange range("tria_accept");
    const char *fn = "tria_accept";
    int rc = validate_cache(v, fn);
    if (!rc) rc = check_ints(fn, "n_rows", n_rows);
    if (!rc) rc = check_ints(fn, "n_rows_out", n_rows_out);
    if (!rc) rc = check_ints(fn, "path", path);
    if (!rc) rc = check_ints(fn, "n_path", n_path);
    if (rc) return rc;
    if (n_tok < 0 || path_stride < 0) FAIL(TRIA_ERR_INVALID, "%s: negative n_tok or path_stride", fn);
    if (v->pos_shared && path_stride) FAIL(TRIA_ERR_INVALID, "%s: shared positions take one path for all caches", fn);
    if (mass && ((uintptr_t)mass & 3)) FAIL(TRIA_ERR_INVALID, "%s: mass misaligned", fn);
    bool alias = false;
    if ((rc = counts_alias(fn, n_rows, n_rows_out, (int64_t)v->n_layer * v->n_head_kv, &alias))) return rc;
    if ((rc = check_written(v, fn, c)) || (rc = check_ctx(c, fn)) || (rc = check_apart(v, fn))) return rc;
    DeviceGuard g(c->device);
    cudaStream_t st = (cudaStream_t)stream;
    if ((rc = note_capture(c, st)) < 0) return rc;
    return for_cache_chunks(v, [&](int l0, int nl) -> int {
        AcceptArgs a;
        memset(&a, 0, sizeof a);
        const int64_t u0 = (int64_t)l0 * v->n_head_kv;
        for (int l = 0; l < nl; l++) { a.k[l] = (uint8_t *)v->k[l0 + l]; a.v[l] = (uint8_t *)v->v[l0 + l]; }
        a.cell_stride = v->cell_stride;
        a.head_stride = v->head_stride;
        a.pos = v->pos_shared ? v->pos : v->pos + u0 * v->n_cells;
        a.pos_shared = v->pos_shared ? 1 : 0;
        a.n_cells = v->n_cells;
        a.n_head_kv = v->n_head_kv;
        a.row_words = (int32_t)(view_row_bytes(v->type, (int)c->hd) / 4);
        a.n_tok = n_tok;
        a.first = l0 == 0;
        a.n_rows = n_rows + u0;
        a.n_rows_out = n_rows_out + u0;
        a.path = path + l0 * path_stride;
        a.n_path = n_path + (path_stride ? l0 : 0);
        a.path_stride = path_stride;
        a.mass = mass ? mass + u0 * v->n_cells : nullptr;
        a.status = c->d_status;
        k_accept<<<nl * v->n_head_kv, ACCEPT_THREADS, 0, st>>>(a);
        CUDA_TRY(cudaGetLastError());
        c->launches++;
        return TRIA_OK;
    });
}

/* ------------------------------------------------------------------ */
/* Eviction by mass                                                     */
/* ------------------------------------------------------------------ */

static int do_evict_mass(tria_ctx *c, const tria_kv_view *s, const tria_kv_view *d,
                         const int32_t *n_rows, const float *mass, float *mass_dst,
                         const tria_evict_params *p, int32_t *n_kept_out, void *stream) {
    NvtxRange range("tria_evict_mass");
    const char *fn = "tria_evict_mass";
    if (!n_rows || !p || !mass) FAIL(TRIA_ERR_INVALID, "%s: null argument", fn);
    if (p->cur_pos < 0) FAIL(TRIA_ERR_INVALID, "%s: cur_pos %d < 0", fn, p->cur_pos);
    if (((uintptr_t)mass & 3) || ((uintptr_t)mass_dst & 3)) FAIL(TRIA_ERR_INVALID, "%s: mass misaligned", fn);
    if (mass == mass_dst) FAIL(TRIA_ERR_INVALID, "%s: mass and mass_dst must be different arrays", fn);
    if (s && d && mass_dst && arrays_meet(mass, view_cells(s), mass_dst, view_cells(d)))
        FAIL(TRIA_ERR_INVALID, "%s: mass and mass_dst overlap", fn);
    if (!c) FAIL(TRIA_ERR_INVALID, "%s: null context", fn);
    int rc = validate_view(c, s, n_rows, "tria_evict_mass src", false);
    if (!rc) rc = validate_view(c, d, nullptr, "tria_evict_mass dst", false);
    if (!rc) rc = check_pair(s, d);
    if (!rc) rc = check_written(d, "tria_evict_mass dst", c);
    if (!rc) rc = check_apart(d, "tria_evict_mass dst");
    if (rc) return rc;
    for (int l = 0; l < s->n_layer; l++)
        if (s->k[l] == d->k[l] || (s->v && s->v[l] == d->v[l]))
            FAIL(TRIA_ERR_INVALID, "%s: src and dst must be different caches", fn);
    const int KV = s->n_head_kv;
    const int64_t units = (int64_t)s->n_layer * KV;
    int max_rows = 0;
    for (int64_t u = 0; u < units; u++) {
        if (n_rows[u] > d->n_cells)   /* the kept count is only known on the device */
            FAIL(TRIA_ERR_INVALID, "dst n_cells %d < n_rows[%lld] = %d", d->n_cells, (long long)u, n_rows[u]);
        max_rows = std::max(max_rows, n_rows[u]);
    }
    DeviceGuard g(c->device);
    cudaStream_t st = (cudaStream_t)stream;
    if ((rc = ensure_scratch(c, units, s->n_cells, st))) return rc;
    std::vector<int32_t> keep;
    keep_requests(c, s, n_rows, p, keep);
    int32_t *cnt = n_kept_out ? n_kept_out : c->cnt;
    if ((rc = launch_select(c, s, n_rows, keep, p, false, mass, c->kept, c->cell_stride, cnt, st, units))) return rc;
    int64_t hint = 0;
    for (int32_t k : keep) hint = std::max<int64_t>(hint, k);
    if (p->window > 0 || p->sink > 0) hint += (int64_t)std::max(0, p->window) + std::max(0, p->sink) + 1;
    hint = std::min<int64_t>(hint, max_rows);
    if ((rc = launch_compact(c, s, d, n_rows, c->kept, c->cell_stride, cnt, st, (int)hint))) return rc;
    if (mass_dst && max_rows > 0) {
        for (int64_t u0 = 0; u0 < units; u0 += TRIA_MAX_UNITS) {
            const int nu = (int)std::min<int64_t>(TRIA_MAX_UNITS, units - u0);
            const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>((hint + 1023) / 1024, 64)), (unsigned)nu);
            k_carry_mass<<<grid, 256, 0, st>>>(mass + u0 * s->n_cells, s->n_cells, mass_dst + u0 * d->n_cells, d->n_cells,
                                               c->kept + u0 * c->cell_stride, c->cell_stride, cnt + u0, c->d_status);
            CUDA_TRY(cudaGetLastError());
            c->launches++;
        }
    }
    c->have_timing = false;
    return read_back_step(c, cnt, units, st);
}

/* ------------------------------------------------------------------ */
/* Attention                                                            */
/* ------------------------------------------------------------------ */

/* Rows of `width` elements at the strides of up to three dimensions. */
struct RowGrid {
    using wide = __int128;               /* strides are the caller's: nothing here may overflow */
    struct Dim { int64_t extent, stride; } dim[3];
    int n = 0;
    int64_t width;
    explicit RowGrid(int64_t w) : width(w) {}
    /* Dimensions of one entry have no stride; the others are kept by ascending stride. */
    RowGrid &add(int64_t extent, int64_t stride) {
        if (extent <= 1) return *this;
        int i = n++;
        for (; i > 0 && dim[i - 1].stride > stride; i--) dim[i] = dim[i - 1];
        dim[i] = {extent, stride};
        return *this;
    }
    /* Elements from the first row's start to the last row's end over the first k dimensions. */
    wide span(int k) const {
        wide s = width;
        for (int i = 0; i < k; i++) s += (wide)(dim[i].extent - 1) * dim[i].stride;
        return s;
    }
    /* Whether each stride steps over all that the smaller ones span. */
    bool nested() const {
        for (int i = 0; i < n; i++)
            if (dim[i].stride < span(i)) return false;
        return true;
    }
    bool same_strides(const RowGrid &o) const {
        if (n != o.n || width != o.width) return false;
        for (int i = 0; i < n; i++)
            if (dim[i].extent != o.dim[i].extent || dim[i].stride != o.dim[i].stride) return false;
        return true;
    }
    /* Whether a row of this nested grid and one of its copy `delta` elements on share one: of each dimension only the
     * two steps around delta come near enough. */
    bool meets_copy(wide delta, int k) const {
        if (delta >= span(k) || -delta >= span(k)) return false;
        if (k == 0) return true;
        const Dim &d = dim[k - 1];
        wide at = delta / d.stride;
        if (delta % d.stride && delta < 0) at--;
        for (int i = 0; i < 2; i++, at++)
            if (at > -d.extent && at < d.extent && meets_copy(delta - at * d.stride, k - 1)) return true;
        return false;
    }
};

/* Whether f16 rows of q and out share elements.  Grids of different strides whose ranges overlap are taken to. */
static bool grids_meet(const RowGrid &q, const void *qp, const RowGrid &o, const void *op) {
    const RowGrid::wide delta = ((int64_t)(uintptr_t)op - (int64_t)(uintptr_t)qp) / 2;
    if (delta >= q.span(q.n) || -delta >= o.span(o.n)) return false;
    return !q.same_strides(o) || o.meets_copy(delta, o.n);
}

/* Grows tria_attend's workspace to `need` bytes. */
static int ensure_attend(tria_ctx *c, size_t need, cudaStream_t st) {
    const int cap = note_capture(c, st);
    if (cap < 0) return cap;
    if (need <= c->attend_cap) return TRIA_OK;
    if (cap) FAIL(TRIA_ERR_INVALID, "tria_attend: the workspace has to grow to %zu bytes inside a stream capture: make "
                  "one eager call with these sizes first", need);
    need += need / 4;
    CUDA_TRY(cudaDeviceSynchronize());        /* earlier calls may still use it, on any stream */
    if (c->d_attend) drop_scratch(c, c->d_attend);
    c->d_attend = nullptr;
    c->attend_cap = 0;
    CUDA_TRY(cudaMalloc(&c->d_attend, need));
    c->attend_cap = need;
    CUDA_TRY(cudaMemset(c->d_attend, 0, need));
    CUDA_TRY(cudaDeviceSynchronize());
    return TRIA_OK;
}

template <int KT>
static int few_blocks_of(int nt) {
    return nt == 1 ? few_blocks<KT, 1>() : few_blocks<KT, 2>();
}

/* Launch plan of one chunk of caches. */
struct AttendPlan {
    bool tile = false;          /* k_attend_tile, else k_attend_few */
    int nt = 1;                 /* k_attend_few: query rows per group, in eights */
    int rows = 8;               /* query rows per group */
    int groups = 0, items = 0, grid = 0;
    bool plan_kernel = false, keep_scores = false;
    size_t steps = 0, span = 0, done = 0, arrived = 0, part_o = 0, part_ml = 0, norm = 0, scores = 0, redo = 0, bytes = 0;
    int64_t score_stride = 0;
};

/* Most blocks of an attention kernel (the workspace's counters). */
constexpr int ATTEND_MAX_GRID = 1024;

/* Query rows of a unit above which the tensor-core tiles are taken.  Groups of
 * 16 on mma read a unit's rows once a group (mostly from L2); tiles of 256 read
 * them once, but start, join and convert q8_0 rows at a higher price.  Measured
 * with 8 units of head_dim 128 over 500 / 4000 / 32000 rows (us, groups against
 * tiles): f16 R = 32: 18 / 35 / 72 against 23 / 38 / 87, R = 64: 19 / 38 / 110
 * against 24 / 39 / 91; q8_0 R = 64: 20 / 40 / 120 against 28 / 50 / 143. */
constexpr int TILE_FROM_F16 = 32, TILE_FROM_Q8_0 = 64;

/* A call with masses and at most 16 query rows a unit keeps its scores (4 bytes
 * a query row and cache row) instead of scoring twice, up to this many bytes.
 * Measured with 8 units over 500 / 4000 / 65000 rows (us, kept against scored
 * again): f16 R = 4: 14 / 24 / 70 against 17 / 27 / 106, R = 16: 22 / 36 / 102
 * against 24 / 40 / 144; q8_0 alike. */
constexpr size_t SCORES_MAX = (size_t)1 << 30;

static int plan_attend(const tria_ctx *c, const tria_kv_view *v, int nl, int T, bool window, bool mass, AttendPlan &pl) {
    const int64_t units = (int64_t)nl * v->n_head_kv, R = (int64_t)T * c->G;
    pl = AttendPlan{};
    pl.tile = R > (v->type == TRIA_TYPE_F16 ? TILE_FROM_F16 : TILE_FROM_Q8_0);
    pl.nt = R <= 8 ? 1 : 2;
    const int rows = pl.rows = pl.tile ? TILE_ROWS : 8 * pl.nt;
    const int step = pl.tile ? TILE_STEP : ATT_STEP;
    const int64_t groups = (R + rows - 1) / rows, items = units * groups;
    if (items * ((v->n_cells + step - 1) / step + 1) > INT32_MAX)
        FAIL(TRIA_ERR_UNSUPPORTED, "tria_attend: %lld query rows over %d cells in one call", (long long)(units * R), v->n_cells);
    pl.groups = (int)groups;
    pl.items = (int)items;
    pl.grid = std::min((v->type == TRIA_TYPE_F16 ? few_blocks_of<KT_F16>(pl.nt) : few_blocks_of<KT_Q8_0>(pl.nt)) * c->sm_count,
                       ATTEND_MAX_GRID);
    if (pl.tile) pl.grid = std::min(c->sm_count, ATTEND_MAX_GRID);
    pl.plan_kernel = pl.tile || window || items > 512;
    pl.score_stride = ((int64_t)v->n_cells + ATT_STEP - 1) / ATT_STEP * ATT_STEP;
    const size_t sb = (size_t)(units * R * pl.score_stride) * 4;
    pl.keep_scores = mass && R <= 16 && sb <= SCORES_MAX;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += align256(bytes); return o; };
    /* the counters come first and keep their place: they are zero between calls, whatever a call lays out behind them */
    pl.done = take(4);
    pl.arrived = take(ATTEND_MAX_GRID * 4);
    if (pl.plan_kernel) {
        pl.steps = take((size_t)items * 4);
        if (window) pl.span = take((size_t)items * 8);
    }
    pl.part_o = take((size_t)2 * pl.grid * rows * c->hd * 4);
    pl.part_ml = take((size_t)2 * pl.grid * rows * 8);
    if (pl.tile) pl.redo = take((size_t)(units * R + 1) * 4);
    if (mass) pl.norm = take((size_t)(units * R) * 8);
    if (pl.keep_scores) pl.scores = take(sb);
    pl.bytes = at;
    return TRIA_OK;
}

template <int KT, int HD, int NT>
static int launch_few(tria_ctx *c, const AttendArgs &a, const AttendPlan &pl, cudaStream_t st) {
    const bool extra = a.softcap > 0.0f || a.window > 0 || a.slopes;
    auto fn = extra ? k_attend_few<KT, HD, NT, true> : k_attend_few<KT, HD, NT, false>;
    constexpr int smem = few_smem<KT, HD, NT>();
    CUDA_TRY(raise_smem_limit((const void *)fn, smem));
    fn<<<pl.grid, FEW_THREADS, smem, st>>>(a);
    CUDA_TRY(cudaGetLastError());
    c->launches++;
    return TRIA_OK;
}

template <int KT, int HD>
static int launch_tile(tria_ctx *c, const AttendArgs &a, const AttendPlan &pl, cudaStream_t st) {
    using L = TileLayout<KT, HD>;
    const bool extra = a.softcap > 0.0f || a.window > 0 || a.slopes;
    auto fn = extra ? k_attend_tile<KT, HD, true> : k_attend_tile<KT, HD, false>;
    CUDA_TRY(raise_smem_limit((const void *)fn, L::BYTES));
    fn<<<pl.grid, L::THREADS, L::BYTES, st>>>(a);
    CUDA_TRY(cudaGetLastError());
    k_attend_redo<KT, HD><<<c->sm_count, ROW_THREADS, 0, st>>>(a);
    CUDA_TRY(cudaGetLastError());
    c->launches += 2;
    return TRIA_OK;
}

template <int KT, int HD>
static int launch_mass_tile(const AttendArgs &a, int units, cudaStream_t st) {
    constexpr int smem = MassTileLayout<KT, HD>::BYTES;
    const bool extra = a.softcap > 0.0f || a.window > 0 || a.slopes;
    auto fn = extra ? k_mass_tile<KT, HD, true> : k_mass_tile<KT, HD, false>;
    CUDA_TRY(raise_smem_limit((const void *)fn, smem));
    const int gx = std::max(1, std::min((a.n_cells + TILE_K - 1) / TILE_K, 65535));
    fn<<<dim3((unsigned)gx, (unsigned)units), MASS_TILE_THREADS, smem, st>>>(a);
    return TRIA_OK;
}

template <int KT, int HD>
static int run_attend(tria_ctx *c, AttendArgs &a, const AttendPlan &pl, cudaStream_t st) {
    const int units = a.n_layer * a.n_head_kv;
    uint8_t *ws = c->d_attend;
    a.groups = pl.groups;
    a.arrived = (int32_t *)(ws + pl.arrived);
    a.part_o = (float *)(ws + pl.part_o);
    a.part_ml = (float2 *)(ws + pl.part_ml);
    a.norm = a.mass_out ? (float2 *)(ws + pl.norm) : nullptr;
    a.scores = pl.keep_scores ? (float *)(ws + pl.scores) : nullptr;
    a.score_stride = pl.score_stride;
    a.redo = pl.tile ? (int32_t *)(ws + pl.redo) : nullptr;
    if (a.T > 0) {
        if (pl.plan_kernel) {
            int32_t *steps = (int32_t *)(ws + pl.steps);
            int2 *span = a.window > 0 ? (int2 *)(ws + pl.span) : nullptr;
            k_attend_plan<<<span ? pl.items : 1, PLAN_THREADS, 0, st>>>(a, pl.rows, pl.tile ? TILE_STEP : ATT_STEP, pl.items, span, steps,
                                                                       (int32_t *)(ws + pl.done));
            CUDA_TRY(cudaGetLastError());
            c->launches++;
            a.steps = steps;
            a.span = span;
        }
        const int rc = pl.tile ? launch_tile<KT, HD>(c, a, pl, st)
                     : pl.nt == 1 ? launch_few<KT, HD, 1>(c, a, pl, st) : launch_few<KT, HD, 2>(c, a, pl, st);
        if (rc) return rc;
    }
    if (a.mass_out) {
        if (pl.keep_scores && a.T > 0) {
            const int gx = std::max(1, std::min((a.n_cells + 255) / 256, 8 * c->sm_count / std::min(units, 8 * c->sm_count)));
            k_mass_scores<<<dim3((unsigned)gx, (unsigned)units), 256, 0, st>>>(a);
        } else if (a.T * a.G > 16) {
            const int rc = launch_mass_tile<KT, HD>(a, units, st);
            if (rc) return rc;
        } else {
            const int gx = std::max(1, std::min((a.n_cells + MASS_KEYS - 1) / MASS_KEYS, 65535));
            k_mass_tiles<KT, HD><<<dim3((unsigned)gx, (unsigned)units), MASS_THREADS, 0, st>>>(a);
        }
        CUDA_TRY(cudaGetLastError());
        c->launches++;
    }
    return TRIA_OK;
}

static int do_attend(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows,
                     const tria_attend_params *p, const void *q, void *out, float *lse,
                     const float *mass_in, float *mass_out, void *stream) {
    NvtxRange range("tria_attend");
    const char *fn = "tria_attend";
    if (!p) FAIL(TRIA_ERR_INVALID, "%s: null parameters", fn);
    int rc = validate_cache(v, fn);
    if (!rc) rc = check_ints(fn, "n_rows", n_rows);
    if (rc) return rc;
    const int T = p->n_tok, KV = v->n_head_kv;
    if (T < 0 || p->window < 0 || p->sink < 0) FAIL(TRIA_ERR_INVALID, "%s: negative n_tok, window or sink", fn);
    if (p->reserved) FAIL(TRIA_ERR_INVALID, "%s: reserved must be 0", fn);
    if (!std::isfinite(p->scale) || !std::isfinite(p->mass_decay) || !std::isfinite(p->softcap) || p->softcap < 0.0f)
        FAIL(TRIA_ERR_INVALID, "%s: scale %g, softcap %g or mass_decay %g not finite, or softcap < 0", fn,
             (double)p->scale, (double)p->softcap, (double)p->mass_decay);
    if (!std::isfinite(p->scale * LOG2E) || !std::isfinite(p->softcap * LOG2E) ||
        (p->softcap > 0.0f && !std::isfinite(p->scale / p->softcap)))
        FAIL(TRIA_ERR_INVALID, "%s: scale %g and softcap %g are out of fp32's range together", fn, (double)p->scale, (double)p->softcap);
    if (mass_in && !mass_out) FAIL(TRIA_ERR_INVALID, "%s: mass_in without mass_out", fn);
    if (((uintptr_t)mass_in & 3) || ((uintptr_t)mass_out & 3) || ((uintptr_t)lse & 3))
        FAIL(TRIA_ERR_INVALID, "%s: lse or mass misaligned", fn);
    if (mass_in && mass_in != mass_out && arrays_meet(mass_in, view_cells(v), mass_out, view_cells(v)))
        FAIL(TRIA_ERR_INVALID, "%s: mass_in and mass_out overlap in part", fn);
    if (T > 0) {
        if (!q || !out || ((uintptr_t)q & 15) || ((uintptr_t)out & 15))
            FAIL(TRIA_ERR_INVALID, "%s: q or out null or not 16-byte aligned", fn);
        if (q == out) FAIL(TRIA_ERR_INVALID, "%s: out must not overlap q", fn);
        const int64_t s[6] = {p->q_cache_stride, p->q_tok_stride, p->q_head_stride,
                              p->o_cache_stride, p->o_tok_stride, p->o_head_stride};
        for (int64_t x : s)
            if (x < 0 || x % 8) FAIL(TRIA_ERR_INVALID, "%s: q and out strides must be multiples of 8 elements, not negative", fn);
        if (p->slopes && ((uintptr_t)p->slopes & 3)) FAIL(TRIA_ERR_INVALID, "%s: slopes misaligned", fn);
        if (p->window > 0 || p->slopes) {
            if ((rc = check_ints(fn, "tok_pos", p->tok_pos))) return rc;
            if (p->tok_pos_stride < 0) FAIL(TRIA_ERR_INVALID, "%s: negative tok_pos_stride", fn);
        }
        if (p->tree) {
            if ((uintptr_t)p->tree & 3) FAIL(TRIA_ERR_INVALID, "%s: tree misaligned", fn);
            if (p->tree_words < (T + 31) / 32 || p->tree_stride < 0)
                FAIL(TRIA_ERR_INVALID, "%s: tree_words %d < %d, or a negative tree_stride", fn, p->tree_words, (T + 31) / 32);
        }
        /* the least rows that any context has; its own follow below */
        if (!RowGrid(64).add(v->n_layer, p->o_cache_stride).add(T, p->o_tok_stride).add(KV, p->o_head_stride).nested())
            FAIL(TRIA_ERR_INVALID, "%s: out strides let outputs overlap", fn);
    }
    if ((rc = check_ctx(c, fn))) return rc;
    const int H = KV * (int)c->G;
    if ((int64_t)v->n_layer * H * T > INT32_MAX / 2)
        FAIL(TRIA_ERR_UNSUPPORTED, "%s: %lld query rows in one call", fn, (long long)v->n_layer * H * T);
    if (T > 0) {
        RowGrid qg((int)c->hd), og((int)c->hd);
        qg.add(v->n_layer, p->q_cache_stride).add(T, p->q_tok_stride).add(H, p->q_head_stride);
        og.add(v->n_layer, p->o_cache_stride).add(T, p->o_tok_stride).add(H, p->o_head_stride);
        if (!og.nested()) FAIL(TRIA_ERR_INVALID, "%s: out strides let outputs overlap", fn);
        if (grids_meet(qg, q, og, out)) FAIL(TRIA_ERR_INVALID, "%s: out must not overlap q", fn);
    }
    if (T == 0 && !mass_out) return TRIA_OK;
    DeviceGuard g(c->device);
    cudaStream_t st = (cudaStream_t)stream;
    /* rows on 16-byte boundaries (q8_0: 8 bytes off them, the same for every cell of a head) */
    const bool copy16 = !(v->cell_stride & 15) && !(v->head_stride & (v->type == TRIA_TYPE_F16 ? 15 : 7));
    size_t need = 0;
    rc = for_cache_chunks(v, [&](int, int nl) -> int {
        AttendPlan pl;
        const int r = plan_attend(c, v, nl, T, p->window > 0, mass_out != nullptr, pl);
        need = std::max(need, pl.bytes);
        return r;
    });
    if (rc) return rc;
    if ((rc = ensure_attend(c, need, st))) return rc;
    return for_cache_chunks(v, [&](int l0, int nl) -> int {
        AttendPlan pl;
        const int r = plan_attend(c, v, nl, T, p->window > 0, mass_out != nullptr, pl);
        if (r) return r;
        AttendArgs a;
        memset(&a, 0, sizeof a);
        const int64_t u0 = (int64_t)l0 * KV;
        for (int l = 0; l < nl; l++) { a.k[l] = (const uint8_t *)v->k[l0 + l]; a.v[l] = (const uint8_t *)v->v[l0 + l]; }
        a.cell_stride = v->cell_stride;
        a.head_stride = v->head_stride;
        a.pos = v->pos_shared ? v->pos : v->pos + u0 * v->n_cells;
        a.pos_shared = v->pos_shared ? 1 : 0;
        a.n_cells = v->n_cells;
        a.n_layer = nl;
        a.n_head_kv = KV;
        a.G = (int32_t)c->G;
        a.T = T;
        a.n_rows = n_rows + u0;
        a.q = (const __half *)q + l0 * p->q_cache_stride;
        a.out = (__half *)out + l0 * p->o_cache_stride;
        a.q_cache = p->q_cache_stride; a.q_tok = p->q_tok_stride; a.q_head = p->q_head_stride;
        a.o_cache = p->o_cache_stride; a.o_tok = p->o_tok_stride; a.o_head = p->o_head_stride;
        a.lse = lse ? lse + (int64_t)l0 * T * H : nullptr;
        a.copy16 = copy16;
        a.mass_in = mass_in ? mass_in + u0 * v->n_cells : nullptr;
        a.mass_out = mass_out ? mass_out + u0 * v->n_cells : nullptr;
        a.mass_decay = p->mass_decay;
        a.scale = p->scale;
        a.softcap = p->softcap;
        a.window = p->window;
        a.sink = p->sink;
        a.slopes = p->slopes;
        a.tok_pos = p->window > 0 || p->slopes ? p->tok_pos + l0 * p->tok_pos_stride : nullptr;
        a.tok_pos_stride = p->tok_pos_stride;
        a.tree = p->tree ? p->tree + l0 * p->tree_stride : nullptr;
        a.tree_stride = p->tree_stride;
        a.tree_words = p->tree_words;
        a.status = c->d_status;
        a.wait_limit = c->wait_limit;
        if (v->type == TRIA_TYPE_F16)
            return c->hd == 128 ? run_attend<KT_F16, 128>(c, a, pl, st) : run_attend<KT_F16, 64>(c, a, pl, st);
        return c->hd == 128 ? run_attend<KT_Q8_0, 128>(c, a, pl, st) : run_attend<KT_Q8_0, 64>(c, a, pl, st);
    });
}

extern "C" TRIA_API int tria_append(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows,
                                    const tria_append_params *p, const void *k, const void *vv, float *mass,
                                    int32_t *n_rows_out, void *stream) {
    return no_throw("tria_append", [&] { return do_append(c, v, n_rows, p, k, vv, mass, n_rows_out, stream); });
}

extern "C" TRIA_API int tria_accept(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows, int32_t n_tok,
                                    const int32_t *path, int64_t path_stride, const int32_t *n_path, float *mass,
                                    int32_t *n_rows_out, void *stream) {
    return no_throw("tria_accept", [&] { return do_accept(c, v, n_rows, n_tok, path, path_stride, n_path, mass, n_rows_out, stream); });
}

extern "C" TRIA_API int tria_evict_mass(tria_ctx *c, const tria_kv_view *s, const tria_kv_view *d,
                                        const int32_t *n_rows, const float *mass, float *mass_dst,
                                        const tria_evict_params *p, int32_t *n_kept_out, void *stream) {
    return no_throw("tria_evict_mass", [&] { return do_evict_mass(c, s, d, n_rows, mass, mass_dst, p, n_kept_out, stream); });
}

extern "C" TRIA_API int tria_attend(tria_ctx *c, const tria_kv_view *v, const int32_t *n_rows,
                                    const tria_attend_params *p, const void *q, void *out, float *lse,
                                    const float *mass_in, float *mass_out, void *stream) {
    return no_throw("tria_attend", [&] { return do_attend(c, v, n_rows, p, q, out, lse, mass_in, mass_out, stream); });
}
