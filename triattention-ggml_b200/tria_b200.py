"""ctypes binding of libtriattention_b200.so (include/triattention.h).

The reference's Python side reimplements the scoring math in torch
(triattention_common.py); this module instead calls the C ABI, so the
Python validate/score scripts can drive the B200 kernels directly:

    st = tria_b200.load("stats.bin")                  # tria_load
    out = tria_b200.score_kv_head(st, k_re, k_im, key_pos, cur_pos, layer, kvh)
    ctx = tria_b200.Context(st, device=0)             # device path
    ctx.evict(src_view, dst_view, n_rows, params, stream)

There is no CPU fallback: if the shared library is missing this module
raises on import of the library, and every device call reports the CUDA
status it got.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import subprocess

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
CHECKED_LIB_PATH = os.path.join(HERE, "libtriattention_b200_checked.so")
# TRIA_B200_LIB=checked loads the checked build (bounds checks in every kernel,
# TRIA_ERR_BOUNDS) instead of the product library
LIB_PATH = CHECKED_LIB_PATH if os.environ.get("TRIA_B200_LIB") == "checked" else \
    os.path.join(HERE, "libtriattention_b200.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "triattention.h")
HEADERS = [HEADER, os.path.join(os.path.dirname(HERE), "include", "triattention_ggml.h")]

TYPE_F16 = 1
TYPE_Q8_0 = 8

OK = 0
ERR_INVALID = -1
ERR_CUDA = -2
ERR_NOMEM = -3
ERR_POSITION = -4
ERR_UNSUPPORTED = -5
ERR_NO_DEVICE = -6
ERR_TIMEOUT = -7
ERR_BOUNDS = -8
ERR_ROWS = -9


class TriaError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"[{status}] {msg}")
        self.status = status


class HeadStats(C.Structure):
    _fields_ = [("q_mean_real", C.POINTER(C.c_float)), ("q_mean_imag", C.POINTER(C.c_float)),
                ("q_abs_mean", C.POINTER(C.c_float)), ("qma", C.POINTER(C.c_float))]


class Stats(C.Structure):
    """struct tria_stats (triattention.h:38-50 of the reference)."""
    _fields_ = [("num_layers", C.c_uint32), ("num_heads", C.c_uint32), ("num_kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("freq_count", C.c_uint32), ("rope_theta", C.c_float),
                ("attn_scale", C.c_float), ("layer_budget_scales", C.POINTER(C.c_float)),
                ("omega", C.POINTER(C.c_float)), ("heads", C.POINTER(HeadStats))]


class KvView(C.Structure):
    """struct tria_kv_view."""
    _fields_ = [("type", C.c_int32), ("n_layer", C.c_int32), ("layer0", C.c_int32),
                ("n_head_kv", C.c_int32), ("head0", C.c_int32), ("n_cells", C.c_int32),
                ("cell_stride", C.c_int64), ("head_stride", C.c_int64),
                ("k", C.POINTER(C.c_void_p)), ("v", C.POINTER(C.c_void_p)),
                ("pos", C.c_void_p), ("pos_shared", C.c_int32), ("flags", C.c_int32)]


VIEW_POST_ROPE = 1      # TRIA_VIEW_POST_ROPE


class GgmlTensor(C.Structure):
    """struct tria_ggml_tensor: the ggml_tensor fields the bridge reads."""
    _fields_ = [("type", C.c_int32), ("reserved", C.c_int32), ("ne", C.c_int64 * 4),
                ("nb", C.c_size_t * 4), ("data", C.c_void_p)]


class GgmlCache(C.Structure):
    """struct tria_ggml_cache."""
    _fields_ = [("k", C.POINTER(C.POINTER(GgmlTensor))), ("v", C.POINTER(C.POINTER(GgmlTensor))),
                ("n_layer", C.c_int32), ("layer0", C.c_int32), ("n_head_kv", C.c_int32),
                ("head_dim", C.c_int32), ("pos", C.c_void_p), ("pos_shared", C.c_int32),
                ("flags", C.c_int32)]


def ggml_tensor(type_id, ne0, ne1, nb1, data, elem=None):
    """A 2-D ggml tensor descriptor [ne0, ne1] with rows nb1 bytes apart."""
    t = GgmlTensor()
    t.type = int(type_id)
    t.ne[:] = [int(ne0), int(ne1), 1, 1]
    e = elem if elem is not None else (2 if type_id == TYPE_F16 else 34)
    t.nb[:] = [e, int(nb1), int(nb1) * int(ne1), int(nb1) * int(ne1)]
    t.data = _ptr(data)
    return t


def ggml_cache(k_tensors, v_tensors, n_head_kv, head_dim, pos, layer0=0, pos_shared=False, flags=0):
    """A GgmlCache over lists of GgmlTensor; keeps its arrays alive."""
    nl = len(k_tensors)
    karr = (C.POINTER(GgmlTensor) * nl)(*[C.pointer(t) for t in k_tensors])
    varr = (C.POINTER(GgmlTensor) * nl)(*[C.pointer(t) for t in v_tensors]) if v_tensors is not None else None
    c = GgmlCache(C.cast(karr, C.POINTER(C.POINTER(GgmlTensor))),
                  C.cast(varr, C.POINTER(C.POINTER(GgmlTensor))) if varr is not None else None,
                  nl, int(layer0), int(n_head_kv), int(head_dim), _ptr(pos), 1 if pos_shared else 0, int(flags))
    c._keep = (karr, varr, k_tensors, v_tensors, pos)
    return c


def ggml_view(cache):
    """tria_ggml_view: (status, KvView) without raising."""
    nl = cache.n_layer
    kp, vp = (C.c_void_p * nl)(), (C.c_void_p * nl)()
    v = KvView()
    r = lib().tria_ggml_view(C.byref(cache), C.byref(v), kp, vp)
    v._keep = (kp, vp, cache)
    return r, v


class EvictParams(C.Structure):
    """struct tria_evict_params."""
    _fields_ = [("cur_pos", C.c_int32), ("budget", C.c_int32), ("ramp_pct", C.c_int32),
                ("window", C.c_int32), ("sink", C.c_int32), ("reserved", C.c_int32)]


class AttendParams(C.Structure):
    """struct tria_attend_params; attend_params() fills one from tensors."""
    _fields_ = [("n_tok", C.c_int32), ("window", C.c_int32), ("sink", C.c_int32), ("tree_words", C.c_int32),
                ("scale", C.c_float), ("softcap", C.c_float), ("mass_decay", C.c_float), ("reserved", C.c_int32),
                ("slopes", C.c_void_p), ("tok_pos", C.c_void_p), ("tree", C.c_void_p),
                ("tok_pos_stride", C.c_int64), ("tree_stride", C.c_int64),
                ("q_cache_stride", C.c_int64), ("q_tok_stride", C.c_int64), ("q_head_stride", C.c_int64),
                ("o_cache_stride", C.c_int64), ("o_tok_stride", C.c_int64), ("o_head_stride", C.c_int64)]
    _keep = (None, None, None)      # slopes, tok_pos, tree
    _sig = None                     # the shapes that the strides were last taken from


class AppendParams(C.Structure):
    """struct tria_append_params."""
    _fields_ = [("n_tok", C.c_int32), ("src_type", C.c_int32), ("cache_stride", C.c_int64), ("tok_stride", C.c_int64),
                ("head_stride", C.c_int64), ("tok_pos", C.c_void_p), ("tok_pos_stride", C.c_int64)]


SRC_F32 = 0
SRC_F16 = 1


def attend_params(scale, softcap=0.0, window=0, sink=0, slopes=None, tok_pos=None, tree=None, mass_decay=1.0):
    """Options of Context.attend that stay the same from call to call (the
    token count and the strides come from the call's q and out).  Device
    tensors: slopes fp32 [heads]; tok_pos int32 [n_tok], or [caches][n_tok]
    for positions of each cache's own; tree int32 [n_tok][words] or
    [caches][n_tok][words], bit j % 32 of word j / 32 of row t set when token t
    sees token j."""
    p = AttendParams()
    p.scale, p.softcap, p.window, p.sink, p.mass_decay = scale, softcap, int(window), int(sink), mass_decay
    p.slopes = _ptr(_ints_or_floats(slopes, "slopes", 1, _torch().float32))
    p.tok_pos = _ptr(_ints_or_floats(tok_pos, "tok_pos", 2, _torch().int32))
    p.tree = _ptr(_ints_or_floats(tree, "tree", 3, _torch().int32))
    if tok_pos is not None and tok_pos.dim() == 2:
        p.tok_pos_stride = tok_pos.stride(0)
    if tree is not None:
        p.tree_words = tree.shape[-1]
        if tree.dim() == 3:
            p.tree_stride = tree.stride(0)
    p._keep = (slopes, tok_pos, tree)
    return p


def _torch():
    """torch, imported by the callers that hand tensors in."""
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


_torch_module = None


def _ints_or_floats(x, name, most_dims, dtype):
    if x is None:
        return None
    if x.dtype != dtype or not 1 <= x.dim() <= most_dims or (x.shape[-1] > 1 and x.stride(-1) != 1):
        raise ValueError(f"{name}: a {dtype} tensor of at most {most_dims} dimensions with a contiguous last one is wanted")
    if x.dim() >= 2 and name == "tree" and x.shape[-2] > 1 and x.stride(-2) != x.shape[-1]:
        raise ValueError("tree: rows must follow one another")
    return x


class Policy(C.Structure):
    """struct tria_policy: the reference runtime's eviction schedule."""
    _fields_ = [("budget_pct", C.c_int32), ("window", C.c_int32), ("interval", C.c_int32),
                ("sink", C.c_int32), ("step", C.c_int32), ("next_pos", C.c_int32)]

    def __init__(self, budget_pct=75, window=512, interval=128, sink=0):
        super().__init__()
        lib().tria_policy_init(C.byref(self), int(budget_pct), int(window), int(interval), int(sink))

    def due(self, n_past: int, n_kv: int):
        """EvictParams when an eviction is due at n_past with n_kv cached rows, else None."""
        out = EvictParams()
        r = lib().tria_policy_due(C.byref(self), int(n_past), int(n_kv), C.byref(out))
        if r < 0:
            check(r)
        return out if r == 1 else None


def n_kv_per_seq(n_kept, seq_of_unit, n_seq):
    """tria_n_kv_per_seq: per-sequence maximum of the kept counts."""
    nk = np.ascontiguousarray(n_kept, np.int32)
    so = np.ascontiguousarray(seq_of_unit, np.int32)
    out = np.zeros(n_seq, np.int32)
    check(lib().tria_n_kv_per_seq(nk.ctypes.data, so.ctypes.data, int(nk.shape[0]), int(n_seq), out.ctypes.data))
    return out


def build() -> str:
    """Compile the library (and the checked build) in-tree (nvcc, sm_100a)."""
    subprocess.run(["make", "-s", "-j4", "-C", HERE, "all", "checked"], check=True)
    return LIB_PATH


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is not built; run `make -C {HERE}`")
        L = C.CDLL(LIB_PATH)
        L.tria_load.restype = C.POINTER(Stats)
        L.tria_load.argtypes = [C.c_char_p]
        L.tria_free.argtypes = [C.POINTER(Stats)]
        L.tria_score_kv_head.argtypes = [C.POINTER(Stats), C.c_void_p, C.c_void_p, C.c_void_p,
                                         C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]
        L.tria_status_str.restype = C.c_char_p
        L.tria_status_str.argtypes = [C.c_int]
        L.tria_last_error.restype = C.c_char_p
        L.tria_ctx_create.argtypes = [C.POINTER(Stats), C.c_int, C.POINTER(C.c_void_p)]
        L.tria_ctx_destroy.argtypes = [C.c_void_p]
        L.tria_score.argtypes = [C.c_void_p, C.POINTER(KvView), C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]
        L.tria_select.argtypes = [C.c_void_p, C.POINTER(KvView), C.c_void_p, C.c_void_p,
                                  C.POINTER(EvictParams), C.c_void_p, C.c_void_p, C.c_void_p]
        L.tria_compact.argtypes = [C.c_void_p, C.POINTER(KvView), C.POINTER(KvView), C.c_void_p,
                                   C.c_void_p, C.c_void_p, C.c_void_p]
        L.tria_evict.argtypes = [C.c_void_p, C.POINTER(KvView), C.POINTER(KvView), C.c_void_p,
                                 C.POINTER(EvictParams), C.c_void_p, C.c_void_p]
        L.tria_get_n_kv.argtypes = [C.c_void_p, C.c_void_p, C.c_int32]
        L.tria_evict_host.argtypes = [C.c_void_p, C.POINTER(KvView), C.POINTER(KvView), C.c_void_p,
                                      C.POINTER(EvictParams), C.c_void_p]
        L.tria_ctx_set_timing.argtypes = [C.c_void_p, C.c_int]
        L.tria_ctx_stage_ms.argtypes = [C.c_void_p, C.c_void_p, C.c_int]
        L.tria_ctx_launches.restype = C.c_int64
        L.tria_ctx_launches.argtypes = [C.c_void_p]
        L.tria_ctx_check.argtypes = [C.c_void_p, C.c_void_p]
        L.tria_ggml_view.argtypes = [C.POINTER(GgmlCache), C.POINTER(KvView), C.c_void_p, C.c_void_p]
        L.tria_ggml_evict.argtypes = [C.c_void_p, C.POINTER(GgmlCache), C.POINTER(GgmlCache), C.c_void_p,
                                      C.POINTER(EvictParams), C.c_void_p]
        L.tria_ctx_set_wait_limit.argtypes = [C.c_void_p, C.c_int64]
        L.tria_ctx_set_select_split.argtypes = [C.c_void_p, C.c_int32]
        L.tria_key_gather.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_uint32,
                                      C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]
        L.tria_checked_build.argtypes = []
        L.tria_select_noalloc.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_int32,
                                          C.c_void_p, C.c_int64, C.c_int32, C.c_int32, C.c_int32,
                                          C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
        L.tria_znorm_stats.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]
        L.tria_policy_init.restype = None
        L.tria_policy_init.argtypes = [C.POINTER(Policy), C.c_int32, C.c_int32, C.c_int32, C.c_int32]
        L.tria_policy_due.argtypes = [C.POINTER(Policy), C.c_int32, C.c_int32, C.POINTER(EvictParams)]
        L.tria_n_kv_per_seq.argtypes = [C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_void_p]
        L.tria_score_key.restype = C.c_uint32
        L.tria_score_key.argtypes = [C.c_float]
        L.tria_key_histogram.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_int32, C.c_uint32,
                                         C.c_void_p, C.c_void_p]
        L.tria_key_count.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_uint32, C.c_void_p,
                                     C.c_void_p]
        L.tria_select_key.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_uint32, C.c_void_p,
                                      C.c_int64, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
        L.tria_attend.argtypes = [C.c_void_p, C.POINTER(KvView), C.c_void_p, C.POINTER(AttendParams)] + [C.c_void_p] * 6
        L.tria_append.argtypes = [C.c_void_p, C.POINTER(KvView), C.c_void_p, C.POINTER(AppendParams)] + [C.c_void_p] * 5
        L.tria_accept.argtypes = [C.c_void_p, C.POINTER(KvView), C.c_void_p, C.c_int32, C.c_void_p, C.c_int64] + \
            [C.c_void_p] * 4
        L.tria_evict_mass.argtypes = [C.c_void_p, C.POINTER(KvView), C.POINTER(KvView), C.c_void_p, C.c_void_p, C.c_void_p,
                                      C.POINTER(EvictParams), C.c_void_p, C.c_void_p]
        L.tria_score_kv_head_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32,
                                             C.c_int32, C.c_int32, C.c_int32, C.c_void_p, C.c_void_p]
        _lib = L
    return _lib


def exported_symbols_in_header(paths=None):
    """Names of every function the public headers declare with TRIA_API."""
    names = set()
    for path in paths or HEADERS:
        txt = open(path).read()
        names |= set(re.findall(r"TRIA_API\s+[^;(]*?\b(tria_\w+)\s*\(", txt))
    return sorted(names)


def last_error() -> str:
    return lib().tria_last_error().decode()


def check(status: int) -> None:
    if status != OK:
        raise TriaError(status, f"{lib().tria_status_str(status).decode()}: {last_error()}")


# ---------------- reference API ----------------

def load(path: str):
    """tria_load: returns a ctypes pointer to Stats (falsy on failure)."""
    p = lib().tria_load(os.fsencode(path))
    return p if p else None


def free(stats) -> None:
    if stats:
        lib().tria_free(stats)


def score_kv_head(stats, k_re, k_im, key_pos, cur_pos, layer, kv_head):
    """tria_score_kv_head on host arrays (fp32 [n, fc] halves, int32 positions)."""
    k_re = np.ascontiguousarray(k_re, np.float32)
    k_im = np.ascontiguousarray(k_im, np.float32)
    key_pos = np.ascontiguousarray(key_pos, np.int32)
    n = int(key_pos.shape[0])
    out = np.empty(max(n, 1), np.float32)
    lib().tria_score_kv_head(stats, k_re.ctypes.data, k_im.ctypes.data, key_pos.ctypes.data,
                             int(cur_pos), n, int(layer), int(kv_head), out.ctypes.data)
    return out[:n]


def layer_budget(stats, layer, base_budget):
    """tria_layer_budget (the header's static inline, restated for Python)."""
    scale = np.float32(stats.contents.layer_budget_scales[layer])
    b = int(np.float32(np.float32(base_budget) * scale))
    return b if b > 0 else 1


# ---------------- device path ----------------

NOALLOC_MAX_KEYS = 1 << 20


def znorm_stats(x, stride, n, mean_std, stream=None):
    """tria_znorm_stats: exact (mean, std) of each row of device array x."""
    nn = np.ascontiguousarray(n, np.int32)
    check(lib().tria_znorm_stats(_ptr(x), int(stride), nn.ctypes.data, int(nn.shape[0]),
                                 _ptr(mean_std), _stream(stream)))


def checked_build() -> bool:
    """tria_checked_build: True when the loaded library is the checked build."""
    return bool(lib().tria_checked_build())


def score_key(x: float) -> int:
    """tria_score_key: the order-preserving 32-bit key of a score."""
    return int(lib().tria_score_key(float(x)))


def key_histogram(scores, score_stride, n_rows, level, prefix, hist, stream=None):
    """tria_key_histogram: add the 16-bit bins of the keys of device `scores`
    ([units][score_stride]) to device `hist` [65536] uint32."""
    nr = np.ascontiguousarray(n_rows, np.int32)
    check(lib().tria_key_histogram(_ptr(scores), int(score_stride), nr.ctypes.data, int(nr.shape[0]),
                                   int(level), int(prefix), _ptr(hist), _stream(stream)))


def key_gather(scores, score_stride, n_rows, key_min, out, cap, count, stream=None):
    """tria_key_gather: scores of the units' rows with key >= key_min into
    device `out` [cap]; device `count` [1] int32 gets how many there were."""
    nr = np.ascontiguousarray(n_rows, np.int32)
    check(lib().tria_key_gather(_ptr(scores), int(score_stride), nr.ctypes.data, int(nr.shape[0]),
                                int(key_min), _ptr(out), int(cap), _ptr(count), _stream(stream)))


def key_count(scores, score_stride, n_rows, key, counts, stream=None):
    """tria_key_count: per-unit counts of rows whose key equals `key`."""
    nr = np.ascontiguousarray(n_rows, np.int32)
    check(lib().tria_key_count(_ptr(scores), int(score_stride), nr.ctypes.data, int(nr.shape[0]),
                               int(key), _ptr(counts), _stream(stream)))


def select_key(scores, score_stride, n_rows, key, counts, tie_allow, kept_idx, kept_stride, n_kept, stream=None):
    """tria_select_key: keep rows with key > `key` and the first `tie_allow`
    rows equal to it (unit order), kept indices ascending per unit."""
    nr = np.ascontiguousarray(n_rows, np.int32)
    check(lib().tria_select_key(_ptr(scores), int(score_stride), nr.ctypes.data, int(nr.shape[0]), int(key),
                                _ptr(counts), int(tie_allow), _ptr(kept_idx), int(kept_stride), _ptr(n_kept),
                                _stream(stream)))


def select_noalloc(scores, score_stride, n_rows, keep, kept_idx, kept_stride, n_kept,
                   pos=None, pos_stride=0, cur_pos=0, window=0, sink=0, stream=None):
    """tria_select_noalloc: rank device scores with no allocation (fixed static
    scratch of NOALLOC_MAX_KEYS keys; see the header)."""
    nr = np.ascontiguousarray(n_rows, np.int32)
    kp = np.ascontiguousarray(keep, np.int32)
    assert nr.shape == kp.shape
    check(lib().tria_select_noalloc(_ptr(scores), int(score_stride), nr.ctypes.data, kp.ctypes.data,
                                    int(nr.shape[0]), _ptr(pos), int(pos_stride), int(cur_pos),
                                    int(window), int(sink), _ptr(kept_idx), int(kept_stride),
                                    _ptr(n_kept), _stream(stream)))

def _ptr(x) -> int:
    """Device pointer of a torch tensor or an int."""
    if x is None:
        return 0
    if isinstance(x, int):
        return x
    return int(x.data_ptr())


def _stream(stream) -> int:
    if stream is None:
        return 0
    if isinstance(stream, int):
        return stream
    return int(stream.cuda_stream)


def make_view(type_id, k_layers, v_layers, pos, n_cells, cell_stride, head_stride,
              n_head_kv, layer0=0, head0=0, pos_shared=False, flags=0):
    """Build a KvView; k_layers / v_layers are lists of torch tensors or device pointers.
    The returned view keeps its pointer arrays alive."""
    nl = len(k_layers)
    karr = (C.c_void_p * nl)(*[_ptr(t) for t in k_layers])
    varr = (C.c_void_p * nl)(*[_ptr(t) for t in v_layers]) if v_layers is not None else None
    v = KvView(type_id, nl, layer0, n_head_kv, head0, n_cells, cell_stride, head_stride,
               C.cast(karr, C.POINTER(C.c_void_p)),
               C.cast(varr, C.POINTER(C.c_void_p)) if varr is not None else None,
               _ptr(pos), 1 if pos_shared else 0, int(flags))
    v._keep = (karr, varr, k_layers, v_layers, pos)
    return v


class Context:
    def __init__(self, stats, device: int = 0):
        h = C.c_void_p()
        check(lib().tria_ctx_create(stats, device, C.byref(h)))
        self.h = h
        self.stats = stats
        s = stats.contents
        self.head_dim, self.gqa, self.device = int(s.head_dim), int(s.num_heads // s.num_kv_heads), int(device)

    def close(self):
        if self.h:
            lib().tria_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def _rows(n_rows):
        a = np.ascontiguousarray(n_rows, np.int32)
        return a, a.ctypes.data

    def score(self, view, n_rows, cur_pos, scores, stream=None):
        a, p = self._rows(n_rows)
        check(lib().tria_score(self.h, C.byref(view), p, int(cur_pos), _ptr(scores), _stream(stream)))

    def select(self, view, n_rows, scores, params, kept_idx, n_kept, stream=None):
        a, p = self._rows(n_rows)
        check(lib().tria_select(self.h, C.byref(view), p, _ptr(scores), C.byref(params),
                                _ptr(kept_idx), _ptr(n_kept), _stream(stream)))

    def compact(self, src, dst, n_rows, kept_idx, n_kept, stream=None):
        a, p = self._rows(n_rows)
        check(lib().tria_compact(self.h, C.byref(src), C.byref(dst), p, _ptr(kept_idx),
                                 _ptr(n_kept), _stream(stream)))

    def evict(self, src, dst, n_rows, params, n_kept_out=None, stream=None):
        a, p = self._rows(n_rows)
        check(lib().tria_evict(self.h, C.byref(src), C.byref(dst), p, C.byref(params),
                               _ptr(n_kept_out), _stream(stream)))

    def ggml_evict(self, src, dst, n_rows, params, stream=None):
        """tria_ggml_evict: one step on ggml-described caches (GgmlCache)."""
        a, p = self._rows(n_rows)
        check(lib().tria_ggml_evict(self.h, C.byref(src), C.byref(dst), p, C.byref(params), _stream(stream)))

    def evict_host(self, src, dst, n_rows, params, stream=None):
        """tria_evict_host: src/dst views over page-locked host buffers."""
        a, p = self._rows(n_rows)
        check(lib().tria_evict_host(self.h, C.byref(src), C.byref(dst), p, C.byref(params), _stream(stream)))

    def get_n_kv(self, units: int = 0):
        buf = np.zeros(max(units, 1), np.int32)
        r = lib().tria_get_n_kv(self.h, buf.ctypes.data if units else None, units)
        if r < 0:
            check(r)
        return r, buf[:units]

    def set_timing(self, on: bool = True):
        check(lib().tria_ctx_set_timing(self.h, 1 if on else 0))

    STAGES = ("table", "score", "znorm", "select", "compact")

    def stage_ms(self):
        """Device ms per stage of the last timed evict: dict stage -> ms."""
        buf = np.zeros(5, np.float32)
        k = lib().tria_ctx_stage_ms(self.h, buf.ctypes.data, 5)
        if k < 0:
            check(k)
        return {n: float(buf[i]) for i, n in enumerate(self.STAGES[:k])}

    def launches(self) -> int:
        return int(lib().tria_ctx_launches(self.h))

    def check(self, stream=None):
        """tria_ctx_check: raise TriaError if a kernel of this context reported a
        bad position or a pipeline timeout since the last check."""
        check(lib().tria_ctx_check(self.h, _stream(stream)))

    def set_wait_limit(self, cycles: int = 0):
        """tria_ctx_set_wait_limit (timeout-path tests): 0 restores the default."""
        check(lib().tria_ctx_set_wait_limit(self.h, int(cycles)))

    def set_select_split(self, max_ctas: int = 0):
        """tria_ctx_set_select_split: CTAs per unit in selection (0 automatic, 1 one block)."""
        check(lib().tria_ctx_set_select_split(self.h, int(max_ctas)))

    def score_kv_head_dev(self, k_re, k_im, key_pos, cur_pos, n, layer, kv_head, out, stream=None):
        check(lib().tria_score_kv_head_dev(self.h, _ptr(k_re), _ptr(k_im), _ptr(key_pos), int(cur_pos),
                                           int(n), int(layer), int(kv_head), _ptr(out), _stream(stream)))

    # ---- serving from an evicted cache ----

    def append(self, view, n_rows, k, v, tok_pos, n_rows_out=None, mass=None, stream=None):
        """tria_append: device tensors k, v [caches][n_tok][kv heads][head_dim]
        (f16 or fp32, contiguous last dimension) behind each unit's n_rows (device
        int32); n_rows_out defaults to n_rows, updated in place."""
        L, KV, T = view.n_layer, view.n_head_kv, _torch()
        shape, stride, dtype = k.shape, k.stride(), k.dtype
        if len(shape) != 4 or stride[3] != 1 or v.shape != shape or v.stride() != stride or v.dtype != dtype:
            raise ValueError("k and v must have the same shape [caches][n_tok][kv heads][head_dim], type and strides, the last "
                             "dimension contiguous")
        f32 = dtype is T.float32
        if not f32 and dtype is not T.float16:
            raise ValueError(f"k and v must be float16 or float32, not {dtype}")
        if shape[0] != L or shape[2] != KV or shape[3] != self.head_dim:
            raise ValueError(f"k of shape {tuple(shape)} for {L} caches of {KV} heads of {self.head_dim}")
        own = tok_pos.dim() == 2
        if tok_pos.dtype is not T.int32 or tok_pos.shape != ((L, shape[1]) if own else (shape[1],)) or \
                (shape[1] > 1 and tok_pos.stride(-1) != 1):
            raise ValueError(f"tok_pos must be int32 [{shape[1]}] or [{L}][{shape[1]}] with a contiguous last dimension")
        if mass is not None:
            self._mass(mass, view)
        rows_out = n_rows if n_rows_out is None else n_rows_out
        self._counts(L * KV, n_rows, rows_out)
        dev = self.device
        if k.get_device() != dev or v.get_device() != dev or tok_pos.get_device() != dev:
            self._elsewhere(k, v, tok_pos)
        p = AppendParams(shape[1], SRC_F32 if f32 else SRC_F16, stride[0], stride[1], stride[2], tok_pos.data_ptr(),
                         tok_pos.stride(0) if own else 0)
        r = _lib.tria_append(self.h, C.byref(view), n_rows.data_ptr(), C.byref(p), k.data_ptr(), v.data_ptr(),
                             0 if mass is None else mass.data_ptr(), rows_out.data_ptr(), _stream(stream))
        if r:
            check(r)

    def attend(self, view, n_rows, q, out, params, lse=None, mass_in=None, mass_out=None, stream=None):
        """tria_attend: device f16 tensors q, out [caches][n_tok][heads][head_dim]
        (any strides that are multiples of 8, the last dimension contiguous)."""
        L, KV = view.n_layer, view.n_head_kv
        sig = (self.device, self.gqa, self.head_dim, L, KV, q.shape, q.stride(), out.shape, out.stride(), q.dtype, out.dtype)
        if params._sig != sig:
            self._attend_shapes(view, q, out, params)
            params._sig = sig
        if lse is not None:
            if lse.dtype is not _torch().float32 or lse.shape != q.shape[:3] or not lse.is_contiguous():
                raise ValueError("lse must be a contiguous fp32 [caches][n_tok][heads]")
            self._here(lse)
        if mass_out is not None:
            self._mass(mass_out, view)
        if mass_in is not None:
            self._mass(mass_in, view)
        self._counts(L * KV, n_rows)
        dev = self.device
        if q.get_device() != dev or out.get_device() != dev:
            self._elsewhere(q, out)
        r = _lib.tria_attend(self.h, C.byref(view), n_rows.data_ptr(), C.byref(params), q.data_ptr(), out.data_ptr(),
                             0 if lse is None else lse.data_ptr(), 0 if mass_in is None else mass_in.data_ptr(),
                             0 if mass_out is None else mass_out.data_ptr(), _stream(stream))
        if r:
            check(r)

    def _attend_shapes(self, view, q, out, params):
        """Checks q and out against the view and the params, and puts their strides into the params."""
        f16 = _torch().float16
        if q.dtype != f16 or out.dtype != f16 or q.dim() != 4 or out.shape != q.shape or q.stride(3) != 1 or out.stride(3) != 1:
            raise ValueError("q and out must be float16 of the same shape [caches][n_tok][heads][head_dim], the last dimension "
                             "contiguous")
        if q.shape[0] != view.n_layer or q.shape[2] != view.n_head_kv * self.gqa or q.shape[3] != self.head_dim:
            raise ValueError(f"q of shape {tuple(q.shape)} for {view.n_layer} caches of {view.n_head_kv} x {self.gqa} heads "
                             f"of {self.head_dim}")
        slopes, tok_pos, tree = params._keep
        self._here(*params._keep)
        if slopes is not None and slopes.shape[0] != q.shape[2]:
            raise ValueError(f"{slopes.shape[0]} slopes for {q.shape[2]} heads")
        self._shared_or_own(tok_pos, "tok_pos", (q.shape[1],), view.n_layer)
        self._shared_or_own(tree, "tree", (q.shape[1], params.tree_words), view.n_layer)
        params.n_tok = q.shape[1]
        params.q_cache_stride, params.q_tok_stride, params.q_head_stride = q.stride()[:3]
        params.o_cache_stride, params.o_tok_stride, params.o_head_stride = out.stride()[:3]

    def accept(self, view, n_rows, n_tok, path, n_path, n_rows_out=None, mass=None, stream=None):
        """tria_accept: device int32 path [caches or 1][entries] and n_path [caches or 1]."""
        L, KV, i32 = view.n_layer, view.n_head_kv, _torch().int32
        if path.dtype is not i32 or path.dim() != 2 or n_path.dtype is not i32 or not n_path.is_contiguous():
            raise ValueError("path must be an int32 [caches or 1][entries], n_path a contiguous int32 [caches or 1]")
        lists, entries = path.shape
        if (lists != 1 and lists != L) or n_path.numel() != lists or (path.stride(1) != 1 and entries > 1):
            raise ValueError("path must be [caches or 1][entries], its rows contiguous, n_path [caches or 1]")
        if entries < n_tok:
            raise ValueError(f"path holds {entries} entries a cache: room for n_tok = {n_tok} is wanted")
        if mass is not None:
            self._mass(mass, view)
        rows_out = n_rows if n_rows_out is None else n_rows_out
        self._counts(L * KV, n_rows, rows_out)
        if path.get_device() != self.device or n_path.get_device() != self.device:
            self._elsewhere(path, n_path)
        r = _lib.tria_accept(self.h, C.byref(view), n_rows.data_ptr(), n_tok, path.data_ptr(), path.stride(0) if lists > 1 else 0,
                             n_path.data_ptr(), 0 if mass is None else mass.data_ptr(), rows_out.data_ptr(), _stream(stream))
        if r:
            check(r)

    def evict_mass(self, src, dst, n_rows, mass, mass_dst, params, n_kept_out=None, stream=None):
        """tria_evict_mass: one eviction step ranked by device `mass`
        [layers][kv heads][n_cells]; n_rows is a host array."""
        a, p = self._rows(n_rows)
        self._mass(mass, src)
        if mass_dst is not None:
            self._mass(mass_dst, dst)
        if a.shape[0] != src.n_layer * src.n_head_kv:
            raise ValueError(f"{a.shape[0]} row counts for {src.n_layer} x {src.n_head_kv} units")
        if n_kept_out is not None:
            self._counts(src.n_layer * src.n_head_kv, n_kept_out)
        check(lib().tria_evict_mass(self.h, C.byref(src), C.byref(dst), p, _ptr(mass), _ptr(mass_dst), C.byref(params),
                                    _ptr(n_kept_out), _stream(stream)))

    def _here(self, *tensors):
        """Tensors that kernels read or write must live on the context's device."""
        for x in tensors:
            if x is not None and x.get_device() != self.device:
                self._elsewhere(x)

    def _elsewhere(self, *tensors):
        raise ValueError(f"a tensor on {', '.join(str(x.device) for x in tensors)} was given to a context of cuda:{self.device}")

    def _counts(self, units, *counts):
        for x in counts:
            if x.dtype is not _torch().int32 or x.numel() != units or x.get_device() != self.device or not x.is_contiguous():
                raise ValueError(f"row counts must be a contiguous int32 tensor of {units} units on cuda:{self.device}")

    @staticmethod
    def _shared_or_own(x, name, shape, caches):
        if x is not None and tuple(x.shape) not in (shape, (caches,) + shape):
            raise ValueError(f"{name} of shape {tuple(x.shape)}: {shape} or {(caches,) + shape} is wanted")

    def _mass(self, x, view):
        if x.dtype is not _torch().float32 or x.shape != (view.n_layer, view.n_head_kv, view.n_cells) \
                or x.get_device() != self.device or not x.is_contiguous():
            raise ValueError(f"mass must be a contiguous fp32 [{view.n_layer}][{view.n_head_kv}][{view.n_cells}] tensor on "
                             f"cuda:{self.device}")
