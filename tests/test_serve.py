"""CPU tests of the serving calls: their symbols and refusals.  The checks that
need no device run before the context is looked at, so they are reached here
without one; a call that passes them all is refused for its null context."""
import ctypes as C

import numpy as np
import pytest

import tria_b200
from tria_b200 import ERR_INVALID, ERR_UNSUPPORTED, EvictParams, TYPE_F16, TYPE_Q8_0

FAKE = 4096            # an aligned address that is never read: the checks come first


@pytest.fixture(scope="module")
def L():
    import os
    if not os.path.exists(tria_b200.LIB_PATH):
        tria_b200.build()
    return tria_b200.lib()


def view(**kw):
    a = dict(type_id=TYPE_F16, k=[FAKE, FAKE], v=[FAKE, FAKE], pos=FAKE, n_cells=64, cell=512, head=256, kv=2,
             shared=False, flags=tria_b200.VIEW_POST_ROPE)
    a.update(kw)
    return tria_b200.make_view(a["type_id"], a["k"], a["v"], a["pos"], a["n_cells"], a["cell"], a["head"], a["kv"],
                               pos_shared=a["shared"], flags=a["flags"])


def attend(L, v=None, n_rows=FAKE, q=FAKE, out=2 * FAKE, lse=None, mass_in=None, mass_out=None, **kw):
    p = tria_b200.AttendParams()
    p.n_tok, p.scale, p.mass_decay = 1, 0.125, 1.0
    p.o_cache_stride, p.o_tok_stride, p.o_head_stride = 512, 512, 128
    for k, x in kw.items():
        setattr(p, k, x)
    return L.tria_attend(None, C.byref(v if v is not None else view()), n_rows, C.byref(p), q, out, lse, mass_in, mass_out, None)


def append(L, v=None, n_rows=FAKE, k=FAKE, vv=FAKE, mass=None, out=2 * FAKE, **kw):
    p = tria_b200.AppendParams()
    p.n_tok, p.src_type, p.tok_pos = 1, tria_b200.SRC_F16, FAKE
    for a, x in kw.items():
        setattr(p, a, x)
    return L.tria_append(None, C.byref(v if v is not None else view()), n_rows, C.byref(p), k, vv, mass, out, None)


def accept(L, v=None, n_rows=FAKE, n_tok=4, path=FAKE, stride=0, n_path=FAKE, mass=None, out=2 * FAKE):
    return L.tria_accept(None, C.byref(v if v is not None else view()), n_rows, n_tok, path, stride, n_path, mass, out, None)


def evict(L, rows=None, mass=FAKE, mass_dst=2 * FAKE, p=None):
    rows = np.full(4, 8, np.int32) if rows is None else rows
    p = EvictParams(100, 4, 100, 0, 0, 0) if p is None else p
    return L.tria_evict_mass(None, C.byref(view()), C.byref(view()), rows.ctypes.data, mass, mass_dst, C.byref(p), None, None)


def refused(r, word, status=ERR_INVALID):
    assert r == status, (r, tria_b200.last_error())
    assert word in tria_b200.last_error(), tria_b200.last_error()


@pytest.mark.parametrize("call", [attend, append, accept, evict])
def test_a_good_call_reaches_the_context_check(L, call):
    refused(call(L), "null context")


@pytest.mark.parametrize("call", [attend, append, accept])
@pytest.mark.parametrize("kw,word,status", [
    (dict(type_id=2), "cache type", ERR_UNSUPPORTED),
    (dict(flags=0), "POST_ROPE", ERR_UNSUPPORTED),
    (dict(flags=3), "flags", ERR_INVALID),
    (dict(kv=0), "kv heads", ERR_INVALID),
    (dict(kv=2049), "kv heads", ERR_INVALID),
    (dict(k=[], v=[]), "caches", ERR_INVALID),
    (dict(n_cells=-1), "n_cells", ERR_INVALID),
    (dict(cell=510), "strides", ERR_INVALID),
    (dict(cell=0), "strides", ERR_INVALID),
    (dict(head=-256), "strides", ERR_INVALID),
    (dict(pos=None), "null", ERR_INVALID),
    (dict(pos=FAKE + 2), "pos misaligned", ERR_INVALID),
    (dict(v=None), "null", ERR_INVALID),
    (dict(k=[FAKE, FAKE + 8]), "k[1]", ERR_INVALID),
    (dict(v=[None, FAKE]), "v[0]", ERR_INVALID),
])
def test_views(L, call, kw, word, status):
    refused(call(L, v=view(**kw)), word, status)


@pytest.mark.parametrize("kw,word", [
    (dict(n_rows=None), "n_rows"), (dict(n_rows=FAKE + 1), "n_rows"),
    (dict(n_tok=-1), "negative"), (dict(window=-1), "negative"), (dict(sink=-1), "negative"),
    (dict(reserved=1), "reserved"), (dict(scale=float("nan")), "finite"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("inf")), "finite"), (dict(mass_decay=float("inf")), "finite"),
    (dict(mass_in=FAKE), "mass_in without"), (dict(mass_out=FAKE + 2), "misaligned"), (dict(lse=FAKE + 2), "misaligned"),
    (dict(o_cache_stride=0), "overlap"), (dict(n_tok=2, o_tok_stride=0), "overlap"), (dict(o_head_stride=0), "overlap"),
    (dict(out=FAKE), "overlap"), (dict(scale=3e38), "range"), (dict(scale=1e10, softcap=1e-30), "range"),
    (dict(q=None), "q or out"), (dict(out=FAKE + 8), "q or out"), (dict(q_tok_stride=4), "strides"),
    (dict(o_head_stride=-8), "strides"), (dict(slopes=FAKE), "tok_pos"), (dict(window=5), "tok_pos"),
    (dict(window=5, tok_pos=FAKE, tok_pos_stride=-1), "tok_pos_stride"), (dict(slopes=FAKE + 1, tok_pos=FAKE), "slopes"),
    (dict(tree=FAKE), "tree_words"), (dict(tree=FAKE, tree_words=1, n_tok=33), "tree_words"),
    (dict(tree=FAKE, tree_words=1, tree_stride=-1), "tree_stride"), (dict(tree=FAKE + 2, tree_words=1), "tree misaligned"),
])
def test_attend(L, kw, word):
    refused(attend(L, **kw), word)


@pytest.mark.parametrize("kw,word,status", [
    (dict(n_rows=None), "n_rows", ERR_INVALID), (dict(out=None), "n_rows_out", ERR_INVALID),
    (dict(n_tok=-1), "n_tok", ERR_INVALID), (dict(src_type=8), "source type", ERR_UNSUPPORTED),
    (dict(tok_pos=None), "tok_pos", ERR_INVALID), (dict(tok_pos_stride=-1), "tok_pos_stride", ERR_INVALID),
    (dict(v=view(shared=True), tok_pos_stride=4), "shared positions", ERR_INVALID),
    (dict(k=None), "k or v", ERR_INVALID), (dict(vv=FAKE + 8), "k or v", ERR_INVALID),
    (dict(tok_stride=4), "strides", ERR_INVALID), (dict(src_type=0, tok_stride=2), "strides", ERR_INVALID),
    (dict(mass=FAKE + 1), "mass", ERR_INVALID), (dict(out=FAKE + 4), "overlap", ERR_INVALID),
])
def test_append(L, kw, word, status):
    refused(append(L, **kw), word, status)


@pytest.mark.parametrize("kw,word", [
    (dict(n_rows=FAKE + 2), "n_rows"), (dict(path=None), "path"), (dict(n_path=None), "n_path"),
    (dict(n_tok=-1), "negative"), (dict(stride=-1), "negative"), (dict(mass=FAKE + 2), "mass"),
    (dict(v=view(shared=True), stride=4), "shared positions"), (dict(out=FAKE + 4), "overlap"),
])
def test_accept(L, kw, word):
    refused(accept(L, **kw), word)


def test_evict_mass(L):
    refused(evict(L, mass=None), "null")
    refused(evict(L, mass=FAKE + 1), "misaligned")
    refused(evict(L, mass_dst=FAKE), "different arrays")
    refused(evict(L, p=EvictParams(-1, 4, 100, 0, 0, 0)), "cur_pos")


def test_status_string(L):
    assert b"row count" in L.tria_status_str(tria_b200.ERR_ROWS)


def test_binding_checks_tensors():
    import torch
    f = torch.zeros
    with pytest.raises(ValueError, match="slopes"):
        tria_b200.attend_params(1.0, slopes=f(4, dtype=torch.float16))
    with pytest.raises(ValueError, match="tok_pos"):
        tria_b200.attend_params(1.0, tok_pos=f(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="tok_pos"):
        tria_b200.attend_params(1.0, tok_pos=f((4, 2), dtype=torch.int32)[:, 0])
    with pytest.raises(ValueError, match="tree"):
        tria_b200.attend_params(1.0, tree=f((4, 2), dtype=torch.int32)[:, :1])
    p = tria_b200.attend_params(0.5, tok_pos=f((3, 4), dtype=torch.int32), tree=f((3, 4, 2), dtype=torch.int32))
    assert (p.tok_pos_stride, p.tree_stride, p.tree_words) == (4, 8, 2)
