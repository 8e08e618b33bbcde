"""CPU tests: writing calls refuse outputs, views and arrays that overlap.  The
rows of a call without a context are at least those of head_dim 64 and one query
head per kv head; test_gpu_serve_calls.py has the contexts' own sizes."""
import pytest

from test_serve import FAKE, L, accept, append, attend, evict, refused, view  # noqa: F401 (L is a fixture)


@pytest.mark.parametrize("kw", [
    dict(o_head_stride=8), dict(o_head_stride=56), dict(o_cache_stride=8), dict(o_cache_stride=128),
    dict(n_tok=3, o_tok_stride=8, o_cache_stride=4096), dict(n_tok=3, o_tok_stride=128, o_cache_stride=4096),
    dict(n_tok=3, o_tok_stride=256, o_cache_stride=512), dict(n_tok=2, o_tok_stride=64, o_head_stride=64),
    dict(o_cache_stride=2 ** 62, n_tok=2, o_tok_stride=2 ** 62),
])
def test_out_strides(L, kw):
    refused(attend(L, **kw), "overlap")


@pytest.mark.parametrize("kw", [
    dict(o_head_stride=64, o_cache_stride=128), dict(n_tok=3, o_tok_stride=64, o_head_stride=192, o_cache_stride=384),
    dict(n_tok=3, o_tok_stride=256, o_head_stride=64, o_cache_stride=704), dict(n_tok=2 ** 20, o_cache_stride=2 ** 30),
    dict(n_tok=2, o_cache_stride=64, o_tok_stride=128, o_head_stride=256), dict(o_tok_stride=0),
])
def test_out_strides_that_keep_rows_apart(L, kw):
    refused(attend(L, **kw), "null context")


@pytest.mark.parametrize("call", [append, accept])
@pytest.mark.parametrize("kw,bad", [
    (dict(head=0), True), (dict(head=64), True), (dict(cell=64), True), (dict(cell=128, head=64), True),
    (dict(cell=192, head=128), True),                      # cells shorter than their two heads
    (dict(cell=128, head=63 * 128), True),                 # head-major, the last row on the next head
    (dict(cell=128, head=64 * 128 - 4), True), (dict(cell=512, head=3 * 512 - 64), True),
    (dict(cell=2 ** 62, head=2 ** 62), True),              # a head on the next cell, past 63 bits
    (dict(cell=256, head=128), False), (dict(cell=128, head=64 * 128), False), (dict(cell=260, head=132), False),
    (dict(cell=384, head=256), False),                     # between the cells of the first head
    (dict(cell=512, head=3 * 512 + 128), False),           # and some cells on
    (dict(kv=1, head=0), False), (dict(n_cells=1, cell=4, head=128), False), (dict(n_cells=0, head=0), False),
    (dict(type_id=8, cell=136, head=68), False), (dict(type_id=8, cell=136, head=64), True),
    (dict(type_id=8, cell=132, head=68), True), (dict(type_id=8, kv=8, cell=8 * 68, head=68), False),
    (dict(type_id=8, kv=8, cell=7 * 68, head=68), True),
])
def test_views_whose_rows_overlap(L, call, kw, bad):
    refused(call(L, v=view(**kw)), "rows of" if bad else "null context")


def test_views_that_are_only_read_may_overlap(L):
    refused(attend(L, v=view(head=0)), "null context")     # one kv head for all


@pytest.mark.parametrize("off,bad", [(4, True), (1020, True), (1024, False), (-4, True), (-1020, True), (-1024, False), (0, False)])
def test_masses_that_overlap_in_part(L, off, bad):
    """Arrays of 2 x 2 x 64 masses: the same one, apart, or neither."""
    refused(attend(L, mass_in=16 * FAKE, mass_out=16 * FAKE + off), "overlap in part" if bad else "null context")
    if off:
        refused(evict(L, mass=16 * FAKE, mass_dst=16 * FAKE + off), "overlap" if bad else "null context")
