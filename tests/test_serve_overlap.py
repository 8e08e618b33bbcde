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
