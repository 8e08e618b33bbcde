"""GPU tests of how the serving calls may be made: steps of other sizes between
a capture and its replay, and views, strides and arrays that the calls refuse."""

import numpy as np
import pytest
import torch

import tria_b200
from serve_cases import Cache, F16, Q8_0, attend_close, attend_oracle
from test_gpu_serve import contexts, kept_oracle, queries  # noqa: F401 (contexts is a fixture)

pytestmark = pytest.mark.gpu


def eviction(L, rows, cells, dev, seed):
    """An evict_mass step over L layers of two kv heads: (caches, masses, call)."""
    c, d = Cache(F16, L, 2, 128, cells, rows, dev, seed=seed), Cache(F16, L, 2, 128, cells, rows, dev, seed=seed + 1)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    mass = torch.rand((L, 2, cells), generator=g, device=dev)
    md = torch.zeros_like(mass)
    prm = tria_b200.EvictParams(10 ** 5, 60 + seed, 100, 0, 0, 0)
    n = np.asarray(rows, np.int32)
    keep = np.minimum(n, 60 + seed)

    def call(ctx, stream):
        ctx.evict_mass(c.view(), d.view(), n, mass, md, prm, stream=stream)

    def check():
        for u in range(2 * L):
            l, h = divmod(u, 2)
            idx = kept_oracle(mass[l, h].cpu().numpy(), c.pos[l, h].cpu().numpy(), int(n[u]), int(keep[u]), 10 ** 5, 0, 0)
            assert torch.equal(md[l, h, :len(idx)], mass[l, h][torch.from_numpy(idx).to(dev)])
    return call, check, keep


def test_replayed_evictions_of_several_sizes(torch_dev, tmp_path):
    """A step of one layer captured, then an eager one of three layers, then one
    of three layers captured: every replay reads back its own counts, whatever
    ran in between, and the read-back buffer stays where the graphs have it."""
    import workloads
    p = str(tmp_path / "s.tria")
    workloads.write_tria(p, 3, 8, 2, 128, seed=1)
    st = tria_b200.load(p)
    ctx = tria_b200.Context(st, 0)
    s = torch.cuda.Stream()
    small, small_ok, small_n = eviction(1, [700, 500], 900, torch_dev, 0)
    large, large_ok, large_n = eviction(3, [100, 200, 300, 40, 0, 128], 128 + 172, torch_dev, 9)
    torch.cuda.synchronize()
    graphs = []
    for call in (small, large):
        with torch.cuda.stream(s):
            call(ctx, s)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(ctx, torch.cuda.current_stream())
        graphs.append(g)
    for i in (0, 1, 0, 0, 1):
        ok, want = ((small_ok, small_n), (large_ok, large_n))[i]
        with torch.cuda.stream(s):
            graphs[i].replay()
        most, counts = ctx.get_n_kv(6)
        assert counts[:len(want)].tolist() == want.tolist() and most == want.max()
        assert (counts[len(want):] == 0).all()
        ok()
    with torch.cuda.stream(s):
        large(ctx, s)
        graphs[0].replay()
    most, counts = ctx.get_n_kv(6)
    assert counts.tolist() == small_n.tolist() + [0] * 4 and most == small_n.max()
    del graphs, g
    ctx.close()
    tria_b200.free(st)


def test_a_larger_step_captured_first(torch_dev, tmp_path):
    """More units than any step before, in scratch that is large enough: nothing has to grow inside the capture."""
    import workloads
    p = str(tmp_path / "s.tria")
    workloads.write_tria(p, 3, 8, 2, 128, seed=1)
    st = tria_b200.load(p)
    ctx = tria_b200.Context(st, 0)
    s = torch.cuda.Stream()
    wide, _, wide_n = eviction(1, [3000, 2900], 3000, torch_dev, 0)
    tall, tall_ok, tall_n = eviction(3, [100, 200, 300, 40, 0, 128], 300, torch_dev, 5)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        wide(ctx, s)
    assert ctx.get_n_kv(2)[1].tolist() == wide_n.tolist()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        tall(ctx, torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g.replay()
    assert ctx.get_n_kv(6)[1].tolist() == tall_n.tolist()
    tall_ok()
    del g
    ctx.close()
    tria_b200.free(st)


def strided(b, *strides, at=0, shape=(2, 3, 8, 128)):
    return torch.as_strided(b, shape, strides + (1,), at)


@pytest.mark.parametrize("kv,heads", [(2, 8), (1, 4)])
def test_outputs_that_overlap_are_refused(contexts, torch_dev, kv, heads):
    """Strides below a row, below what the smaller ones span, and 0, for several
    kv heads and for one with several query heads; q and out that share bytes."""
    c = Cache(F16, 2, kv, 128, 100, [90, 80, 70, 60][:2 * kv], torch_dev)
    ctx, q = contexts(kv, 4, 128), queries(2, 3, heads, 128, torch_dev)
    b = torch.zeros(1 << 16, dtype=torch.float16, device=torch_dev)
    shape = (2, 3, heads, 128)
    p = tria_b200.attend_params(0.1)
    w = heads * 128
    for o in ((3 * w, w, 0), (3 * w, w, 8), (3 * w, w, 120), (3 * w, w - 8, 128), (3 * w - 8, w, 128), (0, w, 128), (3 * w, 0, 128),
              (3 * w, 128, 3 * 128 - 8), (2 * 128 - 8, 2 * w, 128 * 2)):
        with pytest.raises(tria_b200.TriaError, match="overlap"):
            ctx.attend(c.view(), c.rows, q, strided(b, *o, shape=shape), p)
    # one buffer: the same rows, rows half on one another, the last row on the first, another order over the same bytes
    qb = strided(b, 3 * w, w, 128, at=4096, shape=shape)
    for o, at in (((3 * w, w, 128), 4096), ((3 * w, w, 128), 4096 + 64), ((3 * w, w, 128), 4096 - 64), ((3 * w, w, 128), 4096 + 128),
                  ((3 * w, w, 128), 4096 + 6 * w - 8), ((3 * w, 128, 3 * 128), 4096), ((3 * w, w, 128), 4096 - 6 * w + 8 if kv == 1 else 4104)):
        with pytest.raises(tria_b200.TriaError, match="overlap"):
            ctx.attend(c.view(), c.rows, qb, strided(b, *o, at=at, shape=shape), p)


def test_queries_and_outputs_in_one_buffer(contexts, torch_dev):
    """Interleaved head by head, token by token, behind one another, and with one
    cache's outputs before the next one's queries."""
    c = Cache(F16, 2, 2, 128, 300, [290, 222, 150, 151], torch_dev)
    ctx, q = contexts(2, 4, 128), queries(2, 3, 8, 128, torch_dev)
    want = attend_oracle(c, q, 128 ** -0.5)
    p = tria_b200.attend_params(128 ** -0.5)
    w, s = 8 * 128, torch.cuda.current_stream()
    for strides, q_at, o_at in (((6 * w, 2 * w, 256), 0, 128), ((6 * w, 2 * w, 128), w, 0), ((3 * w, w, 128), 0, 6 * w),
                                ((3 * w, w, 128), 6 * w, 0), ((6 * w, w, 128), 3 * w, 0), ((2 * 128, 3 * 512, 512), 0, 128)):
        if strides[0] == 256:
            strides = (256, 8 * 512, 512)                 # caches innermost, q and out side by side in each
        b = torch.full((1 << 15,), 9.0, dtype=torch.float16, device=torch_dev)
        qv, ov = strided(b, *strides, at=q_at), strided(b, *strides, at=o_at)
        qv.copy_(q)
        ctx.attend(c.view(), c.rows, qv, ov, p, stream=s)
        ctx.check(s)
        assert torch.equal(qv, q)
        attend_close(c, ov, None, None, want)


def calls_that_write(ctx, c, view, dev):
    """append, accept and (into `view`) evict_mass, as callables."""
    x = torch.zeros((c.L, 1, c.KV, c.hd), dtype=torch.float16, device=dev)
    one = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    d = Cache(c.type, c.L, c.KV, c.hd, c.cells, c.rows_host, dev)
    mass = torch.zeros((c.L, c.KV, c.cells), device=dev)
    return [lambda: ctx.append(view, c.rows, x, x, torch.zeros(1, dtype=torch.int32, device=dev)),
            lambda: ctx.accept(view, c.rows, 1, one, one[0]),
            lambda: ctx.evict_mass(d.view(), view, c.rows_host.reshape(-1), mass, None, tria_b200.EvictParams(9, 4, 100, 0, 0, 0))]


@pytest.mark.parametrize("type_id,hd", [(F16, 128), (Q8_0, 128), (F16, 64)])
def test_views_that_writing_calls_refuse(contexts, torch_dev, type_id, hd):
    """Rows of this context's head_dim that overlap, and one cache listed twice."""
    ctx = contexts(2, 4, hd, layers=2)
    c = Cache(type_id, 2, 2, hd, 40, [9, 8, 7, 6], torch_dev)
    k, v, rb = [c.k[0], c.k[1]], [c.v[0], c.v[1]], c.rb
    k0, v0 = c.k.clone(), c.v.clone()

    def view(k, v, cell, head):
        return tria_b200.make_view(type_id, k, v, c.pos, 40, cell, head, 2, flags=tria_b200.VIEW_POST_ROPE)

    for cell, head, word in ((2 * rb, rb - 4, "rows of"), (2 * rb - 4, rb, "rows of"), (rb - 4, 20 * rb, "rows of"),
                             (rb, 40 * rb - 4, "rows of")):
        for call in calls_that_write(ctx, c, view(k, v, cell, head), torch_dev):
            with pytest.raises(tria_b200.TriaError, match=word):
                call()
    for kk, vv in (([k[0], k[0]], v), (k, [v[1], v[1]]), (k, [v[0], k[0]]), ([v[1], k[1]], v)):
        for call in calls_that_write(ctx, c, view(kk, vv, 2 * rb, rb), torch_dev):
            with pytest.raises(tria_b200.TriaError, match="twice"):
                call()
    m = torch.zeros((2, 2, 40), device=torch_dev)
    with pytest.raises(tria_b200.TriaError, match="different caches"):
        ctx.evict_mass(c.view(), c.view(), c.rows_host.reshape(-1), m, None, tria_b200.EvictParams(9, 4, 100, 0, 0, 0))
    torch.cuda.synchronize()
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0) and c.rows.tolist() == [[9, 8], [7, 6]]


def test_evicted_masses_that_overlap_are_refused(contexts, torch_dev):
    """mass and mass_dst of different lengths, sharing bytes at either end; side by side they are taken."""
    ctx = contexts(2, 4, 128)
    c, d = Cache(F16, 1, 2, 128, 64, [60, 50], torch_dev), Cache(F16, 1, 2, 128, 96, [60, 50], torch_dev)
    b = torch.rand(1024, device=torch_dev)
    prm = tria_b200.EvictParams(1000, 20, 100, 0, 0, 0)
    n = c.rows_host.reshape(-1)

    def call(m, md):
        ctx.evict_mass(c.view(), d.view(), n, b[m:m + 128].view(1, 2, 64), b[md:md + 192].view(1, 2, 96), prm,
                       stream=torch.cuda.current_stream())

    for m, md in ((0, 127), (0, 1), (192, 1), (192, 300), (200, 150)):
        with pytest.raises(tria_b200.TriaError, match="overlap"):
            call(m, md)
    for m, md in ((0, 128), (192, 0)):
        mass = b[m:m + 128].clone().view(2, 64)
        call(m, md)
        assert ctx.get_n_kv(2)[1].tolist() == [20, 20]
        for h in range(2):
            idx = kept_oracle(mass[h].cpu().numpy(), c.pos[0, h].cpu().numpy(), int(n[h]), 20, 1000, 0, 0)
            assert torch.equal(b[md:md + 192].view(2, 96)[h, :20], mass[h][torch.from_numpy(idx).to(torch_dev)])


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("opt", ["plain", "all"])
@pytest.mark.parametrize("T,G", [(4, 4), (1, 5), (3, 4)])
def test_masses_whose_scores_are_not_kept(contexts, torch_dev, type_id, opt, T, G):
    """Scores are kept for the masses up to 1 GiB: caches of 1.1 million cells,
    a few hundred of them in use, would need more at 16 query rows a unit (and
    with fewer query rows, more cells)."""
    KV, L = 8, 2
    cells = 1_100_000 * 16 // (T * G)
    rows = [290, 17, 64, 203, 130, 299, 65, 128, 16, 33, 300, 256, 100, 4, 211, 48]
    c = Cache(type_id, L, KV, 128, 300, rows, torch_dev, shared=True)
    pos = torch.zeros(cells, dtype=torch.int32, device=torch_dev)
    pos[:300] = c.pos
    view = tria_b200.make_view(type_id, [c.k[0], c.k[1]], [c.v[0], c.v[1]], pos, cells, c.cell_stride, c.head_stride, KV,
                               pos_shared=True, flags=tria_b200.VIEW_POST_ROPE)
    q = queries(L, T, KV * G, 128, torch_dev)
    o = dict(cap=20.0, window=300, sink=8, slopes=torch.linspace(0.001, 0.05, KV * G, device=torch_dev)) if opt == "all" else {}
    tok = (torch.arange(T, device=torch_dev) * 2 + 590).int()
    p = tria_b200.attend_params(128 ** -0.5, o.get("cap", 0.0), o.get("window", 0), o.get("sink", 0), o.get("slopes"), tok,
                                mass_decay=0.5)
    before = torch.rand((L, KV, cells), device=torch_dev)
    mass = before.clone()
    out, lse = torch.empty_like(q), torch.empty((L, T, KV * G), device=torch_dev)
    ctx, s = contexts(KV, G, 128), torch.cuda.current_stream()
    ctx.attend(view, c.rows, q, out, p, lse=lse, mass_in=mass, mass_out=mass, stream=s)
    ctx.check(s)
    want = attend_oracle(c, q, 128 ** -0.5, o.get("cap", 0.0), o.get("window", 0), o.get("sink", 0), o.get("slopes"), tok)
    attend_close(c, out, lse, mass[:, :, :300].contiguous(), want, before[:, :, :300] * 0.5)
    live = torch.arange(cells, device=torch_dev) < c.rows[..., None]
    assert torch.equal(torch.where(live, before, mass), before)
