"""GPU tests of the serving calls against fp64 oracles (serve_cases.py)."""
import numpy as np
import pytest
import torch

import tria_b200
import workloads
from serve_cases import Cache, F16, Q8_0, attend_close, attend_oracle, rows_of_values, tree_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def contexts(torch_dev, tmp_path_factory):
    """context(KV, G, hd, layers): one per geometry, for the module's tests."""
    made = {}

    def get(KV, G, hd, layers=1, scales=None):
        key = (KV, G, hd, layers, None if scales is None else tuple(scales))
        if key not in made:
            p = str(tmp_path_factory.mktemp("serve") / "s.tria")
            workloads.write_tria(p, layers, KV * G, KV, hd, seed=1, scales=scales)
            st = tria_b200.load(p)
            made[key] = (tria_b200.Context(st, torch_dev.index or 0), st)
        return made[key][0]

    yield get
    for ctx, st in made.values():
        ctx.close()
        tria_b200.free(st)


def queries(L, T, H, hd, dev, seed=5, sigma=1.2):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return (torch.randn((L, T, H, hd), generator=g, device=dev) * sigma).half()


def a_tree(T, width=3, seed=0):
    """Ancestor sets of a random tree, itself included."""
    rng = np.random.default_rng(seed)
    sees = np.zeros((T, T), bool)
    depth = np.zeros(T, np.int64)
    for i in range(T):
        if i:
            p = int(rng.integers(max(0, i - width * 2), i))
            sees[i] = sees[p]
            depth[i] = depth[p] + 1
        sees[i, i] = True
    return sees, depth


def run_attend(contexts, c, G, T, opts=None, seed=5, mass=True, sees=None, tok_pos=None, decay=1.0, q=None, sigma=1.2):
    """One call with lse and mass, compared; returns what it gave."""
    opts = dict(opts or {})
    dev = c.dev
    ctx = contexts(c.KV, G, c.hd)
    H = c.KV * G
    q = queries(c.L, T, H, c.hd, dev, seed, sigma) if q is None else q
    if tok_pos is None and (opts.get("window") or opts.get("slopes") is not None):
        tok_pos = (torch.arange(T, device=dev) + 2 * int(c.rows_host.max()) - T).int()
    scale = c.hd ** -0.5
    tree = torch.from_numpy(tree_bits(sees)).to(dev) if sees is not None else None
    p = tria_b200.attend_params(scale, opts.get("cap", 0.0), opts.get("window", 0), opts.get("sink", 0),
                                opts.get("slopes"), tok_pos, tree, decay)
    out = torch.full((c.L, T, H, c.hd), float("nan"), dtype=torch.float16, device=dev)
    lse = torch.full((c.L, T, H), float("nan"), device=dev)
    g = torch.Generator(device=dev)
    g.manual_seed(seed + 1)
    before = torch.rand((c.L, c.KV, c.cells), generator=g, device=dev) * 0.1
    after = torch.full_like(before, -7.0)
    ctx.attend(c.view(), c.rows, q, out, p, lse=lse, mass_in=before if mass else None, mass_out=after if mass else None,
               stream=torch.cuda.current_stream(dev))
    ctx.check(torch.cuda.current_stream(dev))
    want = attend_oracle(c, q, scale, opts.get("cap", 0.0), opts.get("window", 0), opts.get("sink", 0),
                         opts.get("slopes"), tok_pos, sees)
    attend_close(c, out, lse, after if mass else None, want, before * decay if mass else None)
    if mass:
        dead = torch.arange(c.cells, device=dev)[None, None] >= c.rows[..., None]
        assert (after[dead] == -7.0).all(), "rows behind the count were written"
    # without lse and mass: the same outputs
    out2 = torch.full_like(out, float("nan"))
    ctx.attend(c.view(), c.rows, q, out2, p, stream=torch.cuda.current_stream(dev))
    torch.cuda.synchronize()
    fine = torch.isfinite(out)
    assert torch.equal(fine, torch.isfinite(out2))
    err, tol = (out.float() - out2.float()).abs(), 2.0 ** -9 * (want[0].abs() + want[3]) + 2.0 ** -24
    worst = float((err / tol)[fine].max()) if fine.any() else 0.0
    assert worst <= 1.0, worst
    return out, lse, after


def slopes_of(H, dev):
    return torch.exp2(-8.0 * torch.arange(1, H + 1, device=dev) / H).float()


SHAPES = [
    # type, hd, KV, G, rows per unit of two caches, T
    (F16, 128, 2, 4, [1, 17, 64, 203], 1),
    (F16, 64, 2, 1, [0, 1, 2, 15], 1),
    (Q8_0, 128, 2, 4, [1, 16, 65, 1000], 1),
    (Q8_0, 64, 2, 5, [31, 0, 33, 500], 1),
    (F16, 128, 2, 5, [3, 64, 129, 777], 3),
    (Q8_0, 128, 2, 2, [7, 8, 300, 9], 7),
    (F16, 128, 1, 16, [900, 33], 2),
    (F16, 64, 2, 4, [16, 100, 1025, 64], 16),
    (Q8_0, 128, 2, 4, [40, 300, 64, 1111], 33),
    (F16, 128, 2, 4, [64, 300, 1100, 130], 64),
    (Q8_0, 64, 2, 3, [129, 400, 500, 131], 129),
    (F16, 128, 2, 4, [300, 301, 1500, 511], 300),
]


@pytest.mark.parametrize("type_id,hd,KV,G,rows,T", SHAPES)
@pytest.mark.parametrize("opt", ["plain", "cap", "window", "bias", "all"])
def test_attend_causal(contexts, torch_dev, type_id, hd, KV, G, rows, T, opt):
    c = Cache(type_id, 2, KV, hd, max(rows) + 37, rows, torch_dev, seed=T)
    o = {"plain": {}, "cap": dict(cap=15.0), "window": dict(window=60, sink=8),
         "bias": dict(slopes=slopes_of(KV * G, torch_dev)),
         "all": dict(cap=30.0, window=200, sink=0, slopes=slopes_of(KV * G, torch_dev))}[opt]
    run_attend(contexts, c, G, T, o, decay=0.75 if opt == "all" else 1.0)


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("T", [2, 5, 31, 32, 48, 65, 140])
@pytest.mark.parametrize("opt", ["plain", "all"])
def test_attend_tree(contexts, torch_dev, type_id, T, opt):
    rows = [T, T + 1, T + 63, T + 700]
    c = Cache(type_id, 2, 2, 128, T + 750, rows, torch_dev, seed=T)
    sees, depth = a_tree(T, seed=T)
    tok = torch.from_numpy(depth).to(torch_dev).int() + 2 * (T + 700)
    o = {} if opt == "plain" else dict(cap=20.0, window=900, sink=4, slopes=slopes_of(8, torch_dev))
    run_attend(contexts, c, 4, T, o, sees=sees, tok_pos=tok)


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("layout", ["head", "pad"])
@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_layouts_and_shared_positions(contexts, torch_dev, type_id, layout, T, hd):
    c = Cache(type_id, 2, 3, hd, 300, [299, 41, 130, 256, 300, 65], torch_dev, layout=layout, shared=True)
    run_attend(contexts, c, 2, T, dict(window=150, sink=6, slopes=slopes_of(6, torch_dev)))


@pytest.mark.parametrize("T", [1, 4, 40, 130])
@pytest.mark.parametrize("type_id", [F16, Q8_0])
def test_tokens_that_see_nothing(contexts, torch_dev, T, type_id):
    """A window before every position, and tree rows without a bit: 0 and -inf."""
    c = Cache(type_id, 1, 2, 128, 400, [T, 333], torch_dev)
    far = torch.full((T,), 10 ** 6, dtype=torch.int32, device=torch_dev)
    out, lse, _ = run_attend(contexts, c, 4, T, dict(window=5), tok_pos=far)
    assert (out == 0).all() and (lse == -np.inf).all()
    sees = np.eye(T, dtype=bool)
    sees[T // 2] = False
    c.rows_host[0, 0] = T            # nothing before the tokens' own rows
    out, lse, _ = run_attend(contexts, c, 4, T, sees=sees)
    assert (out[0, T // 2, :4] == 0).all() and (lse[0, T // 2, :4] == -np.inf).all()


@pytest.mark.parametrize("T", [1, 3, 40, 150])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_masked_rows_hold_is_without_effect(contexts, torch_dev, T, bad):
    """Non-finite keys and values in rows behind the count, outside the window
    and in drafted rows that other tokens do not see."""
    c = Cache(F16, 1, 2, 128, 500, [401, 260], torch_dev)
    for b in (c.k, c.v):
        for h in range(2):
            u = c.unit(b, 0, h).view(torch.float16)
            u[int(c.rows_host[0, h]):] = bad
            u[30:60] = bad                                       # positions 60..118, before the window
    sees, depth = a_tree(T, seed=3)
    tok = torch.from_numpy(depth).to(torch_dev).int() + 800
    if T > 1:                                                    # a drafted row that only its own token sees
        sees[:, 1] = False
        sees[1, 1] = True
        for h in range(2):
            for b in (c.k, c.v):
                c.unit(b, 0, h).view(torch.float16)[int(c.rows_host[0, h]) - T + 1] = bad
    run_attend(contexts, c, 4, T, dict(window=640, sink=30), sees=sees, tok_pos=tok, mass=T == 1)


@pytest.mark.parametrize("T", [1, 24, 200])
def test_a_visible_infinity_is_not_hidden(contexts, torch_dev, T):
    c = Cache(F16, 1, 2, 64, 500, [450, 300], torch_dev)
    c.unit(c.v, 0, 0).view(torch.float16)[7, 3] = float("inf")
    c.unit(c.v, 0, 1).view(torch.float16)[9, 60] = float("nan")
    out, _, _ = run_attend(contexts, c, 4, T)
    assert torch.isinf(out[0, :, :4, 3]).all() and torch.isnan(out[0, :, 4:, 60]).all()


@pytest.mark.parametrize("T", [1, 20, 160])
def test_scores_far_apart(contexts, torch_dev, T):
    """One key that takes all the weight, late in the rows, and scores of
    several hundred: the running maximum has to carry."""
    c = Cache(F16, 1, 1, 128, 700, [690], torch_dev, sigma=4.0)
    run_attend(contexts, c, 4, T, sigma=4.0)


@pytest.mark.parametrize("T", [1, 12, 150])
def test_strided_queries_and_outputs(contexts, torch_dev, T):
    """q inside a fused projection's output, out with its heads before its tokens."""
    c = Cache(F16, 2, 2, 128, 300, [290, 222, 150, 151], torch_dev)
    ctx = contexts(2, 4, 128)
    H = 8
    q = queries(2, T, H, 128, torch_dev)
    fused = torch.full((2, T, H * 128 + 512), 7.0, dtype=torch.float16, device=torch_dev)
    fused[:, :, 256:256 + H * 128] = q.reshape(2, T, -1)
    qv = fused[:, :, 256:256 + H * 128].unflatten(2, (H, 128))
    store = torch.full((2, H, T, 136), 5.0, dtype=torch.float16, device=torch_dev)
    ov = store[..., :128].permute(0, 2, 1, 3)
    p = tria_b200.attend_params(128 ** -0.5)
    ctx.attend(c.view(), c.rows, qv, ov, p, stream=torch.cuda.current_stream())
    attend_close(c, ov, None, None, attend_oracle(c, q, 128 ** -0.5))
    assert (store[..., 128:] == 5.0).all()


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("G,T", [(6, 3), (8, 3), (4, 8), (3, 11), (8, 6), (4, 16), (5, 13)])
@pytest.mark.parametrize("opt", ["plain", "all"])
def test_attend_between_the_kernels(contexts, torch_dev, type_id, G, T, opt):
    """17 to 65 query rows a unit: several groups of the one kernel, the first tiles of the other."""
    c = Cache(type_id, 1, 2, 128, 900, [880, T + 3], torch_dev, seed=T)
    o = {} if opt == "plain" else dict(cap=25.0, window=700, sink=5, slopes=slopes_of(2 * G, torch_dev))
    run_attend(contexts, c, G, T, o)
    sees, depth = a_tree(T, seed=T)
    tok = torch.from_numpy(depth).to(torch_dev).int() + 1760
    run_attend(contexts, c, G, T, o, sees=sees, tok_pos=tok)


def test_more_units_than_the_kernel_scans_itself(contexts, torch_dev):
    rng = np.random.default_rng(3)
    c = Cache(F16, 70, 8, 64, 80, rng.integers(0, 80, (70, 8)), torch_dev)
    ctx, q = contexts(8, 2, 64), queries(70, 1, 16, 64, torch_dev)
    out, mass = torch.full_like(q, float("nan")), torch.zeros((70, 8, 80), device=torch_dev)
    ctx.attend(c.view(), c.rows, q, out, tria_b200.attend_params(0.125), mass_out=mass, stream=torch.cuda.current_stream())
    ctx.check(torch.cuda.current_stream())
    attend_close(c, out, None, mass, attend_oracle(c, q, 0.125))


@pytest.mark.parametrize("T", [1, 70])
def test_rows_past_two_gigabytes(contexts, torch_dev, T):
    """A cache whose rows lie up to 2.25 GB behind its base.  All keys are 0 but
    one near the end, all values 0 but that row's, so with s its score the
    output is v e^s / (e^s + the other rows that the token sees)."""
    n, cs = 1_100_000, 2048
    k = torch.zeros((n + 8) * cs, dtype=torch.uint8, device=torch_dev)
    v = torch.zeros((n + 8) * cs, dtype=torch.uint8, device=torch_dev)
    pos = torch.zeros((1, 1, n + 8), dtype=torch.int32, device=torch_dev)
    at = n - 200
    kr, vr = k[at * cs:at * cs + 256].view(torch.float16), v[at * cs:at * cs + 256].view(torch.float16)
    q = torch.ones((1, T, 4, 128), dtype=torch.float16, device=torch_dev)
    kr.fill_(1.0)
    vr.copy_(torch.arange(128, device=torch_dev).half() / 64 - 1)
    scale = 14.5 / 128
    view = tria_b200.make_view(F16, [k], [v], pos, n + 8, cs, 256, 1, flags=tria_b200.VIEW_POST_ROPE)
    ctx, s = contexts(1, 4, 128), torch.cuda.current_stream()
    rows = torch.tensor([[n]], dtype=torch.int32, device=torch_dev)
    out, mass = torch.empty_like(q), torch.zeros((1, 1, n + 8), device=torch_dev)
    ctx.attend(view, rows, q, out, tria_b200.attend_params(scale), mass_out=mass, stream=s)
    ctx.check(s)
    others = torch.arange(n - T, n, device=torch_dev).double()                # n - T + t + 1 rows seen, one of them apart
    w = np.exp(14.5) / (np.exp(14.5) + others)
    want = w[None, :, None, None] * vr.double()
    # f16: the weights' and the result's rounding; the score to fp32
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -9 + 2.0 ** -24).all()
    assert abs(float(mass[0, 0, at]) / float(4 * w.sum()) - 1) < 1e-4
    x = torch.full((1, 3, 1, 128), 2.0, dtype=torch.float16, device=torch_dev)
    ctx.append(view, rows, x, x, torch.arange(3, device=torch_dev).int(), stream=s)
    path = torch.tensor([[0, 2, 0]], dtype=torch.int32, device=torch_dev)
    v[(n + 2) * cs:(n + 2) * cs + 256].view(torch.float16).fill_(3.0)
    ctx.accept(view, rows, 3, path, torch.tensor([2], dtype=torch.int32, device=torch_dev), stream=s)
    ctx.check(s)
    assert int(rows) == n + 2
    assert (k[n * cs:n * cs + 256].view(torch.float16) == 2).all()
    assert (v[(n + 1) * cs:(n + 1) * cs + 256].view(torch.float16) == 3).all()
    assert (k[:at * cs] == 0).all()


def test_mass_in_place_and_from_nothing(contexts, torch_dev):
    for T in (1, 20):
        c = Cache(Q8_0, 1, 2, 128, 300, [290, 100], torch_dev)
        ctx, q = contexts(2, 4, 128), queries(1, T, 8, 128, torch_dev)
        out = torch.empty_like(q)
        p = tria_b200.attend_params(128 ** -0.5, mass_decay=0.5)
        a = torch.rand((1, 2, 300), device=torch_dev)
        b = a.clone()
        o2 = torch.zeros_like(a)
        s = torch.cuda.current_stream()
        ctx.attend(c.view(), c.rows, q, out, p, mass_in=b, mass_out=b, stream=s)
        ctx.attend(c.view(), c.rows, q, out, p, mass_out=o2, stream=s)
        want = attend_oracle(c, q, 128 ** -0.5)
        attend_close(c, out, None, b, want, a * 0.5)
        attend_close(c, out, None, o2, want)
        assert torch.equal(b[0, 1, 100:], a[0, 1, 100:])


def test_no_tokens_and_no_rows(contexts, torch_dev):
    ctx = contexts(2, 4, 128)
    c = Cache(F16, 1, 2, 128, 64, [10, 0], torch_dev)
    p = tria_b200.attend_params(0.1, mass_decay=0.5)
    q = queries(1, 0, 8, 128, torch_dev)
    a = torch.ones((1, 2, 64), device=torch_dev)
    ctx.attend(c.view(), c.rows, q, q.clone(), p, stream=torch.cuda.current_stream())
    ctx.attend(c.view(), c.rows, q, q.clone(), p, mass_in=a, mass_out=a, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert (a[0, 0, :10] == 0.5).all() and (a[0, 0, 10:] == 1).all() and (a[0, 1] == 1).all()


def test_many_caches(contexts, torch_dev):
    """More caches than a launch takes, each with a tree and positions of its own."""
    L, T = 131, 3
    rng = np.random.default_rng(1)
    rows = rng.integers(T, 60, (L, 1))
    c = Cache(Q8_0, L, 1, 64, 64, rows, torch_dev)
    ctx = contexts(1, 2, 64)
    q = queries(L, T, 2, 64, torch_dev)
    sees = np.stack([a_tree(T, seed=i)[0] for i in range(L)])
    tok = torch.from_numpy(rng.integers(50, 130, (L, T))).int().to(torch_dev)
    tree = torch.from_numpy(np.stack([tree_bits(s) for s in sees])).to(torch_dev)
    p = tria_b200.attend_params(0.125, window=70, sink=3, tok_pos=tok, tree=tree)
    out, mass = torch.empty_like(q), torch.zeros((L, 1, 64), device=torch_dev)
    ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=torch.cuda.current_stream())
    ctx.check(torch.cuda.current_stream())
    for l in (0, 1, 64, 127, 128, 130):
        one = Cache(Q8_0, 1, 1, 64, 64, rows[l], torch_dev)
        one.k.copy_(c.k[l:l + 1])
        one.v.copy_(c.v[l:l + 1])
        want = attend_oracle(one, q[l:l + 1], 0.125, window=70, sink=3, tok_pos=tok[l], sees=sees[l])
        attend_close(one, out[l:l + 1], None, mass[l:l + 1], want)


def test_bad_counts_are_clamped_and_reported(contexts, torch_dev):
    ctx = contexts(2, 4, 128)
    c = Cache(F16, 1, 2, 128, 64, [64, 0], torch_dev)
    q = queries(1, 1, 8, 128, torch_dev)
    out = torch.empty_like(q)
    bad = torch.tensor([[65, -1]], dtype=torch.int32, device=torch_dev)
    s = torch.cuda.current_stream()
    ctx.attend(c.view(), bad, q, out, tria_b200.attend_params(0.1), stream=s)
    with pytest.raises(tria_b200.TriaError) as e:
        ctx.check(s)
    assert e.value.status == tria_b200.ERR_ROWS
    attend_close(c, out, None, None, attend_oracle(c, q, 0.1))
    ctx.check(s)


@pytest.mark.parametrize("T", [1, 20, 140])
def test_captured_and_replayed_with_other_counts(contexts, torch_dev, T):
    """The counts are read when the graph runs; a later larger eager call does
    not take the workspace away from it."""
    ctx = contexts(2, 4, 128)
    c = Cache(F16, 1, 2, 128, 600, [200, 300], torch_dev)
    q = queries(1, T, 8, 128, torch_dev)
    out, mass = torch.empty_like(q), torch.zeros((1, 2, 600), device=torch_dev)
    p = tria_b200.attend_params(128 ** -0.5)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=st)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=torch.cuda.current_stream())
    big = Cache(F16, 4, 2, 128, 5000, [5000] * 8, torch_dev)
    qb = queries(4, 2 * T + 3, 8, 128, torch_dev)
    ob, mb = torch.empty_like(qb), torch.zeros((4, 2, 5000), device=torch_dev)
    ctx.attend(big.view(), big.rows, qb, ob, p, mass_out=mb, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    for rows in ([200, 300], [600, T], [T, 451], [0, 0]):
        c.rows_host[:] = rows
        c.rows.copy_(torch.tensor([rows], device=torch_dev))
        out.fill_(float("nan"))
        with torch.cuda.stream(st):
            g.replay()
        st.synchronize()
        attend_close(c, out, None, mass, attend_oracle(c, q, 128 ** -0.5))
    ctx.check(st)


def test_two_contexts_on_two_streams(torch_dev, tmp_path):
    p = str(tmp_path / "s.tria")
    workloads.write_tria(p, 1, 8, 2, 128, seed=1)
    st = tria_b200.load(p)
    ctxs = [tria_b200.Context(st, 0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    c = Cache(F16, 1, 2, 128, 9000, [9000, 7777], torch_dev)
    q = queries(1, 2, 8, 128, torch_dev)
    outs = [torch.empty_like(q) for _ in range(2)]
    prm = [tria_b200.attend_params(128 ** -0.5) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            ctxs[i].attend(c.view(), c.rows, q, outs[i], prm[i], stream=streams[i])
    torch.cuda.synchronize()
    want = attend_oracle(c, q, 128 ** -0.5)
    for i in range(2):
        attend_close(c, outs[i], None, None, want)
        ctxs[i].close()
    assert torch.equal(outs[0], outs[1])
    tria_b200.free(st)


def test_repeated_calls_give_the_same_bits(contexts, torch_dev):
    for T, type_id in ((1, F16), (1, Q8_0), (40, F16), (40, Q8_0), (200, F16)):
        c = Cache(type_id, 2, 2, 128, 5000, [5000, 333, 4097, 2000], torch_dev)
        ctx, q = contexts(2, 4, 128), queries(2, T, 8, 128, torch_dev)
        p = tria_b200.attend_params(128 ** -0.5)
        got = []
        for _ in range(3):
            out, mass = torch.empty_like(q), torch.zeros((2, 2, 5000), device=torch_dev)
            ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=torch.cuda.current_stream())
            got.append((out, mass))
        torch.cuda.synchronize()
        for o, m in got[1:]:
            assert torch.equal(o, got[0][0]) and torch.equal(m, got[0][1])


@pytest.mark.parametrize("type_id", [F16, Q8_0])
def test_waits_that_give_up_are_reported(contexts, torch_dev, type_id):
    """With a bound of one cycle the tensor-core kernels' pipeline waits give up:
    the status says so, and the next call is right again."""
    ctx = contexts(2, 4, 128)
    c = Cache(type_id, 2, 2, 128, 3000, [3000, 2500, 1700, 2999], torch_dev)
    T = 80
    q = queries(2, T, 8, 128, torch_dev)
    out, mass = torch.empty_like(q), torch.zeros((2, 2, 3000), device=torch_dev)
    p, s = tria_b200.attend_params(128 ** -0.5), torch.cuda.current_stream()
    ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=s)        # sizes the workspace
    ctx.check(s)
    ctx.set_wait_limit(1)
    try:
        ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=s)
        with pytest.raises(tria_b200.TriaError) as e:
            ctx.check(s)
        assert e.value.status == tria_b200.ERR_TIMEOUT
    finally:
        ctx.set_wait_limit(0)
    for _ in range(2):
        ctx.attend(c.view(), c.rows, q, out, p, mass_out=mass, stream=s)
        ctx.check(s)
        attend_close(c, out, None, mass, attend_oracle(c, q, 128 ** -0.5))


def test_every_value_not_finite(contexts, torch_dev):
    """Values that every token sees: NaN results stand as they are, for any number of rows."""
    for T in (1, 30, 200):
        c = Cache(F16, 1, 2, 128, 2000, [1999, 1500], torch_dev)
        c.unit(c.v, 0, 0).view(torch.float16)[100:200, 5] = float("nan")
        out, _, _ = run_attend(contexts, c, 4, T, mass=False)
        assert torch.isnan(out[0, :, :4, 5]).all() and not torch.isnan(out[0, :, 4:]).any()


def test_binding_refuses_foreign_tensors(contexts, torch_dev):
    ctx = contexts(2, 4, 128)
    c = Cache(F16, 1, 2, 128, 64, [10, 5], torch_dev)
    q = queries(1, 1, 8, 128, torch_dev)
    p = tria_b200.attend_params(0.1)
    with pytest.raises(ValueError, match="cpu"):
        ctx.attend(c.view(), c.rows, q.cpu(), q.clone(), p)
    with pytest.raises(ValueError, match="counts"):
        ctx.attend(c.view(), c.rows.long(), q, q.clone(), p)
    with pytest.raises(ValueError, match="shape"):
        ctx.attend(c.view(), c.rows, q[:, :, :4], q[:, :, :4].clone(), p)
    with pytest.raises(ValueError, match="mass"):
        ctx.attend(c.view(), c.rows, q, q.clone(), p, mass_out=torch.zeros((1, 2, 63), device=torch_dev))
    with pytest.raises(tria_b200.TriaError, match="POST_ROPE"):
        ctx.attend(c.view(flags=0), c.rows, q, q.clone(), p)


# ---------------------------------------------------------------- append, accept, evict by mass

@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layout", ["cell", "head", "pad"])
@pytest.mark.parametrize("src", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,in_place", [(1, True), (1, False), (7, True), (150, True), (150, False), (0, True)])
def test_append(contexts, torch_dev, type_id, hd, layout, src, T, in_place):
    ctx = contexts(2, 4, hd)
    rows = [0, 5, 249 - T, 250 - T]
    c = Cache(type_id, 2, 2, hd, 250, rows, torch_dev, layout=layout)
    g = torch.Generator(device=torch_dev)
    g.manual_seed(T)
    kv = (torch.randn((2, 2, T, 2, hd), generator=g, device=torch_dev) * 3).to(src)
    if T > 3:
        kv[0, 0, 1, 0] = 0                              # a row of zeros: d = 0
        kv[1, 1, 2, 1, :40] = torch.arange(40, device=torch_dev) - 20.0
    tok = (torch.arange(2 * T, device=torch_dev).reshape(2, T) + 900).int()
    mass = torch.full((2, 2, 250), 3.0, device=torch_dev)
    k0, v0, pos0 = c.k.clone(), c.v.clone(), c.pos.clone()
    out = c.rows if in_place else torch.full_like(c.rows, -9)
    ctx.append(c.view(), c.rows, kv[0], kv[1], tok, None if in_place else out, mass=mass,
               stream=torch.cuda.current_stream())
    ctx.check(torch.cuda.current_stream())
    assert torch.equal(out.cpu(), torch.from_numpy(c.rows_host) + T)
    for l in range(2):
        for h in range(2):
            n = int(c.rows_host[l, h])
            for b, b0, x in ((c.k, k0, kv[0]), (c.v, v0, kv[1])):
                want = c.unit(b0, l, h).clone()
                if T:
                    want[n:n + T] = rows_of_values(type_id, x[l, :, h]).reshape(T, -1)
                assert torch.equal(c.unit(b, l, h), want), (l, h)
            wp, wm = pos0[l, h].clone(), torch.full((250,), 3.0, device=torch_dev)
            wp[n:n + T] = tok[l]
            wm[n:n + T] = 0
            assert torch.equal(c.pos[l, h], wp) and torch.equal(mass[l, h], wm)
    if layout == "pad":                                  # the bytes between the cells
        for b, b0 in ((c.k, k0), (c.v, v0)):
            gap = torch.as_strided(b, (2, 250, 4), (b.shape[1], c.cell_stride, 1), 2 * c.rb)
            gap0 = torch.as_strided(b0, (2, 250, 4), (b.shape[1], c.cell_stride, 1), 2 * c.rb)
            assert torch.equal(gap, gap0)


@pytest.mark.parametrize("T", [1, 100])
def test_append_leaves_full_units_alone(contexts, torch_dev, T):
    ctx = contexts(2, 4, 128)
    c = Cache(F16, 1, 2, 128, 250, [251 - T, 250 - T], torch_dev)
    k0 = c.k.clone()
    x = queries(1, T, 2, 128, torch_dev)
    tok = torch.arange(T, device=torch_dev).int()
    s = torch.cuda.current_stream()
    ctx.append(c.view(), c.rows, x, x, tok, stream=s)
    with pytest.raises(tria_b200.TriaError) as e:
        ctx.check(s)
    assert e.value.status == tria_b200.ERR_ROWS
    assert c.rows.tolist() == [[251 - T, 250]]
    assert torch.equal(c.unit(c.k, 0, 0), c.unit(k0, 0, 0))


def test_append_shared_positions_and_strided_sources(contexts, torch_dev):
    ctx = contexts(2, 4, 128)
    c = Cache(Q8_0, 3, 2, 128, 100, [40] * 6, torch_dev, shared=True)
    fused = queries(3, 5, 12, 128, torch_dev)                     # q, k and v heads of one projection
    k, v = fused[:, :, 8:10], fused[:, :, 10:12]
    tok = torch.arange(500, 505, device=torch_dev).int()
    pos0 = c.pos.clone()
    ctx.append(c.view(), c.rows, k, v, tok, stream=torch.cuda.current_stream())
    pos0[40:45] = tok
    torch.cuda.synchronize()
    assert torch.equal(c.pos, pos0) and (c.rows == 45).all()
    for l in range(3):
        for h in range(2):
            assert torch.equal(c.unit(c.v, l, h)[40:45], rows_of_values(Q8_0, v[l, :, h]))


@pytest.mark.parametrize("type_id,hd", [(F16, 128), (Q8_0, 128), (F16, 64), (Q8_0, 64)])
@pytest.mark.parametrize("layout", ["cell", "pad"])
@pytest.mark.parametrize("own", [True, False])
def test_accept(contexts, torch_dev, type_id, hd, layout, own):
    ctx = contexts(2, 4, hd)
    T = 40
    c = Cache(type_id, 3, 2, hd, 200, [40, 41, 100, 200, 160, 77], torch_dev, layout=layout)
    paths = [[0, 1, 2], list(range(40)), [0, 3, 4, 5, 9, 30, 39]] if own else [[1, 2, 7, 8, 39]]
    path = torch.full((len(paths), T), -5, dtype=torch.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = torch.tensor(p)
    n_path = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=torch_dev)
    mass = torch.rand((3, 2, 200), device=torch_dev)
    k0, v0, pos0, m0 = c.k.clone(), c.v.clone(), c.pos.clone(), mass.clone()
    ctx.accept(c.view(), c.rows, T, path.to(torch_dev), n_path, mass=mass, stream=torch.cuda.current_stream())
    ctx.check(torch.cuda.current_stream())
    for l in range(3):
        p = paths[l if own else 0]
        for h in range(2):
            base = int(c.rows_host[l, h]) - T
            assert int(c.rows[l, h]) == base + len(p)
            src = torch.tensor(p, device=torch_dev) + base
            for b, b0 in ((c.k, k0), (c.v, v0)):
                want = c.unit(b0, l, h).clone()
                want[base:base + len(p)] = c.unit(b0, l, h)[src]
                assert torch.equal(c.unit(b, l, h), want)
            for x, x0 in ((c.pos, pos0), (mass, m0)):
                want = x0[l, h].clone()
                want[base:base + len(p)] = x0[l, h][src]
                assert torch.equal(x[l, h], want)


@pytest.mark.parametrize("path,n_path,rows", [
    ([0, 2, 2], 3, 20), ([2, 1], 2, 20), ([0, 8], 2, 20), ([-1, 1], 2, 20), ([0, 1], 9, 20), ([0, 1], -1, 20),
    ([0, 1], 2, 7), ([0, 1], 2, 65), ([0, 1], 2, -1)])
def test_accept_leaves_bad_paths_alone(contexts, torch_dev, path, n_path, rows):
    ctx = contexts(1, 4, 128)
    c = Cache(F16, 1, 1, 128, 64, [rows], torch_dev)
    pt = torch.zeros((1, 9), dtype=torch.int32)
    pt[0, :len(path)] = torch.tensor(path)
    k0 = c.k.clone()
    s = torch.cuda.current_stream()
    ctx.accept(c.view(), c.rows, 8, pt.to(torch_dev), torch.tensor([n_path], dtype=torch.int32, device=torch_dev), stream=s)
    with pytest.raises(tria_b200.TriaError) as e:
        ctx.check(s)
    assert e.value.status == tria_b200.ERR_ROWS
    assert torch.equal(c.k, k0) and c.rows.tolist() == [[rows]]


def test_accept_nothing(contexts, torch_dev):
    ctx = contexts(1, 4, 128)
    c = Cache(F16, 1, 1, 128, 64, [30], torch_dev)
    z = torch.zeros((1, 8), dtype=torch.int32, device=torch_dev)
    ctx.accept(c.view(), c.rows, 8, z, torch.zeros(1, dtype=torch.int32, device=torch_dev),
               stream=torch.cuda.current_stream())
    ctx.check(torch.cuda.current_stream())
    assert c.rows.tolist() == [[22]]


def kept_oracle(mass, pos, n, keep, cur, window, sink):
    """Rows kept of one unit: protected ones, then by (mass desc, row asc)."""
    safe = np.zeros(n, bool)
    if window > 0:
        safe |= pos[:n] >= cur - window
    if sink > 0:
        safe |= pos[:n] < sink
    keep = min(n, max(keep, int(safe.sum())))
    key = np.where(safe, np.inf, mass[:n].astype(np.float64))
    order = np.lexsort((np.arange(n), -key))
    return np.sort(order[:keep])


@pytest.mark.parametrize("type_id,hd,layout", [(F16, 128, "cell"), (Q8_0, 128, "cell"), (Q8_0, 64, "head"), (F16, 64, "pad")])
@pytest.mark.parametrize("ramp,window,sink", [(100, 0, 0), (40, 50, 4), (100, 600, 0)])
def test_evict_mass(contexts, torch_dev, type_id, hd, layout, ramp, window, sink):
    ctx = contexts(2, 4, hd, layers=3, scales=np.array([1.0, 0.5, 1.5], np.float32))
    rows = [300, 0, 1, 299, 700, 123]
    c = Cache(type_id, 3, 2, hd, 700, rows, torch_dev, layout=layout)
    d = Cache(type_id, 3, 2, hd, 700, rows, torch_dev, layout=layout, seed=9)
    mass = torch.rand((3, 2, 700), device=torch_dev)
    mass[:, :, ::3] = 0.25                                        # ties
    mass[0, 0, 5:40] = 0.0
    md = torch.full_like(mass, -1.0)
    kept = torch.full((3, 2), -1, dtype=torch.int32, device=torch_dev)
    k0, p0 = d.k.clone(), d.pos.clone()
    cur = 1400
    prm = tria_b200.EvictParams(cur, 100, ramp, window, sink, 0)
    ctx.evict_mass(c.view(), d.view(), np.asarray(rows, np.int32), mass, md, prm, kept, stream=torch.cuda.current_stream())
    most, counts = ctx.get_n_kv(6)
    assert counts.tolist() == kept.reshape(-1).tolist() and most == counts.max()
    for l, scale in enumerate((1.0, 0.5, 1.5)):
        for h in range(2):
            n = rows[2 * l + h]
            keep = workloads.layer_keep(n, workloads.layer_budget(scale, 100), ramp)
            idx = kept_oracle(mass[l, h].cpu().numpy(), c.pos[l, h].cpu().numpy(), n, keep, cur, window, sink)
            m = len(idx)
            assert int(kept[l, h]) == m
            it = torch.from_numpy(idx).to(torch_dev)
            want = c.unit(k0, l, h).clone()
            want[:m] = c.unit(c.k, l, h)[it]
            assert torch.equal(d.unit(d.k, l, h), want)
            assert torch.equal(d.unit(d.v, l, h)[:m], c.unit(c.v, l, h)[it])
            assert torch.equal(d.pos[l, h, :m], c.pos[l, h][it]) and torch.equal(d.pos[l, h, m:], p0[l, h, m:])
            assert torch.equal(md[l, h, :m], mass[l, h][it]) and (md[l, h, m:] == -1).all()


def test_evict_mass_captured(contexts, torch_dev):
    ctx = contexts(2, 4, 128, layers=3)
    rows = np.asarray([500, 400, 300, 500, 10, 0], np.int32)
    c = Cache(F16, 3, 2, 128, 512, rows, torch_dev)
    d = Cache(F16, 3, 2, 128, 512, rows, torch_dev)
    mass, md = torch.rand((3, 2, 512), device=torch_dev), torch.zeros((3, 2, 512), device=torch_dev)
    prm = tria_b200.EvictParams(1000, 60, 100, 0, 0, 0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    ctx.evict_mass(c.view(), d.view(), rows, mass, md, prm, stream=st)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ctx.evict_mass(c.view(), d.view(), rows, mass, md, prm, stream=torch.cuda.current_stream())
    big = Cache(F16, 3, 2, 128, 4000, [4000] * 6, torch_dev)
    bd = Cache(F16, 3, 2, 128, 4000, [4000] * 6, torch_dev)
    bm = torch.rand((3, 2, 4000), device=torch_dev)
    ctx.evict_mass(big.view(), bd.view(), [4000] * 6, bm, torch.zeros_like(bm), prm, stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    mass.copy_(torch.rand((3, 2, 512), device=torch_dev))
    with torch.cuda.stream(st):
        g.replay()
    st.synchronize()
    for u in range(6):
        n, (l, h) = int(rows[u]), divmod(u, 2)
        idx = kept_oracle(mass[l, h].cpu().numpy(), c.pos[l, h].cpu().numpy(), n, min(n, 60), 1000, 0, 0)
        assert torch.equal(md[l, h, :len(idx)], mass[l, h][torch.from_numpy(idx).to(torch_dev)])


@pytest.mark.parametrize("type_id", [F16, Q8_0])
def test_decode_draft_and_evict_together(contexts, torch_dev, type_id):
    """A prompt, decoded tokens, a drafted tree with its accepted path, and an
    eviction by the mass they left, then a token over what stayed: every
    step's attention against the oracle on the cache as it stands."""
    KV, G, hd, cells = 2, 4, 128, 400
    ctx = contexts(KV, G, hd)
    c = Cache(type_id, 1, KV, hd, cells, [0, 0], torch_dev)
    d = Cache(type_id, 1, KV, hd, cells, [0, 0], torch_dev, seed=3)
    mass, spare = torch.zeros((1, KV, cells), device=torch_dev), torch.zeros((1, KV, cells), device=torch_dev)
    s = torch.cuda.current_stream()
    at = 0

    def step(cache, T, depth=None, sees=None):
        nonlocal at
        k, v = queries(1, T, KV, hd, torch_dev, seed=at + 1), queries(1, T, KV, hd, torch_dev, seed=at + 2)
        q = queries(1, T, KV * G, hd, torch_dev, seed=at + 3)
        tok = (torch.arange(T, device=torch_dev) if depth is None else torch.from_numpy(depth).to(torch_dev)).int() + at
        ctx.append(cache.view(), cache.rows, k, v, tok, mass=mass, stream=s)
        tree = torch.from_numpy(tree_bits(sees)).to(torch_dev) if sees is not None else None
        p = tria_b200.attend_params(hd ** -0.5, softcap=25.0, window=300, sink=2, tok_pos=tok, tree=tree)
        out = torch.empty_like(q)
        before = mass.clone()
        ctx.attend(cache.view(), cache.rows, q, out, p, mass_in=mass, mass_out=mass, stream=s)
        ctx.check(s)
        cache.rows_host = cache.rows.cpu().numpy()
        want = attend_oracle(cache, q, hd ** -0.5, 25.0, 300, 2, None, tok, sees)
        attend_close(cache, out, None, mass, want, before)

    step(c, 200)
    at += 200
    for _ in range(3):
        step(c, 1)
        at += 1
    sees, depth = a_tree(20, seed=2)
    step(c, 20, depth, sees)
    path = [int(i) for i in np.nonzero(sees[19])[0]]
    pt = torch.zeros((1, 20), dtype=torch.int32)
    pt[0, :len(path)] = torch.tensor(path)
    ctx.accept(c.view(), c.rows, 20, pt.to(torch_dev), torch.tensor([len(path)], dtype=torch.int32, device=torch_dev),
               mass=mass, stream=s)
    ctx.check(s)
    at += len(path)
    rows = c.rows.cpu().numpy().reshape(-1)
    assert (rows == 203 + len(path)).all()
    assert torch.equal(c.pos[0, 0, 203:203 + len(path)].cpu(), torch.from_numpy(depth[path]).int() + 203)
    ctx.evict_mass(c.view(), d.view(), rows, mass, spare, tria_b200.EvictParams(at, 50, 100, 16, 2, 0), d.rows, stream=s)
    most, counts = ctx.get_n_kv(KV)
    assert most == 50 and (d.rows == 50).all()
    mass.copy_(spare)
    step(d, 1)
