"""GPU tests of attention over values and scores of every size: small and large
values, rows that take nearly all of the weight and hold none of the value
(attention sinks), and scores that rise late.  Tolerances are attend_close's,
which go by the number formats alone."""
import math

import pytest
import torch

import tria_b200
from serve_cases import Cache, F16, Q8_0, attend_close, attend_oracle, rows_of_values, values_of_rows
from test_gpu_serve import contexts, queries, run_attend  # noqa: F401 (contexts is a fixture)

pytestmark = pytest.mark.gpu

G, HD, SCALE, LEAD = 4, 128, 128 ** -0.5, 16.0


def raised(type_id, dev, T, rows, spread, bits, at, value, alike=False):
    """(cache, q) whose rows at(j) score `bits` (base 2) above the largest of the
    others for every query, by a dimension of their own, and hold values of the
    size `value`; the other rows' values have the size `spread`.  alike: the other
    rows share one key."""
    c = Cache(type_id, 1, 2, HD, max(rows) + 21, rows, dev, seed=T)
    q = queries(1, T, 2 * G, HD, dev, sigma=0.6)
    q[..., 0] = LEAD
    g = torch.Generator(device=dev)
    g.manual_seed(11)
    up = at(torch.arange(c.cells, device=dev))
    for h in range(2):
        k = torch.randn((c.cells, HD), generator=g, device=dev)
        if alike:
            k[:] = k[0]
        k[:, 0] = 0
        top = float((q[0, :, h * G:(h + 1) * G].float().reshape(-1, HD) @ k.T).max()) * SCALE
        k[up] = 0
        k[up, 0] = (top + bits * math.log(2.0)) / (LEAD * SCALE)
        v = torch.randn((c.cells, HD), generator=g, device=dev) * spread
        if alike:
            v = v.abs()
        v[up] *= value / spread
        c.unit(c.k, 0, h).copy_(rows_of_values(type_id, k))
        c.unit(c.v, 0, h).copy_(rows_of_values(type_id, v))
    return c, q


TOKENS = [1, 3, 12, 16, 40, 140]      # 4 to 560 query rows: one group, several, tiles


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("spread", [1e-3, 0.02, 0.3, 4.0, 600.0, 8000.0])
@pytest.mark.parametrize("bits", [12, 20])
def test_sinks_without_value(contexts, torch_dev, type_id, T, spread, bits):
    c, q = raised(type_id, torch_dev, T, [1500, 700], spread, bits, lambda j: j % 16 == 5, 0.0)
    run_attend(contexts, c, G, T, q=q)


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("spread", [1e-3, 4.0, 600.0, 8000.0])
@pytest.mark.parametrize("bits", [2.9, 7.9, 30.0])
def test_scores_that_rise_late(contexts, torch_dev, type_id, T, spread, bits):
    c, q = raised(type_id, torch_dev, T, [2000, 1100], spread, bits, lambda j: (j % 256 >= 128) & (j % 16 == 3), spread)
    run_attend(contexts, c, G, T, q=q)


@pytest.mark.parametrize("type_id", [F16, Q8_0])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("bits", [16, 20, 24, 28])
@pytest.mark.parametrize("spread", [1.0, 600.0])
def test_equal_weights_far_below_a_sink(contexts, torch_dev, type_id, T, bits, spread):
    """The rows that carry the value all have one weight: a rounding of it does
    not average out.  A weight is rounded by 2^-11 of itself or, where that is
    less than half a step of f16's subnormal numbers, by 2^-25 / 2^10 of the
    row's largest (the lift of the weights): in all 2^-35 sum_j |v_j|, since the
    largest weight is at most 1.  attend_close's bound takes it as 2^-24 sum_j
    |v_j| more under the factor 2^-11 of the weights' own rounding."""
    c, q = raised(type_id, torch_dev, T, [1300, 900], spread, bits, lambda j: j % 16 == 9, 0.0, alike=True)
    want = list(attend_oracle(c, q, SCALE))
    for h in range(2):
        n = int(c.rows_host[0, h])
        want[3][0, :, h * G:(h + 1) * G] += 2.0 ** -24 * values_of_rows(type_id, c.unit(c.v, 0, h)[:n], HD).abs().sum(0)
    out, s = torch.empty_like(q), torch.cuda.current_stream(torch_dev)
    lse, mass = torch.empty((1, T, 2 * G), device=torch_dev), torch.empty((1, 2, c.cells), device=torch_dev)
    ctx = contexts(2, G, HD)
    ctx.attend(c.view(), c.rows, q, out, tria_b200.attend_params(SCALE), lse=lse, mass_out=mass, stream=s)
    ctx.check(s)
    attend_close(c, out, lse, mass, want)


@pytest.mark.parametrize("T", TOKENS)
def test_q8_0_scales_of_all_sizes_in_a_row(contexts, torch_dev, T):
    """Blocks of one row from the smallest scale to a large one."""
    c, q = raised(Q8_0, torch_dev, T, [1200, 500], 1.0, 9, lambda j: j % 16 == 2, 0.0)
    for h in range(2):
        v = torch.randn((c.cells, HD), device=torch_dev)
        v *= torch.tensor([2.0 ** -15, 2.0 ** -8, 1.0, 2.0 ** 10], device=torch_dev).repeat_interleave(32)
        c.unit(c.v, 0, h).copy_(rows_of_values(Q8_0, v))
    run_attend(contexts, c, G, T, q=q)


@pytest.mark.parametrize("T", TOKENS)
def test_a_visible_q8_0_infinity(contexts, torch_dev, T):
    """An infinite block scale that every token sees: the stored integers' signs,
    NaN where they are 0, and the other values as they are."""
    c = Cache(Q8_0, 1, 2, HD, 700, [600, 450], torch_dev)
    u = c.unit(c.v, 0, 1)
    u[7, 34:36].view(torch.float16)[0] = float("inf")
    u[7, 36:40].view(torch.int8).copy_(torch.tensor([5, -3, 0, 127], device=torch_dev))
    out, _, _ = run_attend(contexts, c, G, T, mass=False)
    got = out[0, :, G:, 32:36].float()
    assert (got[..., 0] == math.inf).all() and (got[..., 1] == -math.inf).all()
    assert torch.isnan(got[..., 2]).all() and (got[..., 3] == math.inf).all()
    assert torch.isfinite(out[0, :, :G]).all() and torch.isfinite(out[0, :, G:, :32]).all()


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("where", ["keys", "values"])
def test_q8_0_blocks_beyond_f16(contexts, torch_dev, T, where):
    """Scales whose block reaches past 65504 (tria_append stores them from fp32):
    keys along a dimension in which the queries are small, values of rows with
    little weight."""
    c = Cache(Q8_0, 1, 2, HD, 900, [870, 333], torch_dev)
    q = queries(1, T, 2 * G, HD, torch_dev, sigma=0.6)
    q[..., 0] = 2.0 ** -13
    for h, rows in ((0, [3, 200, 869]), (1, [77, 300])):
        for r in rows:
            if where == "keys":
                b = c.unit(c.k, 0, h)[r]
                b[:2].view(torch.float16)[0] = 900.0
                b[2:34] = 0
                b[2] = 120 if r % 2 else 136                       # +120, -120
            else:
                k = torch.zeros((1, HD), device=torch_dev)
                k[0, 0] = -16 * math.log(2.0) / (SCALE * 2.0 ** -13)   # 16 (base 2) below a score of 0
                c.unit(c.k, 0, h)[r:r + 1].copy_(rows_of_values(Q8_0, k))
                b = c.unit(c.v, 0, h)[r]
                b[34:36].view(torch.float16)[0] = 2000.0
    out, lse, mass = run_attend(contexts, c, G, T, q=q)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("T", [1, 12, 40, 140])
@pytest.mark.parametrize("d", [511.75, 512.0])
@pytest.mark.parametrize("side", ["k", "v"])
def test_q8_0_blocks_at_the_edge_of_f16(contexts, torch_dev, T, d, side):
    """-128 (which other writers may store) times 511.75 is f16's largest number, times 512 past it."""
    c = Cache(Q8_0, 1, 2, HD, 500, [470, 333], torch_dev)
    q = queries(1, T, 2 * G, HD, torch_dev, sigma=0.6)
    q[..., 0] = 2.0 ** -13
    b = c.unit(getattr(c, side), 0, 1)[40]
    b[:2].view(torch.float16)[0] = d
    b[2:34] = 0
    b[2] = 128
    out, _, _ = run_attend(contexts, c, G, T, q=q)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("type_id,part", [(F16, 2.0 ** -20), (Q8_0, 2.0 ** -16)])
@pytest.mark.parametrize("T", [1, 3, 8])
@pytest.mark.parametrize("bits", [1, 3.3, 9.6])
def test_few_tokens_keep_the_weights_bits(contexts, torch_dev, type_id, part, T, bits):
    """Up to 32 query rows a unit the weights are not rounded to 11 bits: beyond
    the result's own rounding (2^-11 of it) only the parts' and fp32's are left.
    The rows that carry the value have one weight and positive values, so that
    its rounding shows in full."""
    c, q = raised(type_id, torch_dev, T, [390, 77], 1.0, bits, lambda j: j % 16 == 9, 0.0, alike=True)
    out, s = torch.empty_like(q), torch.cuda.current_stream(torch_dev)
    contexts(2, G, HD).attend(c.view(), c.rows, q, out, tria_b200.attend_params(SCALE), stream=s)
    want, _, _, absum, serr = attend_oracle(c, q, SCALE)
    # attend_close's terms with the weights' 2^-11 replaced by the parts'; the rows' scores share one error, and a
    # factor on all of their weights, e^(2 serr) at most, is in rel
    rel = part + 2 * torch.expm1(serr) + 2.0 ** -20 + 2 * (390 + 32) * 2.0 ** -24
    tol = 2.0 ** -11 * want.abs() * (1 + 2.0 ** -9) + rel[..., None] * absum * (1 + 2.0 ** -9) + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()
