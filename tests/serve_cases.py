"""Inputs and fp64 oracles for the tests of the serving calls (append, attend,
accept, evict by mass): plain loops over units, apart from the kernels."""
import math

import numpy as np
import torch

import tria_b200
import workloads

F16, Q8_0 = workloads.TYPE_F16, workloads.TYPE_Q8_0


def rows_of_values(type_id, x):
    """float values [..., hd] as cache rows [..., row bytes] uint8 (on x's device)."""
    import devcache
    return devcache.quantize_q8_0_torch(x.float()) if type_id == Q8_0 else x.half().contiguous().view(torch.uint8)


def values_of_rows(type_id, rows, hd):
    """Cache rows [n, row bytes] uint8 as fp64 [n, hd]."""
    if type_id == F16:
        return rows.contiguous().view(torch.float16).double()
    b = rows.reshape(rows.shape[0], hd // 32, 34)
    d = b[..., :2].contiguous().view(torch.float16).double()
    return (b[..., 2:].contiguous().view(torch.int8).double() * d).reshape(rows.shape[0], hd)


class Cache:
    """Ragged caches [L][cells][KV] with a choice of layout: "cell" (llama.cpp's,
    heads side by side), "head" (head-major) or "pad" (cells 4 bytes longer
    than their rows, so that rows are only 4-byte aligned)."""

    def __init__(self, type_id, L, KV, hd, cells, rows, dev, seed=0, layout="cell", shared=False, sigma=1.0):
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.type, self.L, self.KV, self.hd, self.cells, self.layout, self.dev = type_id, L, KV, hd, cells, layout, dev
        self.rb = workloads.row_bytes(type_id, hd)
        if layout == "head":
            self.head_stride, self.cell_stride = cells * self.rb, self.rb
        else:
            self.head_stride, self.cell_stride = self.rb, KV * self.rb + (4 if layout == "pad" else 0)
        size = cells * KV * self.rb + (cells * 4 if layout == "pad" else 0)
        size = (size + 15) // 16 * 16
        self.k = torch.zeros((L, size), dtype=torch.uint8, device=dev)
        self.v = torch.zeros((L, size), dtype=torch.uint8, device=dev)
        for b in (self.k, self.v):
            for l in range(L):
                for h in range(KV):
                    self.unit(b, l, h).copy_(rows_of_values(type_id, torch.randn((cells, hd), generator=g, device=dev) * sigma))
        self.shared = shared
        self.rows_host = np.asarray(rows, np.int32).reshape(L, KV)
        self.rows = torch.from_numpy(self.rows_host.copy()).to(dev)
        shape = (cells,) if shared else (L, KV, cells)
        self.pos = (torch.arange(cells, device=dev) * 2).expand(shape).int().contiguous()

    def unit(self, b, l, h):
        """Rows of (l, h) of buffer b, [cells, row bytes], a view."""
        return torch.as_strided(b, (self.cells, self.rb), (self.cell_stride, 1),
                                l * b.shape[1] + h * self.head_stride)

    def pos_of(self, l, h):
        return self.pos if self.shared else self.pos[l, h]

    def view(self, flags=tria_b200.VIEW_POST_ROPE):
        return tria_b200.make_view(self.type, [self.k[l] for l in range(self.L)], [self.v[l] for l in range(self.L)],
                                   self.pos, self.cells, self.cell_stride, self.head_stride, self.KV,
                                   pos_shared=self.shared, flags=flags)


def tree_bits(sees):
    """bool [T, T] as int32 words [T, ceil(T / 32)]."""
    T = sees.shape[0]
    W = (T + 31) // 32
    b = np.zeros((T, W * 32), bool)
    b[:, :T] = sees
    return np.packbits(b, axis=1, bitorder="little").view(np.int32).copy()


def attend_oracle(c, q, scale, cap=0.0, window=0, sink=0, slopes=None, tok_pos=None, sees=None, rows=None):
    """fp64 (out, lse, mass, bound): bound holds, for each output element, what
    the tolerances are built from: (sum_j p_j |v_j|, score error bound)."""
    L, T, H, hd = q.shape
    G = H // c.KV
    dev = q.device
    rows = c.rows_host if rows is None else rows
    out = torch.zeros((L, T, H, hd), dtype=torch.float64, device=dev)
    lse = torch.full((L, T, H), -math.inf, dtype=torch.float64, device=dev)
    mass = torch.zeros((L, c.KV, c.cells), dtype=torch.float64, device=dev)
    absum = torch.zeros_like(out)
    serr = torch.zeros((L, T, H), dtype=torch.float64, device=dev)
    for l in range(L):
        for h in range(c.KV):
            n = int(rows[l, h])
            if n == 0 or T == 0:
                continue
            k = values_of_rows(c.type, c.unit(c.k, l, h)[:n], hd)
            v = values_of_rows(c.type, c.unit(c.v, l, h)[:n], hd)
            own = torch.arange(n, device=dev)[None] - (n - T)
            t = torch.arange(T, device=dev)[:, None]
            if sees is not None:
                sv = torch.as_tensor(sees, device=dev)
                see = (own < 0) | sv[t, own.clamp(0, T - 1)]
            else:
                see = own <= t
            if window or slopes is not None:
                p = c.pos_of(l, h)[:n].long()[None]
                tp = (tok_pos[l] if tok_pos.dim() == 2 else tok_pos).long()[:, None]
            if window:
                see = see & ((p >= tp - window) | (p < sink))
            # rows that no token sees may hold anything
            kk = torch.where(see.any(0)[:, None], k, torch.zeros_like(k))
            for g in range(G):
                hh = h * G + g
                qq = q[l, :, hh].double()
                # a masked row's score may be NaN or infinite: it is replaced, not added to
                s = scale * (qq @ kk.T)
                mag = scale * (qq.abs() @ torch.nan_to_num(kk, nan=0.0, posinf=0.0, neginf=0.0).abs().T)
                if cap:
                    s = cap * torch.tanh(s / cap)
                big = s.abs()
                if slopes is not None:
                    far = slopes[hh].double() * (tp - p).double()
                    s, big = s - far, big + far.abs()
                s = torch.where(see, s, -math.inf)
                top = s.amax(1, keepdim=True)
                top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
                e = torch.where(see, torch.exp(s - top), 0.0)
                tot = e.sum(1, keepdim=True)
                w = torch.where(tot != 0, e / tot, torch.zeros_like(e))
                for i in range(T):
                    # a token sums over its own rows alone, so that 0 * NaN of another's row cannot reach it
                    r = see[i].nonzero()[:, 0]
                    out[l, i, hh] = w[i, r] @ v[r]
                    absum[l, i, hh] = w[i, r] @ v[r].abs()
                lse[l, :, hh] = torch.where(tot[:, 0] != 0, top[:, 0] + torch.log(tot[:, 0]), -math.inf)
                mass[l, h, :n] += w.sum(0)
                # fp32 scores: hd products summed (each sum's rounding 2^-24 of the partial sums, at most mag; tensor
                # cores may truncate: twice that), then scale, log2 e, cap and bias, each a few roundings of the score
                m = torch.where(see, (hd + 8) * 2.0 ** -23 * mag + 2.0 ** -20 * big + (cap or 0.0) * 2.0 ** -20, 0.0)
                serr[l, :, hh] = m.amax(1)
    return out, lse, mass, absum, serr


def attend_close(c, got, lse, mass, want, mass_before=None, rows=None):
    """Asserts the outputs within the bounds of the number formats.

    out: the weights are rounded to f16 for the product (2^-11 of p), the
    result once more (2^-11 of out; 2^-25 where it is subnormal), a weight is
    off by 2 serr from its score (its own and the denominator's) and 2^-20
    from the exponential, and sums of n fp32 terms by n 2^-24 of their
    absolute sum (twice: numerator and denominator)."""
    out, lse64, mass64, absum, serr = want
    rows = c.rows_host if rows is None else rows
    n = int(rows.max()) if rows.size else 0
    rel = 2 * torch.expm1(serr) + 2.0 ** -20 + 2 * (n + 32) * 2.0 ** -24
    tol = 2.0 ** -11 * out.abs() * (1 + 2.0 ** -9) + (2.0 ** -11 + rel)[..., None] * absum * (1 + 2.0 ** -9) + 2.0 ** -25
    fine = torch.isfinite(out)
    assert torch.equal(fine, torch.isfinite(got)), "non-finite outputs elsewhere than the oracle's"
    err = (got.double() - out).abs()
    bad = fine & ~(err <= tol)
    assert not bad.any(), f"out: worst {float((err / tol)[fine].max())} of its tolerance, {int(bad.sum())} of {bad.numel()}"
    if lse is not None:
        same = lse.double() == lse64
        tol = serr + 2.0 ** -20 + (n + 32) * 2.0 ** -24 + 2.0 ** -22 * lse64.abs()
        ok = same | ((lse.double() - lse64).abs() <= tol) | (torch.isnan(lse64) & torch.isnan(lse))
        assert ok.all(), f"lse: worst off by {float((lse.double() - lse64).abs()[~ok].max())}"
    if mass is not None:
        live = torch.arange(c.cells, device=got.device)[None, None] < torch.from_numpy(rows).to(got.device)[..., None]
        before = mass_before.double() if mass_before is not None else torch.zeros_like(mass64)
        w = before + mass64
        tol = mass64 * (2 * torch.expm1(serr.max()) + 2.0 ** -19 + 2 * (n + 32) * 2.0 ** -24) + w.abs() * 2.0 ** -22 + 2.0 ** -100
        err = (mass.double() - w).abs()
        bad = live & ~(err <= tol)
        assert not bad.any(), f"mass: worst {float((err / tol)[live].max())} of its tolerance"
