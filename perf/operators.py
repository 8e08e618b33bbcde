"""Cases of the operators that serve a ragged, evicted KV cache, and their plain forms.

Five operators over the cache of `tria_kv_view` (per (layer, kv head): its own
rows, positions and row count, f16 or ggml q8_0 rows):

  attend       attention of one or many query tokens over the cached rows
  attend mass  the same call, adding each row's attention weight to its mass
  evict        eviction of the rows with the least accumulated mass
  append       new tokens' keys and values written behind each unit's rows
  accept       the accepted path of a tree of drafted tokens kept, the rest dropped

A case's rows, geometry and options are plain values; `prepare` makes the
inputs from the seed on the GPU.
"""
import atexit
import os
import sys
import tempfile

import numpy as np
import torch

own = False

F16, Q8_0 = "f16", "q8_0"
SCALE = {64: 0.125, 128: 0.08838834764831845}


def listed():
    return [
        # one decoded token right after an eviction of a short chat: latency
        dict(name="token short f16", op="attend", caches=1, kv=8, gqa=4, hd=128, type=F16, rows=1003, spread=0,
             tokens=1, mask="causal", cap=0.0, window=0, sink=0, bias=False),
        # a serving batch of 16 sequences under one budget per sequence: each kv head keeps its own count
        dict(name="token batch q8_0", op="attend", caches=16, kv=8, gqa=4, hd=128, type=Q8_0, rows=32768, spread=24571,
             tokens=1, mask="causal", cap=0.0, window=0, sink=0, bias=False),
        # verification of 48 drafted tokens over a long document, model with capped scores
        dict(name="tree capped f16", op="attend", caches=2, kv=8, gqa=4, hd=128, type=F16, rows=30011, spread=4099,
             tokens=48, mask="tree", cap=30.0, window=0, sink=0, bias=False),
        # a prompt's last chunk behind its earlier ones
        dict(name="prompt chunk f16", op="attend", caches=1, kv=8, gqa=4, hd=128, type=F16, rows=8192, spread=0,
             tokens=2048, mask="causal", cap=0.0, window=0, sink=0, bias=False),
        # decoding with the weights watched, long context
        dict(name="mass token f16", op="attend mass", caches=1, kv=8, gqa=4, hd=128, type=F16, rows=65521, spread=0,
             tokens=1, mask="causal", cap=0.0, window=0, sink=0, bias=False),
        # the last 32 tokens of a prompt observe it, model with a distance bias and local attention
        dict(name="mass observe q8_0", op="attend mass", caches=4, kv=8, gqa=5, hd=128, type=Q8_0, rows=12289, spread=1001,
             tokens=32, mask="causal", cap=0.0, window=8192, sink=4, bias=True),
        # a small model's eviction, or one rank's share of the layers
        dict(name="evict share q8_0", op="evict", caches=4, kv=8, gqa=4, hd=128, type=Q8_0, rows=2048, spread=301,
             percent=25, ramp=40, window=128, sink=4),
        # a whole model's eviction to 12 %
        dict(name="evict model f16", op="evict", caches=36, kv=8, gqa=4, hd=128, type=F16, rows=16384, spread=0,
             percent=12, ramp=100, window=512, sink=4),
        # one decoded token of all layers
        dict(name="append token q8_0", op="append", caches=36, kv=8, gqa=4, hd=128, type=Q8_0, rows=4100, spread=1999,
             tokens=1, source="f16"),
        # a prompt chunk of all layers, from the fp32 that the projections of a ggml graph leave
        dict(name="append chunk q8_0", op="append", caches=36, kv=8, gqa=4, hd=128, type=Q8_0, rows=4100, spread=1021,
             tokens=512, source="f32"),
        # a verified path of a small tree, all layers of one sequence
        dict(name="accept path q8_0", op="accept", caches=36, kv=8, gqa=4, hd=128, type=Q8_0, rows=4099, spread=1999,
             tokens=64, width=8, kept=3, shared=True),
        # a batch of sequences at one layer group, each with its own path
        dict(name="accept batch f16", op="accept", caches=64, kv=8, gqa=4, hd=128, type=F16, rows=8191, spread=4001,
             tokens=96, width=9, kept=3, shared=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(2.0 ** rng.uniform(np.log2(lo), np.log2(hi))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "attend mass", "attend mass", "evict", "append", "accept"])
    c = dict(op=op, kv=rng.choice([2, 4, 8]), gqa=rng.choice([1, 2, 4, 5]), hd=rng.choice([64, 128, 128]),
             type=rng.choice([F16, Q8_0]))
    if op in ("attend", "attend mass"):
        t = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 128), _log_int(rng, 128, 1024)])
        c["tokens"] = t
        c["caches"] = 1 if t > 128 else _log_int(rng, 1, 16)
        c["rows"] = t + _log_int(rng, 8, 8192 if t > 128 else 32768 // max(1, c["caches"] * t // 32))
        c["mask"] = rng.choice(["causal", "tree"]) if 1 < t <= 128 else "causal"
        c["cap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
        c["window"] = rng.choice([0, 0, _log_int(rng, 16, 4096)])
        c["sink"] = rng.choice([0, 4]) if c["window"] else 0
        c["bias"] = rng.random() < 0.25
        c["spread"] = rng.randrange(0, max(1, c["rows"] - t))
    elif op == "evict":
        c["caches"] = _log_int(rng, 1, 36)
        c["rows"] = _log_int(rng, 64, 16384)
        c["spread"] = rng.randrange(0, c["rows"])
        c["percent"] = rng.randrange(5, 90)
        c["ramp"] = rng.choice([10, 20, 40, 80, 100])
        c["window"] = rng.choice([0, 32, 512])
        c["sink"] = rng.choice([0, 4])
    elif op == "append":
        c["caches"] = _log_int(rng, 1, 36)
        c["tokens"] = rng.choice([1, _log_int(rng, 2, 512)])
        c["rows"] = c["tokens"] + _log_int(rng, 2, 8000)
        c["spread"] = rng.randrange(0, c["rows"] - c["tokens"])
        c["source"] = rng.choice(["f16", "f32"])
    else:
        c["caches"] = _log_int(rng, 1, 64)
        c["tokens"] = _log_int(rng, 20, 128)
        c["rows"] = c["tokens"] + _log_int(rng, 2, 8000)
        c["spread"] = rng.randrange(0, c["rows"] - c["tokens"])
        c["width"] = rng.choice([4, 5, 8])
        c["kept"] = rng.choice([1, 2, 3]) if c["width"] * (c["width"] + 1) < c["tokens"] else rng.choice([1, 2])
        c["shared"] = rng.random() < 0.5
    return c


# ---------------------------------------------------------------- inputs

def _row_bytes(c):
    return 2 * c["hd"] if c["type"] == F16 else c["hd"] // 32 * 34


def _rows(c):
    """Rows per (cache, kv head), [caches, kv]: from the case alone, between rows - spread and rows."""
    u = np.arange(c["caches"] * c["kv"], dtype=np.int64)
    return (c["rows"] - (u * 7919) % (c["spread"] + 1)).astype(np.int32).reshape(c["caches"], c["kv"])


def _quantize(x):
    """ggml q8_0 blocks of the last axis: d = max|x| / 127 as f16, q = rint(x * (1 / d)), all in fp32."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32).float()
    d = b.abs().amax(dim=-1, keepdim=True) / 127.0
    inv = torch.where(d > 0, 1.0 / torch.where(d > 0, d, torch.ones_like(d)), torch.zeros_like(d))
    q = torch.clamp(torch.round(b * inv), -127, 127).to(torch.int8)
    blk = torch.cat([d.half().view(torch.uint8), q.view(torch.uint8)], dim=-1)
    return blk.reshape(*x.shape[:-1], -1)


def _to_rows(c, x):
    return _quantize(x) if c["type"] == Q8_0 else x.half().view(torch.uint8)


def _fill(c, g, cells, sigma):
    """[caches, cells, kv * row bytes]: normal values, one dimension in a hundred eight times as large."""
    out = torch.empty((c["caches"], cells, c["kv"] * _row_bytes(c)), dtype=torch.uint8, device="cuda")
    for l in range(c["caches"]):
        x = torch.randn((cells, c["kv"], c["hd"]), generator=g, device="cuda") * sigma
        odd = torch.rand((1, c["kv"], c["hd"]), generator=g, device="cuda") < 0.01
        out[l] = _to_rows(c, torch.where(odd, x * 8.0, x)).reshape(cells, -1)
    return out


def _tree(tokens, width):
    """Parents, depths and ancestor sets (itself included) of a complete `width`-ary tree in breadth-first order."""
    parent = np.where(np.arange(tokens) > 0, (np.arange(tokens) - 1) // width, -1)
    depth = np.zeros(tokens, np.int64)
    sees = np.zeros((tokens, tokens), bool)
    for i in range(tokens):
        sees[i, i] = True
        if parent[i] >= 0:
            depth[i] = depth[parent[i]] + 1
            sees[i] |= sees[parent[i]]
    return depth, sees


def _pack(sees):
    t = sees.shape[0]
    words = (t + 31) // 32
    bits = np.zeros((t, words * 32), bool)
    bits[:, :t] = sees
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32).view(np.int32).copy()


def _inputs(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, L, KV, hd = c["op"], c["caches"], c["kv"], c["hd"]
    n, T = _rows(c), c.get("tokens", 0)
    cells = (int(c["rows"]) + 63) // 64 * 64
    s = {"case": c, "cells": cells, "rows_host": n, "rows": torch.from_numpy(n).cuda()}
    # row j's position: rows behind an eviction lie one to three tokens apart, the query tokens follow at `cur`
    cur = 3 * int(c["rows"]) + 8
    before = s["rows"].long()[..., None] - (T if op in ("attend", "attend mass", "accept") else 0)
    gaps = torch.randint(1, 4, (L, KV, cells), generator=g, device="cuda")
    cum = gaps.cumsum(-1)
    last = cum.gather(-1, (before - 1).clamp(min=0))
    pos = cur - 1 - (last - cum)
    s["cur"] = cur
    tree = op == "accept" or c.get("mask") == "tree"
    if T:
        depth, sees = _tree(T, c.get("width", 4)) if tree else (np.arange(T), np.tri(T, dtype=bool))
        tok = torch.from_numpy(cur + depth).cuda()
        s["tok_pos"] = tok.int()
        if op != "append":
            j = torch.arange(cells, device="cuda") - before
            pos = torch.where((j >= 0) & (j < T), tok[j.clamp(0, T - 1)], pos)
        if op in ("attend", "attend mass") and tree:
            s["tree"] = torch.from_numpy(_pack(sees)).cuda()
            s["sees"] = torch.from_numpy(sees).cuda()
    s["pos"] = pos.clamp(0, cur + T).int().contiguous()
    s["k"], s["v"] = _fill(c, g, cells, 1.0), _fill(c, g, cells, 1.0)
    if op in ("attend", "attend mass"):
        H = KV * c["gqa"]
        s["q"] = (torch.randn((L, T, H, hd), generator=g, device="cuda") * 1.2).half()
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda") / H).float() * 0.05 if c["bias"] else None
        s["out"] = torch.zeros_like(s["q"])
        if op == "attend mass":
            # a row's weight in a few calls like this one
            s["mass"] = torch.rand((L, KV, cells), generator=g, device="cuda") * (8.0 * c["gqa"] * T / c["rows"])
            s["mass_out"] = torch.zeros_like(s["mass"])
    elif op == "evict":
        # accumulated weights span decades, and rows that nothing looked at share a mass of zero
        m = torch.exp(torch.randn((L, KV, cells), generator=g, device="cuda") * 2.0)
        s["mass"] = torch.where(torch.rand(m.shape, generator=g, device="cuda") < 0.05, torch.zeros_like(m), m)
        s["dk"], s["dv"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        s["dpos"], s["dmass"] = torch.zeros_like(s["pos"]), torch.zeros_like(s["mass"])
        s["kept"] = torch.zeros((L, KV), dtype=torch.int32, device="cuda")
        s["budget"] = max(1, int(c["rows"]) * c["percent"] // 100)
    elif op == "append":
        x = torch.randn((2, L, T, KV, hd), generator=g, device="cuda")
        x = x.half() if c["source"] == "f16" else x
        s["new_k"], s["new_v"] = x[0].contiguous(), x[1].contiguous()
        s["rows"] = s["rows"] - T
        s["mass"] = torch.rand((L, KV, cells), generator=g, device="cuda")
        s["rows_out"] = torch.zeros_like(s["rows"])
    else:
        w, kept = c["width"], c["kept"]
        one = torch.zeros((1 if c["shared"] else L, T), dtype=torch.int64, device="cuda")
        if kept > 1:
            one[:, 1] = torch.where(torch.rand(one.shape[0], generator=g, device="cuda") < 0.5, 1, w)
        if kept > 2:
            one[:, 2] = w * one[:, 1] + 1 + torch.randint(0, w, (one.shape[0],), generator=g, device="cuda")
            one[:, 2] = torch.where(one[:, 2] < T, one[:, 2], w + 1)
        s["path"] = one.int()
        s["n_path"] = torch.full((one.shape[0],), kept, dtype=torch.int32, device="cuda")
        s["mass"] = torch.rand((L, KV, cells), generator=g, device="cuda")
        s["rows_out"] = torch.zeros_like(s["rows"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handles(s)
    return s


# ---------------------------------------------------------------- the framework's calls

_contexts = {}


def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "triattention-ggml_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tria_b200
    import workloads
    return tria_b200, workloads


def _context(lib, workloads, layers, kv, gqa, hd):
    """The context that a program keeps for its model: one per geometry."""
    key = (layers, kv, gqa, hd)
    if key not in _contexts:
        with tempfile.TemporaryDirectory() as td:
            path = workloads.write_tria(os.path.join(td, "stats.tria"), layers, kv * gqa, kv, hd, seed=1)
            st = lib.load(path)
        ctx = lib.Context(st, torch.cuda.current_device())
        atexit.register(ctx.close)
        _contexts[key] = (ctx, st)
    return _contexts[key][0]


def _view(lib, s, k, v, pos):
    c = s["case"]
    rb = _row_bytes(c)
    return lib.make_view(lib.TYPE_F16 if c["type"] == F16 else lib.TYPE_Q8_0, [k[l] for l in range(c["caches"])],
                         [v[l] for l in range(c["caches"])], pos, s["cells"], c["kv"] * rb, rb, c["kv"],
                         flags=lib.VIEW_POST_ROPE)


def _handles(s):
    lib, workloads = _library()
    c = s["case"]
    s["ctx"] = _context(lib, workloads, c["caches"] if c["op"] == "evict" else 1, c["kv"], c["gqa"], c["hd"])
    s["view"] = _view(lib, s, s["k"], s["v"], s["pos"])
    if c["op"] in ("attend", "attend mass"):
        s["params"] = lib.attend_params(scale=SCALE[c["hd"]], softcap=c["cap"], window=c["window"], sink=c["sink"],
                                        slopes=s["slopes"], tok_pos=s["tok_pos"], tree=s.get("tree"))
    elif c["op"] == "evict":
        s["dst"] = _view(lib, s, s["dk"], s["dv"], s["dpos"])
        s["params"] = lib.EvictParams(s["cur"], s["budget"], c["ramp"], c["window"], c["sink"], 0)


def _run_own(s):
    c, op, ctx, stream = s["case"], s["case"]["op"], s["ctx"], torch.cuda.current_stream()
    if op == "attend":
        ctx.attend(s["view"], s["rows"], s["q"], s["out"], s["params"], stream=stream)
        return s["out"]
    if op == "attend mass":
        ctx.attend(s["view"], s["rows"], s["q"], s["out"], s["params"], mass_in=s["mass"], mass_out=s["mass_out"],
                   stream=stream)
        return s["out"], s["mass_out"]
    if op == "evict":
        ctx.evict_mass(s["view"], s["dst"], s["rows_host"].reshape(-1), s["mass"], s["dmass"], s["params"], s["kept"],
                       stream=stream)
        return s["dk"], s["dv"], s["dpos"], s["dmass"], s["kept"]
    if op == "append":
        ctx.append(s["view"], s["rows"], s["new_k"], s["new_v"], s["tok_pos"], s["rows_out"], mass=s["mass"],
                   stream=stream)
    else:
        ctx.accept(s["view"], s["rows"], c["tokens"], s["path"], s["n_path"], s["rows_out"], mass=s["mass"],
                   stream=stream)
    return s["k"], s["v"], s["pos"], s["mass"], s["rows_out"]


# ---------------------------------------------------------------- plain forms

def _values(c, raw, n):
    """The first n rows as fp32 [caches, kv, n, hd]."""
    L, KV, hd = c["caches"], c["kv"], c["hd"]
    r = raw[:, :n].reshape(L, n, KV, -1)
    if c["type"] == F16:
        x = r.view(torch.float16).float()
    else:
        b = r.reshape(L, n, KV, hd // 32, 34)
        x = (b[..., 2:].contiguous().view(torch.int8).float() * b[..., :2].contiguous().view(torch.float16).float())
        x = x.reshape(L, n, KV, hd)
    return x.permute(0, 2, 1, 3)


def _visible(s, n):
    """[caches, kv, tokens, n]: which rows each query token sees."""
    c, T = s["case"], s["case"]["tokens"]
    j = torch.arange(n, device="cuda")
    rows = s["rows"].long()[..., None, None]
    new = j - (rows - T)                                       # index among the query tokens' own rows
    if "sees" in s:
        t = torch.arange(T, device="cuda")[:, None]
        seen = (new < 0) | (s["sees"][t, new.clamp(0, T - 1)] & (new < T))
    else:
        seen = new <= torch.arange(T, device="cuda")[:, None]
    seen = seen & (j < rows)
    if c["window"]:
        p = s["pos"][:, :, None, :n].long()
        near = p >= s["tok_pos"].long()[:, None] - c["window"]
        seen = seen & (near | (p < c["sink"]))
    return seen


def _attend_plain(s, want_mass):
    c, T, G = s["case"], s["case"]["tokens"], s["case"]["gqa"]
    L, KV, hd, n = c["caches"], c["kv"], c["hd"], int(c["rows"])
    q = s["q"].float().reshape(L, T, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(L, KV, G * T, hd)
    x = (q @ _values(c, s["k"], n).transpose(-1, -2)) * SCALE[hd]
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    x = x.reshape(L, KV, G, T, n)
    if c["bias"]:
        far = (s["tok_pos"][:, None] - s["pos"][:, :, None, :n]).float()
        x = x - s["slopes"].reshape(1, KV, G, 1, 1) * far[:, :, None]
    x = torch.where(_visible(s, n)[:, :, None], x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = p.reshape(L, KV, G * T, n) @ _values(c, s["v"], n)
    o = o.reshape(L, KV, G, T, hd).permute(0, 3, 1, 2, 4).reshape(L, T, KV * G, hd).half()
    s["out"].copy_(o)
    if not want_mass:
        return s["out"]
    live = torch.arange(n, device="cuda") < s["rows"][..., None]
    s["mass_out"][:, :, :n] = torch.where(live, s["mass"][:, :, :n] + p.sum((2, 3)), s["mass_out"][:, :, :n])
    return s["out"], s["mass_out"]


def _evict_plain(s):
    c, n = s["case"], int(s["case"]["rows"])
    L, KV = c["caches"], c["kv"]
    rows = s["rows"].long()[..., None]
    j = torch.arange(n, device="cuda")
    live = j < rows
    p = s["pos"][:, :, :n].long()
    safe = torch.zeros_like(live)
    if c["window"]:
        safe = safe | (p >= s["cur"] - c["window"])
    if c["sink"]:
        safe = safe | (p < c["sink"])
    safe = safe & live
    over = (rows - s["budget"]).clamp(min=0)
    keep = torch.maximum(rows - over * c["ramp"] // 100, safe.sum(-1, keepdim=True)).minimum(rows)
    key = torch.where(safe, float("inf"), torch.where(live, s["mass"][:, :, :n], float("-inf")))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand(L, KV, n))
    kept = rank < keep
    src = torch.sort((~kept).to(torch.uint8), dim=-1, stable=True).indices       # kept rows first, in row order
    # no host read of the counts: what the budget leaves, and every row that the window and the sink may protect
    left = int(s["rows_host"].max()) - s["budget"]
    most = min(n, n - max(0, left) * c["ramp"] // 100 + c["window"] + c["sink"] + 1)
    at = src[..., :most]
    put = j[:most] < keep
    l = torch.arange(L, device="cuda")[:, None, None]
    h = torch.arange(KV, device="cuda")[None, :, None]
    for a, b in (("k", "dk"), ("v", "dv")):
        x, y = s[a].view(L, s["cells"], KV, -1), s[b].view(L, s["cells"], KV, -1)
        moved = x[l, at, h].permute(0, 2, 1, 3)
        y[:, :most] = torch.where(put.permute(0, 2, 1)[..., None], moved, y[:, :most])
    for a, b in (("pos", "dpos"), ("mass", "dmass")):
        s[b][:, :, :most] = torch.where(put, s[a].gather(-1, at), s[b][:, :, :most])
    s["kept"].copy_(keep[..., 0].int())
    return s["dk"], s["dv"], s["dpos"], s["dmass"], s["kept"]


def _append_plain(s):
    c, T = s["case"], s["case"]["tokens"]
    L, KV = c["caches"], c["kv"]
    at = s["rows"].long()[..., None] + torch.arange(T, device="cuda")              # [L, KV, T]
    l = torch.arange(L, device="cuda")[:, None, None]
    h = torch.arange(KV, device="cuda")[None, :, None]
    for a, b in (("new_k", "k"), ("new_v", "v")):
        s[b].view(L, s["cells"], KV, -1)[l, at, h] = _to_rows(c, s[a]).permute(0, 2, 1, 3)
    s["pos"].scatter_(-1, at, s["tok_pos"].expand(L, KV, T))
    s["mass"].scatter_(-1, at, 0.0)
    s["rows_out"].copy_(s["rows"] + T)
    return s["k"], s["v"], s["pos"], s["mass"], s["rows_out"]


def _accept_plain(s):
    c, T = s["case"], s["case"]["tokens"]
    L, KV, m = c["caches"], c["kv"], c["kept"]
    base = s["rows"].long()[..., None] - T
    frm = base + s["path"].long()[:, None, :m]
    to = (base + torch.arange(m, device="cuda")).expand(L, KV, m)
    l = torch.arange(L, device="cuda")[:, None, None]
    h = torch.arange(KV, device="cuda")[None, :, None]
    for b in ("k", "v"):
        x = s[b].view(L, s["cells"], KV, -1)
        x[l, to, h] = x[l, frm.expand(L, KV, m), h]
    for b in ("pos", "mass"):
        s[b].scatter_(-1, to, s[b].gather(-1, frm.expand(L, KV, m)))
    s["rows_out"].copy_(s["rows"] - T + s["n_path"][:, None])
    return s["k"], s["v"], s["pos"], s["mass"], s["rows_out"]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op in ("attend", "attend mass"):
        return _attend_plain(state, op == "attend mass")
    return {"evict": _evict_plain, "append": _append_plain, "accept": _accept_plain}[op](state)


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """Attention unit by unit in fp64.  The other operators move and round
    stored numbers: their outputs have no value beyond those."""
    if case["op"] not in ("attend", "attend mass"):
        return None
    s = _inputs(case, seed)
    L, KV, G, T, hd = case["caches"], case["kv"], case["gqa"], case["tokens"], case["hd"]
    rb, cells = _row_bytes(case), s["cells"]
    out = torch.zeros((L, T, KV * G, hd), dtype=torch.float64, device="cuda")
    mass = torch.zeros((L, KV, cells), dtype=torch.float64, device="cuda")
    for l in range(L):
        for h in range(KV):
            n = int(s["rows_host"][l, h])
            if n == 0:
                continue
            kv = []
            for raw in (s["k"], s["v"]):
                r = raw[l, :n, h * rb:(h + 1) * rb].contiguous()
                if case["type"] == F16:
                    kv.append(r.view(torch.float16).double())
                else:
                    r = r.reshape(n * (hd // 32), 34)
                    d = r[:, :2].contiguous().view(torch.float16).double()
                    kv.append((r[:, 2:].contiguous().view(torch.int8).double() * d).reshape(n, hd))
            k, v = kv
            p = s["pos"][l, h, :n].double()
            t = s["tok_pos"].double()
            hide = torch.zeros((T, n), dtype=torch.bool, device="cuda")
            hide[:, n - T:] = ~s["sees"] if "sees" in s else torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1)
            if case["window"]:
                hide |= (t[:, None] - p[None] > case["window"]) & (p[None] >= case["sink"])
            for g in range(G):
                w = s["q"][l, :, h * G + g].double() @ k.T / hd ** 0.5
                if case["cap"]:
                    w = torch.tanh(w / case["cap"]) * case["cap"]
                if case["bias"]:
                    w = w - s["slopes"][h * G + g].double() * (t[:, None] - p[None])
                w = w.masked_fill(hide, float("-inf"))
                w = torch.exp(w - torch.logsumexp(w, 1, keepdim=True)).nan_to_num(0.0)
                out[l, :, h * G + g] = w @ v
                mass[l, h, :n] += w.sum(0)
            mass[l, h, :n] += s["mass"][l, h, :n].double() if "mass" in s else 0.0
    return out if case["op"] == "attend" else (out, mass)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    n, rb, L, KV = _rows(case).astype(np.float64), _row_bytes(case), case["caches"], case["kv"]
    op, T, hd = case["op"], case.get("tokens", 0), case["hd"]
    if op in ("attend", "attend mass"):
        # rows lie two positions apart on average: a window of w positions holds w / 2 cached rows and the tokens' own
        old = n - T
        seen = np.minimum(old, case["window"] / 2) if case["window"] else old
        among = _tree(T, 4)[1].sum() if case["mask"] == "tree" else T * (T + 1) / 2
        if case["window"]:
            among = min(among, T * (case["window"] + 1.0))
        pairs = float((seen * T + among).sum()) * case["gqa"]
        touched = float((np.minimum(old, seen + T / 2) + T).sum())
        b = touched * 2 * rb + 2 * L * T * KV * case["gqa"] * hd * 2
        f = 4 * hd * pairs
        if op == "attend mass":
            b += float(n.sum()) * 8
            f += pairs
        return {"bytes": b, "flops": f}
    if op == "evict":
        budget = max(1, int(case["rows"]) * case["percent"] // 100)
        kept = float((n - np.floor(np.maximum(n - budget, 0) * case["ramp"] / 100)).sum())
        return {"bytes": float(n.sum()) * 8 + kept * (4 * rb + 16), "flops": 0.0}
    if op == "append":
        src = 2 if case["source"] == "f16" else 4
        return {"bytes": L * T * KV * (2 * (hd * src + rb) + 8.0) + 8 * L * KV, "flops": 0.0}
    m = case["kept"]
    return {"bytes": L * KV * (m * (4 * rb + 16.0) + 8), "flops": 0.0}
