"""The operators of a mixture-of-experts layer as programs use them, one case per call: the router, the exchange of
token rows between token order and expert order, the products grouped by expert with their gradients, and the
products in 8-bit integers.

``listed()`` holds the named cases, ``draw(rng)`` gives further ones of the same ranges.  With ``own`` false ``run``
computes an operator in its plain form, with it the calls of ``sparsetir_b200.ops`` that a program makes.

The number of rows of every group of a case comes from its sizes alone; which group has how many, and all values, come
from the seed.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # router of a decoding step: 24 sequences, one token each; the smallest call, where latency counts
        dict(name="route_step", op="route", tokens=24, experts=64, top_k=6, dtype="float32", renorm=True, masked=0.0, grad=False),
        # router of a training batch with its padding masked, and the gradient to the logits
        dict(name="route_train", op="route", tokens=16384, experts=128, top_k=8, dtype="float32", renorm=False, masked=0.03,
             grad=True),
        # weighted sum of the experts' rows in a decoding step
        dict(name="combine_step", op="combine", tokens=24, top_k=6, groups=64, feat=1024, dtype="float16", grad=False),
        # rows of a long prompt's tokens to the experts' order
        dict(name="dispatch_prompt", op="dispatch", tokens=8192, top_k=8, groups=64, feat=2048, dtype="bfloat16"),
        # gradient of the weighted sum in training, to the rows and to the gates; a width that is no multiple of 16
        dict(name="combine_grad", op="combine", tokens=6007, top_k=4, groups=32, feat=2040, dtype="bfloat16", grad=True),
        # the experts' first product in a decoding step: the weights are read once, for a few rows each
        dict(name="mm_step", op="mm", rows=48, groups=8, feat_in=1024, feat_out=4096, dtype="bfloat16", out_in=True, skew=0.3),
        # a prompt of some thousand tokens through unevenly chosen experts, ragged sizes, the other weight layout
        dict(name="mm_prompt", op="mm", rows=6001, groups=16, feat_in=2048, feat_out=1408, dtype="float16", out_in=False, skew=0.8),
        # a training batch: 8192 tokens with 8 experts each
        dict(name="mm_train", op="mm", rows=65536, groups=64, feat_in=2048, feat_out=2048, dtype="bfloat16", out_in=True, skew=0.5),
        # gradients of the weights: a small layer of odd widths ...
        dict(name="grad_w_small", op="grad_w", rows=1000, groups=8, feat_in=504, feat_out=1000, dtype="float16", skew=0.8),
        # ... and of a training batch
        dict(name="grad_w_train", op="grad_w", rows=32768, groups=64, feat_in=2048, feat_out=1024, dtype="bfloat16", skew=0.5),
        # one token through a dense layer with 8-bit weights, its quantisation included
        dict(name="i8_step", op="mm_i8", tokens=1, top_k=1, groups=1, feat_in=4096, feat_out=8192, dtype="bfloat16", skew=0.0),
        # a prompt through experts with 8-bit weights, quantisation and dispatch included
        dict(name="i8_prompt", op="mm_i8", tokens=4096, top_k=4, groups=32, feat_in=2048, feat_out=2048, dtype="float16", skew=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, hi, unit=1):
    """Features of a layer: powers of two, multiples of 8, and now and then any number."""
    kind = rng.random()
    if kind < 0.4:
        return 2 ** rng.randint(6, int(math.log2(hi)))
    if kind < 0.85:
        return 8 * _log_int(rng, 8, hi // 8)
    return _log_int(rng, 50, hi)


def draw(rng):
    op = rng.choice(["route", "combine", "dispatch", "mm", "mm", "mm", "grad_w", "grad_w", "mm_i8", "mm_i8"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "route":
        experts = rng.choice([8, 16, 64, 128, 256, rng.randint(4, 256)])
        return dict(op=op, tokens=_log_int(rng, 1, 16384), experts=experts, top_k=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]), renorm=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.0, 0.05]), grad=rng.random() < 0.5)
    if op in ("combine", "dispatch"):
        top_k = rng.randint(1, 8)
        feat = _width(rng, 4096)
        tokens = _log_int(rng, 1, min(16384, 8192 * 8 * 2048 // (top_k * feat)))
        c = dict(op=op, tokens=tokens, top_k=top_k, groups=rng.randint(max(2, top_k), 128), feat=feat, dtype=dtype)
        return dict(c, grad=rng.random() < 0.5) if op == "combine" else c
    groups = rng.choice([1, 8, 16, 64, rng.randint(2, 64)])
    fi, fo = _width(rng, 4096), _width(rng, 4096)
    while groups * fi * fo > 64 * 2048 * 2048:
        groups //= 2
    most = min(65536, 65536 * 2048 * 2048 // (fi * fo)) // 2
    c = dict(op=op, groups=groups, feat_in=fi, feat_out=fo, dtype=dtype, skew=round(rng.uniform(0.0, 0.8), 2))
    if op == "mm_i8":
        top_k = 1 if groups == 1 else rng.randint(1, min(4, groups))
        return dict(c, top_k=top_k, tokens=_log_int(rng, 1, max(1, most // top_k)))
    c["rows"] = _log_int(rng, 1, most)
    return dict(c, out_in=rng.random() < 0.5) if op == "mm" else c


# ------------------------------------------------------------------ inputs
def _sizes(case):
    """Rows of every group, before the seed shuffles them over the groups: log-normal popularity."""
    groups = case["groups"]
    rows = case["rows"] if "rows" in case else case["tokens"] * case["top_k"]
    rng = np.random.Generator(np.random.PCG64(rows * 1009 + groups))
    share = np.exp(case["skew"] * rng.standard_normal(groups))
    return rng.multinomial(rows, share / share.sum()).astype(np.int64)


def _pointers(sizes):
    out = torch.zeros(len(sizes) + 1, dtype=torch.int64, device="cuda")
    torch.cumsum(sizes, 0, out=out[1:])
    return out.int()


def _normal(g, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _exchange(case, g):
    """Distinct random experts for every token and the stable places of the pairs by expert."""
    t, k = case["tokens"], case["top_k"]
    chosen = torch.rand(t, case["groups"], device="cuda", generator=g).argsort(1)[:, :k].reshape(-1)
    slots = torch.empty(t * k, dtype=torch.int32, device="cuda")
    slots[chosen.sort(stable=True).indices] = torch.arange(t * k, dtype=torch.int32, device="cuda")
    return slots


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    dtype = TYPES[case["dtype"]]
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        # popular experts, and a spread of a few units within a token
        z = torch.randn(t, e, device="cuda", generator=g) * 1.5 + torch.randn(e, device="cuda", generator=g) * 0.5
        if case["masked"]:  # the padding of a batch: tokens that no expert takes
            z[torch.rand(t, device="cuda", generator=g) < case["masked"]] = -math.inf
        s.update(logits=z.to(dtype).view(-1), d_gates=torch.randn(t * k, device="cuda", generator=g),
                 gates=torch.zeros(t * k, device="cuda"), experts_of=torch.zeros(t * k, **i32), slots=torch.zeros(t * k, **i32),
                 indptr=torch.zeros(e + 1, **i32), d_logits=torch.zeros(t * e, dtype=dtype, device="cuda"))
        return s
    if case["op"] in ("combine", "dispatch"):
        t, k, f = case["tokens"], case["top_k"], case["feat"]
        s["slots"] = _exchange(case, g)
        s["x"] = _normal(g, dtype, t * f)
        s["z"] = _normal(g, dtype, t * k * f) if case["op"] == "combine" else torch.zeros(t * k * f, dtype=dtype, device="cuda")
        s["gates"] = torch.softmax(torch.randn(t, k, device="cuda", generator=g), 1).view(-1)
        s["y"] = torch.zeros(t * f, dtype=dtype, device="cuda")
        s["d_gates"] = torch.zeros(t * k, device="cuda")
        if case.get("grad"):
            s["dz"] = torch.zeros(t * k * f, dtype=dtype, device="cuda")
        return s
    sizes = _sizes(case)
    s["cap"] = int(sizes.max())
    s["indptr"] = _pointers(torch.from_numpy(sizes).cuda()[torch.randperm(len(sizes), device="cuda", generator=g)])
    rows, n, fi, fo = int(sizes.sum()), case["groups"], case["feat_in"], case["feat_out"]
    s["rows"] = rows
    if case["op"] == "mm":
        s.update(x=_normal(g, dtype, rows * fi), w=_normal(g, dtype, n * fi * fo, scale=fi ** -0.5),
                 y=torch.zeros(rows * fo, dtype=dtype, device="cuda"))
    elif case["op"] == "grad_w":
        s.update(x=_normal(g, dtype, rows * fi), dy=_normal(g, dtype, rows * fo), dw=torch.zeros(n * fi * fo, dtype=dtype, device="cuda"))
    else:
        t, k = case["tokens"], case["top_k"]
        # activations with a few large channels, as quantised layers meet them
        x = torch.randn(t, fi, device="cuda", generator=g)
        x *= torch.exp(0.5 * torch.randn(fi, device="cuda", generator=g))
        s["slots"] = torch.randperm(rows, device="cuda", generator=g).int() if k > 1 else None
        s.update(x=x.to(dtype).view(-1), w=torch.randint(-127, 128, (n * fo * fi,), device="cuda", generator=g, dtype=torch.int8),
                 w_scale=torch.rand(n * fo, device="cuda", generator=g) * (0.02 / fi ** 0.5) + 1e-5,
                 xq=torch.zeros(rows * fi, dtype=torch.int8, device="cuda"), x_scale=torch.zeros(rows, device="cuda"),
                 y=torch.zeros(rows * fo, dtype=dtype, device="cuda"))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (OWN if own else PLAIN)[state["op"]](state)


def _own_route(s):
    from sparsetir_b200 import ops

    flags = ops.MOE_RENORMALIZE if s["renorm"] else 0
    ops.moe_route(s["logits"], s["gates"], s["experts_of"], s["slots"], s["indptr"], s["experts"], s["top_k"], flags)
    out = {"gates": s["gates"], "experts": s["experts_of"], "slots": s["slots"], "indptr": s["indptr"]}
    if s["grad"]:
        ops.moe_route_grad(s["logits"], s["gates"], s["experts_of"], s["d_gates"], s["d_logits"], s["experts"], s["top_k"], flags)
        out["d_logits"] = s["d_logits"]
    return out


def _own_dispatch(s):
    from sparsetir_b200 import ops

    ops.moe_dispatch(s["x"], s["slots"], s["z"], s["feat"], s["top_k"])
    return s["z"]


def _own_combine(s):
    from sparsetir_b200 import ops

    if s["grad"]:  # x is the gradient of the sum
        ops.moe_combine_grad(s["x"], s["z"], s["slots"], s["gates"], s["dz"], s["d_gates"], s["feat"], s["top_k"])
        return {"dz": s["dz"], "d_gates": s["d_gates"]}
    ops.moe_combine(s["z"], s["slots"], s["gates"], s["y"], s["feat"], s["top_k"])
    return s["y"]


def _own_mm(s):
    from sparsetir_b200 import ops

    ops.grouped_mm(s["x"], s["w"], s["y"], s["indptr"], s["groups"], s["feat_in"], s["feat_out"],
                   ops.GROUPED_W_OUT_IN if s["out_in"] else 0)
    return s["y"]


def _own_grad_w(s):
    from sparsetir_b200 import ops

    ops.grouped_mm_grad_w(s["x"], s["dy"], s["dw"], s["indptr"], s["groups"], s["feat_in"], s["feat_out"])
    return s["dw"]


def _own_mm_i8(s):
    from sparsetir_b200 import ops

    ops.moe_dispatch_i8(s["x"], s["slots"], s["xq"], s["x_scale"], s["feat_in"], s["top_k"])
    ops.grouped_mm_i8(s["xq"], s["x_scale"], s["w"], s["w_scale"], s["y"], s["indptr"], s["groups"], s["feat_in"], s["feat_out"])
    return s["y"]


def _plain_route(s):
    t, e, k = s["tokens"], s["experts"], s["top_k"]
    z = s["logits"].view(t, e).float()
    top, at = torch.sort(z, dim=1, descending=True, stable=True)  # equal logits: the lowest index first
    top, at = top[:, :k], at[:, :k]
    kept = top > -math.inf
    ex = torch.exp(z - torch.where(kept[:, :1], top[:, :1], 0.0))
    total = ex.sum(1, keepdim=True)
    chosen = torch.where(kept, torch.gather(ex, 1, at), 0.0)
    over = chosen.sum(1, keepdim=True) if s["renorm"] else total
    gates = torch.where(kept, chosen / torch.where(over > 0, over, 1.0), 0.0)
    # the pairs by expert, in the order of the tokens; pairs without an expert come last
    key = torch.where(kept, at, e).view(-1)
    order = torch.sort(key, stable=True).indices
    place = torch.empty(t * k, dtype=torch.int32, device=z.device)
    place[order] = torch.arange(t * k, dtype=torch.int32, device=z.device)
    bounds = torch.arange(e + 1, device=z.device)
    indptr = (key[:, None] < bounds[None, :]).sum(0).int() if t * k < 1024 else torch.searchsorted(key[order], bounds).int()
    out = {"gates": gates.view(-1), "experts": torch.where(kept, at, -1).int().view(-1),
           "slots": torch.where(kept.view(-1), place, -1), "indptr": indptr}
    if s["grad"]:
        dg = torch.where(kept, s["d_gates"].view(t, k), 0.0)
        mean = (dg * gates).sum(1, keepdim=True)
        if s["renorm"]:
            dz = torch.zeros_like(z).scatter_(1, at, gates * (dg - mean))
        else:
            dz = (-mean * ex / torch.where(total > 0, total, 1.0)).scatter_add_(1, at, gates * dg)
        out["d_logits"] = torch.where(z > -math.inf, dz, 0.0).to(s["d_logits"].dtype).view(-1)
    return out


def _plain_dispatch(s):
    t, k, f = s["tokens"], s["top_k"], s["feat"]
    z = torch.zeros_like(s["z"]).view(t * k, f)
    z[s["slots"].long()] = s["x"].view(t, 1, f).expand(t, k, f).reshape(t * k, f)
    return z.view(-1)


def _plain_combine(s):
    t, k, f = s["tokens"], s["top_k"], s["feat"]
    rows = s["z"].view(t * k, f)[s["slots"].long()].float().view(t, k, f)
    gates = s["gates"].view(t, k, 1)
    if not s["grad"]:
        return (rows * gates).sum(1).to(s["y"].dtype).view(-1)
    dy = s["x"].view(t, 1, f).float()
    dz = torch.zeros_like(s["dz"]).view(t * k, f)
    dz[s["slots"].long()] = (gates * dy).view(t * k, f).to(dz.dtype)
    return {"dz": dz.view(-1), "d_gates": (rows * dy).sum(2).view(-1)}


def _by_group(s, x):
    """Rows of every group side by side, groups padded with zeros to the largest: [groups, cap, features]."""
    ptr = s["indptr"].long()
    at = ptr[:-1, None] + torch.arange(s["cap"], device=x.device)
    live = at < ptr[1:, None]
    return torch.where(live[:, :, None], x[at.clamp(max=s["rows"] - 1)], 0)


def _by_row(s, y):
    """The inverse: the rows of [groups, cap, features] in their own order."""
    ptr = s["indptr"].long()
    row = torch.arange(s["rows"], device=y.device)
    group = torch.searchsorted(ptr[1:], row, right=True)
    return y[group, row - ptr[group]]


def _plain_mm(s):
    n, fi, fo = s["groups"], s["feat_in"], s["feat_out"]
    w = s["w"].float()
    w = w.view(n, fo, fi).transpose(1, 2) if s["out_in"] else w.view(n, fi, fo)
    return _by_row(s, torch.bmm(_by_group(s, s["x"].view(-1, fi).float()), w)).to(s["y"].dtype).view(-1)


def _plain_grad_w(s):
    fi, fo = s["feat_in"], s["feat_out"]
    x, dy = _by_group(s, s["x"].view(-1, fi).float()), _by_group(s, s["dy"].view(-1, fo).float())
    return torch.bmm(x.transpose(1, 2), dy).to(s["dw"].dtype).view(-1)


def _plain_mm_i8(s):
    n, fi, fo, k = s["groups"], s["feat_in"], s["feat_out"], s["top_k"]
    x = s["x"].view(-1, fi).float()
    most = x.abs().amax(1, keepdim=True)
    q = torch.round(x * torch.where(most > 0, 127.0 / most, 0.0))
    scale = most / 127.0
    if s["slots"] is not None:
        to = s["slots"].long()
        q = torch.zeros(s["rows"], fi, device=q.device).index_copy_(0, to, q.repeat_interleave(k, 0))
        scale = torch.zeros(s["rows"], 1, device=q.device).index_copy_(0, to, scale.repeat_interleave(k, 0))
    y = torch.bmm(_by_group(s, q), s["w"].float().view(n, fo, fi).transpose(1, 2))
    return (_by_row(s, y * s["w_scale"].view(n, 1, fo)) * scale).to(s["y"].dtype).view(-1)


OWN = {"route": _own_route, "dispatch": _own_dispatch, "combine": _own_combine, "mm": _own_mm, "grad_w": _own_grad_w,
       "mm_i8": _own_mm_i8}
PLAIN = {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "mm": _plain_mm,
         "grad_w": _plain_grad_w, "mm_i8": _plain_mm_i8}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] in ("dispatch", "combine"):
        t, k, f = case["tokens"], case["top_k"], case["feat"]
        slots = s["slots"].view(t, k).long()
        if case["op"] == "dispatch":
            z = torch.zeros(t * k, f, dtype=torch.float64, device="cuda")
            for j in range(k):
                z[slots[:, j]] = s["x"].view(t, f).double()
            return z.view(-1)
        z, gates = s["z"].view(t * k, f), s["gates"].view(t, k).double()
        if not case["grad"]:
            y = torch.zeros(t, f, dtype=torch.float64, device="cuda")
            for j in range(k):
                y += gates[:, j, None] * z[slots[:, j]].double()
            return y.view(-1)
        dy, dz, dg = s["x"].view(t, f).double(), torch.zeros(t * k, f, dtype=torch.float64, device="cuda"), torch.zeros_like(gates)
        for j in range(k):
            dz[slots[:, j]] = gates[:, j, None] * dy
            dg[:, j] = (z[slots[:, j]].double() * dy).sum(1)
        return {"dz": dz.view(-1), "d_gates": dg.view(-1)}
    n, fi, fo, ptr = case["groups"], case["feat_in"], case["feat_out"], s["indptr"].tolist()
    if case["op"] == "grad_w":
        dw = torch.zeros(n, fi, fo, dtype=torch.float64, device="cuda")
        for g in range(n):
            rows = slice(ptr[g], ptr[g + 1])
            dw[g] = s["x"].view(-1, fi)[rows].double().t() @ s["dy"].view(-1, fo)[rows].double()
        return dw.view(-1)
    y = torch.zeros(s["rows"], fo, dtype=torch.float64, device="cuda")
    if case["op"] == "mm":
        for g in range(n):
            w = s["w"].view(n, -1)[g].double()
            w = w.view(fo, fi).t() if case["out_in"] else w.view(fi, fo)
            y[ptr[g]:ptr[g + 1]] = s["x"].view(-1, fi)[ptr[g]:ptr[g + 1]].double() @ w
        return y.view(-1)
    x = s["x"].view(-1, fi).double()
    most = x.abs().max(1).values.clamp(min=1e-300)
    rows = torch.zeros(s["rows"], fi, dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):  # the quantised rows stand for q * most / 127
        to = slice(None) if s["slots"] is None else s["slots"].view(-1, case["top_k"])[:, j].long()
        rows[to] = torch.round(x * 127 / most[:, None]) * most[:, None] / 127
    for g in range(n):
        w = s["w"].view(n, fo, fi)[g].double() * s["w_scale"].view(n, fo)[g].double()[:, None]
        y[ptr[g]:ptr[g + 1]] = rows[ptr[g]:ptr[g + 1]] @ w.t()
    return y.view(-1)


def _exact_route(s):
    t, e, k = s["tokens"], s["experts"], s["top_k"]
    z = s["logits"].view(t, e).double().cpu().numpy()
    at = np.argsort(-z, axis=1, kind="stable")[:, :k]
    dead = np.isneginf(np.take_along_axis(z, at, 1))
    top = z.max(1, keepdims=True)
    p = np.exp(z - np.where(np.isneginf(top), 0.0, top))
    p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
    gates = np.where(dead, 0.0, np.take_along_axis(p, at, 1))
    if s["renorm"]:
        gates = gates / np.maximum(gates.sum(1, keepdims=True), 1e-300)
    out = {"gates": torch.from_numpy(gates.reshape(-1)), "experts": None, "slots": None, "indptr": None}
    if s["grad"]:
        dg = np.where(dead, 0.0, s["d_gates"].view(t, k).double().cpu().numpy())
        mean = (gates * dg).sum(1, keepdims=True)
        dz = np.zeros_like(p) if s["renorm"] else -p * mean
        rows = np.arange(t)
        for j in range(k):
            dz[rows, at[:, j]] += gates[:, j] * (dg[:, j] - (mean[:, 0] if s["renorm"] else 0.0))
        out["d_logits"] = torch.from_numpy(dz.reshape(-1))
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, size = case["op"], 4 if case["dtype"] == "float32" else 2
    if op == "route":
        t, e, pairs = case["tokens"], case["experts"], case["tokens"] * case["top_k"]
        both = 2 if case["grad"] else 1
        # logits in (the gradient's too), gates, experts and places out; d_gates in, d_logits out
        return {"bytes": t * e * size * both + 12 * pairs + 4 * (e + 1) + (4 * pairs + 8 * pairs + 4 * pairs if case["grad"] else 0),
                "flops": 5.0 * t * e * both}
    if op in ("combine", "dispatch"):
        t, pairs, f = case["tokens"], case["tokens"] * case["top_k"], case["feat"]
        if op == "dispatch":
            return {"bytes": size * f * (t + pairs) + 4 * pairs, "flops": 0.0}
        if case["grad"]:
            return {"bytes": size * f * (t + 2 * pairs) + 12 * pairs, "flops": 3.0 * pairs * f}
        return {"bytes": size * f * (t + pairs) + 8 * pairs, "flops": 2.0 * pairs * f}
    sizes, fi, fo = _sizes(case), case["feat_in"], case["feat_out"]
    rows, used = int(sizes.sum()), int((sizes > 0).sum())
    if op == "mm":
        moved = size * (rows * fi + rows * fo + used * fi * fo)
    elif op == "grad_w":
        moved = size * (rows * fi + rows * fo + case["groups"] * fi * fo)
    else:  # 16-bit rows in, 8-bit rows out and in again, 8-bit weights, 16-bit result
        moved = size * case["tokens"] * fi + 2 * rows * fi + used * fi * fo + size * rows * fo + 8 * rows + 4 * used * fo
    return {"bytes": moved + 4 * (case["groups"] + 1), "flops": 2.0 * rows * fi * fo}
