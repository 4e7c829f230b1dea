"""The gated block of an expert with its gradient, and products in 8-bit floating point with a scale for each block of
128, as programs use them, one case per call.

``listed()`` holds the named cases, ``draw(rng)`` gives further ones of the same ranges.  With ``own`` false ``run``
computes an operator in its plain form, with it the calls of ``sparsetir_b200.ops`` that a program makes.

The number of rows of every group of a case comes from its sizes alone; which group has how many, and all values, come
from the seed.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
F8 = torch.float8_e4m3fn  # 448 is its largest number
BLOCK = 128               # elements that share a scale


def listed():
    return [
        # the gated block of a decoding step: 24 tokens, two experts each; the weights are read once, for a few rows
        dict(name="gated_step", op="gated", rows=48, groups=8, feat_in=1024, width=2048, dtype="bfloat16", gelu=False, keep=False,
             skew=0.3),
        # a prompt through unevenly chosen experts, ragged sizes, the other activation
        dict(name="gated_prompt", op="gated", rows=6001, groups=16, feat_in=2048, width=1408, dtype="float16", gelu=True, keep=False,
             skew=0.8),
        # a training batch: 8192 tokens with 8 experts each; both projections are kept for the gradient
        dict(name="gated_train", op="gated", rows=65536, groups=64, feat_in=2048, width=1024, dtype="bfloat16", gelu=False, keep=True,
             skew=0.5),
        # its gradient through the second product, with the activations formed again: a small layer of odd widths ...
        dict(name="gated_grad_small", op="gated_grad", rows=1000, groups=8, feat_in=504, width=1000, dtype="float16", gelu=True,
             keep=True, skew=0.8),
        # ... and the training batch
        dict(name="gated_grad_train", op="gated_grad", rows=65536, groups=64, feat_in=2048, width=1024, dtype="bfloat16", gelu=False,
             keep=True, skew=0.5),
        # activations of a decoding step to 8 bits, in the experts' order; the smallest call, where latency counts
        dict(name="quant_step", op="quant", tokens=24, top_k=2, groups=8, feat=1024, dtype="bfloat16", skew=0.3),
        # and of a long prompt
        dict(name="quant_prompt", op="quant", tokens=8192, top_k=8, groups=64, feat=2048, dtype="bfloat16", skew=0.5),
        # one token through a dense layer, its quantisation included
        dict(name="f8_step", op="mm_f8", tokens=1, top_k=1, groups=1, feat_in=4096, feat_out=8192, dtype="bfloat16", skew=0.0),
        # a prompt through experts, quantisation and dispatch included
        dict(name="f8_prompt", op="mm_f8", tokens=4096, top_k=4, groups=32, feat_in=2048, feat_out=2048, dtype="float16", skew=0.5),
        # a large batch of prompts: 8192 tokens with 8 experts each
        dict(name="f8_batch", op="mm_f8", tokens=8192, top_k=8, groups=64, feat_in=2048, feat_out=2048, dtype="bfloat16", skew=0.5),
        # the gated block in 8 bits: a decoding step and a prompt, quantisation and dispatch included
        dict(name="f8_gated_step", op="gated_f8", tokens=24, top_k=2, groups=8, feat_in=1024, width=2048, dtype="bfloat16", gelu=False,
             skew=0.3),
        dict(name="f8_gated_prompt", op="gated_f8", tokens=4096, top_k=4, groups=32, feat_in=2048, width=1408, dtype="float16",
             gelu=False, skew=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, hi):
    """Features of a layer: powers of two, multiples of 8, and now and then any number."""
    kind = rng.random()
    if kind < 0.4:
        return 2 ** rng.randint(6, int(math.log2(hi)))
    if kind < 0.85:
        return 8 * _log_int(rng, 8, hi // 8)
    return _log_int(rng, 50, hi)


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_grad", "gated_grad", "quant", "mm_f8", "mm_f8", "gated_f8"])
    dtype = rng.choice(["float16", "bfloat16"])
    groups = rng.choice([1, 8, 16, 64, rng.randint(2, 64)])
    skew = round(rng.uniform(0.0, 0.8), 2)
    if op == "quant":
        top_k, feat = (1 if groups == 1 else rng.randint(1, min(8, groups))), _width(rng, 4096)
        tokens = _log_int(rng, 1, min(16384, 8192 * 8 * 2048 // (top_k * feat)))
        return dict(op=op, tokens=tokens, top_k=top_k, groups=groups, feat=feat, dtype=dtype, skew=skew)
    fi, fo = _width(rng, 4096), _width(rng, 4096 if op == "mm_f8" else 2048)
    wide = fo if op in ("mm_f8", "gated_grad") else 2 * fo
    while groups * fi * wide > 64 * 2048 * 2048:
        groups //= 2
    most = min(65536, 65536 * 2048 * 2048 // (fi * wide)) // 2
    c = dict(op=op, groups=groups, feat_in=fi, dtype=dtype, skew=skew)
    if op in ("gated", "gated_grad"):
        return dict(c, width=fo, rows=_log_int(rng, 1, most), gelu=rng.random() < 0.3, keep=rng.random() < 0.5)
    top_k = 1 if groups == 1 else rng.randint(1, min(4, groups))
    c.update(top_k=top_k, tokens=_log_int(rng, 1, max(1, most // top_k)))
    return dict(c, feat_out=fo) if op == "mm_f8" else dict(c, width=fo, gelu=rng.random() < 0.3)


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


def _blocks(n):
    return -(-n // BLOCK)


def _weights_f8(g, groups, fo, fi):
    """Weights in 8 bits, [groups, fo, fi], with a scale for each 128 x 128 of them, as a checkpoint holds them."""
    w = torch.randn(groups, fo, fi, device="cuda", generator=g) * fi ** -0.5
    w *= torch.exp(0.3 * torch.randn(groups, fo, 1, device="cuda", generator=g))
    pad = torch.zeros(groups, _blocks(fo) * BLOCK, _blocks(fi) * BLOCK, device="cuda")
    pad[:, :fo, :fi] = w
    tiles = pad.view(groups, _blocks(fo), BLOCK, _blocks(fi), BLOCK)
    scale = tiles.abs().amax((2, 4)) / 448
    tiles /= scale[:, :, None, :, None].clamp(min=1e-30)
    return pad[:, :fo, :fi].clamp(-448, 448).to(F8).reshape(-1), scale.reshape(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    op, dtype = case["op"], TYPES[case["dtype"]]
    sizes = _sizes(case)
    s["cap"] = int(sizes.max())
    s["indptr"] = _pointers(torch.from_numpy(sizes).cuda()[torch.randperm(len(sizes), device="cuda", generator=g)])
    rows, n = int(sizes.sum()), case["groups"]
    s["rows"] = rows
    if op == "gated":
        fi, width = case["feat_in"], case["width"]
        s.update(x=_normal(g, dtype, rows * fi), w=_normal(g, dtype, n * 2 * width * fi, scale=fi ** -0.5),
                 y=torch.zeros(rows * width, dtype=dtype, device="cuda"),
                 hidden=torch.zeros(rows * 2 * width, dtype=dtype, device="cuda") if case["keep"] else None)
        return s
    if op == "gated_grad":
        fi, width = case["feat_in"], case["width"]
        s.update(dy=_normal(g, dtype, rows * fi, scale=0.1), w=_normal(g, dtype, n * fi * width, scale=width ** -0.5),
                 hidden=_normal(g, dtype, rows * 2 * width), d_hidden=torch.zeros(rows * 2 * width, dtype=dtype, device="cuda"),
                 act=torch.zeros(rows * width, dtype=dtype, device="cuda") if case["keep"] else None)
        return s
    t, k, fi = case["tokens"], case["top_k"], case["feat"] if op == "quant" else case["feat_in"]
    # activations with a few large channels, as quantised layers meet them
    x = torch.randn(t, fi, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(fi, device="cuda", generator=g))
    s["slots"] = torch.randperm(rows, device="cuda", generator=g).int() if k > 1 else None
    s.update(x=x.to(dtype).view(-1), xq=torch.zeros(rows * fi, dtype=F8, device="cuda"),
             x_scale=torch.zeros(_blocks(fi) * rows, device="cuda"))
    if op != "quant":
        fo = case["feat_out"] if op == "mm_f8" else 2 * case["width"]
        s["w"], s["w_scale"] = _weights_f8(g, n, fo, fi)
        s["y"] = torch.zeros(rows * (fo if op == "mm_f8" else case["width"]), dtype=dtype, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (OWN if own else PLAIN)[state["op"]](state)


def _own_gated(s):
    from sparsetir_b200 import ops

    ops.grouped_mm_gated(s["x"], s["w"], s["y"], s["hidden"], s["indptr"], s["groups"], s["feat_in"], s["width"],
                         ops.GATED_GELU if s["gelu"] else 0)
    return {"y": s["y"], "hidden": s["hidden"]} if s["keep"] else {"y": s["y"]}


def _own_gated_grad(s):
    from sparsetir_b200 import ops

    ops.grouped_mm_gated_grad(s["dy"], s["w"], s["hidden"], s["d_hidden"], s["act"], s["indptr"], s["groups"], s["feat_in"],
                              s["width"], ops.GATED_GELU if s["gelu"] else 0)
    return {"d_hidden": s["d_hidden"], "act": s["act"]} if s["keep"] else {"d_hidden": s["d_hidden"]}


def _own_quant(s):
    from sparsetir_b200 import ops

    ops.moe_dispatch_f8(s["x"], s["slots"], s["xq"], s["x_scale"], s["feat"], s["top_k"])
    return {"q": s["xq"], "scale": s["x_scale"]}


def _own_mm_f8(s):
    from sparsetir_b200 import ops

    ops.moe_dispatch_f8(s["x"], s["slots"], s["xq"], s["x_scale"], s["feat_in"], s["top_k"])
    ops.grouped_mm_f8(s["xq"], s["x_scale"], s["w"], s["w_scale"], s["y"], s["indptr"], s["groups"], s["feat_in"], s["feat_out"])
    return s["y"]


def _own_gated_f8(s):
    from sparsetir_b200 import ops

    ops.moe_dispatch_f8(s["x"], s["slots"], s["xq"], s["x_scale"], s["feat_in"], s["top_k"])
    ops.grouped_mm_gated_f8(s["xq"], s["x_scale"], s["w"], s["w_scale"], s["y"], s["indptr"], s["groups"], s["feat_in"], s["width"],
                            ops.GATED_GELU if s["gelu"] else 0)
    return s["y"]


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


def _activate(gate, gelu):
    if gelu:  # the form with tanh
        return 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    return gate / (1 + torch.exp(-gate))


def _plain_gated(s):
    n, fi, width = s["groups"], s["feat_in"], s["width"]
    hidden = _by_row(s, torch.bmm(_by_group(s, s["x"].view(-1, fi).float()), s["w"].float().view(n, 2 * width, fi).transpose(1, 2)))
    out = {"y": (_activate(hidden[:, :width], s["gelu"]) * hidden[:, width:]).to(s["y"].dtype).view(-1)}
    if s["keep"]:
        out["hidden"] = hidden.to(s["y"].dtype).view(-1)
    return out


def _plain_gated_grad(s):
    n, fi, width = s["groups"], s["feat_in"], s["width"]
    d_act = _by_row(s, torch.bmm(_by_group(s, s["dy"].view(-1, fi).float()), s["w"].float().view(n, fi, width)))
    hidden = s["hidden"].view(-1, 2 * width).float()
    gate, up = hidden[:, :width], hidden[:, width:]
    if s["gelu"]:
        inner = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)
        tanh = torch.tanh(inner)
        slope = 0.5 * (1 + tanh) + 0.5 * gate * (1 - tanh * tanh) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * gate * gate)
    else:
        sig = 1 / (1 + torch.exp(-gate))
        slope = sig * (1 + gate * (1 - sig))
    of_gate = _activate(gate, s["gelu"])
    out = {"d_hidden": torch.cat([d_act * up * slope, d_act * of_gate], 1).to(s["d_hidden"].dtype).view(-1)}
    if s["keep"]:
        out["act"] = (of_gate * up).to(s["act"].dtype).view(-1)
    return out


def _quantise(s, feat):
    """Rows in the experts' order, quantised: [rows, blocks, 128] in 8 bits and [rows, blocks] scales."""
    x = s["x"].view(-1, feat).float()
    blocks = _blocks(feat)
    pad = torch.zeros(x.shape[0], blocks * BLOCK, device=x.device)
    pad[:, :feat] = x
    tiles = pad.view(-1, blocks, BLOCK)
    most = tiles.abs().amax(2)
    # 448 x / most: the product is exact for elements of 16 bits, so that a quotient half way between two numbers stays there
    q = (tiles * 0.875 / torch.where(most > 0, most / 512, 1.0)[:, :, None]).to(F8)
    scale = most / 448.0
    if s["slots"] is not None:
        pair_of = torch.empty(s["rows"], dtype=torch.int64, device=x.device)
        pair_of[s["slots"].long()] = torch.arange(s["rows"], device=x.device)
        token = pair_of // s["top_k"]
        q, scale = q.view(torch.int8)[token].view(F8), scale[token]
    return q, scale


def _plain_quant(s):
    q, scale = _quantise(s, s["feat"])
    q = q.view(s["rows"], -1).view(torch.int8)[:, :s["feat"]].contiguous().view(F8)
    return {"q": q.view(-1), "scale": scale.t().contiguous().view(-1)}


def _plain_product_f8(s, fo):
    n, fi = s["groups"], s["feat_in"]
    q, scale = _quantise(s, fi)
    x = (q.float() * scale[:, :, None]).view(s["rows"], -1)[:, :fi]
    to = s["w_scale"].view(n, _blocks(fo), _blocks(fi)).repeat_interleave(BLOCK, 1)[:, :fo].repeat_interleave(BLOCK, 2)[:, :, :fi]
    w = s["w"].float().view(n, fo, fi) * to
    return _by_row(s, torch.bmm(_by_group(s, x), w.transpose(1, 2)))


def _plain_mm_f8(s):
    return _plain_product_f8(s, s["feat_out"]).to(s["y"].dtype).view(-1)


def _plain_gated_f8(s):
    hidden = _plain_product_f8(s, 2 * s["width"])
    return (_activate(hidden[:, :s["width"]], s["gelu"]) * hidden[:, s["width"]:]).to(s["y"].dtype).view(-1)


OWN = {"gated": _own_gated, "gated_grad": _own_gated_grad, "quant": _own_quant, "mm_f8": _own_mm_f8, "gated_f8": _own_gated_f8}
PLAIN = {"gated": _plain_gated, "gated_grad": _plain_gated_grad, "quant": _plain_quant, "mm_f8": _plain_mm_f8,
         "gated_f8": _plain_gated_f8}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _gate64(g, gelu):
    """The activation and its derivative."""
    if gelu:
        c = math.sqrt(2 / math.pi)
        z, dz = 2 * c * (g + 0.044715 * g ** 3), 2 * c * (1 + 3 * 0.044715 * g ** 2)
    else:
        z, dz = g, torch.ones_like(g)
    p = torch.sigmoid(z)
    return g * p, p + g * p * (1 - p) * dz


def _e4m3(v):
    """The number of 4 bits' exponent and 3 bits' fraction next to v, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    op, n, ptr = case["op"], case["groups"], s["indptr"].tolist()
    spans = [slice(ptr[g], ptr[g + 1]) for g in range(n)]
    f64 = dict(dtype=torch.float64, device="cuda")
    if op == "gated_grad":
        fi, width = case["feat_in"], case["width"]
        d_act = torch.zeros(s["rows"], width, **f64)
        for g, rows in enumerate(spans):
            d_act[rows] = s["dy"].view(-1, fi)[rows].double() @ s["w"].view(n, fi, width)[g].double()
        up = s["hidden"].view(-1, 2 * width)[:, width:].double()
        of_gate, slope = _gate64(s["hidden"].view(-1, 2 * width)[:, :width].double(), case["gelu"])
        out = {"d_hidden": torch.stack([d_act * slope * up, d_act * of_gate], 1).view(-1)}
        if case["keep"]:
            out["act"] = (of_gate * up).view(-1)
        return out
    if op == "gated":
        fi, fo = case["feat_in"], 2 * case["width"]
        x, w = s["x"].view(-1, fi).double(), lambda g: s["w"].view(n, fo, fi)[g].double()  # noqa: E731
    else:
        fi = case["feat"] if op == "quant" else case["feat_in"]
        t, k = case["tokens"], case["top_k"]
        tokens = s["x"].view(t, fi).double()
        tiles = [tokens[:, at:at + BLOCK] for at in range(0, fi, BLOCK)]
        most = torch.stack([b.abs().max(1).values for b in tiles], 1)
        parts = torch.cat([b * 448 / torch.where(most > 0, most, 1.0)[:, i, None] for i, b in enumerate(tiles)], 1)
        rows_of = [slice(None)] if s["slots"] is None else [s["slots"].view(t, k)[:, j].long() for j in range(k)]
        x, scale = torch.zeros(s["rows"], fi, **f64), torch.zeros(s["rows"], len(tiles), **f64)
        if op == "quant":  # the numbers that are rounded to 8 bits
            for to in rows_of:
                x[to], scale[to] = parts, most / 448
            return {"q": x.view(-1), "scale": scale.t().reshape(-1)}
        for to in rows_of:
            x[to] = _e4m3(parts) * torch.cat([(most / 448)[:, i, None].expand_as(b) for i, b in enumerate(tiles)], 1)
        fo = case["feat_out"] if op == "mm_f8" else 2 * case["width"]
        w_scale = s["w_scale"].view(n, _blocks(fo), _blocks(fi)).double()
        row, col = torch.arange(fo, device="cuda") // BLOCK, torch.arange(fi, device="cuda") // BLOCK

        def w(g):
            return s["w"].view(n, fo, fi)[g].double() * w_scale[g][row][:, col]
    h = torch.zeros(s["rows"], fo, **f64)
    for g, rows in enumerate(spans):
        h[rows] = x[rows] @ w(g).t()
    if op == "mm_f8":
        return h.view(-1)
    y = (_gate64(h[:, :fo // 2], case["gelu"])[0] * h[:, fo // 2:]).reshape(-1)
    if op == "gated_f8":
        return y
    return {"y": y, "hidden": h.view(-1)} if case["keep"] else {"y": y}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    sizes = _sizes(case)
    rows, used, n = int(sizes.sum()), int((sizes > 0).sum()), case["groups"]
    if op == "quant":  # 16-bit rows in, 8-bit rows and scales out, places
        feat = case["feat"]
        return {"bytes": 2 * case["tokens"] * feat + rows * feat + 4 * rows * _blocks(feat) + (4 * rows if case["top_k"] > 1 else 0),
                "flops": 2.0 * case["tokens"] * feat}
    fi = case["feat_in"]
    if op == "gated":
        width = case["width"]
        return {"bytes": 2 * (rows * fi + used * 2 * width * fi + rows * width * (3 if case["keep"] else 1)) + 4 * (n + 1),
                "flops": 4.0 * rows * fi * width}
    if op == "gated_grad":  # dy, weights and both projections in; their gradients and the activations out
        width = case["width"]
        return {"bytes": 2 * (rows * fi + used * width * fi + rows * width * (5 if case["keep"] else 4)) + 4 * (n + 1),
                "flops": 2.0 * rows * fi * width}
    # 16-bit rows in, 8-bit rows and scales out and in again, 8-bit weights and their scales, 16-bit result
    fo = case["feat_out"] if op == "mm_f8" else 2 * case["width"]
    out = fo if op == "mm_f8" else case["width"]
    moved = 2 * case["tokens"] * fi + 2 * rows * (fi + 4 * _blocks(fi)) + used * (fi * fo + 4 * _blocks(fi) * _blocks(fo))
    return {"bytes": moved + 2 * rows * out + 4 * (n + 1), "flops": 2.0 * rows * fi * fo}
