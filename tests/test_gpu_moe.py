"""The operators of a mixture-of-experts layer against their definitions in 64 bits, at the sizes, masks and values where
they can go wrong.

Tolerances.  u = 2^-24 is the rounding error of one f32 operation; a sum of n products formed in f32 in any order, each
addition rounded or cut off, is off by at most n * 2u times the sum of the products' magnitudes.  A result rounded to f16 or
bf16 is off by half a unit in its last place besides (2^-11 and 2^-8 of it, or half the smallest subnormal number)."""
import math

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}
HALF_TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
NAN, INF = math.nan, math.inf


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def near(got, want, slack, dtype=None):
    """|got - want| <= slack + the rounding of the result, element by element; NaNs and infinities at the same places."""
    got, want = got.double(), want.double()
    dtype = dtype or torch.float32
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    bound = slack + HALF_ULP[dtype] * (want.abs() + slack) + HALF_TINY[dtype]
    off = (got - want).abs()
    worst = torch.where(fine, off - bound, torch.full_like(off, -1.0))
    assert (worst <= 0).all(), f"{int((worst > 0).sum())} of {worst.numel()}, worst {float(off.flatten()[worst.argmax()])}"


def off_by(t, elements):
    """The tensor's values in memory that starts `elements` elements behind an aligned address."""
    flat = torch.empty(t.numel() + elements, dtype=t.dtype, device=t.device)[elements:]
    flat.copy_(t.reshape(-1))
    return flat


# ------------------------------------------------------------------ router
def route(z, k, renorm=False):
    t, e = z.shape
    dev = z.device
    gates = torch.full((t * k,), 7.0, device=dev)
    experts, slots = (torch.full((t * k,), 77, dtype=torch.int32, device=dev) for _ in range(2))
    indptr = torch.full((e + 1,), 77, dtype=torch.int32, device=dev)
    ops.moe_route(z.reshape(-1), gates, experts, slots, indptr, e, k, ops.MOE_RENORMALIZE if renorm else 0)
    return gates.view(t, k), experts.view(t, k), slots.view(t, k), indptr


def route_truth(z, k, renorm):
    """(gates, experts, slots, indptr) from the definition, row by row."""
    z = z.double().cpu()
    t, e = z.shape
    gates, experts = torch.zeros(t, k, dtype=torch.float64), torch.full((t, k), -1, dtype=torch.int64)
    for r in range(t):
        live = [i for i in range(e) if z[r, i] > -INF]
        order = sorted(live, key=lambda i: (-float(z[r, i]), i))[:k]
        if not order:
            continue
        top = float(z[r, order[0]])
        ex = {i: 1.0 if float(z[r, i]) == top else math.exp(float(z[r, i]) - top) for i in live}
        total = sum(ex[i] for i in (order if renorm else live))
        for j, i in enumerate(order):
            gates[r, j], experts[r, j] = ex[i] / total, i
    flat = experts.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=e)
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    nxt, slots = indptr[:-1].clone(), torch.full((t * k,), -1, dtype=torch.int64)
    for p, i in enumerate(flat.tolist()):
        if i >= 0:
            slots[p] = nxt[i]
            nxt[i] += 1
    return gates, experts, slots.view(t, k), indptr


def check_route(z, k, renorm=False):
    got = route(z, k, renorm)
    want = route_truth(z, k, renorm)
    for g, w in zip(got[1:], want[1:]):
        assert torch.equal(g.cpu().long(), w)
    live = z[torch.isfinite(z)]
    spread = float(live.max() - live.min()) if live.numel() else 0.0
    # exp of a rounded difference, two units of expf, a sum over the experts, a quotient
    near(got[0].cpu(), want[0], (min(spread, 200.0) + z.shape[1] + 8) * U * want[0])
    return got


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 4, 4), (5, 7, 3), (33, 32, 1), (70, 33, 8), (40, 64, 6), (257, 128, 8),
                                   (130, 200, 5), (31, 256, 32), (20, 512, 22), (9, 1024, 32), (9, 1000, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("renorm", [False, True])
def test_route(cuda_device, t, e, k, dtype, renorm):
    z = (torch.randn(t, e, generator=gen(t * e + k, cuda_device), device=cuda_device) * 2).to(dtype)
    check_route(z, k, renorm)


@pytest.mark.parametrize("t,e,k", [(3000, 8, 2), (4097, 64, 6), (5000, 256, 8), (2049, 1024, 4), (12345, 16, 1), (8192, 33, 8),
                                   (8195, 128, 8), (9001, 100, 3), (8200, 5, 5), (33, 40, 2)])
def test_route_of_many_tokens_is_a_stable_sort(cuda_device, t, e, k):
    # few distinct logits: mostly ties, and popular experts
    z = torch.randint(-3, 4, (t, e), generator=gen(t, cuda_device), device=cuda_device).float()
    z[:, :e // 4] += 2.0
    z[torch.rand(t, generator=gen(2, cuda_device), device=cuda_device) < 0.1] = -INF
    gates, experts, slots, indptr = (x.cpu() for x in route(z, k))
    top, at = torch.sort(z.cpu(), dim=1, descending=True, stable=True)
    want = torch.where(top[:, :k] > -INF, at[:, :k], -1)
    assert torch.equal(experts.long(), want)
    flat = torch.where(want < 0, e, want).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    kept = int((flat < e).sum())
    place = torch.full((t * k,), -1, dtype=torch.int64)
    place[order[:kept]] = torch.arange(kept)
    assert torch.equal(slots.reshape(-1).long(), place)
    assert torch.equal(indptr.long(), torch.searchsorted(flat[order], torch.arange(e + 1)))
    assert torch.equal(*(torch.stack(list(x)) for x in zip(*[(a.float(), b.cpu().float()) for a, b in
                                                              zip((gates, experts, slots), route(z, k)[:3])])))


def test_route_with_masked_experts(cuda_device):
    low = torch.finfo(torch.float32).min
    rows = [[-INF] * 6, [NAN] * 6, [-INF, 1.0, NAN, 1.0, -INF, 1.0], [low] * 6, [low, -INF, 3e38, low, 0.0, -0.0],
            [-0.0, 0.0, -0.0, 0.0, -INF, -INF], [INF, 1.0, INF, -INF, 0.0, 0.0], [-1e-45, 1e-45, 0.0, -0.0, -1.0, -2.0],
            [5.0, -INF, -INF, -INF, -INF, -INF]]
    z = torch.tensor(rows, device=cuda_device)
    for k in (1, 3, 6):
        for renorm in (False, True):
            check_route(z, k, renorm)
    gates, experts, slots, indptr = check_route(torch.full((40, 6), -INF, device=cuda_device), 2)
    assert int(indptr[-1]) == 0 and (slots == -1).all() and (gates == 0).all()


def test_route_without_tokens(cuda_device):
    assert torch.equal(route(torch.empty(0, 5, device=cuda_device), 2)[3].cpu(), torch.zeros(6, dtype=torch.int32))


def route_grad(z, gates, experts, dg, renorm):
    t, e = z.shape
    k = gates.numel() // max(t, 1)
    dz = torch.full((t * e,), 7.0, dtype=z.dtype, device=z.device)
    ops.moe_route_grad(z.reshape(-1), gates.reshape(-1), experts.reshape(-1), dg.reshape(-1), dz, e, k,
                       ops.MOE_RENORMALIZE if renorm else 0)
    return dz.view(t, e)


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (5, 7, 3), (33, 32, 4), (50, 100, 8), (20, 256, 32), (9, 1000, 2), (3, 1024, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad(cuda_device, t, e, k, dtype, renorm):
    g = gen(t + e, cuda_device)
    z = (torch.randn(t, e, generator=g, device=cuda_device) * 2).to(dtype)
    z[0, :e // 2] = -INF
    dg = torch.randn(t, k, generator=g, device=cuda_device)
    gates, experts, _, _ = route(z, k, renorm)
    got = route_grad(z, gates, experts, dg, renorm)
    p = torch.softmax(z.double(), 1)
    kept = experts >= 0
    d = torch.where(kept, dg, 0.0).double()
    at = experts.clamp(min=0).long()
    chosen = torch.where(kept, torch.gather(p, 1, at), 0.0)
    if renorm:
        chosen = chosen / chosen.sum(1, keepdim=True)
    mean, size = (chosen * d).sum(1, keepdim=True), (chosen * d.abs()).sum(1, keepdim=True)
    want = torch.zeros_like(p) if renorm else -p * mean
    want.scatter_add_(1, at, chosen * (d - mean if renorm else d))
    mags = (chosen * (d.abs() + size) if renorm else chosen * d.abs())
    most = (0 * p if renorm else p * size).scatter_add_(1, at, mags)
    near(got, want, 2 * (40 + e + k) * U * most, dtype)


@pytest.mark.parametrize("t,e,k", [(8192, 64, 6), (8197, 30, 8), (9000, 64, 1)])
@pytest.mark.parametrize("renorm", [False, True])
def test_many_tokens_are_routed_like_few(cuda_device, t, e, k, renorm):
    """Batches from 8,192 tokens on give a token fewer lanes: the same bits but for the order of a sum of e terms."""
    g = gen(t, cuda_device)
    z = torch.randn(t, e, generator=g, device=cuda_device) * 2
    z[torch.rand(t, e, generator=g, device=cuda_device) < 0.1] = -INF
    z[5] = -INF
    dg = torch.randn(t, k, generator=g, device=cuda_device)
    gates, experts, _, _ = route(z, k, renorm)
    dz = route_grad(z, gates, experts, dg, renorm)
    half = t // 2
    for part in (slice(0, half), slice(half, t)):
        some = route(z[part].contiguous(), k, renorm)
        assert torch.equal(experts[part], some[1])
        near(gates[part], some[0].double(), 2 * e * U * some[0].double())
        want = route_grad(z[part].contiguous(), some[0], some[1], dg[part].contiguous(), renorm)
        near(dz[part], want.double(), 8 * (e + k) * U * (dg[part].abs().sum(1, keepdim=True).double() + 0 * want.double()))


@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad_against_differences(cuda_device, renorm):
    """The change of <d_gates, gates> along a direction of logits.  With |d_gates|, |direction| <= 1 the third derivative
    of such a mean is below 4 k, so the central difference is off by h^2 / 6 of that; f32 gates add (E + 60) u k / h."""
    t, e, k, h = 12, 20, 4, 2.0 ** -6
    g = gen(5, cuda_device)
    # logits far enough apart that the step changes no choice
    z = torch.stack([torch.randperm(e, generator=g, device=cuda_device) for _ in range(t)]).float() * 0.25
    z[3, ::2] = -INF
    z[4] = -INF
    dg = torch.rand(t, k, generator=g, device=cuda_device) * 2 - 1
    d = torch.rand(t, e, generator=g, device=cuda_device) * 2 - 1
    gates, experts, _, _ = route(z, k, renorm)
    got = (route_grad(z, gates, experts, dg, renorm).double() * d.double()).sum(1)
    up, down = route(z + h * d, k, renorm), route(z - h * d, k, renorm)
    assert torch.equal(up[1], experts) and torch.equal(down[1], experts)
    step = ((z + h * d) - (z - h * d)).nan_to_num(0.0)  # as rounded: 2 h d but for a few u
    want = ((up[0] - down[0]).double() * dg.double()).sum(1) / (2 * h)
    assert (step - 2 * h * d)[torch.isfinite(z)].abs().max() < 1e-5
    assert ((got - want).abs() <= 4 * k * h * h / 6 + 2 * (e + 60) * U * k / h).all()


# ------------------------------------------------------------------ rows
def some_slots(t, k, rows, seed, device, missing=0.0):
    slots = torch.randperm(rows, generator=gen(seed, device), device=device)[:t * k].int()
    if missing:
        slots[torch.rand(t * k, generator=gen(seed + 1, device), device=device) < missing] = -1
    return slots


ROWS = [(1, 1, 1), (1, 1, 8), (3, 2, 7), (24, 6, 1024), (17, 8, 1001), (5, 32, 130), (64, 3, 2040), (9, 4, 5000), (2, 2, 20000)]


@pytest.mark.parametrize("t,k,f", ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1])
def test_dispatch(cuda_device, t, k, f, dtype, shift):
    rows = t * k + 3
    slots = some_slots(t, k, rows, t + f, cuda_device, missing=0.2)
    x = off_by(torch.randn(t, f, generator=gen(1, cuda_device), device=cuda_device).to(dtype), shift)
    z = off_by(torch.full((rows, f), 9.0, dtype=dtype, device=cuda_device), shift)
    ops.moe_dispatch(x, slots, z, f, k)
    want = torch.full((rows, f), 9.0, dtype=dtype, device=cuda_device)
    kept = slots >= 0
    want[slots[kept].long()] = x.view(t, f).repeat_interleave(k, 0)[kept]
    assert torch.equal(z.view(rows, f), want)


@pytest.mark.parametrize("t,k,f", ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1])
def test_dispatch_in_8_bits(cuda_device, t, k, f, dtype, shift):
    rows = t * k + 3
    slots = some_slots(t, k, rows, t + f, cuda_device, missing=0.2)
    x = off_by((torch.randn(t, f, generator=gen(1, cuda_device), device=cuda_device) * 3).to(dtype), shift).view(t, f)
    x[0, 0] = 0.0 if f == 1 else x[0, 0]
    q = off_by(torch.full((rows, f), 9, dtype=torch.int8, device=cuda_device), shift)
    scale = torch.full((rows,), 9.0, device=cuda_device)
    ops.moe_dispatch_i8(x.reshape(-1), slots, q, scale, f, k)
    most = x.float().abs().amax(1)
    inv = torch.where(most > 0, torch.full_like(most, 127.0) / most, 0.0)
    # a quotient of two tensors: torch multiplies by the reciprocal of a plain number
    want_q, want_s = torch.round(x.float() * inv[:, None]).to(torch.int8), most / torch.full_like(most, 127.0)
    kept = slots >= 0
    to = slots[kept].long()
    all_q, all_s = torch.full((rows, f), 9, dtype=torch.int8, device=cuda_device), torch.full((rows,), 9.0, device=cuda_device)
    all_q[to], all_s[to] = want_q.repeat_interleave(k, 0)[kept], want_s.repeat_interleave(k)[kept]
    assert torch.equal(q.view(rows, f), all_q) and torch.equal(scale, all_s)
    # what the numbers stand for: half a step off, and the roundings of the scale and the quotient
    stands = want_q.double() * want_s.double()[:, None]
    assert ((stands - x.double()).abs() <= want_s.double()[:, None] * (0.5 + 127 * 4 * U)).all()


def test_dispatch_in_8_bits_of_rows_without_a_scale(cuda_device):
    x = torch.tensor([[0.0, -0.0, 0.0], [1.0, INF, 2.0], [NAN, 1.0, INF], [1e-40, 0.0, 2e-40], [-3.0, 1.5, 0.01], [-INF, 0.0, 0.0],
                      [2.0 ** -119, 0.0, -(2.0 ** -119)], [3.4e38, -3.4e38, 1.0]], device=cuda_device)
    q, scale = torch.full((24,), 9, dtype=torch.int8, device=cuda_device), torch.full((8,), 9.0, device=cuda_device)
    ops.moe_dispatch_i8(x.reshape(-1), None, q, scale, 3, 1)
    q = q.view(8, 3).cpu()
    assert (q[[0, 1, 2, 3, 5]] == 0).all()
    assert q[4].tolist() == [-127, 64, 0] and q[6].tolist() == [127, 0, -127] and q[7].tolist() == [127, -127, 0]
    s = scale.cpu().tolist()
    assert s[0] == 0 and s[1] == INF and math.isnan(s[2]) and s[3] == 0 and s[5] == INF
    assert s[4] == float(torch.tensor(3.0) / 127) and s[6] == float(torch.tensor(2.0 ** -119) / 127)


@pytest.mark.parametrize("t,k,f", ROWS)
@pytest.mark.parametrize("dtype,out", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                       (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("weighted", [False, True])
def test_combine(cuda_device, t, k, f, dtype, out, shift, weighted):
    rows = t * k + 3
    slots = some_slots(t, k, rows, t + f, cuda_device, missing=0.2)
    z = off_by(torch.randn(rows, f, generator=gen(1, cuda_device), device=cuda_device).to(dtype), shift)
    gates = torch.randn(t, k, generator=gen(2, cuda_device), device=cuda_device)
    y = off_by(torch.full((t, f), 9.0, dtype=out, device=cuda_device), shift)
    ops.moe_combine(z, slots, gates.reshape(-1) if weighted else None, y, f, k)
    terms = z.view(rows, f)[slots.clamp(min=0).long()].double() * (slots >= 0)[:, None]
    if weighted:
        terms = terms * gates.double().reshape(-1, 1)
    terms = terms.view(t, k, f)
    near(y.view(t, f), terms.sum(1), (k + 1) * U * terms.abs().sum(1), out)


def test_rows_that_no_pair_names_do_not_matter(cuda_device):
    t, k, f, rows = 6, 3, 100, 40
    slots = some_slots(t, k, rows, 3, cuda_device, missing=0.3)
    slots[:k] = -1  # a token without an expert
    z = torch.full((rows, f), NAN, device=cuda_device, dtype=torch.float16)
    x = torch.randn(t, f, generator=gen(4, cuda_device), device=cuda_device).half()
    ops.moe_dispatch(x.reshape(-1), slots, z.view(-1), f, k)
    y = torch.empty(t, f, device=cuda_device)
    ops.moe_combine(z.view(-1), slots, None, y.view(-1), f, k)
    assert torch.equal(y, x.float() * (slots.view(t, k) >= 0).sum(1, keepdim=True))  # up to 3 x: exact
    wild = slots.clone()
    wild[:k] = torch.tensor([rows, -7, 2 ** 31 - 1], dtype=torch.int32)  # outside of the rows: as -1
    again = torch.full_like(z, NAN)
    ops.moe_dispatch(x.reshape(-1), wild, again.view(-1), f, k)
    assert torch.equal(again.isnan(), z.isnan()) and torch.equal(again.nan_to_num(0), z.nan_to_num(0))


@pytest.mark.parametrize("t,k,f", ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1])
def test_combine_grad(cuda_device, t, k, f, dtype, shift):
    rows = t * k + 3
    slots = some_slots(t, k, rows, t + f, cuda_device, missing=0.2)
    g = gen(7, cuda_device)
    dy = off_by(torch.randn(t, f, generator=g, device=cuda_device).to(dtype), shift)
    z = off_by(torch.randn(rows, f, generator=g, device=cuda_device).to(dtype), shift)
    gates = torch.randn(t * k, generator=g, device=cuda_device)
    dz = off_by(torch.full((rows, f), 9.0, dtype=dtype, device=cuda_device), shift)
    dg = torch.full((t * k,), 9.0, device=cuda_device)
    ops.moe_combine_grad(dy, z, slots, gates, dz, dg, f, k)
    kept = slots >= 0
    to = slots.clamp(min=0).long()
    d = dy.view(t, f).double().repeat_interleave(k, 0)
    terms = z.view(rows, f)[to].double() * d * kept[:, None]
    near(dg, terms.sum(1), 2 * f * U * terms.abs().sum(1))
    want = torch.full((rows, f), 9.0, dtype=torch.float64, device=cuda_device)
    want[to[kept]] = (d * gates.double()[:, None])[kept]
    near(dz.view(rows, f), want, U * want.abs(), dtype)


def test_combine_grad_against_differences(cuda_device):
    """<dy, combine(z, gates)> is linear in z and in gates: with small whole numbers the difference of two calls is exact."""
    t, k, f, rows = 5, 3, 40, 17
    g = gen(8, cuda_device)
    slots = some_slots(t, k, rows, 9, cuda_device, missing=0.2)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g, device=cuda_device).half()  # noqa: E731
    z, ez, dy = whole(rows, f), whole(rows, f), whole(t, f)
    gates, eg = whole(t * k).float(), whole(t * k).float()

    def loss(zz, gg):
        y = torch.empty(t * f, device=cuda_device)
        ops.moe_combine(zz.reshape(-1), slots, gg, y, f, k)
        return float((y.view(t, f) * dy.float()).sum())

    dz, dg = torch.zeros(rows * f, dtype=torch.float16, device=cuda_device), torch.empty(t * k, device=cuda_device)
    ops.moe_combine_grad(dy.reshape(-1), z.reshape(-1), slots, gates, dz, dg, f, k)
    assert loss(z + ez, gates) - loss(z - ez, gates) == 2 * float((dz.view(rows, f).float() * ez.float()).sum())
    assert loss(z, gates + eg) - loss(z, gates - eg) == 2 * float((dg * eg).sum())


# ------------------------------------------------------------------ grouped products
def pointers(sizes, device):
    return torch.tensor([0] + sizes, device=device).cumsum(0).int()


GROUPS = {
    "one row": [1], "one": [300], "empty ones": [0, 5, 0, 0, 70, 0], "single rows": [1] * 9, "around a tile": [63, 64, 65, 127, 128, 129],
    "around two": [255, 256, 257, 1, 511, 2], "all in the last": [0, 0, 0, 200], "many": [3, 0, 17, 40] * 20, "long": [1500, 7],
}
FEATS = [(1, 1), (7, 5), (8, 8), (64, 64), (65, 63), (128, 256), (100, 130), (200, 72), (520, 264), (1000, 24), (24, 1000), (33, 257)]


def grouped(x, w, indptr, groups, out_in, out_dtype, y=None, f=None):
    fi, fo = f
    rows = x.numel() // fi
    y = torch.full((rows * fo,), 9.0, dtype=out_dtype, device=x.device) if y is None else y
    ops.grouped_mm(x.reshape(-1), w.reshape(-1), y, indptr, groups, fi, fo, ops.GROUPED_W_OUT_IN if out_in else 0)
    return y.view(rows, fo)


def grouped_truth(x, w, sizes):
    """(product, sum of magnitudes), w as [groups, fi, fo]"""
    x, w = x.double(), w.double()
    parts, mags, at = [], [], 0
    for g, n in enumerate(sizes):
        parts.append(x[at:at + n] @ w[g])
        mags.append(x[at:at + n].abs() @ w[g].abs())
        at += n
    return torch.cat(parts), torch.cat(mags)


def check_grouped(sizes, fi, fo, dtype, out_in, out_dtype, device, shift=0, tail=0):
    g = gen(fi * 7 + fo, device)
    n, rows = len(sizes), sum(sizes)
    x = torch.randn(rows + tail, fi, generator=g, device=device).to(dtype)
    w = (torch.randn(n, fi, fo, generator=g, device=device) / math.sqrt(fi)).to(dtype)
    if tail:
        x[rows:] = NAN
    held = w.transpose(1, 2).contiguous() if out_in else w
    y = off_by(torch.full(((rows + tail) * fo,), 9.0, dtype=out_dtype, device=device), shift)
    got = grouped(off_by(x, shift), off_by(held, shift), pointers(sizes, device), n, out_in, out_dtype, y, (fi, fo))
    want, mags = grouped_truth(x, w, sizes)
    near(got[:rows], want, fi * 2 * U * mags, out_dtype)
    assert (got[rows:] == 9.0).all()


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("fi,fo", [(8, 8), (128, 264), (520, 96)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_sizes(cuda_device, sizes, fi, fo, out_in):
    check_grouped(GROUPS[sizes], fi, fo, torch.bfloat16, out_in, torch.float32, cuda_device)


@pytest.mark.parametrize("fi,fo", FEATS)
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                             (torch.float16, torch.float32)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_features(cuda_device, fi, fo, dtype, out_dtype, out_in):
    check_grouped([70, 0, 33, 129], fi, fo, dtype, out_in, out_dtype, cuda_device, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("out_in", [False, True])
@pytest.mark.parametrize("fi,fo", [(64, 72), (63, 40)])
def test_grouped_operands_at_odd_addresses(cuda_device, shift, out_in, fi, fo):
    for out in (torch.float16, torch.float32):
        check_grouped([30, 100], fi, fo, torch.float16, out_in, out, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,fi,fo", [([2000, 100, 1700], 1024, 1000), ([700] * 8, 2048, 512), ([4096], 512, 2056)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_large(cuda_device, sizes, fi, fo, out_in):
    check_grouped(sizes, fi, fo, torch.bfloat16, out_in, torch.bfloat16, cuda_device)


@pytest.mark.parametrize("sizes,fi,fo", [([100], 4096, 520), ([33, 0, 50, 41], 2056, 200), ([300], 8200, 72)])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_depth_shared_by_several_units(cuda_device, sizes, fi, fo, dtype, out_dtype, out_in):
    check_grouped(sizes, fi, fo, dtype, out_in, out_dtype, cuda_device, tail=9)


@pytest.mark.parametrize("sizes,fi,fo", [([3], 4096, 2000), ([5, 0, 16, 17, 1, 0, 33], 1024, 520), ([1] * 70, 136, 40), ([9], 200, 9)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_few_rows(cuda_device, sizes, fi, fo, dtype, out_in):
    check_grouped(sizes, fi, fo, dtype, out_in, dtype, cuda_device, tail=3)


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5, 2], [9, 16, 12], [1] * 40], ids=str)
@pytest.mark.parametrize("fi,fo", [(1, 1), (7, 9), (63, 130), (264, 257), (1001, 24), (2047, 1111)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_few_rows_of_odd_widths(cuda_device, sizes, fi, fo, dtype, out_in):
    check_grouped(sizes, fi, fo, dtype, out_in, torch.float32, cuda_device)
    check_grouped(sizes, fi, fo, dtype, out_in, dtype, cuda_device, tail=2)


@pytest.mark.parametrize("fi,fo", [(63, 65), (65, 130), (129, 7), (130, 136)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grouped_values_stay_in_rows_of_odd_widths(cuda_device, fi, fo, out_in):
    """What is not a number lies right before and behind the rows of x and W in use, in their own arrays and beyond."""
    sizes, bad = [0, 3, 0, 1, 0], torch.tensor([NAN, INF, -INF], device=cuda_device)
    rows, g = sum(sizes), gen(fi, cuda_device)
    x = bad[torch.arange(rows + 2, device=cuda_device)[:, None].expand(-1, fi) % 3].half()
    w = bad[torch.arange(5, device=cuda_device)[:, None, None].expand(-1, fi, fo) % 3].half()
    x[1:4] = torch.randn(3, fi, generator=g, device=cuda_device).half()
    w[1] = torch.randn(fi, fo, generator=g, device=cuda_device).half()
    want = x[1:4].double() @ w[1].double()
    slack = 2 * fi * U * (x[1:4].double().abs() @ w[1].double().abs())
    flat = (w.transpose(1, 2) if out_in else w).contiguous()
    y = torch.full(((rows + 2) * fo,), 7.0, device=cuda_device)
    indptr = torch.tensor([1, 1, 4, 4, 5, 5], dtype=torch.int32, device=cuda_device)
    ops.grouped_mm(x.view(-1), flat.view(-1), y, indptr, 5, fi, fo, ops.GROUPED_W_OUT_IN if out_in else 0)
    y = y.view(rows + 2, fo)
    near(y[1:4], want, slack)
    assert (y[[0, 5]] == 7).all() and not torch.isfinite(y[4]).any()


def test_grouped_values_stay_in_their_rows_and_groups(cuda_device):
    sizes, fi, fo = [40, 0, 25, 130], 96, 136
    g = gen(3, cuda_device)
    rows = sum(sizes)
    x, w = torch.randn(rows, fi, generator=g, device=cuda_device).half(), torch.randn(4, fi, fo, generator=g, device=cuda_device).half()
    clean = grouped(x, w, pointers(sizes, cuda_device), 4, False, torch.float32, f=(fi, fo))
    x[39, 5], x[64, 0], x[70, 95] = NAN, INF, -INF
    w[1] = NAN  # nobody's expert
    w[3, 0, 135] = INF
    got = grouped(x, w, pointers(sizes, cuda_device), 4, False, torch.float32, f=(fi, fo))
    want, _ = grouped_truth(x, w, sizes)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = torch.isfinite(want)
    assert torch.equal(got[fine], clean[fine])


def test_grouped_without_rows_or_groups(cuda_device):
    e = torch.empty(0, dtype=torch.float16, device=cuda_device)
    w = torch.randn(3 * 64, device=cuda_device).half()
    ops.grouped_mm(e, w, e, torch.zeros(4, dtype=torch.int32, device=cuda_device), 3, 8, 8)
    x, y = torch.randn(16, device=cuda_device).half(), torch.full((16,), 9.0, device=cuda_device).half()
    ops.grouped_mm(x, e, y, torch.zeros(1, dtype=torch.int32, device=cuda_device), 0, 8, 8)
    assert (y == 9).all()
    ops.grouped_mm(x, w, y, torch.tensor([1, 1, 2, 2], dtype=torch.int32, device=cuda_device), 3, 8, 8)
    assert (y[:8] == 9).all() and (y[8:] != 9).any()  # the row ahead of the first group stays as it is
    dw = torch.full((3 * 64,), 9.0, device=cuda_device)
    ops.grouped_mm_grad_w(e, e, dw, torch.zeros(4, dtype=torch.int32, device=cuda_device), 3, 8, 8)
    assert (dw == 0).all()


@pytest.mark.parametrize("bad", [[0, 50, 20, 30], [-5, 10, 99, 2 ** 31 - 1], [40, 30, 20, 10], [-2 ** 31, 0, 30, -1]])
def test_grouped_with_wild_pointers_stays_inside(cuda_device, bad):
    """Pointers that no router writes: what is computed is not defined, but nothing outside of the arrays is touched."""
    fi, fo, rows = 64, 64, 30
    x, w = torch.ones(rows * fi, device=cuda_device).half(), torch.ones(3 * fi * fo, device=cuda_device).half()
    guard = torch.full((1000 + rows * fo + 1000,), 9.0, device=cuda_device)
    ptr = torch.tensor(bad, device=cuda_device).int()
    ops.grouped_mm(x, w, guard[1000:1000 + rows * fo], ptr, 3, fi, fo)
    assert (guard[:1000] == 9).all() and (guard[-1000:] == 9).all()
    dw = torch.full((1000 + 3 * fi * fo + 1000,), 9.0, device=cuda_device)
    ops.grouped_mm_grad_w(x, x, dw[1000:-1000], ptr, 3, fi, fo)
    assert (dw[:1000] == 9).all() and (dw[-1000:] == 9).all()


@pytest.mark.parametrize("fi,rows", [(2048, 30), (64, 3000), (4096, 900)])
def test_grouped_with_wild_pointers_in_every_kernel(cuda_device, fi, rows):
    fo = 264
    x, w = torch.ones(rows * fi, device=cuda_device).half(), torch.ones(3 * fi * fo, device=cuda_device).half()
    for bad in ([0, rows, 5, rows + 9], [-3, rows // 2, 2 ** 31 - 1, 0], [rows, 7, -2 ** 31, rows]):
        guard = torch.full((1000 + rows * fo + 1000,), 9.0, device=cuda_device)
        ptr = torch.tensor(bad, device=cuda_device).int()
        ops.grouped_mm(x, w, guard[1000:1000 + rows * fo], ptr, 3, fi, fo)
        assert (guard[:1000] == 9).all() and (guard[-1000:] == 9).all()


def check_grad_w(sizes, fi, fo, dtype, out_in, out_dtype, device, shift=0, tail=0):
    g = gen(fi * 5 + fo, device)
    n, rows = len(sizes), sum(sizes)
    x, dy = (torch.randn(rows + tail, f, generator=g, device=device).to(dtype) for f in (fi, fo))
    x[rows:], dy[rows:] = NAN, NAN
    dw = off_by(torch.full((n * fi * fo,), 9.0, dtype=out_dtype, device=device), shift)
    ops.grouped_mm_grad_w(off_by(x, shift), off_by(dy, shift), dw, pointers(sizes, device), n, fi, fo,
                          ops.GROUPED_W_OUT_IN if out_in else 0)
    got = dw.view(n, fo, fi).transpose(1, 2) if out_in else dw.view(n, fi, fo)
    at = 0
    for i, k in enumerate(sizes):
        a, b = x[at:at + k].double().t(), dy[at:at + k].double()
        near(got[i], a @ b, k * 2 * U * (a.abs() @ b.abs()), out_dtype)
        at += k


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("fi,fo", [(8, 8), (128, 264), (304, 96)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grad_w_sizes(cuda_device, sizes, fi, fo, out_in):
    check_grad_w(GROUPS[sizes], fi, fo, torch.bfloat16, out_in, torch.float32, cuda_device)


@pytest.mark.parametrize("fi,fo", FEATS)
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                             (torch.float16, torch.float32)])
@pytest.mark.parametrize("out_in", [False, True])
def test_grad_w_features(cuda_device, fi, fo, dtype, out_dtype, out_in):
    check_grad_w([70, 0, 33, 129], fi, fo, dtype, out_in, out_dtype, cuda_device, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("fi,fo", [(64, 72), (63, 40)])
def test_grad_w_operands_at_odd_addresses(cuda_device, shift, fi, fo):
    for out in (torch.float16, torch.float32):
        check_grad_w([30, 100], fi, fo, torch.float16, False, out, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,fi,fo", [([2000, 100, 1700], 1024, 1000), ([700] * 8, 512, 768), ([5000], 264, 520)])
def test_grad_w_large(cuda_device, sizes, fi, fo):
    check_grad_w(sizes, fi, fo, torch.bfloat16, False, torch.bfloat16, cuda_device)


@pytest.mark.parametrize("sizes,fi,fo", [([3000, 0, 130, 2870], 72, 136), ([6001], 40, 8), ([0, 0, 5000], 264, 24)])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_grad_w_depth_shared_by_several_units(cuda_device, sizes, fi, fo, out_dtype):
    check_grad_w(sizes, fi, fo, torch.float16, False, out_dtype, cuda_device, tail=70)


@pytest.mark.parametrize("out_in", [False, True])
@pytest.mark.parametrize("fo", [200, 203])
def test_grad_w_of_groups_without_rows(cuda_device, out_in, fo):
    check_grad_w([0] * 20 + [3] + [0] * 20, 264, fo, torch.bfloat16, out_in, torch.bfloat16, cuda_device)


def test_grad_w_of_many_groups_with_few_rows_repeats(cuda_device):
    """Thousands of launches whose tiles are mostly zeros: every tile is found by all roles alike, every time."""
    groups, fi, fo, rows = 64, 1444, 2024, 9
    g = gen(11, cuda_device)
    sizes = torch.bincount(torch.randint(0, groups, (rows,), generator=g, device=cuda_device), minlength=groups)
    x = torch.randn(rows, fi, generator=g, device=cuda_device).half()
    dy = torch.randn(rows, fo, generator=g, device=cuda_device).half()
    indptr = pointers(sizes.tolist(), cuda_device)
    first, dw = (torch.full((groups * fi * fo,), 9.0, dtype=torch.float16, device=cuda_device) for _ in range(2))
    ops.grouped_mm_grad_w(x.view(-1), dy.view(-1), first, indptr, groups, fi, fo)
    for _ in range(10):
        dw.fill_(9.0)
        for _ in range(200):
            ops.grouped_mm_grad_w(x.view(-1), dy.view(-1), dw, indptr, groups, fi, fo)
        assert torch.equal(dw, first)


def test_grad_w_rows_of_other_groups_do_not_matter(cuda_device):
    """A neighbour's infinities and NaNs, whichever rows of a step they share with this group's."""
    fi, fo, sizes = 72, 136, [5, 0, 58, 1, 100, 64, 20]
    g = gen(6, cuda_device)
    rows = sum(sizes)
    x, dy = (torch.randn(rows, f, generator=g, device=cuda_device).half() for f in (fi, fo))
    ptr = pointers(sizes, cuda_device)

    def grad():
        dw = torch.empty(len(sizes) * fi * fo, device=cuda_device)
        ops.grouped_mm_grad_w(x.reshape(-1), dy.reshape(-1), dw, ptr, len(sizes), fi, fo)
        return dw.view(len(sizes), fi, fo)

    clean = grad()
    for bad in range(len(sizes)):
        keep = x.clone(), dy.clone()
        at = sum(sizes[:bad])
        x[at:at + sizes[bad]], dy[at:at + sizes[bad]] = NAN, INF
        got = grad()
        for i in range(len(sizes)):
            assert got[i].isnan().all() if i == bad and sizes[i] else torch.equal(got[i], clean[i])
        x.copy_(keep[0])
        dy.copy_(keep[1])


def test_grouped_gradients_against_differences(cuda_device):
    """<dy, grouped(x, w)> is linear in x and in w: with small whole numbers the difference of two calls is exact."""
    sizes, fi, fo = [20, 0, 77, 3], 72, 40
    g = gen(11, cuda_device)
    rows, n = sum(sizes), len(sizes)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g, device=cuda_device).half()  # noqa: E731
    x, ex, w, ew, dy = whole(rows, fi), whole(rows, fi), whole(n, fi, fo), whole(n, fi, fo), whole(rows, fo)
    ptr = pointers(sizes, cuda_device)
    loss = lambda a, b: float((grouped(a, b, ptr, n, False, torch.float32, f=(fi, fo)) * dy.float()).sum())  # noqa: E731
    dx = grouped(dy, w, ptr, n, True, torch.float32, f=(fo, fi))
    dw = torch.empty(n * fi * fo, device=cuda_device)
    ops.grouped_mm_grad_w(x.reshape(-1), dy.reshape(-1), dw, ptr, n, fi, fo)
    assert loss(x + ex, w) - loss(x - ex, w) == 2 * float((dx * ex.float()).sum())
    assert loss(x, w + ew) - loss(x, w - ew) == 2 * float((dw.view(n, fi, fo) * ew.float()).sum())


def check_i8(sizes, fi, fo, out_dtype, device, shift=0, tail=0, null=False, full=False):
    g = gen(fi * 3 + fo, device)
    n, rows = len(sizes), sum(sizes)
    lo, hi = (-128, 128) if full else (-127, 128)
    x = torch.randint(lo, hi, (rows + tail, fi), generator=g, device=device, dtype=torch.int8)
    w = torch.randint(lo, hi, (n, fo, fi), generator=g, device=device, dtype=torch.int8)
    if full:
        x[0], w[0, 0] = -128, -128
    xs, ws = torch.rand(rows + tail, generator=g, device=device) * 0.1, torch.rand(n, fo, generator=g, device=device) * 0.01
    y = off_by(torch.full(((rows + tail) * fo,), 9.0, dtype=out_dtype, device=device), shift)
    ops.grouped_mm_i8(off_by(x, shift), xs, off_by(w, shift), ws.reshape(-1), y, None if null else pointers(sizes, device), n, fi, fo)
    want, _ = grouped_truth(x, w.transpose(1, 2), sizes)
    scale = torch.cat([xs[:rows].double()[at:at + k, None] * ws[i].double() for i, (at, k) in
                       enumerate(zip([sum(sizes[:i]) for i in range(n)], sizes))])
    want = want * scale
    # the sum is exact: its conversion, the product of the scales and their product are rounded
    near(y.view(rows + tail, fo)[:rows], want, 3 * U * want.abs(), out_dtype)
    assert (y.view(rows + tail, fo)[rows:] == 9.0).all()


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("fi,fo", [(16, 8), (128, 264), (528, 96)])
def test_i8_sizes(cuda_device, sizes, fi, fo):
    check_i8(GROUPS[sizes], fi, fo, torch.float32, cuda_device)


@pytest.mark.parametrize("fi,fo", FEATS + [(16, 130), (4096, 72), (8200, 16)])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_i8_features(cuda_device, fi, fo, out_dtype):
    check_i8([70, 0, 33, 129], fi, fo, torch.float32 if fi > 1000 and out_dtype is torch.float16 else out_dtype, cuda_device, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("fi,fo", [(64, 72), (63, 40)])
def test_i8_operands_at_odd_addresses(cuda_device, shift, fi, fo):
    check_i8([30, 100], fi, fo, torch.float32, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,fi,fo", [([100], 8200, 520), ([33, 0, 50, 41] * 10, 4112, 72), ([3], 4096, 2000), ([5, 0, 16, 17, 1, 0, 33], 1040, 520)])
def test_i8_depth_shared(cuda_device, sizes, fi, fo):
    check_i8(sizes, fi, fo, torch.float32, cuda_device, tail=9)


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5, 2], [9, 16, 12]], ids=str)
@pytest.mark.parametrize("fi,fo", [(1, 1), (7, 9), (63, 130), (1001, 24), (2047, 1111), (4098, 33)])
def test_i8_few_rows_of_odd_widths(cuda_device, sizes, fi, fo):
    check_i8(sizes, fi, fo, torch.float32, cuda_device, tail=2)


def test_i8_extremes_and_one_dense_product(cuda_device):
    check_i8([200], 131071, 24, torch.float32, cuda_device, full=True)  # -128 * -128 summed 131,071 times: 2^31 - 2^14
    check_i8([1], 4096, 1000, torch.bfloat16, cuda_device, null=True)
    check_i8([333], 512, 777, torch.bfloat16, cuda_device, null=True)


# ------------------------------------------------------------------ how calls behave
def test_null_pointers_mean_all_rows(cuda_device):
    x, w = torch.randn(50, 64, device=cuda_device).half(), torch.randn(64, 40, device=cuda_device).half()
    a = grouped(x, w, None, 1, False, torch.float32, f=(64, 40))
    assert torch.equal(a, grouped(x, w, pointers([50], cuda_device), 1, False, torch.float32, f=(64, 40)))
    dw = [torch.empty(64 * 64, device=cuda_device) for _ in range(2)]
    ops.grouped_mm_grad_w(x.view(-1), x.view(-1), dw[0], None, 1, 64, 64)
    ops.grouped_mm_grad_w(x.view(-1), x.view(-1), dw[1], pointers([50], cuda_device), 1, 64, 64)
    assert torch.equal(*dw)


def test_calls_on_another_stream_and_in_a_graph(cuda_device):
    """The same bits on the default stream, on another one behind a producer, and replayed from a graph."""
    sizes, fi, fo, n = [33, 0, 140, 60], 100, 130, 4  # features that need a copy at aligned rows
    g = gen(2, cuda_device)
    rows = sum(sizes)
    x0, w0 = torch.randn(rows, fi, generator=g, device=cuda_device).half(), torch.randn(n, fi, fo, generator=g, device=cuda_device).half()
    z = torch.randn(500, 40, generator=g, device=cuda_device)
    ptr = pointers(sizes, cuda_device)

    def calls(x, w):
        y = grouped(x, w, ptr, n, False, torch.float16, f=(fi, fo))
        dw = torch.empty(n * fi * fo, dtype=torch.float16, device=cuda_device)
        ops.grouped_mm_grad_w(x.reshape(-1), y.reshape(-1), dw, ptr, n, fi, fo)
        return [y, dw, *route(z, 4)]

    want = calls(x0, w0)
    assert all(torch.equal(a, b) for a, b in zip(want, calls(x0, w0)))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x, w = torch.zeros_like(x0), torch.zeros_like(w0)
        for _ in range(20):
            x.add_(0.0)
        x.copy_(x0)
        w.copy_(w0)
        got = calls(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        x.zero_()
        with torch.cuda.graph(graph, stream=side):
            got = calls(x, w)
        x.copy_(x0)
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = None


def test_bad_indices_are_refused_when_asked(cuda_device):
    lib = L.load()
    x, w = torch.ones(30 * 64, device=cuda_device).half(), torch.ones(2 * 64 * 64, device=cuda_device).half()
    y = torch.zeros(30 * 64, device=cuda_device).half()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    lib.sparsetir_set_validate(1)
    try:
        ops.grouped_mm(x, w, y, i32(0, 10, 25), 2, 64, 64)  # rows past the last group are allowed
        for bad, message in ((i32(0, 20, 10), "decreases"), (i32(0, 10, 31), "out of range"), (i32(1, 10, 30), "expected 0")):
            with pytest.raises(ops.SparseTIRError, match=message):
                ops.grouped_mm(x, w, y, bad, 2, 64, 64)
            with pytest.raises(ops.SparseTIRError, match=message):
                ops.grouped_mm_grad_w(x, x, w, bad, 2, 64, 64)
        with pytest.raises(ops.SparseTIRError, match=r"slots\[1\] = 30 is out of range"):
            ops.moe_dispatch(x[:2 * 64], i32(-1, 30), y, 64, 1)
        with pytest.raises(ops.SparseTIRError, match=r"experts\[0\] = 5 is out of range"):
            ops.moe_route_grad(torch.zeros(5, device=cuda_device), torch.zeros(1, device=cuda_device), i32(5),
                               torch.zeros(1, device=cuda_device), torch.zeros(5, device=cuda_device), 5, 1)
    finally:
        lib.sparsetir_set_validate(0)


def test_no_wait_ran_out(cuda_device):
    import ctypes

    count = ctypes.c_uint(99)
    assert L.load().sparsetir_tc_timeouts(0, ctypes.byref(count)) == 0 and count.value == 0
