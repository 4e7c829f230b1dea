"""The gated block of an expert and its gradient against their definitions in 64 bits, at the sizes, groups and values where they can go
wrong.

Tolerances.  u = 2^-24.  A sum of n products formed in f32 in any order, each addition rounded or cut off, is off by at most
e = 2 n u times the sum of the products' magnitudes.  With f the activation, |f'| <= 1.13:
  act     |f(g) u - f(g~) u~| <= 1.13 e_g |u| + (|f(g)| + 1.13 e_g) e_u, and f itself is evaluated with a relative error of (8 |z| + 32) u (the
          argument of the exponential carries a few roundings, which the exponential multiplies by |z| <= 104; beyond that f is below 2^-140)
  d_gate  e_d |u f'| and |d u| times the error of f' = s + f (1 - s) z': (8 |z| + 32) u (s + |f z'| (1 - s)) + 4 u |f z'|
  d_up    e_d |f| + |d f| (8 |z| + 32) u
and the result's own rounding (`near`)."""
import math

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops
from test_gpu_moe import FEATS, GROUPS, INF, NAN, U, gen, near, off_by, pointers

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -120
TYPES = [torch.float16, torch.bfloat16]


def gate_parts(g, gelu):
    """(f, f', s, z, z') in 64 bits"""
    if gelu:
        c = math.sqrt(2 / math.pi)
        z, dz = 2 * c * (g + 0.044715 * g ** 3), 2 * c * (1 + 3 * 0.044715 * g ** 2)
    else:
        z, dz = g, torch.ones_like(g)
    s = torch.sigmoid(z)
    return g * s, s + g * s * (1 - s) * dz, s, z, dz


def rel(z):
    return (8 * z.abs().clamp(max=104) + 32) * U


def by_group(x, w, sizes):
    """(product, sum of magnitudes), w as [groups, fi, fo]"""
    parts, mags, at = [], [], 0
    for g, n in enumerate(sizes):
        parts.append(x[at:at + n].double() @ w[g].double())
        mags.append(x[at:at + n].double().abs() @ w[g].double().abs())
        at += n
    return torch.cat(parts), torch.cat(mags)


def gated_truth(h, mags, n, gelu):
    """(act, tolerance) from projections with errors of 2 n u mags"""
    w = h.shape[1] // 2
    g, up, eg, eu = h[:, :w], h[:, w:], 2 * n * U * mags[:, :w], 2 * n * U * mags[:, w:]
    f, _, _, z, _ = gate_parts(g, gelu)
    return f * up, 1.13 * eg * up.abs() + (f.abs() + 1.13 * eg) * eu + f.abs() * up.abs() * rel(z) + TINY


def check_gated(sizes, fi, width, dtype, device, gelu=False, keep=True, shift=0, tail=0, null=False, scale=1.0):
    g = gen(fi * 7 + width, device)
    n, rows = len(sizes), sum(sizes)
    x = torch.randn(rows + tail, fi, generator=g, device=device).to(dtype)
    w = (torch.randn(n, 2 * width, fi, generator=g, device=device) * (scale / math.sqrt(fi))).to(dtype)
    if tail:
        x[rows:] = NAN
    y = off_by(torch.full(((rows + tail) * width,), 9.0, dtype=dtype, device=device), shift)
    hidden = off_by(torch.full(((rows + tail) * 2 * width,), 9.0, dtype=dtype, device=device), shift) if keep else None
    ops.grouped_mm_gated(off_by(x, shift), off_by(w, shift), y, hidden, None if null else pointers(sizes, device), n, fi, width,
                         ops.GATED_GELU if gelu else 0)
    h, mags = by_group(x, w.transpose(1, 2), sizes)
    want, slack = gated_truth(h, mags, fi, gelu)
    y = y.view(-1, width)
    near(y[:rows], want, slack, dtype)
    assert (y[rows:] == 9.0).all()
    if keep:
        hidden = hidden.view(-1, 2 * width)
        near(hidden[:rows], h, fi * 2 * U * mags, dtype)
        assert (hidden[rows:] == 9.0).all()


def check_grad(sizes, feat, width, dtype, device, gelu=False, act=True, out_in=False, shift=0, tail=0, null=False):
    g = gen(feat * 5 + width, device)
    n, rows = len(sizes), sum(sizes)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    dy, w = rand(rows + tail, feat).to(dtype), (rand(n, feat, width) / math.sqrt(feat)).to(dtype)
    hidden = (rand(rows + tail, 2 * width) * 2).to(dtype)
    if tail:
        dy[rows:], hidden[rows:] = NAN, NAN
    d_hidden = off_by(torch.full(((rows + tail) * 2 * width,), 9.0, dtype=dtype, device=device), shift)
    a = off_by(torch.full(((rows + tail) * width,), 9.0, dtype=dtype, device=device), shift) if act else None
    held = w.transpose(1, 2).contiguous() if out_in else w
    ops.grouped_mm_gated_grad(off_by(dy, shift), off_by(held, shift), off_by(hidden, shift), d_hidden, a,
                              None if null else pointers(sizes, device), n, feat, width,
                              (ops.GATED_GELU if gelu else 0) | (ops.GROUPED_W_OUT_IN if out_in else 0))
    d, mags = by_group(dy, w, sizes)
    ed = 2 * feat * U * mags
    gate, up = hidden[:rows, :width].double(), hidden[:rows, width:].double()
    f, df, s, z, dz = gate_parts(gate, gelu)
    off_df = rel(z) * (s + (f * dz).abs() * (1 - s)) + 4 * U * (f * dz).abs()
    d_hidden = d_hidden.view(-1, 2 * width)
    near(d_hidden[:rows, :width], d * up * df, ed * (up * df).abs() + (d.abs() + ed) * up.abs() * off_df + TINY, dtype)
    near(d_hidden[:rows, width:], d * f, ed * f.abs() + (d.abs() + ed) * f.abs() * rel(z) + TINY, dtype)
    assert (d_hidden[rows:] == 9.0).all()
    if act:
        a = a.view(-1, width)
        near(a[:rows], f * up, (f * up).abs() * rel(z) + TINY, dtype)
        assert (a[rows:] == 9.0).all()


# ------------------------------------------------------------------ the block
@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("fi,width", [(8, 8), (128, 136), (520, 48)])
@pytest.mark.parametrize("gelu", [False, True])
def test_gated_sizes(cuda_device, sizes, fi, width, gelu):
    check_gated(GROUPS[sizes], fi, width, torch.bfloat16, cuda_device, gelu=gelu, tail=3)


@pytest.mark.parametrize("fi,width", FEATS + [(72, 16), (64, 15), (136, 17), (200, 500), (264, 129)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keep", [False, True])
def test_gated_features(cuda_device, fi, width, dtype, keep):
    check_gated([70, 0, 33, 129], fi, width, dtype, cuda_device, keep=keep, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("fi,width", [(64, 72), (63, 40)])
@pytest.mark.parametrize("sizes", [[70, 0, 130], [2, 3, 0]], ids=str)
def test_gated_operands_at_odd_addresses(cuda_device, shift, fi, width, sizes):
    check_gated(sizes, fi, width, torch.float16, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,fi,width", [([2000, 100, 1700], 1024, 520), ([700] * 8, 2048, 256), ([4096], 512, 1000)])
@pytest.mark.parametrize("gelu", [False, True])
def test_gated_large(cuda_device, sizes, fi, width, gelu):
    check_gated(sizes, fi, width, torch.float16, cuda_device, gelu=gelu)


@pytest.mark.parametrize("sizes,fi,width", [([100], 4096, 264), ([33, 0, 50, 41], 2056, 104), ([300], 8200, 40), ([120], 4096, 33)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keep", [False, True])
def test_gated_depth_shared_by_several_units(cuda_device, sizes, fi, width, dtype, keep):
    check_gated(sizes, fi, width, dtype, cuda_device, keep=keep, tail=2)


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5, 2], [9, 16, 12], [1] * 40, [0, 40, 0, 0, 0, 0, 0, 0]], ids=str)
@pytest.mark.parametrize("fi,width", [(1, 1), (7, 9), (63, 130), (264, 257), (1001, 24), (4096, 1000), (1024, 2048)])
@pytest.mark.parametrize("keep", [False, True])
def test_gated_few_rows(cuda_device, sizes, fi, width, keep):
    check_gated(sizes, fi, width, torch.bfloat16, cuda_device, keep=keep, tail=2)


@pytest.mark.parametrize("rows", [1, 5, 200])
def test_gated_of_one_group_without_pointers(cuda_device, rows):
    check_gated([rows], 136, 72, torch.float16, cuda_device, null=True)


def test_gated_far_from_zero(cuda_device):
    """Gates far on either side: the sigmoid is 0 or 1 to the last bit, and nothing overflows on the way."""
    check_gated([60, 70], 64, 64, torch.bfloat16, cuda_device, scale=60.0)
    check_gated([60, 70], 64, 64, torch.bfloat16, cuda_device, scale=60.0, gelu=True)


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("gelu", [False, True])
def test_gated_infinities_and_nan(cuda_device, rows, gelu):
    """One feature in: the gate is x times its weight.  +inf passes, what is not a number stays where it is."""
    x = torch.zeros(rows, 8, device=cuda_device).half()
    x[0, 0], x[1, 0], x[2, 0] = INF, NAN, 1.0
    w = torch.zeros(1, 16, 8, device=cuda_device).half()
    w[0, :, 0] = 1.0
    y, hidden = torch.full((rows * 8,), 9.0, device=cuda_device).half(), torch.full((rows * 16,), 9.0, device=cuda_device).half()
    ops.grouped_mm_gated(x.view(-1), w.view(-1), y, hidden, None, 1, 8, 8, ops.GATED_GELU if gelu else 0)
    y, hidden = y.view(rows, 8), hidden.view(rows, 16)
    assert (y[0] == INF).all() and y[1].isnan().all() and (hidden[0] == INF).all() and hidden[1].isnan().all()
    one = 0.8412 if gelu else 0.7311  # f(1)
    assert ((y[2].double() - one).abs() < 1e-3).all() and (y[3:] == 0).all()


def test_gated_values_stay_in_their_rows_and_groups(cuda_device):
    sizes, fi, width = [40, 0, 25, 130], 96, 72
    g = gen(3, cuda_device)
    x = torch.randn(195, fi, generator=g, device=cuda_device).half()
    w = torch.randn(4, 2 * width, fi, generator=g, device=cuda_device).half()

    def call():
        y, h = torch.empty(195 * width, device=cuda_device).half(), torch.empty(195 * 2 * width, device=cuda_device).half()
        ops.grouped_mm_gated(x.view(-1), w.view(-1), y, h, pointers(sizes, cuda_device), 4, fi, width)
        return y.view(195, width), h.view(195, 2 * width)

    y0, h0 = call()
    x[39, 5], x[64, 0] = NAN, NAN
    w[1] = NAN             # nobody's expert
    w[3, width - 1] = NAN  # the last gate
    w[3, width + 3] = NAN  # an up projection
    y, h = call()
    bad_y, bad_h = torch.zeros_like(y, dtype=torch.bool), torch.zeros_like(h, dtype=torch.bool)
    bad_y[39], bad_y[64], bad_h[39], bad_h[64] = True, True, True, True
    bad_y[65:, width - 1], bad_y[65:, 3], bad_h[65:, width - 1], bad_h[65:, width + 3] = True, True, True, True
    assert torch.equal(y.isnan(), bad_y) and torch.equal(h.isnan(), bad_h)
    assert torch.equal(y[~bad_y], y0[~bad_y]) and torch.equal(h[~bad_h], h0[~bad_h])


# ------------------------------------------------------------------ its gradient
@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("feat,width", [(8, 8), (128, 264), (520, 96)])
@pytest.mark.parametrize("gelu", [False, True])
def test_grad_sizes(cuda_device, sizes, feat, width, gelu):
    check_grad(GROUPS[sizes], feat, width, torch.bfloat16, cuda_device, gelu=gelu, tail=3)


@pytest.mark.parametrize("feat,width", FEATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("out_in", [False, True])
def test_grad_features(cuda_device, feat, width, dtype, act, out_in):
    check_grad([70, 0, 33, 129], feat, width, dtype, cuda_device, act=act, out_in=out_in, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("feat,width", [(64, 72), (63, 40)])
def test_grad_operands_at_odd_addresses(cuda_device, shift, feat, width):
    check_grad([70, 0, 130], feat, width, torch.float16, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,feat,width", [([2000, 100, 1700], 1024, 1000), ([700] * 8, 2048, 512), ([4096], 512, 2056), ([900, 5], 264, 4100)])
@pytest.mark.parametrize("gelu", [False, True])
def test_grad_large(cuda_device, sizes, feat, width, gelu):
    check_grad(sizes, feat, width, torch.bfloat16, cuda_device, gelu=gelu)


@pytest.mark.parametrize("sizes,feat,width", [([100], 4096, 520), ([33, 0, 50, 41], 2056, 200), ([300], 8200, 72), ([120], 4096, 33)])
@pytest.mark.parametrize("out_in", [False, True])
@pytest.mark.parametrize("act", [False, True])
def test_grad_depth_shared_by_several_units(cuda_device, sizes, feat, width, out_in, act):
    check_grad(sizes, feat, width, torch.float16, cuda_device, out_in=out_in, act=act, tail=2)


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5, 2], [1] * 40], ids=str)
@pytest.mark.parametrize("feat,width", [(1, 1), (63, 130), (2048, 1024)])
def test_grad_few_rows(cuda_device, sizes, feat, width):
    check_grad(sizes, feat, width, torch.bfloat16, cuda_device, tail=2)


@pytest.mark.parametrize("rows", [1, 200])
def test_grad_of_one_group_without_pointers(cuda_device, rows):
    check_grad([rows], 136, 72, torch.float16, cuda_device, null=True)


@pytest.mark.parametrize("gelu", [False, True])
def test_gradient_against_differences(cuda_device, gelu):
    """The whole block x -> f(x Wg^T) * (x Wu^T) -> D, a scalar product with a fixed tensor: the gradient to `hidden` moves it as a central
    difference in 64 bits says.  The difference is off by its third derivative times step^2 (1e-8 here), the operator's result by its
    float16 rounding, 2^-11 of it, and that of dy W: within 3 * 2^-11 of the largest."""
    g = gen(11, cuda_device)
    rows, feat, width, step = 6, 16, 8, 1e-4
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device)  # noqa: E731
    hidden, down, dy = rand(rows, 2 * width).half(), (rand(1, feat, width) / 4).half(), rand(rows, feat).half()
    d_hidden = torch.empty(rows * 2 * width, dtype=torch.float16, device=cuda_device)
    ops.grouped_mm_gated_grad(dy.view(-1), down.view(-1), hidden.view(-1), d_hidden, None, None, 1, feat, width,
                              ops.GATED_GELU if gelu else 0)

    def loss(h):
        f = gate_parts(h[:, :width], gelu)[0]
        return float(((f * h[:, width:]) @ down[0].double().t() * dy.double()).sum())

    want = torch.zeros(rows, 2 * width, dtype=torch.float64, device=cuda_device)
    for r in range(rows):
        for c in range(2 * width):
            h = hidden.double().clone()
            h[r, c] += step
            hi = loss(h)
            h[r, c] -= 2 * step
            want[r, c] = (hi - loss(h)) / (2 * step)
    off = (d_hidden.view(rows, -1).double() - want).abs().max()
    assert off <= 3 * 2.0 ** -11 * want.abs().max()


def test_grad_values_stay_in_their_rows(cuda_device):
    sizes, feat, width = [40, 0, 25, 130], 96, 72
    g = gen(3, cuda_device)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device).half()  # noqa: E731
    dy, w, hidden = rand(195, feat), rand(4, feat, width), rand(195, 2 * width)

    def call():
        d, a = torch.empty(195 * 2 * width, device=cuda_device).half(), torch.empty(195 * width, device=cuda_device).half()
        ops.grouped_mm_gated_grad(dy.view(-1), w.view(-1), hidden.view(-1), d, a, pointers(sizes, cuda_device), 4, feat, width)
        return d.view(195, 2 * width), a.view(195, width)

    d0, a0 = call()
    dy[39, 5], hidden[64, 3], hidden[70, width + 7] = NAN, NAN, NAN
    w[1] = NAN
    d, a = call()
    bad_d, bad_a = torch.zeros_like(d, dtype=torch.bool), torch.zeros_like(a, dtype=torch.bool)
    bad_d[39], bad_d[64, 3], bad_d[64, width + 3], bad_d[70, 7] = True, True, True, True
    bad_a[64, 3], bad_a[70, 7] = True, True
    assert torch.equal(d.isnan(), bad_d) and torch.equal(a.isnan(), bad_a)
    assert torch.equal(d[~bad_d], d0[~bad_d]) and torch.equal(a[~bad_a], a0[~bad_a])


@pytest.mark.parametrize("sizes,feat,width", [([70, 0, 300, 1], 200, 136), ([90], 4096, 72), ([40, 500], 65, 33), ([60] * 40, 72, 520)], ids=str)
def test_gradient_in_the_place_of_the_projections(cuda_device, sizes, feat, width):
    g = gen(8, cuda_device)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    rows, n = sum(sizes), len(sizes)
    dy, w, hidden, ptr = rand(rows * feat), rand(n * feat * width), rand(rows * 2 * width), pointers(sizes, cuda_device)
    d, act, act2 = torch.empty_like(hidden), torch.empty_like(hidden[:rows * width]), torch.empty_like(hidden[:rows * width])
    ops.grouped_mm_gated_grad(dy, w, hidden, d, act, ptr, n, feat, width)
    ops.grouped_mm_gated_grad(dy, w, hidden, hidden, act2, ptr, n, feat, width)
    assert torch.equal(hidden, d) and torch.equal(act, act2)


# ------------------------------------------------------------------ both
@pytest.mark.parametrize("fi,rows,width", [(64, 30, 64), (2048, 30, 136), (64, 3000, 132), (4096, 900, 136)])
def test_wild_pointers_stay_inside(cuda_device, fi, rows, width):
    """Pointers that no router writes: what is computed is not defined, but nothing outside of the arrays is touched."""
    x, w = torch.ones(rows * fi, device=cuda_device).half(), torch.ones(3 * 2 * width * fi, device=cuda_device).half()
    h = torch.ones(rows * 2 * width, device=cuda_device).half()
    for bad in ([0, rows, 5, rows + 9], [-3, rows // 2, 2 ** 31 - 1, 0], [rows, 7, -2 ** 31, rows]):
        ptr = torch.tensor(bad, device=cuda_device).int()
        for n in (width, 2 * width):
            guard = [torch.full((1000 + rows * m + 1000,), 9.0, device=cuda_device).half() for m in (width, 2 * width)]
            y, hid = (t[1000:-1000] for t in guard)
            ops.grouped_mm_gated(x, w, y, hid if n == width else None, ptr, 3, fi, width)
            ops.grouped_mm_gated_grad(x, w[:3 * width * fi], h, hid, y if n == width else None, ptr, 3, fi, width)
            for t in guard:
                assert (t[:1000] == 9).all() and (t[-1000:] == 9).all()


def test_a_row_ahead_of_the_first_group_is_left(cuda_device):
    x, w = torch.ones(16, device=cuda_device).half(), torch.ones(3 * 16 * 8, device=cuda_device).half()
    y, h = torch.full((16,), 9.0, device=cuda_device).half(), torch.full((32,), 9.0, device=cuda_device).half()
    ptr = torch.tensor([1, 1, 2, 2], dtype=torch.int32, device=cuda_device)
    ops.grouped_mm_gated(x, w, y, h, ptr, 3, 8, 8)
    assert (y[:8] == 9).all() and (y[8:] != 9).all() and (h[:16] == 9).all() and (h[16:] == 8).all()


def test_results_repeat(cuda_device):
    """The same bits from call to call, whatever the order in which blocks run."""
    g = gen(5, cuda_device)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    for sizes, fi, width in (([100], 4096, 264), ([5, 300, 0, 41], 520, 200), ([3, 1], 2048, 512)):
        rows, n = sum(sizes), len(sizes)
        x, w, down, h, ptr = rand(rows * fi), rand(n * 2 * width * fi), rand(n * fi * width), rand(rows * 2 * width), pointers(sizes, cuda_device)
        seen = []
        for _ in range(20):
            y, hid, d, a = (torch.empty(rows * m, device=cuda_device).bfloat16() for m in (width, 2 * width, 2 * width, width))
            ops.grouped_mm_gated(x, w, y, hid, ptr, n, fi, width)
            ops.grouped_mm_gated_grad(x, down, h, d, a, ptr, n, fi, width)
            seen.append((y, hid, d, a))
        assert all(torch.equal(p, q) for s in seen[1:] for p, q in zip(s, seen[0]))


@pytest.mark.parametrize("rows,fi,width", [(100, 4096, 264), (200, 135, 71), (4, 264, 136)])
def test_in_a_graph_and_on_two_streams(cuda_device, rows, fi, width):
    """Captured calls own their scratch memory: two graphs replayed side by side, beside an eager call, on other inputs than captured."""
    g = gen(6, cuda_device)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device).half()  # noqa: E731
    w, down = rand(2 * width * fi) / 30, rand(fi * width) / 30
    inputs = [(rand(rows * fi), rand(rows * 2 * width)) for _ in range(3)]

    def calls(x, h):
        y, d = torch.empty(rows * width, device=cuda_device).half(), torch.empty(rows * 2 * width, device=cuda_device).half()
        ops.grouped_mm_gated(x, w, y, None, None, 1, fi, width)
        ops.grouped_mm_gated_grad(x, down, h, d, None, None, 1, fi, width)
        return y, d

    want = [calls(*i) for i in inputs]
    torch.cuda.synchronize()
    sides, graphs, held, outs = [], [], [], []
    for _ in range(2):
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream())
        h = tuple(torch.zeros_like(t) for t in inputs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            outs.append(calls(*h))
        sides.append(side), graphs.append(graph), held.append(h)
    torch.cuda.synchronize()
    for i in range(2):
        for t, v in zip(held[i], inputs[i]):
            t.copy_(v)
    torch.cuda.synchronize()
    for _ in range(5):
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        eager = calls(*inputs[2])
    torch.cuda.synchronize()
    for got, exp in zip(outs + [eager], want):
        assert all(torch.equal(a, b) for a, b in zip(got, exp))


def test_bad_indices_are_refused_when_asked(cuda_device):
    lib = L.load()
    x, w = torch.ones(30 * 64, device=cuda_device).half(), torch.ones(2 * 128 * 64, device=cuda_device).half()
    y, h = torch.zeros(30 * 64, device=cuda_device).half(), torch.zeros(30 * 128, device=cuda_device).half()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    lib.sparsetir_set_validate(1)
    try:
        ops.grouped_mm_gated(x, w, y, h, i32(0, 10, 25), 2, 64, 64)
        for bad, message in ((i32(0, 20, 10), "decreases"), (i32(0, 10, 31), "out of range"), (i32(1, 10, 30), "expected 0")):
            with pytest.raises(ops.SparseTIRError, match=message):
                ops.grouped_mm_gated(x, w, y, h, bad, 2, 64, 64)
            with pytest.raises(ops.SparseTIRError, match=message):
                ops.grouped_mm_gated_grad(x, w[:2 * 64 * 64], h, h.clone(), None, bad, 2, 64, 64)
    finally:
        lib.sparsetir_set_validate(0)


def test_no_wait_ran_out(cuda_device):
    import ctypes

    count = ctypes.c_uint(99)
    assert L.load().sparsetir_tc_timeouts(0, ctypes.byref(count)) == 0 and count.value == 0
