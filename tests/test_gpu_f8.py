"""Rows in 8-bit floating point with a scale for each block of 128, and the products of such operands, against their definitions in 64
bits.

Tolerances.  u = 2^-24.  The sums of a block's products are formed in f32, scaled by the rounded product of two scales and added in
f32: n products in all are off by at most (2 n + 8) u times the sum of the scaled products' magnitudes; act as in
test_gpu_gated.py.  The numbers of 8 bits themselves are exact for 16-bit rows: 448 x / max has a place between two of them that one
rounded division of exact operands does not move."""
import math

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops
from test_gpu_gated import gate_parts, rel, TINY
from test_gpu_moe import FEATS, GROUPS, INF, NAN, ROWS, U, gen, near, off_by, pointers, some_slots

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
N = 128


def blocks(n):
    return -(-n // N)


def e4m3(v):
    """To the nearest number of 4 bits' exponent and 3 bits' fraction, in 64 bits, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def quantised(x):
    """(numbers, scales [rows, blocks]) of rows, in 64 bits"""
    r, f = x.shape
    pad = torch.zeros(r, blocks(f) * N, dtype=torch.float64, device=x.device)
    pad[:, :f] = x.double()
    most = pad.view(r, -1, N).abs().amax(2)
    q = e4m3(pad.view(r, -1, N) * 448 / torch.where(most > 0, most, 1.0)[:, :, None])
    return q.view(r, -1)[:, :f], most / 448


@pytest.mark.parametrize("t,k,f", ROWS + [(4, 2, 128), (4, 1, 256), (3, 2, 129), (7, 3, 1152), (2, 1, 127)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1])
def test_dispatch(cuda_device, t, k, f, dtype, shift):
    rows = t * k + 3
    slots = some_slots(t, k, rows, t + f, cuda_device, missing=0.2)
    x = torch.randn(t, f, generator=gen(1, cuda_device), device=cuda_device) * 3
    x = off_by((x * torch.exp(torch.randn(f, generator=gen(2, cuda_device), device=cuda_device))).to(dtype), shift).view(t, f)
    q = off_by(torch.full((rows, f), 9.0, device=cuda_device).to(F8).view(torch.int8), shift).view(F8)
    scale = torch.full((blocks(f) * rows,), 9.0, device=cuda_device)
    ops.moe_dispatch_f8(x.reshape(-1), slots, q, scale, f, k)
    want_q, want_s = quantised(x)
    kept = slots >= 0
    to = slots[kept].long()
    all_q = torch.full((rows, f), 9.0, dtype=torch.float64, device=cuda_device)
    all_s = torch.full((rows, blocks(f)), 9.0, dtype=torch.float64, device=cuda_device)
    all_q[to], all_s[to] = want_q.repeat_interleave(k, 0)[kept], want_s.repeat_interleave(k, 0)[kept]
    got = q.view(rows, f).double()
    if dtype is torch.float32:  # 0.875 x is rounded: a quotient within 2^-22 of the middle may go either way, by one step
        off = (got - all_q).abs()
        assert (off <= all_q.abs().clamp(min=2.0 ** -6) * 2.0 ** -3 * 1.0001).all() and (off > 0).float().mean() < 1e-3
    else:
        assert torch.equal(got, all_q)
    near(scale.view(-1, rows).t(), all_s, 0.0, torch.float32)


def test_every_quotient_of_two_short_numbers(cuda_device):
    """All fractions a bfloat16 has over all that its largest has: every tie is among them."""
    m = torch.arange(128, 256, device=cuda_device).double()
    for e in (0, -3, -7, -9):
        x = torch.zeros(128 * 128, N, device=cuda_device)
        x[:, 0] = m.repeat_interleave(128).float()
        x[:, 1] = (m.repeat(128) * 2.0 ** e).clamp(max=255).float()
        x[:, 1] = torch.minimum(x[:, 0], x[:, 1])
        x[:, 2] = -x[:, 1]
        for dtype in (torch.bfloat16, torch.float16):
            v = x.to(dtype)
            assert torch.equal(v.double(), x.double())
            q, scale = torch.zeros(v.numel(), dtype=torch.int8, device=cuda_device).view(F8), torch.zeros(len(v), device=cuda_device)
            ops.moe_dispatch_f8(v.view(-1), None, q, scale, N, 1)
            assert torch.equal(q.view(len(v), N).double(), quantised(v)[0])


def test_dispatch_of_blocks_without_a_scale(cuda_device):
    x = torch.zeros(8, 2 * N, device=cuda_device)
    x[:, N:] = 1.0  # the second block has its own
    x[1, 0], x[2, 0], x[2, 1], x[3, 0], x[4, 5], x[4, 6], x[5, 0], x[6, 0], x[6, 1], x[7, 0], x[7, 1] = \
        INF, NAN, INF, 2.0 ** -111, -3.0, 1.5, -INF, 2.0 ** -110, -(2.0 ** -111), 3.4e38, -3.4e38
    q, scale = torch.full((8 * 2 * N,), 9.0, device=cuda_device).to(F8), torch.full((16,), 9.0, device=cuda_device)
    ops.moe_dispatch_f8(x.view(-1), None, q, scale, 2 * N, 1)
    q, s = q.view(8, 2 * N).float().cpu(), scale.view(2, 8).cpu()
    assert (q[[0, 1, 2, 3, 5], :N] == 0).all() and (q[:, N:] == 448).all() and (s[1] == torch.tensor(1.0) / 448).all()
    assert q[4, 5:7].tolist() == [-448, 224] and q[6, :2].tolist() == [448, -224] and q[7, :2].tolist() == [448, -448]
    assert s[0, 0] == 0 and s[0, 1] == INF and s[0, 2].isnan() and s[0, 3] == 0 and s[0, 5] == INF
    assert s[0, 6] == torch.tensor(2.0 ** -110) / 448 and s[0, 4] == torch.tensor(3.0) / 448


# ------------------------------------------------------------------ products
def operands(rows, n, fi, fo, device, tail=0, seed=0):
    """(x, x_scale, w, w_scale) as the operators take them, and x and w [groups, fi, fo] as they stand for"""
    g = gen(fi * 7 + fo + seed, device)
    all_rows = rows + tail
    x = torch.randn(all_rows, fi, generator=g, device=device).mul(60).clamp(-448, 448).to(F8)
    w = torch.randn(n, fo, fi, generator=g, device=device).mul(60).clamp(-448, 448).to(F8)
    xs = torch.rand(blocks(fi), all_rows, generator=g, device=device) * 0.03 + 0.003
    ws = (torch.rand(n, blocks(fo), blocks(fi), generator=g, device=device) * 0.03 + 0.003) / math.sqrt(fi)
    if tail:
        xs[:, rows:] = NAN
    xd = x.double() * xs.double().repeat_interleave(N, 0)[:fi].t()
    wd = w.double() * ws.double().repeat_interleave(N, 1)[:, :fo].repeat_interleave(N, 2)[:, :, :fi]
    return x, xs, w, ws, xd[:rows], wd.transpose(1, 2)


def odd(t, shift):
    return off_by(t.view(torch.int8), shift).view(F8)


def truth(x, w, sizes):
    parts, mags, at = [], [], 0
    for g, n in enumerate(sizes):
        parts.append(x[at:at + n] @ w[g])
        mags.append(x[at:at + n].abs() @ w[g].abs())
        at += n
    return torch.cat(parts), torch.cat(mags)


def check_mm(sizes, fi, fo, dtype, device, shift=0, tail=0, null=False):
    n, rows = len(sizes), sum(sizes)
    x, xs, w, ws, xd, wd = operands(rows, n, fi, fo, device, tail)
    y = off_by(torch.full(((rows + tail) * fo,), 9.0, dtype=dtype, device=device), shift)
    ops.grouped_mm_f8(odd(x, shift), off_by(xs, shift), odd(w, shift), off_by(ws, shift), y, None if null else pointers(sizes, device), n, fi, fo)
    want, mags = truth(xd, wd, sizes)
    y = y.view(-1, fo)
    near(y[:rows], want, (2 * fi + 8) * U * mags, dtype)
    assert (y[rows:] == 9.0).all()


def check_gated(sizes, fi, width, dtype, device, gelu=False, shift=0, tail=0, null=False):
    n, rows = len(sizes), sum(sizes)
    x, xs, w, ws, xd, wd = operands(rows, n, fi, 2 * width, device, tail)
    y = off_by(torch.full(((rows + tail) * width,), 9.0, dtype=dtype, device=device), shift)
    ops.grouped_mm_gated_f8(odd(x, shift), off_by(xs, shift), odd(w, shift), off_by(ws, shift), y, None if null else pointers(sizes, device), n,
                            fi, width, ops.GATED_GELU if gelu else 0)
    h, mags = truth(xd, wd, sizes)
    e = (2 * fi + 8) * U * mags
    g, up, eg, eu = h[:, :width], h[:, width:], e[:, :width], e[:, width:]
    f, _, _, z, _ = gate_parts(g, gelu)
    y = y.view(-1, width)
    near(y[:rows], f * up, 1.13 * eg * up.abs() + (f.abs() + 1.13 * eg) * eu + (f * up).abs() * rel(z) + TINY, dtype)
    assert (y[rows:] == 9.0).all()


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("fi,fo", [(16, 8), (128, 264), (528, 96)])
def test_mm_sizes(cuda_device, sizes, fi, fo):
    check_mm(GROUPS[sizes], fi, fo, torch.bfloat16, cuda_device, tail=3)


@pytest.mark.parametrize("fi,fo", FEATS + [(16, 130), (4096, 72), (8200, 16), (127, 129), (129, 127)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_mm_features(cuda_device, fi, fo, dtype):
    check_mm([70, 0, 33, 129], fi, fo, dtype, cuda_device, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("fi,fo", [(64, 72), (63, 40), (272, 136)])
@pytest.mark.parametrize("sizes", [[70, 0, 130], [2, 3, 0]], ids=str)
def test_mm_operands_at_odd_addresses(cuda_device, shift, fi, fo, sizes):
    check_mm(sizes, fi, fo, torch.float16, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,fi,fo", [([2000, 100, 1700], 1024, 1000), ([700] * 8, 2048, 512), ([4096], 528, 2056), ([256] * 30, 640, 768)])
def test_mm_large(cuda_device, sizes, fi, fo):
    check_mm(sizes, fi, fo, torch.bfloat16, cuda_device)


@pytest.mark.parametrize("sizes,fi,fo", [([100], 8200, 520), ([33, 0, 50, 41] * 10, 4112, 72), ([3], 4096, 2000), ([5, 0, 16, 17, 1, 0, 33], 1040, 520),
                                         ([300], 16400, 72)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_mm_depth_shared(cuda_device, sizes, fi, fo, dtype):
    check_mm(sizes, fi, fo, dtype, cuda_device, tail=2)


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5, 2], [9, 16, 12], [1] * 40, [0, 40, 0, 0, 0, 0, 0, 0]], ids=str)
@pytest.mark.parametrize("fi,fo", [(1, 1), (7, 9), (63, 130), (264, 257), (1001, 24), (4096, 1000), (1024, 2048)])
def test_mm_few_rows(cuda_device, sizes, fi, fo):
    check_mm(sizes, fi, fo, torch.bfloat16, cuda_device, tail=2)


@pytest.mark.parametrize("rows", [1, 5, 200])
def test_one_group_without_pointers(cuda_device, rows):
    check_mm([rows], 144, 72, torch.float16, cuda_device, null=True)
    check_gated([rows], 144, 72, torch.float16, cuda_device, null=True)


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("fi,width", [(16, 8), (128, 136), (528, 48)])
@pytest.mark.parametrize("gelu", [False, True])
def test_gated_sizes(cuda_device, sizes, fi, width, gelu):
    check_gated(GROUPS[sizes], fi, width, torch.bfloat16, cuda_device, gelu=gelu, tail=3)


@pytest.mark.parametrize("fi,width", FEATS + [(72, 16), (64, 15), (136, 17), (200, 500), (264, 129), (4096, 72)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gated_features(cuda_device, fi, width, dtype):
    check_gated([70, 0, 33, 129], fi, width, dtype, cuda_device, tail=5)


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("fi,width", [(64, 72), (63, 40), (272, 136)])
@pytest.mark.parametrize("sizes", [[70, 0, 130], [2, 3, 0]], ids=str)
def test_gated_operands_at_odd_addresses(cuda_device, shift, fi, width, sizes):
    check_gated(sizes, fi, width, torch.float16, cuda_device, shift=shift)


@pytest.mark.parametrize("sizes,fi,width", [([2000, 100, 1700], 1024, 520), ([700] * 8, 2048, 256), ([4096], 528, 1000)])
def test_gated_large(cuda_device, sizes, fi, width):
    check_gated(sizes, fi, width, torch.bfloat16, cuda_device)


@pytest.mark.parametrize("sizes,fi,width", [([100], 8200, 264), ([33, 0, 50, 41], 4112, 104), ([300], 16400, 40), ([120], 8192, 33)])
def test_gated_depth_shared(cuda_device, sizes, fi, width):
    check_gated(sizes, fi, width, torch.float16, cuda_device, tail=2)


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5, 2], [9, 16, 12], [1] * 40, [0, 40, 0, 0, 0, 0, 0, 0]], ids=str)
@pytest.mark.parametrize("fi,width", [(1, 1), (7, 9), (63, 130), (264, 257), (1001, 24), (4096, 1000), (1024, 2048)])
def test_gated_few_rows(cuda_device, sizes, fi, width):
    check_gated(sizes, fi, width, torch.bfloat16, cuda_device, tail=2)


def test_sums_are_kept_in_32_bits(cuda_device):
    """Products of one size and an odd one out, 2^-20 of their sum: whole numbers, so that f32 holds every partial sum and the result is
    exact.  Sums with fewer bits would lose the odd one."""
    for rows in (2, 300):
        fi, fo = 1024, 16
        x, w = torch.full((rows, fi), 16.0, device=cuda_device), torch.full((1, fo, fi), 16.0, device=cuda_device)
        x[:, 700], w[:, :, 700] = 1.0, 0.5
        x[:, 701], w[:, :, 701] = 0.0, 1.0
        y = torch.zeros(rows * fo, device=cuda_device)
        ops.grouped_mm_f8(x.to(F8).view(-1), torch.ones(8 * rows, device=cuda_device), w.to(F8).view(-1), torch.ones(8, device=cuda_device), y, None, 1,
                          fi, fo)
        assert (y == 256.0 * (fi - 2) + 0.5).all()


def test_values_stay_in_their_rows_blocks_and_groups(cuda_device):
    sizes, fi, fo = [40, 0, 25, 130], 400, 264
    x, xs, w, ws, _, _ = operands(195, 4, fi, fo, cuda_device)

    def call():
        y = torch.empty(195 * fo, device=cuda_device)
        ops.grouped_mm_f8(x.view(-1), xs.view(-1), w.view(-1), ws.view(-1), y, pointers(sizes, cuda_device), 4, fi, fo)
        return y.view(195, fo)

    y0 = call()
    xs[2, 39], xs[0, 64] = NAN, INF
    ws[1] = NAN        # nobody's expert
    ws[3, 1, 3] = NAN  # features 128 to 255 of the last group
    x.view(torch.int8)[70, 399] = 0x7f  # not a number
    y = call()
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[39], bad[64], bad[70], bad[65:, 128:256] = True, True, True, True
    assert torch.equal(~torch.isfinite(y), bad) and torch.equal(y[~bad], y0[~bad])


@pytest.mark.parametrize("fi,rows", [(64, 30), (2048, 30), (64, 3000), (4096, 900)])
def test_wild_pointers_stay_inside(cuda_device, fi, rows):
    width = 132
    x, w = torch.ones(rows * fi, device=cuda_device).to(F8), torch.ones(3 * 2 * width * fi, device=cuda_device).to(F8)
    xs, ws = torch.ones(blocks(fi) * rows, device=cuda_device), torch.ones(3 * blocks(2 * width) * blocks(fi), device=cuda_device)
    for bad in ([0, rows, 5, rows + 9], [-3, rows // 2, 2 ** 31 - 1, 0], [rows, 7, -2 ** 31, rows]):
        ptr = torch.tensor(bad, device=cuda_device).int()
        guard = [torch.full((1000 + rows * m + 1000,), 9.0, device=cuda_device).half() for m in (width, 2 * width)]
        ops.grouped_mm_gated_f8(x, xs, w, ws, guard[0][1000:-1000], ptr, 3, fi, width)
        ops.grouped_mm_f8(x, xs, w, ws, guard[1][1000:-1000], ptr, 3, fi, 2 * width)
        for t in guard:
            assert (t[:1000] == 9).all() and (t[-1000:] == 9).all()


def test_results_repeat(cuda_device):
    for sizes, fi, fo in (([100], 8200, 264), ([5, 300, 0, 41], 528, 200), ([3, 1], 2048, 512)):
        rows, n = sum(sizes), len(sizes)
        x, xs, w, ws, _, _ = operands(rows, n, fi, fo, cuda_device)
        seen = []
        for _ in range(20):
            y, a = torch.empty(rows * fo, device=cuda_device), torch.empty(rows * fo // 2, device=cuda_device).half()
            ops.grouped_mm_f8(x.view(-1), xs.view(-1), w.view(-1), ws.view(-1), y, pointers(sizes, cuda_device), n, fi, fo)
            ops.grouped_mm_gated_f8(x.view(-1), xs.view(-1), w.view(-1), ws.view(-1), a, pointers(sizes, cuda_device), n, fi, fo // 2)
            seen.append((y, a))
        assert all(torch.equal(p, q) for s in seen[1:] for p, q in zip(s, seen[0]))


@pytest.mark.parametrize("rows,fi,width", [(100, 8200, 264), (200, 135, 71), (4, 264, 136)])
def test_in_a_graph_and_on_two_streams(cuda_device, rows, fi, width):
    """A captured step quantises and multiplies its new inputs, beside another one and an eager one."""
    g = gen(6, cuda_device)
    _, _, w, ws, _, _ = operands(1, 1, fi, 2 * width, cuda_device)
    inputs = [torch.randn(rows * fi, generator=g, device=cuda_device).bfloat16() for _ in range(3)]

    def calls(x):
        q, s = torch.empty(rows * fi, dtype=F8, device=cuda_device), torch.empty(blocks(fi) * rows, device=cuda_device)
        y, a = torch.empty(rows * 2 * width, device=cuda_device), torch.empty(rows * width, device=cuda_device).half()
        ops.moe_dispatch_f8(x, None, q, s, fi, 1)
        ops.grouped_mm_f8(q, s, w.view(-1), ws.view(-1), y, None, 1, fi, 2 * width)
        ops.grouped_mm_gated_f8(q, s, w.view(-1), ws.view(-1), a, None, 1, fi, width)
        return y, a

    want = [calls(x) for x in inputs]
    torch.cuda.synchronize()
    sides, graphs, held, outs = [], [], [], []
    for _ in range(2):
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream())
        x, graph = torch.zeros_like(inputs[0]), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            outs.append(calls(x))
        sides.append(side), graphs.append(graph), held.append(x)
    torch.cuda.synchronize()
    for x, v in zip(held, inputs):
        x.copy_(v)
    torch.cuda.synchronize()
    for _ in range(5):
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        eager = calls(inputs[2])
    torch.cuda.synchronize()
    for got, exp in zip(outs + [eager], want):
        assert all(torch.equal(a, b) for a, b in zip(got, exp))


def test_bad_indices_are_refused_when_asked(cuda_device):
    lib = L.load()
    x, w = torch.ones(30 * 64, device=cuda_device).to(F8), torch.ones(2 * 128 * 64, device=cuda_device).to(F8)
    xs, ws = torch.ones(30, device=cuda_device), torch.ones(2, device=cuda_device)
    y, a = torch.zeros(30 * 128, device=cuda_device).half(), torch.zeros(30 * 64, device=cuda_device).half()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    lib.sparsetir_set_validate(1)
    try:
        ops.grouped_mm_f8(x, xs, w, ws, y, i32(0, 10, 25), 2, 64, 128)
        for bad, message in ((i32(0, 20, 10), "decreases"), (i32(0, 10, 31), "out of range"), (i32(1, 10, 30), "expected 0")):
            with pytest.raises(ops.SparseTIRError, match=message):
                ops.grouped_mm_f8(x, xs, w, ws, y, bad, 2, 64, 128)
            with pytest.raises(ops.SparseTIRError, match=message):
                ops.grouped_mm_gated_f8(x, xs, w, ws, a, bad, 2, 64, 64)
        with pytest.raises(ops.SparseTIRError, match=r"slots\[1\] = 30 is out of range"):
            ops.moe_dispatch_f8(y[:2 * 64], i32(-1, 30), x, xs, 64, 1)
    finally:
        lib.sparsetir_set_validate(0)


def test_no_wait_ran_out(cuda_device):
    import ctypes

    count = ctypes.c_uint(99)
    assert L.load().sparsetir_tc_timeouts(0, ctypes.byref(count)) == 0 and count.value == 0
