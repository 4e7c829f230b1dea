"""The gated products and those of 8-bit floating point where every pair of thread blocks has several tiles, where a batch meets in a few
groups, launched a thousand times, from several threads, and over more than 2^31 elements."""
import threading

import pytest
import torch

from sparsetir_b200 import ops
from test_gpu_f8 import F8, blocks, operands, truth
from test_gpu_f8 import check_gated as check_gated_f8
from test_gpu_f8 import check_mm as check_mm_f8
from test_gpu_gated import by_group, check_gated, check_grad, gate_parts, gated_truth, rel, TINY
from test_gpu_moe import U, gen, near, pointers
from test_gpu_moe_hot import SIZES as HOT
from test_gpu_moe_tiles import LARGE, PAIRS, SMALL, every_launch, mostly_empty, no_wait_ran_out, tiles

pytestmark = pytest.mark.gpu


def name(s):
    return f"{sum(s)}-{len(s)}" if isinstance(s, list) else str(s)


@pytest.mark.parametrize("sizes", LARGE + SMALL, ids=name)
@pytest.mark.parametrize("fi,width,dtype,gelu", [(64, 512, torch.float16, False), (136, 520, torch.bfloat16, True), (328, 505, torch.bfloat16, False)])
def test_gated(cuda_device, sizes, fi, width, dtype, gelu):
    assert tiles(sizes, 2 * width, 256) >= 4 * PAIRS
    check_gated(sizes, fi, width, dtype, cuda_device, gelu=gelu, keep=width != 505, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes", LARGE + SMALL, ids=name)
@pytest.mark.parametrize("feat,width,dtype,gelu,out_in", [(64, 1024, torch.float16, False, False), (136, 1000, torch.bfloat16, True, True),
                                                          (328, 1009, torch.bfloat16, False, False)])
def test_gradient(cuda_device, sizes, feat, width, dtype, gelu, out_in):
    assert tiles(sizes, width, 256) >= 4 * PAIRS
    check_grad(sizes, feat, width, dtype, cuda_device, gelu=gelu, out_in=out_in, act=width != 1009, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes", LARGE + SMALL, ids=name)
@pytest.mark.parametrize("fi,fo,out", [(128, 1024, torch.float16), (272, 1000, torch.float32), (656, 1001, torch.bfloat16)])
def test_products_of_8_bit_floating_point(cuda_device, sizes, fi, fo, out):
    assert tiles(sizes, fo, 256) >= 4 * PAIRS
    check_mm_f8(sizes, fi, fo, out, cuda_device, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes", LARGE + SMALL, ids=name)
@pytest.mark.parametrize("fi,width,gelu", [(128, 512, False), (272, 520, True), (656, 505, False)])
def test_gated_of_8_bit_floating_point(cuda_device, sizes, fi, width, gelu):
    """Widths of which the other projection's rows lie in whole blocks of W, of which they do not, and of which 16 of them do not."""
    check_gated_f8(sizes, fi, width, torch.bfloat16, cuda_device, gelu=gelu, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes", HOT, ids=lambda s: f"{sum(s)}-{len(s)}-{max(s)}")
@pytest.mark.parametrize("fi,width", [(272, 40), (528, 257)])
def test_rows_in_a_few_groups(cuda_device, sizes, fi, width):
    check_gated(sizes, fi, width, torch.float16, cuda_device, tail=9)
    check_mm_f8(sizes, fi, width, torch.bfloat16, cuda_device, tail=9)
    check_gated_f8(sizes, fi, width, torch.float16, cuda_device, tail=9)


def f8_calls(sizes, fi, width, device):
    n, rows = len(sizes), sum(sizes)
    x, xs, w, ws, xd, wd = operands(rows, n, fi, 2 * width, device)
    ptr = pointers(sizes, device)
    flat = [t.reshape(-1) for t in (x, xs, w, ws)]
    return (lambda y: ops.grouped_mm_f8(*flat, y, ptr, n, fi, 2 * width), lambda y: ops.grouped_mm_gated_f8(*flat, y, ptr, n, fi, width)), xd, wd


@pytest.mark.parametrize("sizes", [mostly_empty(128, 9, 20000, 3), mostly_empty(300, 150, 4000, 4), [3000, 1], [100]], ids=name)
@pytest.mark.parametrize("fi,width", [(384, 256), (1296, 72)])
def test_8_bit_floating_point_every_launch(cuda_device, sizes, fi, width):
    rows = sum(sizes)
    (mm, gated), xd, wd = f8_calls(sizes, fi, width, cuda_device)
    y, a = torch.empty(rows * 2 * width, dtype=torch.bfloat16, device=cuda_device), torch.empty(rows * width, dtype=torch.bfloat16, device=cuda_device)
    h, mags = truth(xd, wd, sizes)
    e = (2 * fi + 8) * U * mags
    near(every_launch(lambda: mm(y), y, 1000).view(rows, -1), h, e, torch.bfloat16)
    g, up, eg, eu = h[:, :width], h[:, width:], e[:, :width], e[:, width:]
    f, _, _, z, _ = gate_parts(g, False)
    near(every_launch(lambda: gated(a), a, 1000).view(rows, -1), f * up,
         1.13 * eg * up.abs() + (f.abs() + 1.13 * eg) * eu + (f * up).abs() * rel(z) + TINY, torch.bfloat16)


@pytest.mark.parametrize("sizes", [mostly_empty(128, 9, 20000, 3), mostly_empty(300, 150, 4000, 4)], ids=name)
def test_gated_every_launch(cuda_device, sizes):
    fi, width, n, rows = 200, 264, len(sizes), sum(sizes)
    g = gen(4, cuda_device)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device)  # noqa: E731
    x, w, down, h = rand(rows, fi).half(), (rand(n, 2 * width, fi) / fi ** 0.5).half(), (rand(n, fi, width) / fi ** 0.5).half(), rand(rows, 2 * width).half()
    ptr = pointers(sizes, cuda_device)
    y, d = torch.empty(rows * width, dtype=torch.float16, device=cuda_device), torch.empty(rows * 2 * width, dtype=torch.float16, device=cuda_device)
    first = every_launch(lambda: ops.grouped_mm_gated(x.view(-1), w.view(-1), y, None, ptr, n, fi, width), y, 1000)
    want, slack = gated_truth(*by_group(x, w.transpose(1, 2), sizes), fi, False)
    near(first.view(rows, width), want, slack, torch.float16)
    every_launch(lambda: ops.grouped_mm_gated_grad(x.view(-1), down.view(-1), h.view(-1), d, None, ptr, n, fi, width), d, 1000)


def test_offsets_beyond_32_bits(cuda_device):
    """Tensors of more than 2^31 elements: rows far apart have the values of rows at the start."""
    rows, fi, width = 540_000, 8, 2048
    assert rows * 2 * width > 2 ** 31
    g = gen(9, cuda_device)
    few = torch.randn(500, fi, generator=g, device=cuda_device).half()
    x = few.repeat(rows // 500, 1)
    w, down = torch.randn(2 * width, fi, generator=g, device=cuda_device).half(), torch.randn(fi, width, generator=g, device=cuda_device).half()
    y, hidden = torch.zeros(rows * width, device=cuda_device, dtype=torch.float16), torch.zeros(rows * 2 * width, device=cuda_device, dtype=torch.float16)
    ops.grouped_mm_gated(x.view(-1), w.view(-1), y, hidden, None, 1, fi, width)
    small_y, small_h = torch.zeros(500 * width, device=cuda_device).half(), torch.zeros(500 * 2 * width, device=cuda_device).half()
    ops.grouped_mm_gated(few.view(-1), w.view(-1), small_y, small_h, None, 1, fi, width)
    for at in (0, 250_000, 262_000, 524_000, 539_500):
        assert torch.equal(y.view(rows, width)[at:at + 500], small_y.view(500, width))
        assert torch.equal(hidden.view(rows, 2 * width)[at:at + 500], small_h.view(500, 2 * width))
    d, small_d = torch.empty_like(hidden), torch.empty_like(small_h)
    ops.grouped_mm_gated_grad(x.view(-1), down.view(-1), hidden, d, y, None, 1, fi, width)
    ops.grouped_mm_gated_grad(few.view(-1), down.view(-1), small_h, small_d, None, None, 1, fi, width)
    for at in (0, 250_000, 262_000, 524_000, 539_500):
        assert torch.equal(d.view(rows, 2 * width)[at:at + 500], small_d.view(500, 2 * width))
    del y, hidden, d
    q, scale = torch.zeros(rows * 4096, dtype=torch.int8, device=cuda_device).view(F8), torch.zeros(blocks(4096) * rows, device=cuda_device)
    wide = torch.randn(500, 4096, generator=g, device=cuda_device).bfloat16()
    slots = torch.arange(rows, device=cuda_device).view(-1, 500).t().contiguous().int()  # each row to 1,080 places
    one_q, one_s = torch.zeros(500 * 4096, dtype=torch.int8, device=cuda_device).view(F8), torch.zeros(blocks(4096) * 500, device=cuda_device)
    ops.moe_dispatch_f8(wide.view(-1), None, one_q, one_s, 4096, 1)
    for k in range(0, rows // 500, 30):
        ops.moe_dispatch_f8(wide.view(-1), slots[:, k:k + 30].reshape(-1).contiguous(), q, scale, 4096, 30)
    for at in (0, 524_000, 539_500):
        assert torch.equal(q.view(torch.int8).view(rows, 4096)[at:at + 500], one_q.view(torch.int8).view(500, 4096))
        assert torch.equal(scale.view(-1, rows)[:, at:at + 500], one_s.view(-1, 500))
    wq, ws = torch.randint(-100, 100, (16 * 4096,), device=cuda_device, dtype=torch.int8, generator=g).view(F8), torch.rand(blocks(4096), generator=g, device=cuda_device)
    out, small = torch.zeros(rows * 16, device=cuda_device), torch.zeros(500 * 16, device=cuda_device)
    ops.grouped_mm_f8(q, scale, wq, ws, out, None, 1, 4096, 16)
    want = (one_q.view(500, 32, 128).double() * one_s.view(32, 500).t().double()[:, :, None]).view(500, 4096) @ \
        (wq.view(16, 32, 128).double() * ws.view(1, 32, 1).double()).view(16, 4096).t()
    mags = (one_q.view(500, 32, 128).double().abs() * one_s.view(32, 500).t().double()[:, :, None]).view(500, 4096) @ \
        (wq.view(16, 32, 128).double().abs() * ws.view(1, 32, 1).double()).view(16, 4096).t()
    for at in (0, 524_000, 539_500):
        near(out.view(rows, 16)[at:at + 500], want, (2 * 4096 + 8) * U * mags)
    assert small.numel() == 500 * 16


def test_threads_on_one_stream(cuda_device):
    """Calls of several launches, which hand data to each other through the stream's scratch memory: operands that are copied to aligned
    rows, and a depth that several units share."""
    stream = torch.cuda.Stream(cuda_device)

    def job(seed, rows, fi, width):
        g = gen(seed, cuda_device)
        rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device).half()  # noqa: E731
        x, w, down, h = rand(rows * fi), rand(2 * width * fi) / 20, rand(fi * width) / 20, rand(rows * 2 * width)
        q, qs, wq, ws, _, _ = operands(rows, 1, fi, 2 * width, cuda_device)

        def calls():
            y, d = torch.zeros(rows * width, device=cuda_device).half(), torch.zeros(rows * 2 * width, device=cuda_device).half()
            z, a = torch.zeros(rows * 2 * width, device=cuda_device), torch.zeros(rows * width, device=cuda_device).half()
            ops.grouped_mm_gated(x, w, y, None, None, 1, fi, width)
            ops.grouped_mm_gated_grad(x, down, h, d, None, None, 1, fi, width)
            ops.grouped_mm_f8(q.view(-1), qs.view(-1), wq.view(-1), ws.view(-1), z, None, 1, fi, 2 * width)
            ops.grouped_mm_gated_f8(q.view(-1), qs.view(-1), wq.view(-1), ws.view(-1), a, None, 1, fi, width)
            return y, d, z, a

        return calls

    jobs = [job(1, 100, 4099, 131), job(2, 700, 203, 67), job(3, 40, 2051, 200)]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    errors, gate = [], threading.Barrier(len(jobs))

    def work(j, expected):
        try:
            torch.cuda.set_device(cuda_device)
            with torch.cuda.stream(stream):
                gate.wait()
                for _ in range(40):
                    got = j()
                    stream.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, expected))
        except Exception as e:  # surfaced by the main thread
            errors.append(repr(e))
            gate.abort()

    threads = [threading.Thread(target=work, args=pair) for pair in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("rows,fi,width", [(100, 4099, 131), (200, 4096, 264)])
def test_calls_on_a_reserved_stream_allocate_nothing(cuda_device, rows, fi, width):
    """What the query answers is enough for each of the products."""
    import ctypes

    from sparsetir_b200 import _lib as L

    lib, need = L.load(), 0
    for size in ((2 * width, 2, ops.GROUPED_W_OUT_IN), (2 * width, 1, 0), (width, 2, 0)):
        out = ctypes.c_size_t(0)
        assert lib.sparsetir_grouped_mm_workspace(rows, 1, fi, size[0], size[1], size[2], ctypes.byref(out)) == 0
        need = max(need, out.value)
    g = gen(3, cuda_device)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device).half()  # noqa: E731
    x, w, down, h = rand(rows * fi), rand(2 * width * fi), rand(fi * width), rand(rows * 2 * width)
    q, qs, wq, ws, _, _ = operands(rows, 1, fi, 2 * width, cuda_device)
    y, d, z = torch.empty(rows * width, device=cuda_device).half(), torch.empty(rows * 2 * width, device=cuda_device).half(), torch.empty(rows * 2 * width, device=cuda_device)
    stream = torch.cuda.Stream(cuda_device)
    calls = [lambda: ops.grouped_mm_gated(x, w, y, None, None, 1, fi, width), lambda: ops.grouped_mm_gated_grad(x, down, h, d, None, None, 1, fi, width),
             lambda: ops.grouped_mm_f8(q.view(-1), qs.view(-1), wq.view(-1), ws.view(-1), z, None, 1, fi, 2 * width),
             lambda: ops.grouped_mm_gated_f8(q.view(-1), qs.view(-1), wq.view(-1), ws.view(-1), y, None, 1, fi, width)]
    for c in calls:  # kernels are loaded, and with them what memory they take
        c()
    torch.cuda.synchronize()
    assert lib.sparsetir_reserve_workspace(0, ctypes.c_void_p(stream.cuda_stream), need, 0) == 0
    free = torch.cuda.mem_get_info(cuda_device)[0]
    with torch.cuda.stream(stream):
        for c in calls:
            c()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info(cuda_device)[0] == free
