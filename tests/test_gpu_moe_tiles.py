"""The grouped products where every pair of thread blocks has several tiles: the ring of stages and the two accumulators go
round, their phases flip, and tiles of one step, of many and of none follow each other.  A pair has the tiles of its number, of its number plus
the pairs, and so on: 74 pairs with tiles of 256 rows or columns, 148 with tiles of 128 rows."""
import ctypes
import random

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops
from test_gpu_moe import check_grad_w, check_grouped, check_i8, gen, grouped_truth, near, pointers, U

pytestmark = pytest.mark.gpu

PAIRS, FEATURES = 74, 256  # with tiles of 256; features of a tile


def tiles(sizes, features, n):
    """Non-empty tiles of a product, of n rows each."""
    return sum(-(-s // n) for s in sizes) * -(-features // FEATURES)


def spread(groups, mean, seed, empty=0.1):
    rng = random.Random(seed)
    return [0 if rng.random() < empty else max(1, int(mean * rng.lognormvariate(0, 0.8))) for _ in range(groups)]


# few groups of many rows: tiles of 256 rows.  At least four to a pair, some of them a single row
LARGE = [[5000, 0, 300, 9000, 257, 5000, 1, 511], [700] * 31 + [0, 1, 2], [256] * 76, [19000]]
# many groups of few rows (128 at most on average): tiles of 128 rows
SMALL = [spread(180, 60, 1) + [129, 128, 127] + [1] * 20, [100] * 150, [0, 1, 0, 128, 3, 0] * 60, [1] * 260]


def no_wait_ran_out():
    count = ctypes.c_uint(99)
    assert L.load().sparsetir_tc_timeouts(0, ctypes.byref(count)) == 0 and count.value == 0


@pytest.mark.parametrize("sizes", LARGE, ids=lambda s: f"{sum(s)}-{len(s)}")
@pytest.mark.parametrize("fi,fo,dtype,out", [(64, 1024, torch.float16, torch.float16), (136, 1000, torch.bfloat16, torch.float32),
                                             (520, 1001, torch.bfloat16, torch.bfloat16), (65, 1024, torch.float16, torch.float16)])
@pytest.mark.parametrize("out_in", [False, True])
def test_products(cuda_device, sizes, fi, fo, dtype, out, out_in):
    assert tiles(sizes, fo, 256) >= 4 * PAIRS and sum(sizes) > 128 * len(sizes)
    check_grouped(sizes, fi, fo, dtype, out_in, out, cuda_device, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes", SMALL, ids=lambda s: f"{sum(s)}-{len(s)}")
@pytest.mark.parametrize("fi,dtype,out", [(64, torch.float16, torch.float16), (200, torch.bfloat16, torch.float32), (520, torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("out_in", [False, True])
def test_products_in_tiles_of_128(cuda_device, sizes, fi, dtype, out, out_in):
    fo = 1024
    assert tiles(sizes, fo, 128) >= 4 * 2 * PAIRS and 256 < sum(sizes) <= 128 * len(sizes)
    check_grouped(sizes, fi, fo, dtype, out_in, out, cuda_device, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes,n", [(s, 256) for s in LARGE] + [(s, 128) for s in SMALL], ids=lambda s: f"{sum(s)}-{len(s)}" if isinstance(s, list) else str(s))
@pytest.mark.parametrize("fi,fo,out", [(128, 1024, torch.float16), (272, 1000, torch.float32), (1040, 1001, torch.bfloat16)])
def test_products_in_8_bits(cuda_device, sizes, n, fi, fo, out):
    assert tiles(sizes, fo, n) >= 4 * PAIRS * 256 // n
    check_i8(sizes, fi, fo, out, cuda_device, tail=7)
    no_wait_ran_out()


@pytest.mark.parametrize("sizes", [[70] * 19 + [1], spread(24, 130, 3, empty=0), spread(60, 200, 4, empty=0.5), [64, 128, 640, 65, 127, 1] * 4],
                         ids=lambda s: f"{sum(s)}-{len(s)}")
@pytest.mark.parametrize("fi,fo", [(1000, 1024), (1024, 776)])
@pytest.mark.parametrize("dtype,out", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("out_in", [False, True])
def test_gradients(cuda_device, sizes, fi, fo, dtype, out, out_in):
    assert sum(s > 0 for s in sizes) * (-(-fi // FEATURES)) * (-(-fo // FEATURES)) >= 4 * PAIRS
    check_grad_w(sizes, fi, fo, dtype, out_in, out, cuda_device, tail=70)
    no_wait_ran_out()


# ------------------------------------------------------------------ every launch of many
def every_launch(call, out, times):
    """The first result; the others have the same bits, each written over 9s."""
    out.fill_(9.0)
    call()
    first, differs = out.clone(), torch.zeros((), dtype=torch.bool, device=out.device)
    for _ in range(times):
        out.fill_(9.0)
        call()
        differs |= (out != first).any()
    assert not differs
    no_wait_ran_out()
    return first


def mostly_empty(groups, used, rows, seed):
    rng = random.Random(seed)
    sizes = [0] * groups
    for _ in range(rows):
        sizes[rng.randrange(used) * groups // used] += 1
    return sizes


@pytest.mark.parametrize("sizes", [mostly_empty(64, 64, 9, 1), mostly_empty(64, 20, 700, 2)], ids=lambda s: f"{sum(s)}-{len(s)}")
def test_gradient_every_launch(cuda_device, sizes):
    """Tiles that are mostly zeros."""
    groups, fi, fo, rows = len(sizes), 712, 1000, sum(sizes)
    g = gen(1, cuda_device)
    x, dy = (torch.randn(rows, f, generator=g, device=cuda_device).half() for f in (fi, fo))
    ptr, dw = pointers(sizes, cuda_device), torch.empty(groups * fi * fo, dtype=torch.float16, device=cuda_device)
    first = every_launch(lambda: ops.grouped_mm_grad_w(x.view(-1), dy.view(-1), dw, ptr, groups, fi, fo), dw, 1000).view(groups, fi, fo)
    at = 0
    for i, n in enumerate(sizes):
        a, b = x[at:at + n].double().t(), dy[at:at + n].double()
        near(first[i], a @ b, n * 2 * U * (a.abs() @ b.abs()), torch.float16)
        at += n


@pytest.mark.parametrize("sizes,n", [(mostly_empty(128, 9, 20000, 3), 256), (mostly_empty(300, 150, 4000, 4), 128), (mostly_empty(400, 2, 9000, 5), 128)],
                         ids=lambda s: f"{sum(s)}-{len(s)}" if isinstance(s, list) else str(s))
@pytest.mark.parametrize("fi,fo", [(64, 1024), (328, 520)])
def test_product_every_launch(cuda_device, sizes, n, fi, fo):
    """Groups are mostly empty, their tiles found by sums over 32 pointers at a time."""
    groups, rows = len(sizes), sum(sizes)
    used = min(groups, rows)
    assert (rows <= 128 * used) == (n == 128)
    g = gen(2, cuda_device)
    x, w = torch.randn(rows, fi, generator=g, device=cuda_device).half(), (torch.randn(groups, fi, fo, generator=g, device=cuda_device) / fi ** 0.5).half()
    ptr, y = pointers(sizes, cuda_device), torch.empty(rows * fo, dtype=torch.float16, device=cuda_device)
    first = every_launch(lambda: ops.grouped_mm(x.view(-1), w.view(-1), y, ptr, groups, fi, fo), y, 1000)
    want, mags = grouped_truth(x, w, sizes)
    near(first.view(rows, fo), want, fi * 2 * U * mags, torch.float16)
