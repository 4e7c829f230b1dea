"""Decoding batches whose rows meet in a few groups (grouped_mm, grouped_mm_i8)."""
import random

import pytest
import torch

from sparsetir_b200 import ops
from test_gpu_moe import check_grouped, check_i8, pointers

pytestmark = pytest.mark.gpu


def uneven(rows, groups, seed):
    """A batch in which a few groups have most of the rows, in the order of the groups or against it, with empty ones between."""
    rng = random.Random(seed)
    cuts = sorted(min(rows, int(rows * rng.random() ** 4)) for _ in range(groups - 1))
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    return sizes[::-1] if seed % 2 else sizes


# rows of a group around the 8 and 16 of one block, groups that begin and end at, before and behind their multiples
SIZES = [[0, 17, 0], [8, 9, 7, 8], [16, 17, 15, 16, 1], [7, 25, 0, 0, 32, 0], [0] * 15 + [120] + [0] * 16, [1] * 7 + [64] + [1] * 9,
         [3, 0, 90, 0, 0, 2, 1, 40], uneven(256, 64, 1), uneven(256, 64, 2), uneven(200, 40, 3), uneven(100, 70, 4), uneven(77, 10, 5)]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{sum(s)}-{len(s)}-{max(s)}")
@pytest.mark.parametrize("fi,fo", [(264, 72), (520, 257)])
@pytest.mark.parametrize("out_in", [False, True])
def test_rows_in_a_few_groups(cuda_device, sizes, fi, fo, out_in):
    check_grouped(sizes, fi, fo, torch.float16, out_in, torch.float32, cuda_device, tail=9)
    check_grouped(sizes, fi, fo, torch.bfloat16, out_in, torch.bfloat16, cuda_device)


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{sum(s)}-{len(s)}-{max(s)}")
@pytest.mark.parametrize("fi,fo", [(272, 72), (528, 257)])
def test_rows_in_a_few_groups_in_8_bits(cuda_device, sizes, fi, fo):
    check_i8(sizes, fi, fo, torch.float32, cuda_device, tail=9)


def time_of(sizes, fi, fo, device):
    rows, groups = sum(sizes), len(sizes)
    x, w = torch.randn(rows * fi, device=device).half(), torch.randn(groups * fi * fo, device=device).half()
    y, ptr = torch.zeros(rows * fo, device=device).half(), pointers(sizes, device)
    call = ops.grouped_mm.prepare(x, w, y, ptr, groups, fi, fo, ops.GROUPED_W_OUT_IN)
    best = []
    for _ in range(6):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(20):
            call()
        end.record()
        torch.cuda.synchronize()
        best.append(start.elapsed_time(end))
    return min(best[1:])


@pytest.mark.parametrize("hot", [64, 256])
def test_one_hot_group_does_not_hold_up_the_batch(cuda_device, hot):
    """256 rows in 64 groups, spread evenly and with 64 or all of them in one group.  The weights to be read are the same or
    fewer; when a group's blocks walked its rows 8 at a time the calls took 3.5 and 8.8 times as long."""
    even = [4] * 64
    uneven = [(256 - hot) // 63] * 30 + [hot] + [(256 - hot) // 63] * 33
    uneven[0] += 256 - sum(uneven)
    assert time_of(uneven, 2048, 1024, cuda_device) < 2 * time_of(even, 2048, 1024, cuda_device)
