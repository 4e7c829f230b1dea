"""How many bits the sums of products of 8-bit floating point keep inside one block of 128 of K, where they are formed by the tensor core.

2^16 and 2^-7 are the highest and the lowest bit of a number of 24 bits: f32 holds 2^16 + k 2^-7 for every k up to 2^23, so that no partial sum here
is rounded, in any order, and the results are exact.  Sums of fewer bits lose the small products."""
import pytest
import torch

from sparsetir_b200 import ops

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
PLACES = [(0, 1), (0, 31), (0, 32), (5, 127), (31, 30), (63, 64), (64, 63), (100, 6), (127, 0), (127, 126)]  # of the large product, of the small one
ROWS = [1, 12, 300]  # the kernels for few rows, with 8 and with 16 at a time, and for tiles
SMALL = 2.0 ** -7


def product(x, w):
    rows, fi = x.shape
    fo = len(w)
    y = torch.zeros(rows * fo, device=x.device)
    ops.grouped_mm_f8(x.to(F8).view(-1), torch.ones(-(-fi // 128) * rows, device=x.device), w.to(F8).view(-1),
                      torch.ones(-(-fo // 128) * -(-fi // 128), device=x.device), y, None, 1, fi, fo)
    return y


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("block", [0, 2])
def test_the_lowest_of_24_bits_is_kept(cuda_device, rows, block):
    fi, fo = 384, 40
    for large, small in PLACES:
        large, small = large + 128 * block, small + 128 * block
        other = 128 * block + (large - 128 * block + 7) % 128
        x, w = torch.zeros(rows, fi, device=cuda_device), torch.zeros(fo, fi, device=cuda_device)
        x[:, small], w[:, small] = 2.0 ** -4, 2.0 ** -3
        x[:, large], w[:, large] = 256.0, 256.0
        assert (product(x, w) == 2.0 ** 16 + SMALL).all(), (large, small)
        x[:, other], w[:, other] = -256.0, 256.0  # what is left when the large ones are gone
        assert other != small and (product(x, w) == SMALL).all(), (large, small)
        each = slice(128 * block, 128 * block + 128)
        x[:, each], w[:, each] = 2.0 ** -4, 2.0 ** -3
        x[:, large], w[:, large] = 256.0, 256.0
        assert (product(x, w) == 2.0 ** 16 + 127 * SMALL).all(), (large, small)


@pytest.mark.parametrize("rows", ROWS)
def test_of_a_gated_block(cuda_device, rows):
    """The other projection is 2^16 - 2^16 + 2^-7 and the gate 64, whose sigmoid is 1 but for 2^-92: y = 64 * 2^-7, off by the rounding to
    16 bits and by the (8 * 64 + 32) units of 2^-24 that the gate may be off, 2^-14: less than 2^-8 in all; 0 were the small product lost."""
    fi = width = 128
    for large, small in PLACES:
        other = (large + 7) % 128
        x, w = torch.zeros(rows, fi, device=cuda_device), torch.zeros(2 * width, fi, device=cuda_device)
        x[:, small], w[width:, small] = 2.0 ** -4, 2.0 ** -3
        x[:, large], w[width:, large] = 256.0, 256.0
        x[:, other], w[width:, other] = -256.0, 256.0
        w[:width, small] = 64.0  # times 2^-4 and its scale of 16
        y = torch.zeros(rows * width, dtype=torch.bfloat16, device=cuda_device)
        ops.grouped_mm_gated_f8(x.to(F8).view(-1), torch.ones(rows, device=cuda_device), w.to(F8).view(-1),
                                torch.tensor([16.0, 1.0], device=cuda_device), y, None, 1, fi, width)
        assert ((y.double() / (64 * SMALL) - 1).abs() <= 2.0 ** -8).all(), (large, small)
