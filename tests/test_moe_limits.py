"""Sizes at the end of 32 bits: kernels round them up to whole tiles and steps, so that those without room for it are refused."""
import ctypes

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops

LARGEST = 2 ** 31 - 1 - 4096  # of any size


def refused(match, name, *args):
    assert getattr(L.load(), name)(*args) == -1
    assert match in L.last_error(), L.last_error()


@pytest.mark.parametrize("at", ["rows", "num_groups", "feat_in", "feat_out"])
def test_sizes_of_products(at):
    for n, match in ((LARGEST, "null pointer"), (LARGEST + 1, "too large"), (2 ** 31 - 1, "too large")):
        size = dict(rows=4, num_groups=1, feat_in=8, feat_out=8)
        size[at] = n
        r, g, fi, fo = size.values()
        ptr = ctypes.c_void_p(0x1000)  # of the row pointers: never read
        refused(match, "sparsetir_grouped_mm_raw", None, None, 1, None, 1, ptr, r, g, fi, fo, 0, 0, None)
        refused(match, "sparsetir_grouped_mm_grad_w_raw", None, None, 1, None, 1, ptr, r, g, fi, fo, 0, 0, None)
        if at != "feat_in":  # 131,071 at most
            refused(match, "sparsetir_grouped_mm_i8_raw", None, None, None, None, None, 0, ptr, r, g, fi, fo, 0, None)


def test_weights_beyond_64_bits():
    ptr = ctypes.c_void_p(0x1000)
    n = 2 ** 30
    refused("too large", "sparsetir_grouped_mm_raw", None, None, 1, None, 1, ptr, 4, n, n, n, 0, 0, None)
    refused("too large", "sparsetir_grouped_mm_grad_w_raw", None, None, 1, None, 1, ptr, 4, n, n, n, 0, 0, None)


def test_scratch_query():
    out = ctypes.c_size_t(0)
    for sizes in ((2 ** 31 - 1, 1, 8, 8), (4, 2 ** 31 - 1, 8, 8), (4, 1, 8, 2 ** 31 - 1), (4, 2 ** 30, 2 ** 30, 2 ** 30)):
        refused("too large", "sparsetir_grouped_mm_workspace", *sizes, 2, 0, ctypes.byref(out))


@pytest.mark.parametrize("at", ["tokens", "rows", "feat"])
def test_sizes_of_rows(at):
    for n, match in ((LARGEST, "null pointer"), (LARGEST + 1, "too large"), (2 ** 31 - 1, "too large")):
        t, r, f = (n if at == name else 4 for name in ("tokens", "rows", "feat"))
        refused(match, "sparsetir_moe_dispatch_raw", None, None, None, 1, t, r, f, 1, 0, None)
        refused(match, "sparsetir_moe_dispatch_i8_raw", None, 1, ctypes.c_void_p(0x1000), None, None, t, r, f, 1, 0, None)
        refused(match, "sparsetir_moe_combine_raw", None, 1, None, None, None, 1, t, r, f, 1, 0, None)
        refused(match, "sparsetir_moe_combine_grad_raw", None, None, 1, None, None, None, None, t, r, f, 1, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_row_of_2_gigabytes(cuda_device, dtype):
    """The bytes of the depth pass 31 bits.  Zeros but for a few small whole numbers, from the first element to the last: the
    sum is exact."""
    fi = 2 ** 30 + 64
    at = torch.tensor([0, 1, 63, 64, 4097, 2 ** 28 + 5, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 77, 2 ** 30 - 1, 2 ** 30, fi - 2, fi - 1], device=cuda_device)
    x, w = (torch.zeros(fi, dtype=dtype, device=cuda_device) for _ in range(2))
    a = torch.arange(1, len(at) + 1, device=cuda_device)
    x[at], w[at] = a.to(dtype), (2 * a - 7).to(dtype)
    w[at[3] + 1], x[at[5] + 1] = 9.0, 9.0  # of one operand alone
    y = torch.full((1,), 7.0, device=cuda_device)
    ops.grouped_mm(x, w, y, None, 1, fi, 1, ops.GROUPED_W_OUT_IN)
    assert int(y) == int((a * (2 * a - 7)).sum())
