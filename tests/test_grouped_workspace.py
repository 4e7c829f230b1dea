"""The scratch that `sparsetir_grouped_mm_workspace` answers covers the copies of operands that every product may make, asked with the flags
of the product's own call.  On the CPU: the query reads no device."""
import ctypes

import pytest

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops

GELU, OUT_IN = ops.GATED_GELU, ops.GROUPED_W_OUT_IN


def ask(*args):
    out = ctypes.c_size_t(0)
    assert L.load().sparsetir_grouped_mm_workspace(*args, ctypes.byref(out)) == 0, L.last_error()
    return out.value


def copy(rows, cols, element_bytes):
    """Rows of a multiple of 16 bytes, as many as make a multiple of 256."""
    return -(-(-(-cols * element_bytes // 16) * 16 * rows) // 256) * 256


SIZES = [(500, 64, 1001, 704), (500, 64, 1, 704), (3, 2, 7, 9), (700, 5, 203, 67), (1000, 8, 4099, 131), (1, 1, 1, 1)]


@pytest.mark.parametrize("rows,groups,feat_in,width", SIZES)
def test_gated_product(rows, groups, feat_in, width):
    """W is [groups, 2 * width, feat_in] whatever the flags."""
    need = copy(rows, feat_in, 2) + copy(groups * 2 * width, feat_in, 2)
    for flags in (0, GELU, OUT_IN):
        assert ask(rows, groups, feat_in, 2 * width, 2, flags) >= need
    need = copy(rows, feat_in, 1) + copy(groups * 2 * width, feat_in, 1)
    for flags in (0, GELU):
        assert ask(rows, groups, feat_in, 2 * width, 1, flags) >= need


@pytest.mark.parametrize("rows,groups,feat,width", SIZES)
def test_gradient(rows, groups, feat, width):
    for flags in (0, GELU, OUT_IN, GELU | OUT_IN):
        rows_of_w, cols = (width, feat) if flags & OUT_IN else (feat, width)
        assert ask(rows, groups, feat, width, 2, flags) >= copy(rows, feat, 2) + copy(groups * rows_of_w, cols, 2)


def test_the_size_that_was_too_small():
    assert copy(500, 1001, 2) + copy(64 * 2 * 704, 1001, 2) == 182_673_920
    assert ask(500, 64, 1001, 2 * 704, 2, 0) >= 182_673_920


@pytest.mark.parametrize("element_bytes", [1, 2])
def test_flags_that_no_product_has_are_refused(element_bytes):
    out = ctypes.c_size_t(0)
    for flags in (4, 8, -1):
        assert L.load().sparsetir_grouped_mm_workspace(4, 2, 8, 8, element_bytes, flags, ctypes.byref(out)) == -1
        assert f"unknown flags {flags}" in L.last_error()
