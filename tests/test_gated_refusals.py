"""What the gated products and those of 8-bit floating point refuse, and calls with nothing to do.  No device work: every call ends
before any CUDA call."""
import ctypes

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import moe, ops
from test_abi import _fake_cuda, f16, f32, i32
from test_moe_empty import empty
from test_moe_refusals import bf16, i8, refused

LARGEST = 2 ** 31 - 1 - 4096  # of any size


def f8(n, **kw):
    return _fake_cuda(n, L.kDLFloat8E4M3, 8, **kw)


def test_tensors_of_8_bit_floating_point_reach_the_new_operators_alone():
    t = torch.zeros(4, dtype=torch.float8_e4m3fn)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.csrmm(t)
    args = [t, torch.zeros(2), t, torch.zeros(1), torch.zeros(4, dtype=torch.float16), None, 1, 2, 2]
    refused("no CPU path", ops.grouped_mm_f8, *args)
    refused("no CPU path", ops.grouped_mm_f8.prepare(*args))
    with pytest.raises(TypeError, match="float8_e5m2"):
        ops.grouped_mm_f8(torch.zeros(4, dtype=torch.float8_e5m2), *args[1:])


@pytest.mark.parametrize("fn,nargs", [(ops.grouped_mm_gated, 7), (ops.grouped_mm_gated, 10), (ops.grouped_mm_gated_grad, 8),
                                      (ops.grouped_mm_gated_grad, 11), (ops.moe_dispatch_f8, 5), (ops.grouped_mm_f8, 8),
                                      (ops.grouped_mm_f8, 10), (ops.grouped_mm_gated_f8, 8), (ops.grouped_mm_gated_f8, 11)])
def test_wrong_argument_count(fn, nargs):
    refused("num_args should be", fn, *[torch.zeros(2)] * nargs)


def replaced(args, i, v):
    return [v if j == i else a for j, a in enumerate(args)]


def common(fn, good, indptr_at, of_x, size_names):
    """The groups of a product: row pointers, their number, two sizes."""
    refused("indptr.shape", fn, *replaced(good, indptr_at, i32(5)))
    refused("indptr.dtype is expected to be int32", fn, *replaced(good, indptr_at, f32(4)))
    refused("null with num_groups 1 only", fn, *replaced(good, indptr_at, None))
    refused("num_groups = -1 does not fit", fn, *replaced(good, indptr_at + 1, -1))
    refused("must be positive", fn, *replaced(good, indptr_at + 2, 0))
    refused(f"{size_names[0]} = 3000000000 does not fit", fn, *replaced(good, indptr_at + 2, 3_000_000_000))
    refused(f"{size_names[1]} = 3000000000 does not fit", fn, *replaced(good, indptr_at + 3, 3_000_000_000))
    refused("to be int", fn, *replaced(good, indptr_at + 3, 2.0))
    refused("not a multiple of 8 features", fn, *replaced(good, 0, of_x(41)))
    refused("device_id", fn, *replaced(good, 2, _fake_cuda(96, good[2].dtype.code, good[2].dtype.bits, device_id=1)))


def test_gated():
    good = [f16(5 * 8), f16(3 * 8 * 8), f16(5 * 4), f16(5 * 8), i32(4), 3, 8, 4]
    with_ = lambda i, v: replaced(good, i, v)  # noqa: E731
    common(ops.grouped_mm_gated, good, 4, f16, ("feat_in", "width"))
    refused("x.dtype is expected to be float16 bfloat16", ops.grouped_mm_gated, *with_(0, f32(40)))
    refused("w.dtype is expected to be float16, got", ops.grouped_mm_gated, *with_(1, bf16(192)))
    refused("w.shape", ops.grouped_mm_gated, *with_(1, f16(96)))
    refused("y.dtype is expected to be float16, got", ops.grouped_mm_gated, *with_(2, f32(20)))
    refused("y.shape", ops.grouped_mm_gated, *with_(2, f16(40)))
    refused("hidden.shape", ops.grouped_mm_gated, *with_(3, f16(20)))
    refused("hidden.dtype", ops.grouped_mm_gated, *with_(3, f32(40)))
    for flags in (1, 3, 4, -1):  # the layout of the weights is not to be chosen
        refused(f"unknown flags {flags}", ops.grouped_mm_gated, *good, flags)


def test_gated_grad():
    good = [bf16(5 * 8), bf16(3 * 8 * 4), bf16(5 * 8), bf16(5 * 8), bf16(5 * 4), i32(4), 3, 8, 4]
    with_ = lambda i, v: replaced(good, i, v)  # noqa: E731
    common(ops.grouped_mm_gated_grad, good, 5, bf16, ("feat", "width"))
    refused("dy.dtype is expected to be float16 bfloat16", ops.grouped_mm_gated_grad, *with_(0, f32(40)))
    refused("w.shape", ops.grouped_mm_gated_grad, *with_(1, bf16(192)))
    refused("hidden is a null handle", ops.grouped_mm_gated_grad, *with_(2, None))
    refused("hidden.shape", ops.grouped_mm_gated_grad, *with_(2, bf16(20)))
    refused("d_hidden.shape", ops.grouped_mm_gated_grad, *with_(3, bf16(41)))
    refused("d_hidden.dtype is expected to be bfloat16, got", ops.grouped_mm_gated_grad, *with_(3, f16(40)))
    refused("act.shape", ops.grouped_mm_gated_grad, *with_(4, bf16(40)))
    refused("unknown flags 4", ops.grouped_mm_gated_grad, *good, 4)


def test_dispatch_f8():
    good = [f16(2 * 136), i32(4), f8(4 * 136), f32(2 * 4), 136, 2]
    with_ = lambda i, v: replaced(good, i, v)  # noqa: E731
    refused("x.dtype is expected to be float32 float16 bfloat16", ops.moe_dispatch_f8, *with_(0, i8(272)))
    refused("slots.shape", ops.moe_dispatch_f8, *with_(1, i32(5)))
    refused("q.dtype is expected to be e4m3 float8", ops.moe_dispatch_f8, *with_(2, i8(4 * 136)))
    refused("scale.shape", ops.moe_dispatch_f8, *with_(3, f32(4)))
    refused("not a multiple of 136", ops.moe_dispatch_f8, *with_(2, f8(300)))
    refused("features must be positive", ops.moe_dispatch_f8, *with_(4, 0))
    refused("top_k = 33", ops.moe_dispatch_f8, *with_(5, 33))
    refused("null with top_k 1 only", ops.moe_dispatch_f8, *with_(1, None))
    refused("q.shape", ops.moe_dispatch_f8, f16(272), None, f8(4 * 136), f32(8), 136, 1)


def test_products_of_8_bit_floating_point():
    good = [f8(5 * 8), f32(5), f8(3 * 8 * 4), f32(3), bf16(5 * 4), i32(4), 3, 8, 4]
    with_ = lambda i, v: replaced(good, i, v)  # noqa: E731
    common(ops.grouped_mm_f8, good, 5, f8, ("feat_in", "feat_out"))
    refused("x.dtype is expected to be e4m3 float8", ops.grouped_mm_f8, *with_(0, i8(40)))
    refused("x_scale.shape", ops.grouped_mm_f8, *with_(1, f32(6)))
    refused("w.shape", ops.grouped_mm_f8, *with_(2, f8(95)))
    refused("w_scale.shape", ops.grouped_mm_f8, *with_(3, f32(12)))
    refused("y.dtype is expected to be float32 float16 bfloat16", ops.grouped_mm_f8, *with_(4, f8(20)))
    refused("y.shape", ops.grouped_mm_f8, *with_(4, bf16(21)))
    gated = [f8(5 * 8), f32(5), f8(3 * 8 * 8), f32(3), bf16(5 * 4), i32(4), 3, 8, 4]
    common(ops.grouped_mm_gated_f8, gated, 5, f8, ("feat_in", "width"))
    refused("y.dtype is expected to be float16 bfloat16", ops.grouped_mm_gated_f8, *replaced(gated, 4, f32(20)))
    refused("unknown flags 1", ops.grouped_mm_gated_f8, *gated, 1)
    # scales of 2 * width rows of weights in blocks of 128, not of width
    refused("w_scale.shape", ops.grouped_mm_gated_f8, f8(8), f32(1), f8(8 * 200), f32(1), bf16(100), None, 1, 8, 100)


def raw(match, name, *args):
    assert getattr(L.load(), name)(*args) == -1
    assert match in L.last_error(), L.last_error()


@pytest.mark.parametrize("at", ["rows", "num_groups", "feat_in", "width"])
def test_sizes_at_the_end_of_32_bits(at):
    ptr = ctypes.c_void_p(0x1000)  # of the row pointers: never read
    for n in (LARGEST, LARGEST + 1, 2 ** 31 - 1):
        size = dict(rows=4, num_groups=1, feat_in=8, width=8)
        size[at] = n
        r, g, fi, fo = size.values()
        match = "null pointer" if n == LARGEST else "too large"
        raw(match, "sparsetir_grouped_mm_f8_raw", None, None, None, None, None, 0, ptr, r, g, fi, fo, 0, None)
        if at == "width":
            match = "too large"
        raw(match, "sparsetir_grouped_mm_gated_raw", None, None, None, None, 1, ptr, r, g, fi, fo, 0, 0, None)
        raw(match, "sparsetir_grouped_mm_gated_grad_raw", None, None, None, None, None, 1, ptr, r, g, fi, fo, 0, 0, None)
        raw(match, "sparsetir_grouped_mm_gated_f8_raw", None, None, None, None, None, 1, ptr, r, g, fi, fo, 0, 0, None)
    raw("null pointer", "sparsetir_grouped_mm_gated_raw", None, None, None, None, 1, ptr, 4, 1, 8, LARGEST // 2, 0, 0, None)
    raw("too large", "sparsetir_grouped_mm_gated_raw", None, None, None, None, 1, ptr, 4, 2 ** 30, 2 ** 30, 2 ** 30 - 4096, 0, 0, None)


def test_plain_pointer_forms():
    ptr = ctypes.c_void_p(0x1000)
    raw("negative size", "sparsetir_grouped_mm_gated_raw", None, None, None, None, 1, None, -4, 1, 8, 8, 0, 0, None)
    raw("f16 or bf16", "sparsetir_grouped_mm_gated_raw", ptr, ptr, ptr, None, 0, None, 4, 1, 8, 8, 0, 0, None)
    raw("unknown flags", "sparsetir_grouped_mm_gated_raw", ptr, ptr, ptr, None, 1, None, 4, 1, 8, 8, 1, 0, None)
    raw("num_groups 1 only", "sparsetir_grouped_mm_gated_raw", ptr, ptr, ptr, None, 1, None, 4, 2, 8, 8, 0, 0, None)
    raw("null pointer", "sparsetir_grouped_mm_gated_grad_raw", ptr, ptr, None, ptr, None, 1, None, 4, 1, 8, 8, 0, 0, None)
    raw("f16 or bf16", "sparsetir_grouped_mm_gated_grad_raw", ptr, ptr, ptr, ptr, None, 3, None, 4, 1, 8, 8, 0, 0, None)
    raw("unknown element type", "sparsetir_grouped_mm_f8_raw", ptr, ptr, ptr, ptr, ptr, 3, None, 4, 1, 8, 8, 0, None)
    raw("f16 or bf16", "sparsetir_grouped_mm_gated_f8_raw", ptr, ptr, ptr, ptr, ptr, 0, None, 4, 1, 8, 8, 0, 0, None)
    raw("a row per token", "sparsetir_moe_dispatch_f8_raw", None, 1, None, None, None, 4, 5, 8, 1, 0, None)
    raw("a row per token", "sparsetir_moe_dispatch_f8_raw", None, 1, None, None, None, 4, 8, 8, 2, 0, None)
    raw("null pointer", "sparsetir_moe_dispatch_f8_raw", None, 1, ptr, None, None, 4, 8, 8, 2, 0, None)
    for n in (LARGEST + 1, 2 ** 31 - 1):
        raw("too large", "sparsetir_moe_dispatch_f8_raw", None, 1, ptr, None, None, n, 4, 8, 1, 0, None)
        raw("too large", "sparsetir_moe_dispatch_f8_raw", None, 1, ptr, None, None, 4, n, 8, 1, 0, None)
        raw("too large", "sparsetir_moe_dispatch_f8_raw", None, 1, ptr, None, None, 4, 4, n, 1, 0, None)


def test_nothing_to_do():
    half, one, ints, eight = (lambda: empty(L.kDLFloat, 16)), (lambda: empty(L.kDLFloat, 32)), (lambda: i32(4)), (lambda: empty(L.kDLFloat8E4M3, 8))
    ops.grouped_mm_gated(half(), f16(3 * 16 * 8), half(), half(), ints(), 3, 8, 8)
    ops.grouped_mm_gated(half(), f16(3 * 16 * 8), half(), None, ints(), 3, 8, 8)
    ops.grouped_mm_gated_grad(half(), f16(3 * 8 * 8), half(), half(), None, ints(), 3, 8, 8)
    ops.grouped_mm_f8(eight(), one(), f8(3 * 8 * 4), f32(3), half(), ints(), 3, 8, 4)
    ops.grouped_mm_gated_f8(eight(), one(), f8(3 * 8 * 8), f32(3), half(), ints(), 3, 8, 4)
    for k in (1, 2, 32):
        ops.moe_dispatch_f8(half(), empty(L.kDLInt, 32), eight(), one(), 8, k)
    ops.moe_dispatch_f8(half(), None, eight(), one(), 8, 1)
    # rows but no groups: rows of no group, which nothing is written to
    ops.grouped_mm_gated(f16(16), empty(L.kDLFloat, 16), f16(16), None, i32(1), 0, 8, 8)
    ops.grouped_mm_f8(f8(16), f32(2), eight(), one(), f16(8), i32(1), 0, 8, 4)


def test_layers():
    router, gate_up, down = torch.zeros(4, 8), torch.zeros(4, 6, 8).half(), torch.zeros(4, 8, 3).half()
    with pytest.raises(ValueError, match="gated must be None or one of \\['gelu', 'silu'\\], got 'relu'"):
        moe.ExpertLayer(router, gate_up, down, 2, gated="relu")
    with pytest.raises(ValueError, match='kind must be "int8" or "float8"'):
        moe.ExpertLayer(router, gate_up, down, 2).quantized("float16")


@pytest.mark.parametrize("out,features", [(1, 1), (128, 128), (129, 127), (300, 520)])
def test_weights_in_blocks(out, features):
    """Each 128 x 128 has its own scale, its largest value becomes 448, and none is off by more than half a step: 2^-4 of it, or half
    of the smallest number, 2^-10, times the scale (and the rounding of the scale and of the quotient, 2^-22)."""
    w = torch.randn(2, out, features, generator=torch.Generator().manual_seed(out)).half()
    w[0, : out // 2] = 0
    w *= torch.exp(3 * torch.randn(2, out, 1, generator=torch.Generator().manual_seed(1))).half()
    q, scale = moe.quantize_blocks(w)
    rb, cb = -(-out // 128), -(-features // 128)
    assert q.shape == w.shape and q.dtype == torch.float8_e4m3fn and scale.shape == (2, rb, cb)
    for b in range(2):
        for i in range(rb):
            for j in range(cb):
                part = w[b, 128 * i:128 * i + 128, 128 * j:128 * j + 128].double()
                got = q[b, 128 * i:128 * i + 128, 128 * j:128 * j + 128].double() * float(scale[b, i, j])
                assert abs(float(part.abs().max()) / 448 - float(scale[b, i, j])) <= 2.0 ** -24 * float(part.abs().max())
                assert ((got - part).abs() <= 2.0 ** -4 * part.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * float(scale[b, i, j]) * (1 + 2.0 ** -20)).all()
