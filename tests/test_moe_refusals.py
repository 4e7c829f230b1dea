"""What the operators of a mixture-of-experts layer refuse, with the messages of the argument checks.  No device work:
every call is rejected before any CUDA call."""
import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import ops
from test_abi import _fake_cuda, f16, f32, i32
from test_pycall import record


def bf16(n, **kw):
    return _fake_cuda(n, L.kDLBfloat, 16, **kw)


def i8(n, **kw):
    return _fake_cuda(n, L.kDLInt, 8, **kw)


def refused(match, fn, *args):
    with pytest.raises(ops.SparseTIRError, match=match):
        fn(*args)


def test_tensors_of_more_types_reach_the_new_operators_alone():
    for dtype, name in ((torch.bfloat16, "bfloat16"), (torch.int8, "int8")):
        t = torch.zeros(4, dtype=dtype)
        assert record((t,)) == (None, [])
        with pytest.raises(TypeError, match=name):
            ops.csrmm(t)
        with pytest.raises(TypeError, match=name):
            ops.csrmm.prepare(t)
    refused("no CPU path", ops.grouped_mm, *[torch.zeros(4, dtype=torch.bfloat16)] * 3, torch.zeros(2, dtype=torch.int32), 1, 2, 2)
    refused("no CPU path", ops.grouped_mm.prepare(*[torch.zeros(4, dtype=torch.bfloat16)] * 3, None, 1, 2, 2))
    refused("no CPU path", ops.grouped_mm_i8, torch.zeros(4, dtype=torch.int8), *[torch.zeros(2)] * 5, 1, 2, 2)


@pytest.mark.parametrize("fn,nargs", [(ops.moe_route, 6), (ops.moe_route_grad, 9), (ops.moe_dispatch, 6), (ops.moe_dispatch_i8, 5),
                                      (ops.moe_combine, 5), (ops.moe_combine_grad, 7), (ops.grouped_mm, 6), (ops.grouped_mm_grad_w, 9),
                                      (ops.grouped_mm_i8, 8)])
def test_wrong_argument_count(fn, nargs):
    refused("num_args should be", fn, *[torch.zeros(2)] * nargs)


def test_router():
    good = lambda t=3, e=8, k=2: [f32(t * e), f32(t * k), i32(t * k), i32(t * k), i32(e + 1), e, k]  # noqa: E731
    with_ = lambda i, v, **kw: [v if j == i else a for j, a in enumerate(good(**kw))]  # noqa: E731
    refused("logits.dtype is expected to be float32 float16 bfloat16", ops.moe_route, *with_(0, i32(24)))
    refused("gates.dtype is expected to be float32", ops.moe_route, *with_(1, f16(6)))
    refused("not a multiple of 8 features", ops.moe_route, *with_(0, f32(25)))
    refused("gates.shape", ops.moe_route, *with_(1, f32(5)))
    refused("experts.shape", ops.moe_route, *with_(2, i32(7)))
    refused("slots.shape", ops.moe_route, *with_(3, i32(7)))
    refused("indptr.shape", ops.moe_route, *with_(4, i32(8)))
    refused("num_experts = 0", ops.moe_route, *with_(5, 0))
    refused("num_experts = 1025", ops.moe_route, *good(e=1025))
    refused("top_k = 0", ops.moe_route, *with_(6, 0))
    refused("top_k = 33", ops.moe_route, *good(e=64, k=33))
    refused("top_k = 9 exceeds num_experts = 8", ops.moe_route, *good(k=9))
    refused("unknown flags 2", ops.moe_route, *good(), 2)
    refused("to be int", ops.moe_route, *with_(6, 2.0))
    refused("device_id", ops.moe_route, *with_(3, i32(6, device_id=1)))
    refused("compact", ops.moe_route, *with_(0, f32(24, strides=[2])))
    grad = lambda: [bf16(24), f32(6), i32(6), f32(6), bf16(24), 8, 2]  # noqa: E731
    refused("d_logits.dtype is expected to be bfloat16, got", ops.moe_route_grad, *grad()[:4], f32(24), 8, 2)
    refused("d_logits.shape", ops.moe_route_grad, *grad()[:4], bf16(32), 8, 2)
    refused("d_gates.shape", ops.moe_route_grad, *grad()[:3], f32(7), *grad()[4:])


def test_rows():
    refused("x.dtype is expected to be float32 float16 bfloat16", ops.moe_dispatch, i8(16), i32(4), i8(32), 8, 2)
    refused("z.dtype is expected to be float16, got", ops.moe_dispatch, f16(16), i32(4), bf16(32), 8, 2)
    refused("len\\(x\\) = 17 is not a multiple of 8", ops.moe_dispatch, f16(17), i32(4), f16(32), 8, 2)
    refused("len\\(z\\) = 33 is not a multiple of 8", ops.moe_dispatch, f16(16), i32(4), f16(33), 8, 2)
    refused("slots.shape", ops.moe_dispatch, f16(16), i32(5), f16(32), 8, 2)
    refused("features must be positive", ops.moe_dispatch, f16(16), i32(4), f16(32), 0, 2)
    refused("top_k = 33", ops.moe_dispatch, f16(16), i32(66), f16(32), 8, 33)
    refused("slots is a null handle", ops.moe_dispatch, f16(16), None, f16(32), 8, 2)
    refused("q.dtype is expected to be int8", ops.moe_dispatch_i8, f16(16), i32(4), f16(32), f32(4), 8, 2)
    refused("scale.shape", ops.moe_dispatch_i8, f16(16), i32(4), i8(32), f32(5), 8, 2)
    refused("null with top_k 1 only", ops.moe_dispatch_i8, f16(16), None, i8(32), f32(4), 8, 2)
    refused("q.shape", ops.moe_dispatch_i8, f16(16), None, i8(32), f32(4), 8, 1)
    refused("y.dtype is expected to be float32 bfloat16, got", ops.moe_combine, bf16(32), i32(4), f32(4), f16(16), 8, 2)
    refused("gates.shape", ops.moe_combine, bf16(32), i32(4), f32(5), bf16(16), 8, 2)
    refused("slots.shape", ops.moe_combine, bf16(32), i32(4), None, bf16(24), 8, 2)
    refused("z.dtype is expected to be float16, got", ops.moe_combine_grad, f16(16), f32(32), i32(4), f32(4), f16(32), f32(4), 8, 2)
    refused("dz.shape", ops.moe_combine_grad, f16(16), f16(32), i32(4), f32(4), f16(40), f32(4), 8, 2)
    refused("gates is a null handle", ops.moe_combine_grad, f16(16), f16(32), i32(4), None, f16(32), f32(4), 8, 2)


def test_grouped_products():
    good = lambda: [f16(5 * 8), f16(3 * 8 * 4), f16(5 * 4), i32(4), 3, 8, 4]  # noqa: E731
    with_ = lambda i, v: [v if j == i else a for j, a in enumerate(good())]  # noqa: E731
    for fn in (ops.grouped_mm, ops.grouped_mm_grad_w):
        refused("x.dtype is expected to be float16 bfloat16", fn, *with_(0, f32(40)))
        refused("indptr.shape", fn, *with_(3, i32(5)))
        refused("null with num_groups 1 only", fn, *with_(3, None))
        refused("must be positive", fn, *with_(5, 0))
        refused("num_groups = -1 does not fit", fn, *with_(4, -1))
        refused("feat_out = 3000000000 does not fit", fn, *with_(6, 3_000_000_000))
        refused("unknown flags 6", fn, *good(), 6)
        refused("not a multiple of 8 features", fn, *with_(0, f16(41)))
    refused("w.dtype is expected to be float16, got", ops.grouped_mm, *with_(1, bf16(96)))
    refused("y.dtype is expected to be float32 float16, got", ops.grouped_mm, *with_(2, bf16(20)))
    refused("w.shape", ops.grouped_mm, *with_(1, f16(97)))
    refused("y.shape", ops.grouped_mm, *with_(2, f16(24)))
    refused("w is too large", ops.grouped_mm, f16(0), f16(96), f16(0), i32(2_000_000_001), 2_000_000_000, 2_000_000_000,
            2_000_000_000)
    refused("dy.shape", ops.grouped_mm_grad_w, f16(40), f16(24), f16(96), i32(4), 3, 8, 4)
    refused("dw.shape", ops.grouped_mm_grad_w, f16(40), f16(20), f16(97), i32(4), 3, 8, 4)
    refused("dw.dtype is expected to be float32 float16, got", ops.grouped_mm_grad_w, f16(40), f16(20), bf16(96), i32(4), 3, 8, 4)
    int8 = lambda: [i8(40), f32(5), i8(96), f32(12), bf16(20), i32(4), 3, 8, 4]  # noqa: E731
    q = lambda i, v: [v if j == i else a for j, a in enumerate(int8())]  # noqa: E731
    refused("x.dtype is expected to be int8", ops.grouped_mm_i8, *q(0, _fake_cuda(40, L.kDLUInt, 8)))
    refused("x_scale.shape", ops.grouped_mm_i8, *q(1, f32(6)))
    refused("w_scale.shape", ops.grouped_mm_i8, *q(3, f32(3)))
    refused("w.shape", ops.grouped_mm_i8, *q(2, i8(95)))
    refused("y.dtype is expected to be float32 float16 bfloat16", ops.grouped_mm_i8, *q(4, i8(20)))
    refused("may not fit 32 bits", ops.grouped_mm_i8, i8(131072), f32(1), i8(131072), f32(1), f32(1), i32(2), 1, 131072, 1)


def test_plain_pointer_forms():
    lib = L.load()

    def raw(match, name, *args):
        assert getattr(lib, name)(*args) == -1
        assert match in L.last_error(), L.last_error()

    raw("null pointer", "sparsetir_grouped_mm_raw", None, None, 1, None, 1, None, 4, 1, 8, 8, 0, 0, None)
    raw("negative size", "sparsetir_grouped_mm_raw", None, None, 1, None, 1, None, -4, 1, 8, 8, 0, 0, None)
    raw("f16 or bf16", "sparsetir_grouped_mm_raw", None, None, 0, None, 0, None, 4, 1, 8, 8, 0, 0, None)
    raw("the type of x", "sparsetir_grouped_mm_raw", None, None, 1, None, 2, None, 4, 1, 8, 8, 0, 0, None)
    raw("num_groups 1 only", "sparsetir_grouped_mm_grad_w_raw", None, None, 1, None, 1, None, 4, 2, 8, 8, 0, 0, None)
    raw("unknown flags", "sparsetir_grouped_mm_grad_w_raw", None, None, 1, None, 1, None, 4, 1, 8, 8, 4, 0, None)
    raw("32 bits", "sparsetir_grouped_mm_i8_raw", None, None, None, None, None, 0, None, 4, 1, 1 << 17, 8, 0, None)
    raw("top_k = 0", "sparsetir_moe_dispatch_raw", None, None, None, 1, 4, 4, 8, 0, 0, None)
    raw("unknown element type", "sparsetir_moe_combine_raw", None, 5, None, None, None, 5, 4, 4, 8, 1, 0, None)
    raw("a row per token", "sparsetir_moe_dispatch_i8_raw", None, 1, None, None, None, 4, 5, 8, 1, 0, None)
    raw("num_experts = 3", "sparsetir_moe_route_raw", None, 0, None, None, None, None, 4, 3, 4, 0, 0, None)
    assert lib.sparsetir_grouped_mm_raw(None, None, 1, None, 1, None, 0, 1, 8, 8, 0, 0, None) == 0  # no rows: nothing to do


def test_scratch_queries():
    import ctypes

    out = ctypes.c_size_t(99)

    def ask(name, *sizes):
        assert getattr(L.load(), name)(*sizes, ctypes.byref(out)) == 0, L.last_error()
        return out.value

    assert ask("sparsetir_moe_route_workspace", 0, 8) == ask("sparsetir_moe_route_workspace", 32, 1024) == 0
    assert ask("sparsetir_moe_route_workspace", 33, 8) == 2 * 8 * 4
    assert ask("sparsetir_moe_route_workspace", 2 ** 31 - 1, 1024) <= 148 * 1024 * 4
    # copies at rows of a multiple of 16 bytes
    assert ask("sparsetir_grouped_mm_workspace", 100, 4, 9, 16, 2, 1) == 100 * 32 + 128 + max(4 * 16 * 32, 100 * 32 + 128)
    assert ask("sparsetir_grouped_mm_workspace", 100, 4, 17, 16, 1, 0) == 100 * 32 + 128 + 4 * 16 * 32
    assert ask("sparsetir_grouped_mm_workspace", 0, 4, 17, 16, 1, 0) == ask("sparsetir_grouped_mm_workspace", 4, 0, 17, 16, 2, 0) == 0
    # sums of units that share a tile: of the gradient, of the product; of no more units than run at a time
    assert ask("sparsetir_grouped_mm_workspace", 64000, 1, 256, 256, 2, 0) == 2 * 64000 * 512 + 74 * 256 * 256 * 4
    assert ask("sparsetir_grouped_mm_workspace", 300, 1, 4096, 256, 2, 1) == 300 * 8192 + 256 * 8192 + 16 * 300 * 256 * 4
    for rows in (1, 100, 10_000, 1_000_000):
        for sizes in ((1, 64, 64), (1, 4096, 64), (8, 512, 512), (64, 2048, 2048), (1, 100_000, 8)):
            copies = 2 * (rows * sizes[1] + max(sizes[0] * sizes[1] * sizes[2], rows * sizes[2])) + 512
            assert ask("sparsetir_grouped_mm_workspace", rows, *sizes, 2, 1) <= copies + (20 << 20)
    for name, sizes in (("sparsetir_moe_route_workspace", (-1, 8)), ("sparsetir_moe_route_workspace", (4, 0)),
                        ("sparsetir_grouped_mm_workspace", (4, 4, 0, 8, 2, 0)), ("sparsetir_grouped_mm_workspace", (4, 4, 8, 8, 3, 0))):
        assert getattr(L.load(), name)(*sizes, ctypes.byref(out)) == -1
