"""Batches without tokens through the operators of a mixture-of-experts layer: an empty tensor has a null pointer, which is
not an absent argument."""
import ctypes

import pytest
import torch

from sparsetir_b200 import _lib as L
from sparsetir_b200 import moe, ops
from test_abi import _fake_cuda


def empty(code, bits):
    t = _fake_cuda(0, code, bits)
    t.data = ctypes.c_void_p(None)  # as torch has it
    return t


@pytest.mark.parametrize("top_k", [1, 2, 32])
def test_operators_without_tokens(top_k):
    """Nothing to do, and no CUDA call: whatever the number of choices."""
    f16, f32, i32, i8 = (lambda: empty(L.kDLFloat, 16)), (lambda: empty(L.kDLFloat, 32)), (lambda: empty(L.kDLInt, 32)), (lambda: empty(L.kDLInt, 8))
    ops.moe_route_grad(f32(), f32(), i32(), f32(), f32(), 40, top_k)
    ops.moe_dispatch(f16(), i32(), f16(), 8, top_k)
    ops.moe_dispatch_i8(f16(), i32(), i8(), f32(), 8, top_k)
    ops.moe_combine(f16(), i32(), f32(), f16(), 8, top_k)
    ops.moe_combine(f16(), i32(), None, f32(), 8, top_k)
    ops.moe_combine_grad(f16(), f16(), i32(), f32(), f16(), f32(), 8, top_k)
    w = _fake_cuda(3 * 8 * 4, L.kDLFloat, 16)
    ops.grouped_mm(f16(), w, f16(), _fake_cuda(4, L.kDLInt, 32), 3, 8, 4)
    ops.grouped_mm_i8(i8(), f32(), _fake_cuda(3 * 8 * 4, L.kDLInt, 8), _fake_cuda(12, L.kDLFloat, 32), f16(),
                      _fake_cuda(4, L.kDLInt, 32), 3, 8, 4)


def test_what_is_absent_is_still_refused():
    one = lambda: _fake_cuda(8, L.kDLFloat, 16)  # noqa: E731
    with pytest.raises(ops.SparseTIRError, match="null with top_k 1 only"):
        ops.moe_dispatch_i8(one(), None, _fake_cuda(16, L.kDLInt, 8), _fake_cuda(2, L.kDLFloat, 32), 8, 2)
    lib = L.load()
    assert lib.sparsetir_moe_dispatch_i8_raw(None, 1, None, None, None, 4, 5, 8, 1, 0, None) == -1
    assert "a row per token" in L.last_error()
    assert lib.sparsetir_moe_dispatch_i8_raw(None, 1, None, None, None, 4, 8, 8, 2, 0, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("top_k", [1, 3])
@pytest.mark.parametrize("renormalize", [False, True])
def test_layers_without_tokens(cuda_device, top_k, renormalize):
    g = torch.Generator(device=cuda_device).manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device)  # noqa: E731
    layer = moe.ExpertLayer(rand(5, 64), rand(5, 80, 64).half(), rand(5, 64, 40).half(), top_k, renormalize)
    x = rand(0, 64).half()
    for padding in (None, torch.zeros(0, dtype=torch.bool, device=cuda_device)):
        y, saved = layer.forward(x, padding)
        assert y.shape == (0, 64) and saved.routing.indptr.tolist() == [0] * 6
        grads = layer.backward(x, saved)
        assert grads["x"].shape == (0, 64)
        assert all((grads[n] == 0).all() for n in ("router", "gate_up", "down"))
        assert layer.quantized()(x, padding).shape == (0, 64)
