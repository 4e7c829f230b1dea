"""The mixture-of-experts layer that runs the operators together, against torch's own automatic differentiation in 64 bits.

Tolerances, of the 2-norm: a 16-bit tensor carries its rounding u (2^-11 for float16, 2^-8 for bfloat16, relative and in the worst case), and
a result behind n roundings of 16-bit tensors, each met by sums of independent errors, n u of its norm at most.  The result
passes three (hidden, act, out) and its own, the gradients of the weights up to seven: forward's three, d_out, d_act, d_hidden and their own."""
import pytest
import torch
import torch.nn.functional as F

from sparsetir_b200 import moe, ops

pytestmark = pytest.mark.gpu


def make(tokens, experts, features, width, top_k, dtype, renormalize, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    layer = moe.ExpertLayer(rand(experts, features) * 0.1, (rand(experts, 2 * width, features) / features ** 0.5).to(dtype),
                            (rand(experts, features, width) / width ** 0.5).to(dtype), top_k, renormalize)
    return layer, rand(tokens, features).to(dtype), rand(tokens, features).to(dtype)


def reference(layer, x, dy, padding, experts_of):
    """Result and gradients in 64 bits, with the choice of experts as the layer made it."""
    leaf = lambda t: t.double().requires_grad_(True)  # noqa: E731
    x, router, gate_up, down = leaf(x), leaf(layer.router), leaf(layer.gate_up), leaf(layer.down)
    p = torch.softmax(x @ router.t(), 1)
    kept = experts_of >= 0
    gates = torch.gather(p, 1, experts_of.clamp(min=0).long()) * kept
    if layer.renormalize:
        gates = gates / gates.sum(1, keepdim=True).clamp(min=1e-300)
    y = torch.zeros_like(x)
    for e in range(layer.experts):
        h = x @ gate_up[e].t()
        out = (F.silu(h[:, :layer.width]) * h[:, layer.width:]) @ down[e].t()
        y = y + (gates * (experts_of == e)).sum(1, keepdim=True) * out
    y.backward(dy.double())
    return y.detach(), {"x": x.grad, "router": router.grad, "gate_up": gate_up.grad, "down": down.grad}


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("tokens,experts,features,width,top_k", [(1, 4, 64, 32, 2), (24, 8, 96, 40, 3), (300, 16, 128, 72, 4),
                                                                 (1000, 6, 264, 136, 1)])
@pytest.mark.parametrize("dtype,u", [(torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)])
@pytest.mark.parametrize("renormalize", [False, True])
def test_result_and_gradients(cuda_device, tokens, experts, features, width, top_k, dtype, u, renormalize):
    layer, x, dy = make(tokens, experts, features, width, top_k, dtype, renormalize, cuda_device)
    padding = torch.zeros(tokens, dtype=torch.bool, device=cuda_device)
    padding[tokens // 2 + 1::3] = True
    y, saved = layer.forward(x, padding)
    assert (saved.routing.experts[padding] == -1).all() and (y[padding] == 0).all()
    grads = layer.backward(dy, saved)
    want, want_grads = reference(layer, x, dy, padding, saved.routing.experts)
    assert off(y, want) <= 4 * u
    for name, g in grads.items():
        assert g.shape == want_grads[name].shape
        if name == "router" and renormalize and top_k == 1:
            assert (g == 0).all()  # the only gate is 1 whatever the logits: the reference has its own rounding here
        else:
            assert off(g, want_grads[name]) <= 8 * u, name
    used = torch.bincount(saved.routing.experts[saved.routing.experts >= 0].long(), minlength=experts) > 0
    assert (grads["down"][~used] == 0).all() and (grads["gate_up"][~used] == 0).all()


def test_8_bit_layer(cuda_device):
    """A row's quantisation moves each value by half a step of max / 127 at most, 1 / 508 of the largest; of normal values whose
    largest is about 3.5 deviations that is an error of 3.5 / (127 sqrt(12)) = 0.8 % of the norm per tensor.  Four
    tensors of the result are quantised, two of them products of two: 3 % in all, and twice that is allowed."""
    for tokens in (3, 200):
        layer, x, _ = make(tokens, 8, 512, 256, 2, torch.bfloat16, True, cuda_device, seed=tokens)
        q = layer.quantized()
        assert off(q(x), layer(x).double()) <= 0.06


def test_step_in_a_graph(cuda_device):
    """A captured step follows the routing of new inputs, whose groups have other sizes."""
    layer, x, dy = make(200, 8, 128, 64, 2, torch.bfloat16, False, cuda_device)
    other = make(200, 8, 128, 64, 2, torch.bfloat16, False, cuda_device, seed=1)[1]
    held = x.clone()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            y, saved = layer.forward(held)
            grads = layer.backward(dy, saved)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, saved = layer.forward(held)
            grads = layer.backward(dy, saved)
    torch.cuda.current_stream().wait_stream(side)
    for inputs in (other, x):
        held.copy_(inputs)
        graph.replay()
        want, want_saved = layer.forward(inputs)
        want_grads = layer.backward(dy, want_saved)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(grads[k], want_grads[k]) for k in grads)


def test_refusals(cuda_device):
    layer, x, _ = make(8, 4, 64, 32, 2, torch.float16, False, cuda_device)
    with pytest.raises(ValueError, match="contiguous \\[tokens, 64\\]"):
        layer(x[:, ::2])
    with pytest.raises(ValueError, match="gate_up must be"):
        moe.ExpertLayer(layer.router, layer.gate_up[:, :-1], layer.down, 2)
    with pytest.raises(ops.SparseTIRError, match="float16, got"):
        layer(x.bfloat16())
