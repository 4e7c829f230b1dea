"""The mixture-of-experts layer with its gated block as one operator, and in 8-bit floating point, as a program runs them: a training
step and a serving step, against torch's automatic differentiation in 64 bits and against the layer itself.

Tolerances as in test_gpu_moe_layer.py: the gated block rounds once where the passes round twice, so the bounds there hold here."""
import pytest
import torch
import torch.nn.functional as F

from sparsetir_b200 import moe
from test_gpu_moe_layer import off

pytestmark = pytest.mark.gpu


def make(tokens, experts, features, width, top_k, dtype, device, gated="silu", renormalize=False, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    layer = moe.ExpertLayer(rand(experts, features) * 0.1, (rand(experts, 2 * width, features) / features ** 0.5).to(dtype),
                            (rand(experts, features, width) / width ** 0.5).to(dtype), top_k, renormalize, gated=gated)
    return layer, rand(tokens, features).to(dtype), rand(tokens, features).to(dtype)


def activation(x, name):
    return F.gelu(x, approximate="tanh") if name == "gelu" else F.silu(x)


def reference(layer, x, dy, experts_of):
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
        out = (activation(h[:, :layer.width], layer.gated) * h[:, layer.width:]) @ down[e].t()
        y = y + (gates * (experts_of == e)).sum(1, keepdim=True) * out
    y.backward(dy.double())
    return y.detach(), {"x": x.grad, "router": router.grad, "gate_up": gate_up.grad, "down": down.grad}


@pytest.mark.parametrize("tokens,experts,features,width,top_k", [(1, 4, 64, 32, 2), (24, 8, 96, 40, 3), (300, 16, 128, 72, 4),
                                                                 (1000, 6, 264, 136, 2), (40, 5, 77, 33, 2)])
@pytest.mark.parametrize("dtype,u", [(torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)])
@pytest.mark.parametrize("gated", ["silu", "gelu"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_result_and_gradients(cuda_device, tokens, experts, features, width, top_k, dtype, u, gated, renormalize):
    layer, x, dy = make(tokens, experts, features, width, top_k, dtype, cuda_device, gated, renormalize)
    padding = torch.zeros(tokens, dtype=torch.bool, device=cuda_device)
    padding[tokens // 2 + 1::3] = True
    y, saved = layer.forward(x, padding)
    assert saved.act is None and (y[padding] == 0).all()
    assert torch.equal(layer(x, padding), y)  # without what the gradient needs
    grads = layer.backward(dy, saved)
    want, want_grads = reference(layer, x, dy, saved.routing.experts)
    assert off(y, want) <= 4 * u
    for name, g in grads.items():
        assert g.shape == want_grads[name].shape
        assert off(g, want_grads[name]) <= 8 * u, name
    used = torch.bincount(saved.routing.experts[saved.routing.experts >= 0].long(), minlength=experts) > 0
    assert (grads["down"][~used] == 0).all() and (grads["gate_up"][~used] == 0).all()


@pytest.mark.parametrize("gated", [None, "silu", "gelu"])
@pytest.mark.parametrize("tokens,features,width", [(3, 512, 256), (200, 512, 256), (70, 200, 136)])
def test_8_bit_floating_point(cuda_device, gated, tokens, features, width):
    """A number of 4 bits' fraction (3 stored) is off by 2^-4 of it at most, and by 2^-4 / sqrt(3) / 1.4 = 2.6 % of the norm on
    average over the fractions.  Four tensors of the result are quantised, in two products one after the other: sqrt(4) * 2.6 % = 5.2 %
    of independent errors, and twice that is allowed."""
    layer, x, _ = make(tokens, 8, features, width, 2, torch.bfloat16, cuda_device, gated, True, seed=tokens)
    q = layer.quantized("float8")
    assert off(q(x), layer(x).double()) <= 0.104


def test_8_bit_integers_take_the_activation_of_the_layer(cuda_device):
    layer, x, _ = make(60, 8, 512, 256, 2, torch.bfloat16, cuda_device, "gelu", True)
    assert off(layer.quantized()(x), layer(x).double()) <= 0.06


def test_default_layer_is_unchanged(cuda_device):
    """Without `gated` the block runs in passes: the same bits as from the operators called one by one."""
    from sparsetir_b200 import ops

    layer, x, _ = make(50, 4, 64, 40, 2, torch.float16, cuda_device, None)
    y, s = layer.forward(x)
    hidden = torch.empty_like(s.hidden)
    ops.grouped_mm(s.rows.view(-1), layer.gate_up.view(-1), hidden.view(-1), s.routing.indptr, 4, 64, 80, ops.GROUPED_W_OUT_IN)
    assert torch.equal(hidden, s.hidden) and torch.equal(s.act, F.silu(hidden[:, :40]) * hidden[:, 40:])


def test_steps_in_a_graph(cuda_device):
    """Captured training and serving steps follow the routing of new inputs, whose groups have other sizes; an eager step of the same
    layer between replays changes nothing."""
    layer, x, dy = make(200, 8, 128, 64, 2, torch.bfloat16, cuda_device)
    other = make(200, 8, 128, 64, 2, torch.bfloat16, cuda_device, seed=1)[1]
    f8, held = layer.quantized("float8"), x.clone()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            y, saved = layer.forward(held)
            grads, z = layer.backward(dy, saved), f8(held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, saved = layer.forward(held)
            grads, z = layer.backward(dy, saved), f8(held)
    torch.cuda.current_stream().wait_stream(side)
    for inputs in (other, x):
        held.copy_(inputs)
        graph.replay()
        want, want_saved = layer.forward(inputs)
        want_grads, want_z = layer.backward(dy, want_saved), f8(inputs)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want_z) and all(torch.equal(grads[k], want_grads[k]) for k in grads)


@pytest.mark.parametrize("gated", ["silu", "gelu"])
def test_without_tokens_or_with_none_kept(cuda_device, gated):
    layer, x, dy = make(6, 5, 64, 40, 2, torch.float16, cuda_device, gated)
    y, saved = layer.forward(x[:0])
    grads = layer.backward(dy[:0], saved)
    assert y.shape == (0, 64) and (grads["gate_up"] == 0).all() and layer.quantized("float8")(x[:0]).shape == (0, 64)
    padding = torch.ones(6, dtype=torch.bool, device=cuda_device)
    y, saved = layer.forward(x, padding)
    grads = layer.backward(dy, saved)
    assert (y == 0).all() and all((grads[n] == 0).all() for n in grads)
    assert (layer.quantized("float8")(x, padding) == 0).all()
