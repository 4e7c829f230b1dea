"""The gate and its gradient at every number of 16 bits, not only where projections usually are.

With a depth of 1 and a weight of 1 the gradient of the activations is dy itself, exactly.  Tolerances as in test_gpu_gated.py."""
import pytest
import torch

from sparsetir_b200 import ops
from test_gpu_gated import TINY, TYPES, U, gate_parts, rel
from test_gpu_moe import near

pytestmark = pytest.mark.gpu

WIDTH = 64


def every_number(dtype, device):
    v = torch.arange(-32768, 32768, device=device, dtype=torch.int32).to(torch.int16).view(dtype)
    return torch.where(v.isfinite(), v, torch.zeros_like(v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_gradient(cuda_device, dtype, gelu, shift):
    """shift: the form for rows at any address."""
    gate = every_number(dtype, cuda_device).view(-1, WIDTH)
    rows = len(gate)
    up = torch.tensor([1.0, -0.375, 2.0, 0.0625], device=cuda_device, dtype=dtype).repeat(rows, WIDTH // 4)
    dy = torch.tensor([1.0, -0.5, 0.75], device=cuda_device, dtype=dtype).repeat(rows)[:rows].contiguous()
    hidden = torch.cat([gate, up], 1)
    w = torch.ones(WIDTH, device=cuda_device, dtype=dtype)
    memory = [torch.full((rows * n * WIDTH + shift,), 9.0, device=cuda_device, dtype=dtype)[shift:] for n in (2, 2, 1)]
    memory[0].copy_(hidden.view(-1))
    ops.grouped_mm_gated_grad(dy, w, memory[0], memory[1], memory[2], None, 1, 1, WIDTH, ops.GATED_GELU if gelu else 0)
    g, u, d = gate.double(), up.double(), dy.double()[:, None]
    f, df, s, z, dz = gate_parts(g, gelu)
    far = rel(z)
    top = torch.finfo(dtype).max
    off_df = far * (s + (f * dz).abs() * (1 - s)) + 4 * U * (f * dz).abs() * (z.abs() < 104)
    d_gate, d_up = memory[1].view(rows, 2 * WIDTH).split(WIDTH, 1)
    near(d_gate, d * u * df, (d * u).abs() * off_df + TINY, dtype)
    fits = (d * f).abs() <= top, (f * u).abs() <= top
    near(d_up[fits[0]], (d * f)[fits[0]], ((d * f).abs() * far + TINY)[fits[0]], dtype)
    near(memory[2].view(rows, WIDTH)[fits[1]], (f * u)[fits[1]], ((f * u).abs() * far + TINY)[fits[1]], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("rows", [200, 65536])
def test_product(cuda_device, dtype, gelu, rows):
    """One feature in, weights of 1 and 0.5: both projections are exact in 32 bits.  In one call, and 200 rows of 13 groups at a time (few to a
    group, the kernel for them)."""
    x = every_number(dtype, cuda_device)
    groups = 1 if rows == len(x) else 13
    w = torch.cat([torch.ones(8, device=cuda_device, dtype=dtype), torch.full((8,), 0.5, device=cuda_device, dtype=dtype)]).repeat(groups)
    ptr = torch.linspace(0, rows, groups + 1, device=cuda_device).int() if groups > 1 else None
    y = torch.full((len(x), 8), 9.0, device=cuda_device, dtype=dtype)
    for at in range(0, len(x), rows):
        at = min(at, len(x) - rows)
        ops.grouped_mm_gated(x[at:at + rows].contiguous(), w, y[at:at + rows].view(-1), None, ptr, groups, 1, 8, ops.GATED_GELU if gelu else 0)
    g = x.double()
    f, _, _, z, _ = gate_parts(g, gelu)
    want = f * 0.5 * g
    fits = want.abs() <= torch.finfo(dtype).max
    near(y[fits], want[fits, None].expand(-1, 8), ((want.abs() * rel(z))[fits] + TINY)[:, None], dtype)
