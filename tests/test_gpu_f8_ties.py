"""Rows of 32-bit numbers in 8-bit floating point: the nearest number of 8 bits, however near the quotient is to the middle of two.

In 64 bits 448 x is exact, and the quotient by a, of 24 bits each, is either a middle (5 bits) itself or 2^-29 of it away or more, so that the
rounded quotient lies on its side of the middle: the expected numbers are exact."""
import pytest
import torch

from sparsetir_b200 import ops
from test_gpu_f8 import F8, N, quantised
from test_gpu_moe import gen, off_by

pytestmark = pytest.mark.gpu


def middles():
    """Of two neighbours among the numbers of 8 bits, and the middle of 0 and the smallest."""
    normal = [(2 * m + 1) / 16 * 2.0 ** e for e in range(-6, 9) for m in range(8, 16)]
    return [v for v in normal if v < 448] + [(2 * m + 1) * 2.0 ** -10 for m in range(8)]


def test_middles_are_in_the_middle():
    numbers = torch.arange(127, dtype=torch.uint8).view(F8).double()
    assert sorted(middles()) == ((numbers[1:] + numbers[:-1]) / 2).tolist()


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("largest", [1.0, 3e38, 2.0 ** -109])
def test_beside_the_middles(cuda_device, largest, shift):
    m = torch.tensor(middles(), device=cuda_device, dtype=torch.float64)  # 126 of them
    assert len(m) < N
    a = largest / 2 * (1 + torch.rand(3000, generator=gen(1, cuda_device), device=cuda_device, dtype=torch.float32))
    a[:8] = largest / 2 * torch.tensor([1, 1.75, 1.125, 1.5, 1 + 2.0 ** -23, 2 - 2.0 ** -23, 1.25, 1.875], device=cuda_device)
    for step in (-2, -1, 0, 1, 2):
        x = torch.zeros(len(a), N, device=cuda_device)
        x[:, :len(m)] = (m * a.double()[:, None] / 448).float()
        for _ in range(abs(step)):
            x = torch.nextafter(x, torch.full_like(x, float("inf") if step > 0 else 0.0))
        x[:, len(m):] = a[:, None]
        x[::2] *= -1
        assert (x.abs() <= a[:, None]).all()
        x = off_by(x, shift).view(len(a), N)
        q, scale = torch.zeros(x.numel(), dtype=torch.int8, device=cuda_device).view(F8), torch.zeros(len(a), device=cuda_device)
        ops.moe_dispatch_f8(x.view(-1), None, q, scale, N, 1)
        assert torch.equal(q.view(len(a), N).double(), quantised(x)[0])


@pytest.mark.parametrize("t,f", [(5000, 200), (64, 4096), (300, 129)])
def test_random_rows(cuda_device, t, f):
    x = torch.randn(t, f, generator=gen(t, cuda_device), device=cuda_device)
    q, scale = torch.zeros(x.numel(), dtype=torch.int8, device=cuda_device).view(F8), torch.zeros(-(-f // N) * t, device=cuda_device)
    ops.moe_dispatch_f8(x.view(-1), None, q, scale, f, 1)
    assert torch.equal(q.view(t, f).double(), quantised(x)[0])
