"""What `ExpertLayer.forward` keeps and what `backward` asks for, without a device."""
import pytest
import torch

from sparsetir_b200 import moe


@pytest.mark.parametrize("gated", ["silu", "gelu"])
def test_backward_of_a_forward_that_kept_nothing_is_refused(gated):
    """Before any operator is called, with what is missing and how to have it."""
    layer = moe.ExpertLayer(torch.zeros(4, 8), torch.zeros(4, 6, 8).half(), torch.zeros(4, 8, 3).half(), 2, gated=gated)
    x, rows = torch.zeros(5, 8).half(), torch.zeros(10, 8).half()
    routing = moe.Routing(torch.zeros(5, 4), torch.zeros(5, 2), torch.zeros(5, 2).int(), torch.zeros(5, 2).int(), torch.zeros(5).int())
    with pytest.raises(ValueError, match="forward.* train=True"):
        layer.backward(x, moe.Saved(x, routing, rows, None, None, rows))
