"""The gated linear layer at the ends of its range: layers without outputs and gradients far from one in size."""
import pytest
import torch

from forge_b200 import _forge_C as C
from forge_b200.nn import GatedLinear, gated_linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_no_outputs():
    """The gradient of x is an empty sum: zeros, whatever the memory held before."""
    for M, lead in ((5, (5,)), (6, (2, 3)), (0, (0,))):
        x = torch.randn(*lead, 64, device=DEV).half().requires_grad_()
        trash = torch.full((M, 64), 7.0, device=DEV).half()
        del trash   # what the allocator hands out next
        m = GatedLinear(64, 0, bias=True, device=DEV)
        h = m(x)
        assert h.shape == (*lead, 0)
        h.sum().backward()
        assert x.grad.shape == x.shape and (x.grad == 0).all()
        assert m.w_gate.grad.shape == (0, 64) and m.b_up.grad.shape == (0,)
    torch.cuda.synchronize()
    assert C.device_status() == 0
