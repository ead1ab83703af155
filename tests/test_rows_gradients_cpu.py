"""What the ops without a gradient ask of their tensors."""
import pytest
import torch
from torch.autograd import forward_ad

from jit_kernel.norm_rope import _no_grad


def test_no_grad():
    x, y = torch.zeros(3), torch.zeros(3, dtype=torch.uint8).view(torch.float8_e4m3fn)
    _no_grad(x, None, y)
    for t in (torch.zeros(3, requires_grad=True), (torch.zeros(3, requires_grad=True) * 2)):
        with pytest.raises(RuntimeError, match="gradient"):
            _no_grad(x, t)
        with torch.no_grad():
            _no_grad(x, t)
    with forward_ad.dual_level():
        _no_grad(x, None, y)
        dual = forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(RuntimeError, match="tangent"):
            _no_grad(y, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
            _no_grad(dual * 2)
    _no_grad(x)
