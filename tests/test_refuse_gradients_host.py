"""What an operator without derivatives refuses (no GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


def test_gradients_and_tangents(pkg):
    refuse, x = pkg._lib.refuse_gradients, torch.ones(3)
    refuse(x=x, y=None, z=1.0, ids=torch.ones(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="y asks for a gradient"):
        refuse(x=x, y=x.clone().requires_grad_())
    with torch.no_grad():
        refuse(y=x.clone().requires_grad_())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        refuse(x=x)
        for mode in (torch.enable_grad, torch.no_grad):   # (forward derivatives go on without grad mode)
            with mode(), pytest.raises(RuntimeError, match="z has a tangent"):
                refuse(x=x, z=dual * 2)
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(lambda x: refuse(x=x), (x,), (torch.ones(3),))


def test_a_differentiated_call_reaches_neither_path(pkg):
    """Wrapped tensors of torch.func are refused for their derivative, before the device is."""
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(lambda x: pkg.block_norm(x, x)[0], (x,), (x,))
    with pytest.raises(RuntimeError, match="gradient"):
        torch.func.grad(lambda x: pkg.block_norm(x, x)[0].sum())(x)
