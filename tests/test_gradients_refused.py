"""The operators have no derivative: inputs that ask for one are refused, in reverse
mode (requires_grad) and in forward mode (a tangent), not detached (no GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_reverse_mode():
    from eraserdit_b200._native import refuse_gradients
    x, leaf = torch.ones(3), torch.ones(3, requires_grad=True)
    refuse_gradients("op", x, None)
    with pytest.raises(ValueError):
        refuse_gradients("op", x, None, leaf)
    with torch.no_grad():
        refuse_gradients("op", leaf)


def test_forward_mode():
    from eraserdit_b200._native import refuse_gradients
    x = torch.ones(3)
    with fwd.dual_level():
        refuse_gradients("op", x, None)
        dual = fwd.make_dual(x, torch.ones(3))
        with pytest.raises(ValueError):
            refuse_gradients("op", None, dual)
        with torch.no_grad():  # stops reverse mode alone
            with pytest.raises(ValueError):
                refuse_gradients("op", dual)
        refuse_gradients("op", fwd.unpack_dual(dual).primal)
    refuse_gradients("op", x)


def test_func_jvp():
    from eraserdit_b200._native import refuse_gradients
    with pytest.raises(ValueError):
        torch.func.jvp(lambda t: refuse_gradients("op", t) or t, (torch.ones(3),), (torch.ones(3),))
