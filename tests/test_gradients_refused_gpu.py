"""Every entry point refuses a tangent (tests/test_gradients_refused.py), under no_grad too."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad_mode", [False, True])
def test_every_operator_refuses_tangents(grad_mode):
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    from eraserdit_b200.linear import linear_act
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    x = torch.ones(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(8, 64, device="cuda", dtype=torch.bfloat16)
    rotary = RotaryPositions(64)
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    calls = [lambda a, b: linear_act(a, w), lambda a, b: linear_act(b, w, residual=a @ w.T),
             lambda a, b: apply_rotary(a, b, rotary, 0), lambda a, b: apply_rotary(b, a, rotary, 0),
             lambda a, b: apply_fused_qk_head_rmsnorm_rotary(a, b, norm, norm, rotary),
             lambda a, b: block_topk_attention(a, b, b, 0.125, 1),
             lambda a, b: block_topk_attention(b, b, a, 0.125, 1), lambda a, b: pool_key_blocks(a)]
    with torch.set_grad_enabled(grad_mode), fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in calls:
            call(x, x)
            with pytest.raises(ValueError, match="backward"):
                call(dual, x)


def test_destinations_that_want_a_gradient_are_refused():
    """Writing over a tensor that records gradients would go past its graph, as torch's
    own out= arguments refuse to."""
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    from eraserdit_b200.linear import linear_act
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    x = torch.ones(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, 64, device="cuda", dtype=torch.bfloat16)
    rotary = RotaryPositions(64)
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    pool = pool_key_blocks(x)
    calls = [(x, lambda out: linear_act(x, w, out=out)),
             (x, lambda out: apply_rotary(x, x, rotary, 0, query_out=out)),
             (x, lambda out: apply_rotary(x, x, rotary, 0, key_out=out)),
             (x, lambda out: apply_fused_qk_head_rmsnorm_rotary(x, x, norm, norm, rotary, key_out=out)),
             (x, lambda out: block_topk_attention(x, x, x, 0.125, 1, out=out)),
             (pool, lambda out: pool_key_blocks(x, out=out))]
    for like, call in calls:
        out = torch.zeros_like(like, requires_grad=True)
        with pytest.raises(ValueError, match="backward"):
            call(out)
        with torch.no_grad():
            call(out)
