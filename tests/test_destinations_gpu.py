"""A caller's destination counts as written in place: autograd must not use what it
saved of that tensor before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    from eraserdit_b200.linear import linear_act
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    x = torch.ones(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, 64, device="cuda", dtype=torch.bfloat16)
    rotary = RotaryPositions(64)
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    pool = pool_key_blocks(x)
    return {"linear": (x, lambda out: linear_act(x, w, out=out)),
            "linear in slots": (x.view(2, 2, 2, 64).transpose(0, 1),
                                lambda out: linear_act(x.view(2, 2, 2, 64).transpose(0, 1), w, out=out)),
            "query": (x, lambda out: apply_rotary(x, x, rotary, 0, query_out=out)),
            "key": (x, lambda out: apply_rotary(x, x, rotary, 0, key_out=out)),
            "norm": (x, lambda out: apply_fused_qk_head_rmsnorm_rotary(x, x, norm, norm, rotary, query_out=out)),
            "attention": (x, lambda out: block_topk_attention(x, x, x, 0.125, 1, out=out)),
            "no keys": (x, lambda out: block_topk_attention(x, x[:, :0], x[:, :0], 0.125, 1, out=out)),
            "means": (pool, lambda out: pool_key_blocks(x, out=out))}


@pytest.mark.parametrize("name", ["linear", "linear in slots", "query", "key", "norm", "attention", "no keys",
                                  "means"])
def test_saved_tensors_are_known_to_have_changed(name):
    like, call = _calls()[name]
    leaf = torch.ones_like(like, requires_grad=True)
    out = leaf * 2
    square = (out * out).sum()
    version = out._version
    with torch.no_grad():
        call(out)
    assert out._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.backward()


def test_inference_tensors_have_no_version():
    for like, call in _calls().values():
        with torch.inference_mode():
            call(torch.zeros_like(like))
