"""Calls from host threads that have made no CUDA call before (a server's workers)."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _in_a_new_thread(call):
    """call()'s result or exception, from a thread of its own."""
    got = []

    def work():
        try:
            got.append(call())
        except Exception as error:  # handed to the caller
            got.append(error)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("rows", [1, 50, 3000])
def test_linear(rows):
    from eraserdit_b200.linear import linear_act, linear_bf16
    x = torch.randn(rows, 512, device="cuda").bfloat16()
    w = torch.randn(1024, 512, device="cuda").bfloat16()
    for op in (linear_act, linear_bf16):
        want = op(x, w)
        out = torch.zeros_like(want)
        torch.cuda.synchronize()
        _in_a_new_thread(lambda: op(x, w, out=out))
        assert torch.equal(out, want)


@pytest.mark.parametrize("query_block", [1, 128])
def test_block_attention(query_block):
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    q, k = (torch.randn(1, n, 2, 64, device="cuda").bfloat16() for n in (130, 600))
    pool = pool_key_blocks(k)
    want = block_topk_attention(q, k, k, 0.125, 3, query_block=query_block, key_pool=pool)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    _in_a_new_thread(lambda: block_topk_attention(q, k, k, 0.125, 3, query_block=query_block, key_pool=pool,
                                                  out=out))
    assert torch.equal(out, want)


def test_rotation_and_norm():
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions
    x = torch.randn(1, 40, 4, 64, device="cuda").bfloat16()
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    rotary = RotaryPositions(64)
    want, _ = apply_fused_qk_head_rmsnorm_rotary(x, None, norm, None, rotary, 3)
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    _in_a_new_thread(lambda: apply_fused_qk_head_rmsnorm_rotary(x, None, norm, None, rotary, 3, query_out=out))
    assert torch.equal(out, want)


def test_attention():
    from eraserdit_b200.attention import attention_bshd
    q, k, v = (torch.randn(1, 300, 2, 64, device="cuda").bfloat16() for _ in range(3))
    want = attention_bshd(q, k, v, 0.125)
    torch.cuda.synchronize()
    assert torch.equal(_in_a_new_thread(lambda: attention_bshd(q, k, v, 0.125)), want)
