"""The block operators run together, as a transformer block uses them: projection,
per-head norms and rotation in place in the projection's buffer, attention over
selected blocks, gated output projection onto the residual stream, and the feed-forward
products; then the same block for one new token against kept keys."""
import pytest
import torch

from tests.test_block_topk_gpu import _check as check_attention
from tests.test_head_rotary_gpu import _close, _want
from tests.test_linear_act_gpu import _check as check_linear

pytestmark = pytest.mark.gpu

HEADS, DIM, HIDDEN, FFN = 32, 64, 2048, 8192
FRAMES, ROWS, COLS = 2, 8, 12


class Block:
    def __init__(self, dtype, seed):
        from eraserdit_b200.rotary import RotaryPositions
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda n, k: (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).to(dtype)
        v = lambda n: (torch.randn(n, generator=g, device="cuda") * 0.1).to(dtype)
        self.w_qkv, self.b_qkv = w(3 * HIDDEN, HIDDEN), v(3 * HIDDEN)
        self.w_out, self.b_out = w(HIDDEN, HIDDEN), v(HIDDEN)
        self.w_up, self.b_up = w(FFN, HIDDEN), v(FFN)
        self.w_down, self.b_down = w(HIDDEN, FFN), v(HIDDEN)
        self.norms = [torch.nn.RMSNorm(DIM, eps=1e-6, device="cuda", dtype=dtype).requires_grad_(False)
                      for _ in range(2)]
        self.rotary = RotaryPositions(DIM, layout="interleaved", axes_dim=(24, 20, 20))

    def heads(self, x, positions):
        """Queries, keys and values of x, normalised and turned in place."""
        from eraserdit_b200.linear import linear_act
        from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
        qkv = linear_act(x, self.w_qkv, self.b_qkv)
        self.raw = qkv.clone()
        q, k, v = (t.unflatten(-1, (HEADS, DIM)) for t in qkv.split(HIDDEN, -1))
        apply_fused_qk_head_rmsnorm_rotary(q, k, *self.norms, self.rotary, positions, query_out=q, key_out=k)
        return q, k, v

    def rest(self, x, attended, gate):
        from eraserdit_b200.linear import linear_act
        self.h = linear_act(attended.flatten(2), self.w_out, self.b_out, gate=gate, residual=x)
        self.up = linear_act(self.h, self.w_up, self.b_up, activation="gelu_tanh")
        return linear_act(self.up, self.w_down, self.b_down, residual=self.h)


def _positions():
    s = torch.arange(FRAMES * ROWS * COLS, device="cuda")
    return torch.stack([s // (ROWS * COLS), s // COLS % ROWS, s % COLS])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_clip(dtype):
    from eraserdit_b200 import _native
    from eraserdit_b200.block_topk import block_topk_attention
    block, pos = Block(dtype, 1), _positions()
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, pos.shape[1], HIDDEN, generator=g, device="cuda").to(dtype)
    gate = torch.randn(2, HIDDEN, generator=g, device="cuda").to(dtype)

    def run():
        q, k, v = block.heads(x, pos)
        a, sel = block_topk_attention(q, k, v, DIM ** -0.5, 2, return_selection=True)
        return q, k, v, a, sel, block.rest(x, a, gate)

    q, k, v, a, sel, y = run()
    assert _native.read_status(x.device) == 0
    check_linear(block.raw, x, block.w_qkv, block.b_qkv, "none", None, None)
    table = pos.T[None].expand(2, -1, 3)
    for got, raw, norm in ((q, block.raw[..., :HIDDEN], block.norms[0]),
                           (k, block.raw[..., HIDDEN:2 * HIDDEN], block.norms[1])):
        _close(got, _want(raw.unflatten(-1, (HEADS, DIM)), block.rotary, table, weight=norm.weight, eps=1e-6))
    assert torch.equal(v.flatten(2), block.raw[..., 2 * HIDDEN:])
    check_attention(a, sel, q, k, v, 2, 128, 64)
    check_linear(block.h, a.flatten(2), block.w_out, block.b_out, "none", gate, x)
    check_linear(block.up, block.h, block.w_up, block.b_up, "gelu_tanh", None, None)
    check_linear(y, block.up, block.w_down, block.b_down, "none", None, block.h)
    # captured whole, replayed on other input
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    x.mul_(0.5)
    graph.replay()
    again = run()
    for i in (3, 4, 5):
        assert torch.equal(out[i], again[i])


def test_next_token():
    """One token more: its key and value are appended to kept buffers, the last
    block's mean is renewed, and it attends the blocks it picks."""
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    block, pos = Block(torch.bfloat16, 3), _positions()
    g = torch.Generator(device="cuda").manual_seed(4)
    n = pos.shape[1]
    x = torch.randn(2, n, HIDDEN, generator=g, device="cuda").bfloat16()
    keys = torch.full((2, 256, HEADS, DIM), float("nan"), device="cuda", dtype=torch.bfloat16)
    values = torch.full_like(keys, float("nan"))
    lengths = torch.tensor([n - 1, n - 1], dtype=torch.int32, device="cuda")
    _, k, v = block.heads(x[:, :n - 1], pos[:, :n - 1])
    keys[:, :n - 1], values[:, :n - 1] = k, v
    pool = pool_key_blocks(keys, key_lengths=lengths)
    new = x[:, n - 1:].contiguous()
    q, k, v = block.heads(new, pos[:, n - 1:])
    keys[:, n - 1:n], values[:, n - 1:n] = k, v
    lengths += 1
    last = (n - 1) // 64
    pool[:, :, last:last + 1] = pool_key_blocks(keys[:, last * 64:n])
    a, sel = block_topk_attention(q, keys, values, DIM ** -0.5, 2, query_block=1, key_lengths=lengths,
                                  key_pool=pool, return_selection=True)
    check_attention(a, sel, q, keys, values, 2, 1, 64, lengths)
    y = block.rest(new, a, torch.ones(HIDDEN, device="cuda", dtype=torch.bfloat16))
    check_linear(y, block.up, block.w_down, block.b_down, "none", None, block.h)
