"""Host side of the block-selecting attention: workspace sizes and refusals (no GPU)."""
import pytest
import torch


def test_host_tensors_are_refused():
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    x = torch.zeros(1, 128, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        block_topk_attention(x, x, x, 0.125, 1)
    with pytest.raises(ValueError):
        pool_key_blocks(x)


def test_workspace_bytes():
    from eraserdit_b200 import _native
    f = _native.load().erd_block_topk_workspace_bytes
    # key means, query sums and scores, 8 bytes each
    assert f(2, 8, 2, 300, 1000, 128, 64, 0) == 8 * (2 * 2 * 16 * 64 + 2 * 8 * 3 * 64 + 2 * 8 * 3 * 16)
    assert f(2, 8, 2, 300, 1000, 128, 64, 1) == 8 * (2 * 8 * 3 * 64 + 2 * 8 * 3 * 16)
    assert f(2, 8, 2, 1, 1000, 1, 128, 0) == 8 * (2 * 2 * 8 * 64)
    assert f(2, 8, 2, 1, 1000, 1, 128, 1) == 0
    assert f(0, 8, 2, 1, 1000, 1, 128, 0) == 0 and f(2, 8, 2, 1, 1000, 2, 128, 0) == 0
    # beyond 32 bits
    assert f(16, 64, 64, 1 << 20, 1 << 20, 128, 64, 1) > 1 << 37


def test_entries_reject_bad_arguments_before_any_device_call():
    from eraserdit_b200 import _native
    lib = _native.load()
    p = 1 << 20

    def call(dtype=0, q=p, k=p, v=p, qt=64, ot=64, batch=1, heads=2, kv_heads=1, q_len=5, kv_len=70,
             dim=64, lengths=None, means=None, topk=1, qb=1, kb=64, out=p, sel=p, ws=p, nbytes=1 << 20,
             scale=0.125):
        fields = (q, k, v, lengths, means, out, sel, ws, qt, *([64] * 8), ot, 64, 64, nbytes, dtype,
                  batch, heads, kv_heads, q_len, kv_len, dim, topk, qb, kb, scale)
        return lib.erd_block_topk_attn(
            _native.pack("erd_block_topk_attn", *(0 if f is None else f for f in fields)), None, None)

    assert lib.erd_block_topk_attn(None, None, None) == -1
    other = _native.STRUCTS["erd_block_topk_attn"].pack(8, *([0] * 32))
    assert lib.erd_block_topk_attn(other, None, None) == -2
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(sel=None), dict(ws=None)):
        assert call(**kw) == -1, kw
    for kw in (dict(dtype=2), dict(dim=128), dict(batch=0), dict(heads=3, kv_heads=2), dict(kv_heads=0),
               dict(q_len=0), dict(kv_len=0), dict(topk=0), dict(qb=64), dict(kb=32),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
               dict(nbytes=8 * 2 * 64 - 1)):
        assert call(**kw) == -2, kw
    for kw in (dict(q=p + 8), dict(v=p + 2), dict(out=p + 8), dict(qt=60), dict(ot=65), dict(means=p + 8),
               dict(lengths=p + 2), dict(sel=p + 1)):
        assert call(**kw) == -3, kw
    for kw in (dict(batch=300, heads=300, nbytes=1 << 40), dict(kv_len=64 * 18774, nbytes=1 << 40),
               dict(q_len=1 << 28, nbytes=1 << 60)):
        assert call(**kw) == -6, kw

    def means(dtype=0, k=p, kt=64, batch=1, heads=1, kv_len=70, kb=64, lengths=None, out=p):
        return lib.erd_block_key_means(dtype, k, kt, 64, 64, batch, heads, kv_len, kb, lengths, out, None)

    assert means(k=None) == -1 and means(out=None) == -1
    assert means(dtype=2) == -2 and means(kb=63) == -2 and means(kv_len=0) == -2 and means(heads=0) == -2
    assert means(kt=4) == -3 and means(out=p + 8) == -3 and means(lengths=p + 1) == -3


def test_topk_whose_loops_would_wrap_is_refused():
    """The loops over topk run in steps of 32: an int32 index passes 2^31 behind the last
    of them and the kernel would write in front of the selection."""
    from eraserdit_b200 import _native
    fn = _native.load().erd_block_topk_attn
    p = 1 << 20
    for qb in (1, 128):
        for topk in (0x7fff0001, 0x7fffffe1, 0x7fffffff):
            fields = (p, p, p, 0, 0, p, p, p, *([64] * 12), 1 << 20, 0, 1, 2, 1, 5, 70, 64, topk, qb, 64, 0.125)
            assert fn(_native.pack("erd_block_topk_attn", *fields), None, None) == -6


def test_means_of_as_many_keys_as_would_wrap_are_refused():
    """A block's end, first key + 64 (or 128), has to fit int32."""
    from eraserdit_b200 import _native
    fn = _native.load().erd_block_key_means
    p = 1 << 20
    for kb in (64, 128):
        for kv_len in (0x7fff0001, 0x7fffffc1, 0x7fffffff):
            assert fn(0, p, 64, 64, 64, 1, 1, kv_len, kb, None, p, None) == -6


def test_only_inputs_are_read_as_constant():
    """Kernels of one call start before the one in front has ended, so what that one
    writes (means, sums, scores, choice) is not constant while they run: of all
    pointers only the lengths, complete before the call, are read with __ldg."""
    import re
    from tests.conftest import ROOT
    text = (ROOT / "eraserdit_b200" / "csrc" / "block_topk.cu").read_text()
    reads = re.findall(r"__ldg\(([^;]*)", text)
    assert reads and all(r.startswith("lengths + b)") for r in reads)
    assert "__restrict__" not in text  # which would let the compiler choose such reads


def test_scales_whose_base_2_form_is_infinite_are_refused():
    """The kernels multiply by scale / ln 2: above 2.35e38 that leaves FP32's range, and
    scores of 0 times it are NaN."""
    from eraserdit_b200 import _native
    fn = _native.load().erd_block_topk_attn
    p = 1 << 20
    for qb in (1, 128):
        for scale in (2.4e38, 3.0e38, 3.4e38):
            fields = (p, p, p, 0, 0, p, p, p, *([64] * 12), 1 << 20, 0, 1, 2, 1, 5, 70, 64, 3, qb, 64, scale)
            assert fn(_native.pack("erd_block_topk_attn", *fields), None, None) == -2
