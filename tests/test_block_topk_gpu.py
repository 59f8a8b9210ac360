"""block_topk_attention (erd_block_topk_attn) against its definition in 64 bits:
the chosen blocks exactly, the values within their roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 0.125


def _inputs(batch, q_len, kv_len, heads, kv_heads, dtype, seed, amp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: torch.randn(batch, n, h, 64, generator=g, device="cuda")
    k = r(kv_len, kv_heads)
    k += 0.5 * torch.randn(batch, -(-kv_len // 64), kv_heads, 64, generator=g,
                           device="cuda").repeat_interleave(64, 1)[:, :kv_len]
    return (amp * r(q_len, heads)).to(dtype), (amp * k).to(dtype), r(kv_len, kv_heads).to(dtype)


def _choose(q, k, topk, query_block, key_block, lengths):
    """bool [B, H, groups, blocks] and the padded index lists."""
    batch, q_len, heads, _ = q.shape
    kv_len, per = k.shape[1], heads // k.shape[2]
    groups, blocks = -(-q_len // query_block), -(-kv_len // key_block)
    keep = torch.zeros(batch, heads, groups, blocks, dtype=torch.bool, device=q.device)
    lists = torch.full((batch, heads, groups, topk), -1, dtype=torch.int32, device=q.device)
    for b in range(batch):
        length = kv_len if lengths is None else min(max(int(lengths[b]), 0), kv_len)
        n = -(-length // key_block)
        if n == 0:
            continue
        means = torch.stack([x.double().mean(0) for x in k[b, :length].split(key_block)])  # [n, Hkv, 64]
        sums = torch.stack([x.double().sum(0) for x in q[b].split(query_block)])           # [groups, H, 64]
        score = torch.einsum("ghd,nhd->hgn", sums, means.repeat_interleave(per, 1))
        order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :topk].sort(-1).values
        lists[b, :, :, :order.shape[-1]] = order.int()
        keep[b].scatter_(-1, order, True)
    return keep, lists


def _check(out, sel, q, k, v, topk, query_block, key_block, lengths=None, scale=SCALE):
    keep, lists = _choose(q, k, topk, query_block, key_block, lengths)
    assert torch.equal(sel, lists)
    fi = torch.finfo(q.dtype)
    per = q.shape[2] // k.shape[2]
    for b in range(q.shape[0]):
        length = k.shape[1] if lengths is None else min(max(int(lengths[b]), 0), k.shape[1])
        if length == 0:
            assert bool((out[b] == 0).all())
            continue
        for h in range(q.shape[2]):
            kf, vf, qf = (t.double() for t in (k[b, :length, h // per], v[b, :length, h // per], q[b, :, h]))
            mask = keep[b, h].repeat_interleave(key_block, 1)[:, :length]
            mask = mask.repeat_interleave(query_block, 0)[:q.shape[1]]
            s = (qf @ kf.T * scale).masked_fill(~mask, -math.inf)
            p = torch.softmax(s, -1)
            y = p @ vf
            spread = p @ vf.abs()
            # relative error of a weight: its rounding to the type, the exponential
            # (2^-21), the FP32 score (64 products, a truncation of 2^-23 each, and
            # the two roundings of its scaling); an FP16 weight below the normal range
            # is off by 2^-25 of the greatest, which the sum is at least
            size = (qf.abs() @ kf.abs().T * abs(scale)).masked_fill(~mask, 0).amax(-1, keepdim=True)
            share = fi.eps / 2 + 2.0 ** -20 + 68 * 2.0 ** -23 * size
            tol = share * (spread + y.abs()) * 1.01
            if q.dtype == torch.float16:
                tol = tol + mask.sum(-1, keepdim=True) * 2.0 ** -25 * vf.abs().amax()
            half = (y.abs() * fi.eps / 2).clamp(min=fi.smallest_normal * fi.eps / 2)
            bad = ((out[b, :, h].double() - y).abs() > (half + tol) * 1.001) | torch.isnan(out[b, :, h])
            assert int(bad.sum()) == 0, f"batch {b} head {h}: {int(bad.sum())} values off"


def _run(q, k, v, topk, **kw):
    from eraserdit_b200 import _native
    from eraserdit_b200.block_topk import block_topk_attention
    out, sel = block_topk_attention(q, k, v, kw.pop("scale", SCALE), topk, return_selection=True, **kw)
    assert _native.read_status(q.device) == 0
    return out, sel


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("query_block", [1, 128])
@pytest.mark.parametrize("key_block", [64, 128])
@pytest.mark.parametrize("q_len,kv_len", [(1, 1), (1, 64), (2, 65), (127, 63), (128, 128), (129, 127),
                                          (5, 1000), (300, 641), (200, 2049)])
@pytest.mark.parametrize("topk", [1, 3, 64])
def test_matches_definition(dtype, query_block, key_block, q_len, kv_len, topk):
    q, k, v = _inputs(2, q_len, kv_len, 4, 2, dtype, q_len + kv_len + topk)
    out, sel = _run(q, k, v, topk, query_block=query_block, key_block=key_block)
    _check(out, sel, q, k, v, topk, query_block, key_block)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (6, 3), (32, 32)])
@pytest.mark.parametrize("query_block", [1, 128])
def test_head_layouts_in_a_projection_buffer(heads, kv_heads, query_block):
    """Views of an interleaved Q|K|V buffer, the result into a strided buffer whose
    other bytes stay."""
    g = torch.Generator(device="cuda").manual_seed(heads)
    n = 700
    buf = torch.randn(2, n, (heads + 2 * kv_heads) * 64, generator=g, device="cuda").bfloat16()
    q = buf[..., :heads * 64].unflatten(-1, (heads, 64))
    k = buf[..., heads * 64:(heads + kv_heads) * 64].unflatten(-1, (kv_heads, 64))
    v = buf[..., (heads + kv_heads) * 64:].unflatten(-1, (kv_heads, 64))
    if query_block == 1:
        q = q[:, -3:]
    wide = torch.full((2, q.shape[1], heads, 80), 7.0, device="cuda", dtype=torch.bfloat16)
    out, sel = _run(q, k, v, 4, query_block=query_block, out=wide[..., 8:72])
    _check(out, sel, q, k, v, 4, query_block, 64)
    assert bool((wide[..., :8] == 7).all()) and bool((wide[..., 72:] == 7).all())
    # BHSD storage
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    again, sel2 = _run(qt, kt, vt, 4, query_block=query_block)
    assert torch.equal(again, out) and torch.equal(sel, sel2)


@pytest.mark.parametrize("query_block", [1, 128])
@pytest.mark.parametrize("key_block", [64, 128])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf, -3.0e38])
def test_lengths_and_what_lies_behind_them(query_block, key_block, poison):
    """Ragged sequences, one of them empty; keys and values behind a length hold
    NaN, infinities or the type's lowest values and change nothing; lengths beyond
    the buffer or below zero are clamped."""
    lengths = torch.tensor([700, 0, 1, 64, 65, 333, 10 ** 9, -5], dtype=torch.int32, device="cuda")
    q, k, v = _inputs(8, 140 if query_block > 1 else 3, 700, 2, 1, torch.bfloat16, 5)
    for b, n in enumerate(lengths.clamp(0, 700).tolist()):
        k[b, n:] = poison
        v[b, n:] = poison
    out, sel = _run(q, k, v, 3, query_block=query_block, key_block=key_block, key_lengths=lengths)
    _check(out, sel, q, k, v, 3, query_block, key_block, lengths)
    # queries behind the last one of a tile are not read either
    if query_block > 1:
        wide = torch.full((8, 256, 2, 64), poison, device="cuda", dtype=torch.bfloat16)
        wide[:, :140] = q
        again, sel2 = _run(wide[:, :140], k, v, 3, query_block=128, key_block=key_block, key_lengths=lengths)
        assert torch.equal(again, out) and torch.equal(sel, sel2)


@pytest.mark.parametrize("query_block", [1, 128])
def test_bad_values_in_one_place_stay_there(query_block):
    """A NaN in a key spoils its block's score (it ranks last) and the rows that
    attend it all the same; blocks that are not chosen may hold NaN values."""
    q, k, v = _inputs(1, 128, 640, 1, 1, torch.bfloat16, 6)
    out, sel = _run(q, k, v, 4, query_block=query_block)
    k2, v2 = k.clone(), v.clone()
    chosen = set(sel.unique().tolist())
    for block in range(10):
        if block not in chosen:
            v2[0, block * 64:block * 64 + 64] = math.nan
    again, sel2 = _run(q, k, v2, 4, query_block=query_block)
    assert torch.equal(sel, sel2) and torch.equal(again, out)
    k2[0, 5 * 64 + 3, 0, 7] = math.nan
    _, sel3 = _run(q, k2, v, 4, query_block=query_block)
    assert not bool((sel3 == 5).any())
    out4, sel4 = _run(q, k2, v, 10, query_block=query_block)
    assert bool(torch.isnan(out4).all()) and bool((sel4 == torch.arange(10, device="cuda")).all())


@pytest.mark.parametrize("query_block", [1, 128])
@pytest.mark.parametrize("blocks,topk", [(9, 4), (300, 17), (700, 64), (1100, 33)])
def test_ties_go_to_the_lowest_index(query_block, blocks, topk):
    """Equal scores (zeros of either sign), scores that differ in their last bits
    only, and every size of the selection (registers and memory)."""
    kv_len = blocks * 64 - 5
    q = torch.zeros(1, 3, 1, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(1, kv_len, 1, 64, device="cuda", dtype=torch.bfloat16)
    k[0, 64:, 0, 1] = -0.0
    v = torch.randn(1, kv_len, 1, 64, device="cuda").bfloat16()
    q[..., 0] = 1
    k[..., 0] = 1.0
    want = torch.arange(topk, device="cuda", dtype=torch.int32)
    _, sel = _run(q, k, v, topk, query_block=query_block)
    assert bool((sel == want).all())
    # score 1 + code * 2^-45: the upper words tie, the lower ones decide
    code = (torch.arange(blocks, device="cuda") * 37) % 101
    q[..., 1] = 2.0 ** -45
    k[..., 1] = code.repeat_interleave(64)[:kv_len, None].to(torch.bfloat16)
    out, sel = _run(q, k, v, topk, query_block=query_block)
    order = torch.sort(code, descending=True, stable=True).indices[:topk].sort().values.int()
    assert bool((sel == order).all())
    _check(out, sel, q, k, v, topk, query_block, 64)


@pytest.mark.parametrize("q_len", [1, 2048, 2177])
@pytest.mark.parametrize("kv_len", [4032, 4096, 4097])
def test_rows_of_one_tile_of_scores_and_of_two(q_len, kv_len):
    """63, 64 and 65 key blocks; one, 16 and 18 query blocks."""
    q, k, v = _inputs(2, q_len, kv_len, 2, 1, torch.bfloat16, q_len + kv_len)
    lengths = torch.tensor([kv_len, 1000], device="cuda", dtype=torch.int32)
    for given in (None, lengths):
        out, sel = _run(q, k, v, 40, query_block=128, key_lengths=given)
        _check(out, sel, q, k, v, 40, 128, 64, lengths=given)


def test_large_scores_and_far_rows():
    """Sharp softmaxes (scores of several hundred, so the running maximum moves);
    scales that masked keys' -inf cannot be multiplied with are refused."""
    q, k, v = _inputs(1, 256, 1500, 2, 2, torch.bfloat16, 7, amp=6.0)
    for query_block in (1, 128):
        for scale in (0.125, 1.0):
            out, sel = _run(q, k, v, 8, query_block=query_block, scale=scale)
            _check(out, sel, q, k, v, 8, query_block, 64, scale=scale)
        for scale in (-0.125, 0.0, math.inf, math.nan):
            with pytest.raises(ValueError):
                _run(q, k, v, 8, query_block=query_block, scale=scale)


@pytest.mark.parametrize("batch,kv_len,topk", [(1, 40000, 32), (4, 5000, 64), (1, 300, 64), (64, 700, 2)])
def test_single_tokens(batch, kv_len, topk):
    """One to eight CTAs a row."""
    q, k, v = _inputs(batch, 1, kv_len, 8, 4, torch.float16, 8)
    out, sel = _run(q, k, v, topk, query_block=1)
    _check(out, sel, q, k, v, topk, 1, 64)


@pytest.mark.parametrize("key_block", [64, 128])
def test_kept_means(key_block):
    """Means computed once, kept, and extended by an append, give what the call
    computes itself."""
    from eraserdit_b200.block_topk import pool_key_blocks
    q, k, v = _inputs(2, 130, 1000, 4, 2, torch.bfloat16, 9)
    lengths = torch.tensor([900, 130], dtype=torch.int32, device="cuda")
    pool = pool_key_blocks(k, key_block, key_lengths=lengths)
    for b, n in enumerate((900, 130)):
        means = torch.stack([x.double().mean(0) for x in k[b, :n].split(key_block)], 1)
        assert torch.allclose(pool[b, :, :means.shape[1]], means, rtol=1e-14, atol=1e-15)
        assert bool((pool[b, :, means.shape[1]:] == 0).all())
    for query_block in (1, 128):
        own = _run(q, k, v, 3, query_block=query_block, key_block=key_block, key_lengths=lengths)
        kept = _run(q, k, v, 3, query_block=query_block, key_block=key_block, key_lengths=lengths, key_pool=pool)
        assert torch.equal(own[0], kept[0]) and torch.equal(own[1], kept[1])
    # one sequence grows by 70 keys: only the blocks from the first changed one on
    first = 900 // key_block
    part = pool_key_blocks(k[:1, first * key_block:970], key_block)
    pool[:1, :, first:first + part.shape[2]] = part
    lengths[0] = 970
    assert torch.equal(pool, pool_key_blocks(k, key_block, key_lengths=lengths))


def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_graph():
    q, k, v = _inputs(2, 200, 3000, 4, 2, torch.bfloat16, 10)
    from eraserdit_b200.block_topk import block_topk_attention
    for query_block, qq in ((128, q), (1, q[:, :2])):
        call = lambda: block_topk_attention(qq, k, v, SCALE, 9, query_block=query_block, return_selection=True)
        want = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        outs = []
        for _ in range(8):  # two streams at once, each with its workspace
            with torch.cuda.stream(side):
                outs.append(call())
            outs.append(call())
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                o = call()
            graphs.append((g, o))
        k.neg_()
        for g, _ in graphs:
            g.replay()
        want = call()
        for _, o in graphs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_offsets_beyond_32_bits():
    """Keys 2^23 values apart: the last one lies 5 * 10^9 values in (10 GB)."""
    step, n = 2 ** 23, 600
    buf = torch.empty(step * n, device="cuda", dtype=torch.bfloat16)
    q, k0, v0 = _inputs(1, 130, n, 1, 1, torch.bfloat16, 11)
    k, v = (buf.as_strided((1, n, 1, 64), (step * n, step, 64, 1), off) for off in (0, 64))
    k.copy_(k0)
    v.copy_(v0)
    for query_block in (1, 128):
        out, sel = _run(q, k, v, 4, query_block=query_block)
        want, sel2 = _run(q, k0, v0, 4, query_block=query_block)
        assert torch.equal(out, want) and torch.equal(sel, sel2)
    del buf, k, v
    torch.cuda.empty_cache()


def test_empty_and_refusals():
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    q, k, v = _inputs(2, 130, 200, 4, 2, torch.bfloat16, 12)
    out, sel = block_topk_attention(q, k[:, :0], v[:, :0], SCALE, 3, return_selection=True)
    assert bool((out == 0).all()) and bool((sel == -1).all())
    assert block_topk_attention(q[:, :0], k, v, SCALE, 3).shape == (2, 0, 4, 64)
    assert block_topk_attention(q[:0], k[:0], v[:0], SCALE, 3).shape == (0, 130, 4, 64)
    assert pool_key_blocks(k[:, :0]).shape == (2, 2, 0, 64)
    lengths = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    pool = pool_key_blocks(k)
    bad = [dict(query=q.float()), dict(query=q[0]), dict(query=q[..., :32]), dict(key=k.half()),
           dict(value=v[:, :100]), dict(query=q[:1]), dict(query=q[:, :, :3]), dict(topk=0), dict(topk=2.0),
           dict(query_block=64), dict(key_block=32), dict(key_lengths=lengths.long()),
           dict(key_lengths=lengths[:1]), dict(key_lengths=lengths.cpu()), dict(key_pool=pool.float()),
           dict(key_pool=pool[:, :, :2]), dict(key_pool=pool, key_block=128), dict(out=q.half()),
           dict(out=q[:, :1]), dict(key=k[:, :, :1].expand(2, 200, 2, 64)),
           dict(query=torch.zeros(2, 130, 4, 68, device="cuda", dtype=torch.bfloat16)[..., 4:]),
           dict(query=q.transpose(2, 3).contiguous().transpose(2, 3))]
    for kw in bad:
        args = dict(dict(query=q, key=k, value=v, topk=3), **kw)
        rest = {n: args.pop(n) for n in list(args) if n not in ("query", "key", "value", "topk")}
        with pytest.raises(ValueError):
            block_topk_attention(args["query"], args["key"], args["value"], SCALE, args["topk"], **rest)
    with pytest.raises(ValueError):
        block_topk_attention(q.requires_grad_(), k, v, SCALE, 3)


@pytest.mark.parametrize("query_block", [1, 128])
def test_destination_over_the_queries_but_not_the_keys(query_block):
    from eraserdit_b200.block_topk import block_topk_attention
    q, k, v = _inputs(2, 140, 300, 4, 4, torch.bfloat16, 13)
    want = block_topk_attention(q, k, v, SCALE, 2, query_block=query_block)
    own = q.clone()
    assert block_topk_attention(own, k, v, SCALE, 2, query_block=query_block, out=own) is own
    assert torch.equal(own, want)
    for out in (k[:, :140], v[:, 20:160]):
        with pytest.raises(ValueError):
            block_topk_attention(q, k, v, SCALE, 2, query_block=query_block, out=out)


@pytest.mark.parametrize("query_block", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_that_are_not_finite(query_block, dtype):
    """Valid keys whose scores are NaN or infinite, in every kind of place of a block:
    NaN and +inf make the row NaN, -inf weighs nothing, and a row with nothing but -inf
    is zeros."""
    q = torch.rand(1, 130, 1, 64, device="cuda").to(dtype) + 0.5  # positive: q . inf = inf
    _, k0, v = _inputs(1, 1, 192, 1, 1, dtype, 14)
    for place in (0, 1, 2, 7, 8, 9, 31, 62, 63, 64, 100, 191):
        for bad in (math.nan, math.inf, -math.inf):
            k = k0.clone()
            k[0, place, 0, 5] = bad
            out, _ = _run(q, k, v, 3, query_block=query_block)
            if bad == -math.inf:
                s = (q[0, :, 0].double() @ k[0, :, 0].double().T * SCALE)
                want = torch.softmax(s, -1) @ v[0, :, 0].double()
                assert float((out[0, :, 0].double() - want).abs().max()) <= 0.05
            else:
                assert bool(torch.isnan(out).all())
    k = k0.clone()
    k[..., 5] = -math.inf
    out, _ = _run(q, k, v, 3, query_block=query_block)
    assert bool((out == 0).all())
    k[0, 150, 0, 5] = 0.0  # one finite score behind two blocks of -inf
    out, _ = _run(q, k, v, 3, query_block=query_block)
    assert torch.equal(out, v[:, 150:151].expand_as(out))


def test_many_blocks_in_the_first_call_of_a_process():
    """5816 and 6112 blocks with 64 chosen: scores and choice take just below 48 KB of
    shared memory, which the kernel's own 2.4 KB lift above it."""
    import subprocess
    import sys
    from tests.conftest import ROOT
    code = ("import torch\n"
            "from eraserdit_b200.block_topk import block_topk_attention\n"
            "for n in (5816, 6112):\n"
            "    k = torch.randn(1, n * 64, 1, 64, device='cuda').bfloat16()\n"
            "    block_topk_attention(k[:, :1], k, k, 0.125, 64, query_block=1)\n"
            "torch.cuda.synchronize()\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("blocks,topk", [(1536, 7), (1537, 64), (5815, 64), (5816, 64), (6112, 64), (6113, 64),
                                         (18773, 64), (18773, 18773)])
def test_single_queries_over_very_many_blocks(blocks, topk):
    """The choice from shared memory instead of registers (above 1536 blocks), up to the
    stated limit; one block more is refused."""
    from eraserdit_b200.block_topk import block_topk_attention, pool_key_blocks
    kv_len = blocks * 64 - 3
    q, k, v = _inputs(1, 2, kv_len, 1, 1, torch.bfloat16, blocks)
    pool = pool_key_blocks(k)
    for given in (pool, None):
        out, sel = _run(q, k, v, topk, query_block=1, key_pool=given)
        _check(out, sel, q, k, v, topk, 1, 64)
    # ties, so that the bits of the scores decide
    k[:, 64:] = k[:, :64].repeat(1, blocks - 1, 1, 1)[:, :kv_len - 64]
    _, sel = _run(q, k, v, topk, query_block=1)
    full = torch.arange(topk, device="cuda", dtype=torch.int32)
    if topk < blocks:  # every whole block scores alike; the last, shorter one may lead
        assert bool(((sel == full) | ((full == topk - 1) & (sel == blocks - 1))).all())
    else:
        assert bool((sel == full).all())
    if blocks == 18773:
        more = torch.zeros(1, blocks * 64 + 1, 1, 64, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(RuntimeError):
            block_topk_attention(q, more, more, SCALE, topk, query_block=1)


@pytest.mark.parametrize("query_block", [1, 128])
def test_topk_far_above_the_blocks_costs_nothing(query_block):
    """"All blocks" asked for by a large number: without the selection in the result no
    list of that width is made."""
    from eraserdit_b200.block_topk import MAX_TOPK, block_topk_attention
    q, k, v = _inputs(2, 130, 700, 4, 2, torch.bfloat16, 15)
    want = block_topk_attention(q, k, v, SCALE, 11, query_block=query_block)
    for topk in (2 ** 20, MAX_TOPK):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = block_topk_attention(q, k, v, SCALE, topk, query_block=query_block)
        assert torch.cuda.max_memory_allocated() - before < 1 << 21
        assert torch.equal(out, want)
    _, sel = block_topk_attention(q, k, v, SCALE, 5000, query_block=query_block, return_selection=True)
    assert sel.shape[-1] == 5000 and bool((sel[..., 11:] == -1).all())
    for topk in (MAX_TOPK + 1, 2 ** 31 - 1, 2 ** 40):
        with pytest.raises(ValueError):
            block_topk_attention(q, k, v, SCALE, topk, query_block=query_block)


def test_means_renewed_from_a_block_on_in_a_ragged_batch():
    """An append to kept keys whose rest holds anything: the blocks from the first that
    changed are renewed with what is left of each length there."""
    from eraserdit_b200.block_topk import pool_key_blocks
    keys = torch.full((3, 512, 2, 64), math.nan, device="cuda", dtype=torch.bfloat16)
    old, new = [200, 70, 0], [330, 75, 64]
    _, k, _ = _inputs(3, 1, 512, 2, 2, torch.bfloat16, 16)
    for b, n in enumerate(old):
        keys[b, :n] = k[b, :n]
    pool = pool_key_blocks(keys, key_lengths=torch.tensor(old, dtype=torch.int32, device="cuda"))
    for b, n in enumerate(new):
        keys[b, :n] = k[b, :n]
    lengths = torch.tensor(new, dtype=torch.int32, device="cuda")
    i = min(n // 64 for n in old)
    pool[:, :, i:] = pool_key_blocks(keys[:, i * 64:], key_lengths=lengths - i * 64)
    assert torch.equal(pool, pool_key_blocks(keys, key_lengths=lengths))
    assert bool(torch.isfinite(pool).all())


@pytest.mark.parametrize("query_block", [1, 128])
def test_scales_at_the_ends_of_their_range(query_block):
    from eraserdit_b200.block_topk import block_topk_attention
    q, k, v = _inputs(1, 130, 200, 1, 1, torch.bfloat16, 17)
    for scale in (1e39, 2.4e38, 1e-50):
        with pytest.raises(ValueError):
            block_topk_attention(q, k, v, scale, 2, query_block=query_block)
    # scores that all but vanish, and scores of 0 under the greatest scale: the mean of v
    want = torch.stack([v[0, :, 0].double().mean(0)] * 130)
    for scale, queries in ((1e-44, q), (2e38, torch.zeros_like(q))):
        out = block_topk_attention(queries, k, v, scale, 4, query_block=query_block)
        assert float((out[0, :, 0].double() - want).abs().max()) < 2.0 ** -8
