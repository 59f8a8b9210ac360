"""Rotary positions and per-head RMS norms (erd_head_norm_rotary) against the
formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# FP32 arithmetic on a pair (y0, y1), as a share of |y0| + |y1|.  Rotation: the
# reduced angle is rounded to 32 bits (at most 2^-26 turns, 2 pi 2^-26 < 2^-23),
# sincospif is within 2 ulp (2^-23), the amplitude and the two products and
# their sum round by 2^-24 each: below 2^-21.
ROTATE = 2.0 ** -21
# Norm: the sum of squares accumulates at most 16 terms a lane, then 5 shuffles
# (or 32 terms a lane, 1024 channels): 37 half-steps, halved by the root, plus
# rsqrtf (2 ulp), the mean and two products: below 25 * 2^-24 < 2^-19.
NORM = 2.0 ** -19


def _randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _want(x, rotary=None, pos=None, inverse=False, weight=None, eps=None):
    """(value, tolerance before the last rounding) in 64 bits; pos [B or 1, S, axes]."""
    y = x.double()
    share = 0.0
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
        share = NORM
    if rotary is None:
        return y, share * y.abs()
    r = rotary.rotary_dim
    ends = [0, rotary.second_axis, rotary.third_axis, r // 2]
    axis = torch.zeros(r // 2, dtype=torch.long, device=x.device)
    axis[ends[1]:] += 1
    axis[ends[2]:] += 1
    angle = pos.double()[..., axis.clamp(max=pos.shape[-1] - 1)] * rotary.frequencies.to(x.device)
    angle = angle[:, :, None]
    c, s = angle.cos() * rotary.amplitude, angle.sin() * rotary.amplitude
    if inverse:
        s = -s
    sel = (slice(0, r // 2), slice(r // 2, r)) if rotary.layout == "half" else \
        (slice(0, r, 2), slice(1, r, 2))
    a, b = y[..., sel[0]], y[..., sel[1]]
    out, tol = y.clone(), share * y.abs()
    out[..., sel[0]], out[..., sel[1]] = a * c - b * s, a * s + b * c
    both = (ROTATE + share) * rotary.amplitude * (a.abs() + b.abs())
    tol[..., sel[0]], tol[..., sel[1]] = both, both
    return out, tol


def _close(got, want_tol):
    want, tol = want_tol
    fi = torch.finfo(got.dtype)
    # one rounding to the output type: half a step of the value (of the smallest
    # subnormal below the normal range)
    half = torch.maximum(want.abs() * fi.eps / 2, torch.tensor(fi.smallest_normal * fi.eps / 2,
                                                               device=got.device))
    bad = ((got.double() - want).abs() > (half + tol) * (1 + 1e-3)) | torch.isnan(got)
    assert int(bad.sum()) == 0, f"{int(bad.sum())} of {bad.numel()} values off"


def _pos(batch, tokens, axes=1, start=0):
    p = torch.arange(tokens, device="cuda")[None, :, None] + torch.arange(axes, device="cuda") * 7
    return (p + start).expand(batch, tokens, axes)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (128, 64), (80, 32), (40, 40), (2, 2), (33, 22),
                                            (96, 90), (256, 256), (512, 16), (1024, 1024), (72, 72)])
def test_rotation_matches_formula(dtype, layout, dim, rotary_dim):
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(dim, rotary_dim=rotary_dim, layout=layout)
    q, k = _randn((2, 19, 5, dim), dtype, 1), _randn((2, 19, 3, dim), dtype, 2)
    pos = _pos(2, 19, start=1000)
    qo, ko = apply_rotary(q, k, rotary, pos[0, :, 0].contiguous())
    _close(qo, _want(q, rotary, pos))
    _close(ko, _want(k, rotary, pos))
    assert torch.equal(qo[..., rotary_dim:], q[..., rotary_dim:])  # passed through


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (128, 64), (80, 32), (33, 22), (1024, 6)])
@pytest.mark.parametrize("weights", ["same", "fp32", "none"])
def test_norm_and_rotation_match_formula(dtype, layout, dim, rotary_dim, weights):
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions
    rotary = RotaryPositions(dim, rotary_dim=rotary_dim, layout=layout,
                             scaling={"type": "yarn", "factor": 4, "original_length": 64})
    q, k = _randn((3, 7, 9, dim), dtype, 3), 20 * _randn((3, 7, 2, dim), dtype, 4)
    q[0, 0, 0] = 0  # a head of zeros stays zero
    norms = []
    for seed, eps in ((5, 1e-6), (6, 1e-5)):
        n = torch.nn.RMSNorm(dim, eps=eps, device="cuda", elementwise_affine=weights != "none",
                             dtype=torch.float32 if weights == "fp32" else dtype)
        if n.weight is not None:
            n.requires_grad_(False)
            n.weight.copy_(_randn((dim,), torch.float32, seed))
        norms.append(n)
    pos = _pos(3, 7, start=-3) * torch.tensor([1, 50, 7], device="cuda")[:, None, None]
    qo, ko = apply_fused_qk_head_rmsnorm_rotary(q, k, *norms, rotary, pos[..., 0].int())
    _close(qo, _want(q, rotary, pos, weight=norms[0].weight, eps=1e-6))
    _close(ko, _want(k, rotary, pos, weight=norms[1].weight, eps=1e-5))
    assert bool((qo[0, 0, 0] == 0).all())
    qn, none = apply_fused_qk_head_rmsnorm_rotary(q, None, norms[0], None, None)
    assert none is None
    _close(qn, _want(q, weight=norms[0].weight, eps=1e-6))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim", [(44, 40), (80, 12), (16, 8), (24, 6), (60, 60), (6, 2)])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_every_width_of_reads(dtype, layout, dim, rotary_dim, offset):
    """Heads and weights that allow 16, 8 and 4 bytes at a time or single values, with
    plain channels beside turned ones in a lane; infinities in plain channels of the
    rotation stay."""
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(dim, rotary_dim=rotary_dim, layout=layout)
    q, k = _randn((2, 11, 7, dim), dtype, 13), _randn((2, 11, 2, dim), dtype, 14)
    norms = []
    for seed in (15, 16):
        n = torch.nn.RMSNorm(dim, eps=1e-6, device="cuda", dtype=dtype).requires_grad_(False)
        n.weight.data = _randn((dim + 8,), dtype, seed)[offset:offset + dim]
        norms.append(n)
    pos = _pos(2, 11, start=70)
    qo, ko = apply_fused_qk_head_rmsnorm_rotary(q, k, *norms, rotary, 70)
    _close(qo, _want(q, rotary, pos, weight=norms[0].weight, eps=1e-6))
    _close(ko, _want(k, rotary, pos, weight=norms[1].weight, eps=1e-6))
    wide = _randn((2, 11, 7, dim + 8), dtype, 17)
    q = wide[..., offset:offset + dim]
    if rotary_dim < dim:
        q[0, 0, 0, rotary_dim:] = math.inf
    qo, ko = apply_rotary(q, k, rotary, 70)
    _close(qo[1], tuple(t[1] for t in _want(q, rotary, pos)))
    _close(qo[..., :rotary_dim], tuple(t[..., :rotary_dim] for t in _want(q, rotary, pos)))
    _close(ko, _want(k, rotary, pos))
    assert torch.equal(qo[..., rotary_dim:], q[..., rotary_dim:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(4600, 61, 17), (2501, 157, 13), (9500, 62, 0)])
def test_many_heads_of_many_tokens(layout, norm, tokens, heads, kv_heads):
    """Warps that walk over eleven or eight head groups, one or two warps a token, with
    the keys behind the queries of one of them, in place."""
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64, layout=layout)
    q = _randn((1, tokens, heads, 64), torch.bfloat16, 18)
    k = _randn((1, tokens, kv_heads, 64), torch.bfloat16, 19) if kv_heads else None
    q0, k0 = q.clone(), None if k is None else k.clone()
    w, eps = None, None
    if norm:
        n = torch.nn.RMSNorm(64, eps=1e-6, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
        n.weight.copy_(_randn((64,), torch.float32, 20))
        w, eps = n.weight, 1e-6
        apply_fused_qk_head_rmsnorm_rotary(q, k, n, n, rotary, 3, query_out=q, key_out=k)
    else:
        apply_rotary(q, k, rotary, 3, query_out=q, key_out=k)
    pos = _pos(1, tokens, start=3)
    _close(q, _want(q0, rotary, pos, weight=w, eps=eps))
    if k is not None:
        _close(k, _want(k0, rotary, pos, weight=w, eps=eps))


@pytest.mark.parametrize("tokens", [1, 2, 33, 1777])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (32, 8), (33, 1)])
def test_views_of_a_projection_buffer_in_place(tokens, heads, kv_heads):
    """Heads inside an interleaved Q|K|V buffer, turned in place; V and the
    neighbouring bytes stay."""
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64)
    buf = _randn((2, tokens, (heads + 2 * kv_heads) * 64), torch.bfloat16, 9)
    before = buf.clone()
    view = lambda t, h0, n: t[..., h0 * 64:(h0 + n) * 64].unflatten(-1, (n, 64))
    q, k = view(buf, 0, heads), view(buf, heads, kv_heads)
    qo, ko = apply_rotary(q, k, rotary, 5, query_out=q, key_out=k)
    assert qo.data_ptr() == q.data_ptr()
    pos = _pos(2, tokens, start=5)
    _close(view(buf, 0, heads), _want(view(before, 0, heads), rotary, pos))
    _close(view(buf, heads, kv_heads), _want(view(before, heads, kv_heads), rotary, pos))
    assert torch.equal(buf[..., (heads + kv_heads) * 64:], before[..., (heads + kv_heads) * 64:])


@pytest.mark.parametrize("offset,dim", [(1, 64), (4, 64), (8, 60)])
def test_unaligned_rows(offset, dim):
    """Heads that start off a 16-byte boundary go value by value."""
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(dim)
    buf = _randn((2, 5, 3, dim + 13), torch.float16, 11)
    q = buf[..., offset:offset + dim]
    qo, _ = apply_rotary(q, None, rotary, 2)
    _close(qo, _want(q, rotary, _pos(2, 5, start=2)))


def test_orders_and_broadcast_inputs():
    """BHSD storage, and one head expanded over eight."""
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64, layout="interleaved")
    q = _randn((2, 6, 50, 64), torch.bfloat16, 12).transpose(1, 2)
    k = _randn((2, 50, 1, 64), torch.bfloat16, 13).expand(2, 50, 8, 64)
    pos = _pos(2, 50)
    qo, ko = apply_rotary(q, k, rotary, pos[..., 0])
    _close(qo, _want(q, rotary, pos))
    _close(ko, _want(k, rotary, pos))
    with pytest.raises(ValueError):
        apply_rotary(q, k, rotary, 0, key_out=k)  # an expanded destination


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 8.0},
                                     {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 8.0, "original_length": 4096}])
@pytest.mark.parametrize("start", [0, 10 ** 6, 2 ** 31 - 4, -(2 ** 31), 2 ** 40 + 1])
def test_far_positions(scaling, start):
    """FP32 outputs hold their tolerance at any position (the 64-bit reference
    itself is off by |angle| 2^-53: 2^-12 at 2^40, so that start is compared
    through the reduced turns)."""
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64, scaling=scaling)
    q = _randn((1, 8, 2, 64), torch.float32, 14)
    pos = torch.arange(8, device="cuda")[None, :, None] + start
    got, _ = apply_rotary(q, None, rotary, pos[0, :, 0])
    again, _ = apply_rotary(q, None, rotary, start)
    assert torch.equal(got, again)
    if abs(start) < 2 ** 33:
        # 2^31 radians: the 64-bit angle of the reference and the kernel's turns
        # are each within 2^31 * 2^-52 < 2^-20, below what FP32 angles cost
        want, tol = _want(q, rotary, pos)
        _close(got, (want, tol + 2.0 ** -20 * q.abs().max()))
        if start <= 10 ** 6:
            _close(got, (want, tol))
    else:
        turned = got.double()[..., :32] ** 2 + got.double()[..., 32:] ** 2
        kept = (q.double()[..., :32] ** 2 + q.double()[..., 32:] ** 2) * rotary.amplitude ** 2
        assert torch.allclose(turned, kept, rtol=1e-5)


@pytest.mark.parametrize("axes_dim", [(64,), (40, 24), (24, 20, 20), (2, 60, 2)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("per_batch", [False, True])
def test_position_axes(axes_dim, layout, per_batch):
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64, layout=layout, axes_dim=axes_dim)
    n = len(axes_dim)
    q = _randn((2, 30, 4, 64), torch.float32, 15)
    g = torch.Generator(device="cuda").manual_seed(16)
    pos = torch.randint(0, 60, (n, 2 if per_batch else 1, 30), generator=g, device="cuda")
    given = pos if n > 1 else pos[0]
    got, _ = apply_rotary(q, None, rotary, given if per_batch else given.squeeze(-2))
    _close(got, _want(q, rotary, pos.permute(1, 2, 0).expand(2, 30, n)))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_transpose_and_the_gradient(layout):
    """<R x, y> = <x, R^T y>, and R^T is what autograd gives for the formula and
    what central differences give for the kernel."""
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(48, rotary_dim=32, layout=layout)
    x, y = _randn((2, 9, 3, 48), torch.float32, 17), _randn((2, 9, 3, 48), torch.float32, 18)
    rx, _ = apply_rotary(x, None, rotary, 100)
    rty, _ = apply_rotary(y, None, rotary, 100, inverse=True)
    a, b = (rx.double() * y.double()).sum(), (x.double() * rty.double()).sum()
    assert abs(float(a - b)) <= 4 * ROTATE * float((x.double().abs() * y.double().abs()).sum() * 2)
    leaf = x.double().requires_grad_()
    out, _ = _want(leaf, rotary, _pos(2, 9, start=100))
    grad, = torch.autograd.grad(out, leaf, y.double())
    _, tol = _want(y, rotary, _pos(2, 9, start=100), inverse=True)
    _close(rty, (grad, tol))
    # central differences of the kernel along a random direction (it is linear,
    # so a step of 1 has no truncation error)
    d = _randn(x.shape, torch.float32, 19)
    up, _ = apply_rotary(x + d, None, rotary, 100)
    down, _ = apply_rotary(x - d, None, rotary, 100)
    slope = ((up.double() - down.double()) / 2 * y.double()).sum()
    assert abs(float(slope - (d.double() * rty.double()).sum())) <= \
        8 * ROTATE * float(((x.abs() + d.abs()).double() * y.abs().double()).sum() * 2)


def test_values_beyond_the_range_stay_theirs():
    """An infinity or NaN touches its own pair (rotation) or head (norm) only."""
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64)
    q = _randn((1, 4, 8, 64), torch.bfloat16, 20)
    clean, _ = apply_rotary(q, None, rotary, 3)
    norm = torch.nn.RMSNorm(64, eps=1e-6, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    clean_n, _ = apply_fused_qk_head_rmsnorm_rotary(q, None, norm, None, rotary, 3)
    bad = q.clone()
    bad[0, 2, 5, 7] = math.inf
    bad[0, 1, 0, 40] = math.nan
    got, _ = apply_rotary(bad, None, rotary, 3)
    keep = torch.ones_like(q, dtype=torch.bool)
    keep[0, 2, 5, [7, 39]] = False
    keep[0, 1, 0, [8, 40]] = False
    assert torch.equal(got[keep], clean[keep]) and not bool(torch.isfinite(got[~keep]).any())
    got, _ = apply_fused_qk_head_rmsnorm_rotary(bad, None, norm, None, rotary, 3)
    keep[0, 2, 5] = False
    keep[0, 1, 0] = False
    assert torch.equal(got[keep], clean_n[keep])


def test_empty_inputs_and_refusals():
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64)
    z = torch.zeros(2, 0, 4, 64, device="cuda", dtype=torch.bfloat16)
    q, _ = apply_rotary(z, z, rotary, 0)
    assert q.shape == z.shape
    x = torch.zeros(2, 6, 4, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.zeros(6, device="cuda", dtype=torch.int64)
    bad = [dict(query=x[0]), dict(query=x.double()), dict(query=x.transpose(2, 3)),
           dict(key=x.half()), dict(key=x[:, :5]), dict(key=x[..., :32]), dict(rotary=None),
           dict(positions=pos.float()), dict(positions=pos[:5]), dict(positions=pos.cpu()),
           dict(positions=pos[None].expand(3, 6)), dict(query_out=x[:1]),
           dict(query_out=x.half()), dict(key=None, key_out=x),
           dict(rotary=RotaryPositions(128)), dict(rotary=RotaryPositions(64, axes_dim=(32, 32)))]
    for kw in bad:
        args = dict(dict(query=x, key=x, rotary=rotary, positions=pos), **kw)
        extra = {n: args.pop(n) for n in ("query_out", "key_out") if n in args}
        if args["rotary"] is None:
            continue
        with pytest.raises(ValueError):
            apply_rotary(args["query"], args["key"], args["rotary"], args["positions"], **extra)
    with pytest.raises(ValueError):
        apply_rotary(x.float().requires_grad_(), None, rotary, 0)
    with torch.no_grad():
        apply_rotary(x.float().requires_grad_(), None, rotary, 0)
    norm = lambda d, **kw: torch.nn.RMSNorm(d, device="cuda", **kw).requires_grad_(False)
    for n in (norm(32), norm(64, dtype=torch.float16),
              torch.nn.LayerNorm(64, device="cuda").requires_grad_(False)):
        with pytest.raises(ValueError):
            apply_fused_qk_head_rmsnorm_rotary(x, None, n, None, rotary, 0)
    with pytest.raises(ValueError):  # two weight types
        apply_fused_qk_head_rmsnorm_rotary(x, x, norm(64), norm(64, dtype=torch.bfloat16), rotary, 0)


def test_another_stream_and_a_replayed_graph():
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import RotaryPositions
    rotary = RotaryPositions(64)
    norm = torch.nn.RMSNorm(64, eps=1e-6, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    q, k = _randn((2, 40, 8, 64), torch.bfloat16, 21), _randn((2, 40, 2, 64), torch.bfloat16, 22)
    pos = torch.arange(40, device="cuda")
    want = apply_fused_qk_head_rmsnorm_rotary(q, k, norm, norm, rotary, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = apply_fused_qk_head_rmsnorm_rotary(q, k, norm, norm, rotary, pos)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_fused_qk_head_rmsnorm_rotary(q, k, norm, norm, rotary, pos)
    q.copy_(_randn(q.shape, q.dtype, 23))
    pos += 9
    graph.replay()
    want = apply_fused_qk_head_rmsnorm_rotary(q, k, norm, norm, rotary, pos)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_offsets_beyond_32_bits():
    """A batch stride of 2^32 elements (an 8.6 GB buffer)."""
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64)
    far = 2 ** 32
    buf = torch.empty(far + 4 * 128, device="cuda", dtype=torch.bfloat16)
    q = buf.as_strided((2, 4, 2, 64), (far, 128, 64, 1))
    src = _randn((2, 4, 2, 64), torch.bfloat16, 24)
    q.copy_(src)
    got, _ = apply_rotary(q, None, rotary, 1, query_out=q)
    _close(got, _want(src, rotary, _pos(2, 4, start=1)))
    del buf, q, got
    torch.cuda.empty_cache()


def test_overlapping_destinations_are_refused():
    from eraserdit_b200.rotary import RotaryPositions, apply_rotary
    rotary = RotaryPositions(64)
    buf = _randn((2, 6, 8 * 64), torch.bfloat16, 25)
    heads = lambda a, b: buf[..., a * 64:b * 64].unflatten(-1, (b - a, 64))
    apply_rotary(heads(0, 2), heads(2, 4), rotary, 0, query_out=heads(4, 6), key_out=heads(6, 8))
    for kw in (dict(query_out=heads(1, 3)), dict(query_out=heads(2, 4)), dict(key_out=heads(0, 2)),
               dict(query_out=heads(4, 6), key_out=heads(5, 7))):
        with pytest.raises(ValueError):
            apply_rotary(heads(0, 2), heads(2, 4), rotary, 0, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rms", [1e-4, 0.05, 1.0])
def test_a_norm_with_torchs_default_eps(dtype, rms):
    """torch.nn.RMSNorm(D) without eps: FP32's epsilon for every type, as torch computes it."""
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    eps = torch.finfo(torch.float32).eps
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=dtype).requires_grad_(False)
    norm.weight.copy_(_randn((64,), torch.float32, 25))
    q, k = (rms * _randn((2, 6, 3, 64), torch.float32, s).to(dtype) for s in (26, 27))
    qo, ko = apply_fused_qk_head_rmsnorm_rotary(q, k, norm, norm, None)
    for x, y in ((q, qo), (k, ko)):
        _close(y, _want(x, weight=norm.weight, eps=eps))
        # torch's own result: one more rounding where it rounds before the weight
        torchs = torch.nn.functional.rms_norm(x, (64,), norm.weight).double()
        assert bool(((y.double() - torchs).abs() <= 2 * torch.finfo(dtype).eps * torchs.abs()
                     + 4 * NORM * torchs.abs() + 1e-30).all())


def test_norms_without_an_eps_are_refused():
    """Nothing stands in for an epsilon that goes by another name, or for no norm."""
    from types import SimpleNamespace
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    x = torch.zeros(2, 6, 4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    good = SimpleNamespace(weight=w, eps=1e-6)
    apply_fused_qk_head_rmsnorm_rotary(x, x, good, good, None)
    for bad in (None, SimpleNamespace(weight=w), SimpleNamespace(weight=w, eps=None),
                SimpleNamespace(weight=w, variance_epsilon=1e-6)):
        with pytest.raises(ValueError):
            apply_fused_qk_head_rmsnorm_rotary(x, x, bad, good, None)
        with pytest.raises(ValueError):
            apply_fused_qk_head_rmsnorm_rotary(x, x, good, bad, None)


def test_what_is_no_rms_norm_of_one_head_is_refused():
    """Norms that subtract a mean, or that go over more or fewer channels than a head has,
    also where no weight's shape shows it."""
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    x = torch.zeros(2, 6, 4, 64, device="cuda", dtype=torch.bfloat16)
    kw = dict(device="cuda", dtype=torch.bfloat16)
    good = torch.nn.RMSNorm(64, elementwise_affine=False, **kw)
    apply_fused_qk_head_rmsnorm_rotary(x, x, good, good, None)
    for bad in (torch.nn.LayerNorm(64, bias=False, **kw), torch.nn.LayerNorm(64, elementwise_affine=False, **kw),
                torch.nn.GroupNorm(1, 64, affine=False, **kw), torch.nn.BatchNorm1d(64, affine=False, **kw),
                torch.nn.RMSNorm(32, elementwise_affine=False, **kw),
                torch.nn.RMSNorm((4, 64), elementwise_affine=False, **kw)):
        for p in bad.parameters():
            p.requires_grad_(False)
        for pair in ((bad, good), (good, bad)):
            with pytest.raises(ValueError):
                apply_fused_qk_head_rmsnorm_rotary(x, x, *pair, None)


def test_a_rotation_without_positions_is_refused():
    """None stands for the norm alone, in the operator that has a norm."""
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import apply_rotary
    x = torch.zeros(2, 6, 4, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        apply_rotary(x, x, None, 0)
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    apply_fused_qk_head_rmsnorm_rotary(x, x, norm, norm, None)
