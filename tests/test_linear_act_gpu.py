"""linear_act (erd_linear_act) against the formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def _operands(m, n, k, dtype, seed, bias=True, groups=0, residual=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w = r(m, k).to(dtype), (r(n, k) * k ** -0.5).to(dtype)
    b = (r(n) * 0.5).to(dtype) if bias else None
    gate = r(groups, n).to(dtype) if groups else None
    res = r(m, n).to(dtype) if residual else None
    return x, w, b, gate, res


def _act(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def _check(got, x, w, b, act, gate, res):
    """Every value within one rounding plus what FP32 sums cost, and the whole
    within one rounding."""
    k = x.shape[-1]
    xd, wd = x.double().flatten(0, -2), w.double()
    v = xd @ wd.T
    # k products (exact in FP32) meet the accumulator with at most one FP32
    # truncation (2^-23) each, of sums that stay below sum |x| |w|
    tol = k * 2.0 ** -23 * (xd.abs() @ wd.abs().T)
    if b is not None:
        v = v + b.double()
    y = _act(v, act)
    # |act'| < 1.13; the FP32 activations are good to 2^-20 of their argument
    tol = 1.13 * tol + 2.0 ** -20 * v.abs()
    if gate is not None:
        g = gate.double().view(-1, y.shape[1]).repeat_interleave(y.shape[0] // max(1, gate.numel() // y.shape[1]), 0)
        y, tol = y * g, tol * g.abs()
    if res is not None:
        y = y + res.double().flatten(0, -2)
    fi = torch.finfo(got.dtype)
    got = got.double().flatten(0, -2)
    half = (y.abs() * fi.eps / 2).clamp(min=fi.smallest_normal * fi.eps / 2)
    bad = ((got - y).abs() > (half + tol) * 1.001 + 2.0 ** -22 * y.abs()) | torch.isnan(got)
    assert int(bad.sum()) == 0, f"{int(bad.sum())} of {bad.numel()} values off"
    assert float((got - y).norm()) <= float(y.norm()) * (fi.eps / 2 + 2.0 ** -16) + 1e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 64), (1, 8192, 2048), (3, 7, 40), (8, 1999, 1048),
                                   (9, 256, 8192), (77, 130, 72), (127, 64, 512), (128, 65, 520),
                                   (129, 512, 2048), (300, 1000, 200), (640, 2048, 1024)])
def test_small_products(m, n, k, dtype):
    """Tails in every dimension, one to several parts of the reduction."""
    from eraserdit_b200 import _native
    from eraserdit_b200.linear import linear_act
    if k % 8 and m > 1:
        pytest.skip("k is a row stride")
    x, w, b, _, _ = _operands(m, n, k, dtype, m + n + k)
    if k % 8:  # one row each: no stride follows
        w = w[:1]
        b = b[:1]
    got = linear_act(x, w, b, activation="silu")
    assert _native.read_status(x.device) == 0
    _check(got, x, w, b, "silu", None, None)


@pytest.mark.parametrize("m,n,k", [(2500, 2304, 264), (5000, 2048, 1000), (65280, 264, 64), (257, 38000, 128),
                                   (4097, 2055, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_products(m, n, k, dtype):
    """256-row tiles with ragged edges, one and several tiles a CTA pair."""
    from eraserdit_b200 import _native
    from eraserdit_b200.linear import linear_act
    x, w, b, gate, res = _operands(m, n, k, dtype, m + n, groups=1, residual=True)
    got = linear_act(x, w, b, activation="gelu_tanh", gate=gate[0], residual=res)
    assert _native.read_status(x.device) == 0
    _check(got, x, w, b, "gelu_tanh", gate, res)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 20, 200, 3000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias,groups,residual", [(False, 0, False), (True, 1, False), (False, 4, True),
                                                  (True, 0, True)])
def test_epilogues(act, m, dtype, bias, groups, residual):
    """Every activation with every mixture of the other parts; the gate's groups
    (m / 4 rows) also end inside a tile and inside a warp's rows."""
    from eraserdit_b200.linear import linear_act
    groups = groups if groups and m % groups == 0 else min(groups, 1)
    x, w, b, gate, res = _operands(m, 1544, 320, dtype, m + 1, bias, groups, residual)
    x *= 3  # arguments out to the tails of the activations
    got = linear_act(x, w, b, activation=act, gate=gate, residual=res)
    _check(got, x, w, b, act, gate, res)


@pytest.mark.parametrize("act", ACTS)
def test_activation_values_far_out(act):
    """x W^T is the argument itself (a one-hot weight): the activations' values
    from -60000 to 60000, beyond the range where exponentials overflow."""
    from eraserdit_b200.linear import linear_act
    v = torch.cat([torch.linspace(-12, 12, 481), torch.tensor([-6e4, -300.0, -100.0, -90.0, 90.0, 100.0,
                                                               300.0, 6e4])]).half().cuda()
    x = torch.zeros(v.numel(), 64, device="cuda", dtype=torch.float16)
    x[:, 5] = v
    w = torch.zeros(8, 64, device="cuda", dtype=torch.float16)
    w[:, 5] = 1
    got = linear_act(x, w, activation=act)
    want = _act(v.double(), act)[:, None].expand(-1, 8)
    fi = torch.finfo(torch.float16)
    half = (want.abs() * fi.eps / 2).clamp(min=fi.smallest_normal * fi.eps / 2)
    # the exponent's argument is good to 2^-24 of itself, at most 2^-24 * 64 where the
    # result is above FP16's smallest value
    assert bool(((got.double() - want).abs() <= (half + want.abs() * 2.0 ** -17) * 1.001).all())


@pytest.mark.parametrize("m", [5, 3000])
def test_views_and_in_place_residual(m):
    """x inside a wider buffer, an output with an odd row stride, and the result
    written over the residual; nothing else is written."""
    from eraserdit_b200.linear import linear_act
    x, w, b, gate, res = _operands(m, 1100, 320, torch.bfloat16, 3, groups=1, residual=True)
    wide = torch.randn(m, 1024, device="cuda").bfloat16()
    wide[:, 512:832] = x
    wcut = torch.randn(1100, 400, device="cuda").bfloat16()
    wcut[:, 80:400] = w
    for off, width in ((0, 1112), (3, 1107)):
        buf = torch.full((m, width), 7.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:, off:off + 1100]
        linear_act(wide[:, 512:832], wcut[:, 80:400], b, gate=gate, residual=res, out=out)
        _check(out, x, w, b, "none", gate, res)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[:, off:off + 1100] = False
        assert bool((buf[mask] == 7.0).all())
    own = res.clone()
    assert linear_act(x, w, b, residual=own, out=own) is own
    _check(own, x, w, b, "none", None, res)


@pytest.mark.parametrize("m", [37, 200, 3001])
@pytest.mark.parametrize("n", [65, 190, 1099, 1102])
@pytest.mark.parametrize("res_at", [(0, 0), (2, 6), (1, 5), (3, 4)])
@pytest.mark.parametrize("out_at", [(0, 0), (2, 6), (1, 5)])
def test_rows_on_two_and_four_bytes(m, n, res_at, out_at):
    """Residual and result whose rows start on 4 bytes or on 2, with even and odd
    strides and numbers of columns; what lies around the result stays."""
    from eraserdit_b200.linear import linear_act
    x, w, b, gate, res = _operands(m, n, 136, torch.float16, m + n, groups=1, residual=True)
    (ro, rp), (oo, op) = res_at, out_at  # columns in front, and in front and behind together
    wide = torch.full((m, n + rp), 9.0, device="cuda", dtype=torch.float16)
    wide[:, ro:ro + n] = res
    buf = torch.full((m, n + op), 7.0, device="cuda", dtype=torch.float16)
    out = buf[:, oo:oo + n]
    linear_act(x, w, b, activation="silu", gate=gate, residual=wide[:, ro:ro + n], out=out)
    _check(out, x, w, b, "silu", gate, res)
    assert bool((buf[:, :oo] == 7.0).all()) and bool((buf[:, oo + n:] == 7.0).all())


def test_leading_dimensions_and_slots():
    from eraserdit_b200.linear import linear_act
    x, w, b, gate, res = _operands(2 * 70, 136, 128, torch.bfloat16, 4, groups=2, residual=True)
    want = linear_act(x, w, b, activation="gelu", gate=gate, residual=res)
    got = linear_act(x.view(2, 7, 10, 128), w, b, activation="gelu", gate=gate,
                     residual=res.view(2, 7, 10, 136))
    assert got.shape == (2, 7, 10, 136) and torch.equal(got.view(-1, 136), want)
    part = linear_act(x.view(2, 70, 128)[:, :33], w, b, activation="gelu", gate=gate,
                      residual=res.view(2, 70, 136)[:, :33])
    for i in range(2):
        _check(part[i], x.view(2, 70, 128)[i, :33], w, b, "gelu", gate[i:i + 1], res.view(2, 70, 136)[i, :33])
    one = linear_act(x[0], w, b)
    assert one.shape == (136,)
    _check(one[None], x[:1], w, b, "none", None, None)


def test_the_same_call_gives_the_same_bits():
    """The parts of a reduction are added in one order."""
    from eraserdit_b200.linear import linear_act
    for m, n, k in ((7, 2048, 8192), (3000, 1024, 512)):
        x, w, b, _, _ = _operands(m, n, k, torch.bfloat16, 6)
        first = linear_act(x, w, b)
        for _ in range(20):
            assert torch.equal(linear_act(x, w, b), first)


def test_infinities_and_nan_stay_in_their_rows_and_columns():
    from eraserdit_b200.linear import linear_act
    for m in (9, 2600):
        x, w, b, _, _ = _operands(m, 2049, 136, torch.bfloat16, 7)
        clean = linear_act(x, w, b)
        x2, w2 = x.clone(), w.clone()
        x2[m - 1, 135] = math.nan
        w2[2048, 3] = math.inf
        got = linear_act(x2, w2, b)
        assert torch.equal(got[:-1, :-1], clean[:-1, :-1])
        assert not bool(torch.isfinite(got[-1]).any()) and not bool(torch.isfinite(got[:, -1]).any())


def test_streams_and_graphs():
    from eraserdit_b200.linear import linear_act
    cases = [_operands(m, 2048, 1024, torch.bfloat16, m, residual=True) for m in (1, 130, 3000)]
    side = torch.cuda.Stream()
    for x, w, b, _, res in cases:
        want = linear_act(x, w, b, activation="silu", residual=res)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = linear_act(x, w, b, activation="silu", residual=res)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_act(x, w, b, activation="silu", residual=res)
        x.mul_(-0.5)
        graph.replay()
        assert torch.equal(out, linear_act(x, w, b, activation="silu", residual=res))
    # two at once
    (x1, w1, b1, _, r1), (x2, w2, b2, _, r2) = cases[1], cases[2]
    want1, want2 = linear_act(x1, w1, b1, residual=r1), linear_act(x2, w2, b2, residual=r2)
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):
        with torch.cuda.stream(side):
            outs.append((linear_act(x1, w1, b1, residual=r1), want1))
        outs.append((linear_act(x2, w2, b2, residual=r2), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)


def test_offsets_beyond_32_bits():
    """An output of 2^31 + values (a 4.3 GB buffer) is right in its last rows."""
    from eraserdit_b200.linear import linear_act
    m, n = 270000, 8200
    x, w, b, _, _ = _operands(m, n, 8, torch.bfloat16, 8)
    assert m * n > 2 ** 31
    got = linear_act(x, w, b)
    _check(got[-300:], x[-300:], w, b, "none", None, None)
    _check(got[:300], x[:300], w, b, "none", None, None)


def test_empty_and_refusals():
    from eraserdit_b200.linear import linear_act
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, w, b = torch.zeros(6, 64, **bf), torch.zeros(16, 64, **bf), torch.zeros(16, **bf)
    assert linear_act(x[:0], w, b).shape == (0, 16)
    assert linear_act(x, w[:0]).shape == (6, 0)
    res = torch.zeros(6, 16, **bf)
    for args, kw in [((x.float(), w), {}), ((x, w.half()), {}), ((x, w[:, :32]), {}), ((x, w, b[:8]), {}),
                     ((x, w, b), dict(activation="tanh")), ((x, w, b), dict(residual=res[:, :8])),
                     ((x, w, b), dict(gate=torch.zeros(4, 16, **bf))),
                     ((x, w, b), dict(gate=torch.zeros(2, 3, 16, **bf))),
                     ((x, w, b), dict(out=res.float())), ((x, w, b), dict(out=res[:1].expand(6, 16))),
                     ((x[:, :60], w[:, :60].contiguous(), b), {}),  # rows of W not on 16 bytes
                     ((torch.zeros(6, 65, **bf)[:, 1:], w, b), {}),
                     ((x.t()[:, :6].contiguous().t(), w[:, :], b), {}),  # strided last dimension
                     ((x[:, :0], w[:, :0]), {}), ((x, w.cpu()), {})]:
        with pytest.raises(ValueError):
            linear_act(*args, **kw)
    with pytest.raises(ValueError):
        linear_act(x, w.clone().requires_grad_(), b)
    with torch.no_grad():
        linear_act(x, w.clone().requires_grad_(), b)


def test_overlapping_destinations_are_refused():
    """The result may replace the residual, but nothing that other tiles still read."""
    from eraserdit_b200.linear import linear_act
    buf = torch.zeros(300, 256, device="cuda", dtype=torch.bfloat16)
    x, w = buf[:, :128], torch.zeros(128, 128, device="cuda", dtype=torch.bfloat16)
    linear_act(x, w, out=buf[:, 128:])  # other columns of the same rows
    for kw in (dict(out=x), dict(out=buf[:, 64:192]), dict(out=buf[:, 128:], residual=buf[:, 120:248]),
               dict(residual=buf[:1, :128].expand(300, 128))):
        with pytest.raises(ValueError):
            linear_act(x, w, **kw)
    with pytest.raises(ValueError):
        linear_act(x[:1].expand(300, 128), w)
    with pytest.raises(ValueError):
        linear_act(x[:128], w, out=w)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 20, 3000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activations_of_infinities_and_nan(act, m, dtype):
    """From an operand, from the bias and from a product that leaves FP32's range: what
    the formula gives (+inf stays +inf under every activation)."""
    from eraserdit_b200.linear import linear_act
    values = torch.tensor([math.inf, -math.inf, math.nan, 1.0, -1.0, 0.0, 40.0, -40.0], device="cuda").to(dtype)
    x = torch.zeros(m, 64, device="cuda", dtype=dtype)
    w = torch.zeros(8, 64, device="cuda", dtype=dtype)
    bias = values.clone()

    def check(got, v):
        want = _act(v.double(), act).expand(m, -1).to(dtype)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got.sign()[want.isinf()], want.sign()[want.isinf()])
        finite = want.isfinite()
        assert torch.allclose(got[finite].double(), want[finite].double(), rtol=0.01, atol=1e-6)

    check(linear_act(x, w, bias, activation=act), bias)
    x[:, 3] = 1
    w[:, 3] = values
    check(linear_act(x, w, activation=act), values)
    if dtype == torch.bfloat16:
        x[:, 3], w[:, 3] = 3e38, torch.tensor([3e38, -3e38, 1, 2, 3, 4, 5, 6], device="cuda").to(dtype)
        got = linear_act(x, w, activation=act)
        assert bool((got[:, 0] == math.inf).all())
        assert bool((got[:, 1] == 0).all() if act == "relu" else (~got[:, 1].isfinite()).all())


@pytest.mark.parametrize("lead,groups", [(4, 1), (4, 2), (4, 4), (4, 8), (3, 6)])
def test_gates_of_slots(lead, groups):
    """Rows that no single stride walks (prefixes of wider slots), with every number of
    gate groups that the rows divide into at a slot's end or within one."""
    from eraserdit_b200.linear import linear_act
    x, w, b, gate, res = _operands(lead * 30, 136, 128, torch.bfloat16, 31, groups=groups, residual=True)
    wide = torch.randn(lead, 50, 128, device="cuda").bfloat16()
    wide[:, :30] = x.view(lead, 30, 128)
    got = linear_act(wide[:, :30], w, b, activation="silu", gate=gate, residual=res.view(lead, 30, 136))
    assert got.shape == (lead, 30, 136)
    _check(got, x, w, b, "silu", gate, res)
    # two leading dimensions
    if lead == 4:
        deep = wide.view(2, 2, 50, 128)[:, :, :30]
        again = linear_act(deep, w, b, activation="silu", gate=gate, residual=res.view(2, 2, 30, 136))
        assert torch.equal(again.view(lead, 30, 136), got)


def test_gate_groups_across_slots_are_refused():
    from eraserdit_b200.linear import linear_act
    wide = torch.zeros(3, 50, 128, device="cuda", dtype=torch.bfloat16)
    w, gate = (torch.zeros(s, 128, device="cuda", dtype=torch.bfloat16) for s in (128, 2))
    with pytest.raises(ValueError):
        linear_act(wide[:, :30], w, gate=gate)  # 45 rows each: one and a half slots
    linear_act(wide[:, :30].contiguous(), w, gate=gate)
