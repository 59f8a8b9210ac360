"""Host side of the head rotation: frequencies, refusals and the C entry's
argument errors (no GPU)."""
import ctypes
import math

import pytest
import torch


def test_frequencies_follow_their_formulas():
    from eraserdit_b200.rotary import rotary_frequencies
    f, a = rotary_frequencies(8, 10000.0)
    want = torch.tensor([10000.0 ** (-2 * i / 8) for i in range(4)], dtype=torch.float64)
    assert a == 1.0 and torch.allclose(f, want, rtol=1e-14, atol=0)
    assert torch.allclose(rotary_frequencies(8, scaling={"type": "linear", "factor": 4})[0],
                          want / 4, rtol=1e-14, atol=0)
    ntk, _ = rotary_frequencies(8, scaling={"type": "ntk", "factor": 8})
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(want[-1]) / 8, rel_tol=1e-12)
    spec = {"type": "yarn", "factor": 16, "original_length": 4096}
    yarn, amp = rotary_frequencies(64, scaling=spec)
    plain, _ = rotary_frequencies(64)
    assert math.isclose(amp, 0.1 * math.log(16) + 1)
    turns = plain * 4096 / (2 * math.pi)  # turns of each pair within the trained length
    ratio = plain / yarn
    # one pair index of rounding on either side of the ramp's ends
    fast = turns >= 32 * 10000.0 ** (2 / 64)
    slow = turns <= 10000.0 ** (-2 / 64)
    assert bool((ratio[fast] == 1).all()) and int(fast.sum()) > 0
    assert torch.allclose(ratio[slow], torch.full_like(ratio[slow], 16.0)) and int(slow.sum()) > 0
    assert bool((ratio[1:] >= ratio[:-1]).all())  # monotone between
    assert rotary_frequencies(64, scaling=dict(spec, attention_factor=1.5))[1] == 1.5


@pytest.mark.parametrize("dim,scaling", [
    (0, None), (7, None), (8, {"type": "cubic", "factor": 2}), (8, {"type": "linear"}),
    (8, {"type": "linear", "factor": 0.5}), (8, {"type": "linear", "factor": math.inf}),
    (2, {"type": "ntk", "factor": 2}), (8, {"type": "yarn", "factor": 2}),
    (8, {"type": "yarn", "factor": 2, "original_length": 10, "beta_fast": 1, "beta_slow": 2}),
    (8, {"type": "linear", "factor": 2, "original_length": 10})])
def test_frequencies_refuse(dim, scaling):
    from eraserdit_b200.rotary import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(dim, scaling=scaling)


@pytest.mark.parametrize("kw", [dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=31),
                                dict(head_dim=1026), dict(head_dim=64, layout="both"),
                                dict(head_dim=64, axes_dim=(32, 16)),
                                dict(head_dim=64, axes_dim=(16, 16, 16, 16)),
                                dict(head_dim=64, axes_dim=(31, 33)),
                                dict(head_dim=64, device="cpu")])
def test_rotary_positions_refuse(kw):
    from eraserdit_b200.rotary import RotaryPositions
    with pytest.raises(ValueError):
        RotaryPositions(**kw)


def test_host_tensors_are_refused():
    from eraserdit_b200.operator_fusion import apply_fused_qk_head_rmsnorm_rotary
    from eraserdit_b200.rotary import apply_rotary
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(ValueError):
        apply_rotary(x, None, None, 0)
    norm = torch.nn.RMSNorm(64)
    with pytest.raises(ValueError):
        apply_fused_qk_head_rmsnorm_rotary(x, x, norm, norm, None)


def test_entry_rejects_bad_arguments_before_any_device_call():
    from eraserdit_b200 import _native
    fn = _native.load().erd_head_norm_rotary
    p = 1 << 20

    def call(dtype=0, q=p, k=p, batch=1, tokens=1, heads=1, kv_heads=1, dim=64, rotary=64,
             turns=p, q_out=p, k_out=p, weight=None, weight_fp32=0, pos=None, wide=0):
        fields = (q, k, weight, weight, turns, pos, q_out, k_out, *([64] * 12), 0, 0, 1, 0, dtype,
                  batch, tokens, heads, kv_heads, dim, rotary, 0, 1, weight_fp32, 0, rotary // 2,
                  rotary // 2, wide, 1e-6, 1e-6, 1.0)
        return fn(_native.pack("erd_head_norm_rotary", *(0 if f is None else f for f in fields)), None)

    assert fn(None, None) == -1
    assert fn(_native.STRUCTS["erd_head_norm_rotary"].pack(8, *([0] * 41)), None) == -2  # another struct
    with pytest.raises(ValueError):
        call(tokens=2 ** 31)
    assert call(q=None) == -1 and call(q_out=None) == -1 and call(k_out=None) == -1
    assert call(turns=None) == -1
    assert call(dtype=3) == -2 and call(batch=0) == -2 and call(tokens=0) == -2
    assert call(heads=0) == -2 and call(kv_heads=-1) == -2 and call(rotary=66) == -2
    assert call(rotary=63) == -2
    assert call(dim=1026) == -6
    assert call(q=p + 1) == -3 and call(dtype=2, k_out=p + 2) == -3
    assert call(weight=p + 2, weight_fp32=1) == -3
    assert call(pos=p + 4, wide=1) == -3 and call(turns=p + 4) == -3
