"""Host side of linear_act: refusals of the C entry and of host tensors (no GPU)."""
import pytest
import torch


def test_host_tensors_are_refused():
    from eraserdit_b200.linear import linear_act
    with pytest.raises(ValueError):
        linear_act(torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16))


def test_entry_rejects_bad_arguments_before_any_device_call():
    from eraserdit_b200 import _native
    fn = _native.load().erd_linear_act
    p = 1 << 20

    def call(dtype=0, x=p, ldx=64, w=p, ldw=64, bias=None, act=0, gate=None, gate_rows=0, res=None,
             ldr=0, y=p, ldy=48, m=4, n=48, k=64):
        fields = (x, w, bias, gate, res, y, ldx, ldw, ldr, ldy, dtype, act, gate_rows, m, n, k)
        return fn(_native.pack("erd_linear_act", *(0 if f is None else f for f in fields)), None, None)

    assert fn(None, None, None) == -1
    assert fn(_native.STRUCTS["erd_linear_act"].pack(8, *([0] * 16)), None, None) == -2  # another struct

    assert call(x=None) == -1 and call(w=None) == -1 and call(y=None) == -1
    assert call(dtype=2) == -2 and call(dtype=-1) == -2 and call(act=5) == -2 and call(act=-1) == -2
    assert call(m=0) == -2 and call(n=0) == -2 and call(k=0) == -2
    assert call(ldx=63) == -2 and call(ldw=56) == -2 and call(ldy=47) == -2
    assert call(res=p, ldr=40) == -2 and call(gate=p, gate_rows=0) == -2
    assert call(x=p + 8) == -3 and call(w=p + 2) == -3 and call(ldx=68) == -3 and call(ldw=66) == -3
    assert call(bias=p + 1) == -3 and call(y=p + 1) == -3
    assert call(m=0x7fffffff) == -6
