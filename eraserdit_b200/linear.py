"""The self-attention path's linear layers on ``erd_linear_bf16``.

``linear_bf16(x, weight, bias)`` computes ``F.linear(x, weight, bias)`` for
BF16 tensors (FP32 accumulation, bias added in FP32, one rounding to BF16) on
the sm_100a tensor cores.  It serves the Q/K/V projections of
``EraserDiTAttentionProcessor.self_attn``
(``models/dits/eraserdit_attention.py:248-253``; one product over the
concatenated weights) and its output projection ``_project_output``
(``:216-229``).  There is no fallback: an unsupported shape raises.

``linear_act(x, weight, bias, activation=, gate=, residual=)`` is a product of any
size with the rest of a block's step in its epilogue: ``residual + gate *
act(x @ weight.T + bias)``, BF16 or FP16 (``erd_linear_act``).
"""

from __future__ import annotations

import torch

from . import _native

TILE_N = 256  # output columns per tile: n must be a multiple
TILE_K = 64   # reduction depth per pipeline stage: k must be a multiple


def _rows(t: torch.Tensor) -> tuple[int, int] | None:
    """(rows, row stride) of a tensor viewed as [rows, last dim], or None when
    its leading dimensions do not form one strided row axis."""
    lead = t.shape[:-1]
    rows = 1
    for d in lead:
        rows *= d
    stride = t.stride(-2) if t.dim() >= 2 else t.shape[-1]
    expect = stride
    for d, s in zip(reversed(lead), reversed(t.stride()[:-1])):
        if d > 1 and s != expect:
            return None
        expect *= d
    return rows, stride


def _launch(x, weight, bias, out) -> None:
    n, k = weight.shape
    m, ldx = _rows(x)
    _, ldy = _rows(out)
    if m == 0:
        return
    lib = _native.load()
    device = x.device
    with torch.cuda.device(device):
        rc = lib.erd_linear_bf16(x.data_ptr(), ldx, weight.data_ptr(), weight.stride(0),
                                 _native.ptr(bias), out.data_ptr(), ldy, m, n, k,
                                 _native.status_word(device).data_ptr(),
                                 _native.stream_handle(device))
    _native.check(rc, "erd_linear_bf16")


def linear_bf16(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` for BF16 CUDA tensors: x [..., k], weight [n, k],
    bias [n] (or None); the result [..., n] (written into ``out`` when given)."""
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or not x.is_cuda:
        raise ValueError("linear_bf16 needs CUDA bfloat16 tensors")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError("weight must be [n, k] with k = x.shape[-1]")
    n, k = weight.shape
    if n % TILE_N or k % TILE_K:
        raise ValueError(f"linear_bf16 needs n % {TILE_N} == 0 and k % {TILE_K} == 0")
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (n,)
                             or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous BF16 [n] tensor")
    if weight.stride(1) != 1:
        raise ValueError("weight must have a contiguous last dimension")
    if out is None:
        out = torch.empty(*x.shape[:-1], n, device=x.device, dtype=torch.bfloat16)
    elif out.shape != (*x.shape[:-1], n) or out.dtype != torch.bfloat16:
        raise ValueError("out must be BF16 [..., n]")
    if x.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError("x and out need a contiguous last dimension")
    if _rows(x) is not None and _rows(out) is not None:
        _launch(x, weight, bias, out)
    elif x.dim() >= 3:
        # e.g. [B, L, k] rows of wider [B, L_slot, k] slots: one product per
        # leading index (rows within it are evenly strided)
        for xs, ys in zip(x.unbind(0), out.unbind(0)):
            linear_bf16(xs, weight, bias, out=ys)
    else:
        raise ValueError("x and out must be viewable as [rows, last dim] with one row stride")
    return out


def linear_bf16_scatter(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                        out: torch.Tensor, scatter_col0: int, dest_bases: list[int],
                        group_cols: int, batch_stride: int, token_stride: int) -> None:
    """``linear_bf16`` of ``x`` [B, L, k] with the output columns from
    ``scatter_col0`` on stored into ``dest_bases`` (``erd_linear_bf16_scatter``):
    column j of token (b, t) goes to ``dest_bases[(j - scatter_col0) //
    group_cols]`` at element ``b * batch_stride + t * token_stride +
    (j - scatter_col0) % group_cols``; the columns below go to ``out`` [B, L, n]."""
    import ctypes
    if x.dim() != 3 or x.dtype != torch.bfloat16 or not x.is_contiguous():
        raise ValueError("x must be a contiguous BF16 [B, L, k] tensor")
    n, k = weight.shape
    if out.shape != (*x.shape[:-1], n) or not out.is_contiguous():
        raise ValueError("out must be a contiguous BF16 [B, L, n] tensor")
    m = x.shape[0] * x.shape[1]
    if m == 0:
        return
    lib = _native.load()
    device = x.device
    bases = (ctypes.c_void_p * len(dest_bases))(*dest_bases)
    with torch.cuda.device(device):
        rc = lib.erd_linear_bf16_scatter(
            x.data_ptr(), k, weight.data_ptr(), weight.stride(0), _native.ptr(bias),
            out.data_ptr(), n, m, n, k, scatter_col0, bases, len(dest_bases), group_cols,
            x.shape[1], batch_stride, token_stride, _native.status_word(device).data_ptr(),
            _native.stream_handle(device))
    _native.check(rc, "erd_linear_bf16_scatter")


ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


_LINEAR_TYPES = (torch.bfloat16, torch.float16)


def _row_stride(what: str, t: torch.Tensor) -> int | None:
    """Stride of ``t``'s rows, one that fits where no row follows, or None when its
    leading dimensions do not form one strided row axis."""
    last = t.shape[-1]
    if t.is_contiguous():
        return last if t.dim() > 1 and t.numel() > last else -(-last // 8) * 8
    if last > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what} needs a contiguous last dimension")
    if t.numel() == last:
        return -(-last // 8) * 8
    if t.dim() == 2:
        return t.stride(0)
    # the stride of the last dimension that has several entries, met by all others
    stride = expect = None
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size > 1:
            if stride is None:
                stride = expect = step
            if step != expect:
                return None
            expect *= size
    return stride


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               activation: str = "none", gate: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, out: torch.Tensor | None = None
               ) -> torch.Tensor:
    """``residual + gate * act(x @ weight.T + bias)`` for BF16 or FP16 CUDA tensors.

    x [..., k], weight [n, k], bias [n]; ``activation``: ``"none"``, ``"relu"``,
    ``"silu"``, ``"gelu"`` (with the normal distribution function) or
    ``"gelu_tanh"``; ``gate`` [n], or [g, n] with g dividing the number of rows
    (one gate per batch entry: consecutive rows / g share one); ``residual`` and
    ``out`` [..., n], where ``out`` may be ``residual``.  Everything is added up
    in FP32 and rounded once.  Any sizes; rows of ``x`` and ``weight`` start on 16
    bytes (row strides, and so a contiguous k, are multiples of 8).
    """
    dtype, device = x.dtype, x.device
    if dtype not in _LINEAR_TYPES or device.type != "cuda" or x.dim() < 1:
        raise ValueError("linear_act needs a CUDA BF16 or FP16 x")
    shape = x.shape
    if weight.dim() != 2 or weight.shape[1] != shape[-1] or shape[-1] == 0:
        raise ValueError("weight must be [n, k] with k = x.shape[-1] > 0")
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
    n, k = weight.shape
    shape = shape[:-1] + (n,)
    for what, t in (("weight", weight), ("bias", bias), ("gate", gate), ("residual", residual),
                    ("out", out)):
        if t is not None and (t.dtype != dtype or t.device != device):
            raise ValueError(f"{what} must have x's type and device")
    _native.refuse_gradients("linear_act", x, weight, bias, gate, residual, out)
    if bias is not None and (bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous [n] tensor")
    if residual is not None and residual.shape != shape:
        raise ValueError("residual must be [..., n]")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
    elif out.shape != shape or any(s == 0 and d > 1 for s, d in zip(out.stride(), out.shape)):
        raise ValueError("out must be [..., n] and no expanded view")
    else:
        _native.refuse_overlap("out", out, (x, weight, bias, gate), residual)
        _native.written(out)
    m = x.numel() // k
    gate_rows = 0
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != n or not gate.is_contiguous():
            raise ValueError("gate must be a contiguous [n] or [g, n] tensor")
        groups = 1 if gate.dim() == 1 else gate.shape[0]
        if m and (groups == 0 or m % groups):
            raise ValueError("the gate's groups must divide the rows")
        gate_rows = m // max(groups, 1)
    if m == 0 or n == 0:
        return out
    ldx, ldy, ldw = _row_stride("x", x), _row_stride("out", out), _row_stride("weight", weight)
    ldr = 0 if residual is None else _row_stride("residual", residual)
    if ldx is None or ldy is None or ldr is None:
        # rows that no single stride walks, e.g. prefixes [B, L, k] of wider slots:
        # one product per leading index, each with its part of the gate
        lead, groups = x.shape[0], 1 if gate is None or gate.dim() == 1 else gate.shape[0]
        if x.dim() < 3:
            raise ValueError("x, residual and out must be viewable as [rows, last dim] with one "
                             "row stride")
        if groups % lead and lead % groups:
            raise ValueError("a gate's group may not end within one leading index of rows "
                             "without a common stride")
        for i in range(lead):
            part = gate
            if groups > 1:
                part = gate[i * groups // lead:max((i + 1) * groups // lead, i * groups // lead + 1)]
            linear_act(x[i], weight, bias, activation=activation, gate=part,
                       residual=None if residual is None else residual[i], out=out[i])
        return out
    if ldx < k or ldw < k or ldy < n or (residual is not None and ldr < n):
        raise ValueError("rows must not overlap (an expanded view is given in full)")
    xp, wp = x.data_ptr(), weight.data_ptr()
    if (xp | wp) % 16 or (ldx | ldw) % 8:
        raise ValueError("rows of x and weight must start on 16 bytes (strides multiples of 8)")
    _native.call("erd_linear_act", device, _native.pack(
        "erd_linear_act", xp, wp, 0 if bias is None else bias.data_ptr(),
        0 if gate is None else gate.data_ptr(), 0 if residual is None else residual.data_ptr(),
        out.data_ptr(), ldx, ldw, ldr, ldy, _native.DTYPE_CODES[dtype], code, gate_rows, m, n, k),
        _native.status_pointer(device))
    return out
