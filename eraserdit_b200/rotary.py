"""LTX 3D rotary embedding in factored (per-axis) form.

Mirrors ``LTXVideoRotaryPosEmbed`` (``models/dits/eraserdit_transformer.py:115-214``,
instantiated at ``:402-410`` with dim 2048, base (20, 2048, 2048), theta 1e4).
The reference materialises cos/sin tables of shape [B, F*H*W, 2048] in fp32
(267 MB each at 2 x 32640 tokens).  Every entry is cos/sin of
``freq[k] * (2 * coord_axis - 1)`` for one of three axes, so the same values
are stored here once per (axis, coordinate, frequency): (F + H + W) * 341
float2 entries (300 KB at 16 x 34 x 60), built on the device by
``erd_rope_axis_table`` and read by the fused QK-norm/RoPE kernel.

The 341 base frequencies are computed with the reference's own torch
expression (``:194-201``) on the host, once per table, so that they are
bit-identical to the reference's; all per-token work runs on the device.

``RotaryPositions`` and ``apply_rotary`` are the rotation of single heads by
token positions (``erd_head_norm_rotary``): interleaved or half layout, all or
part of the head, one to three position axes, frequencies scaled for contexts
longer than the trained one.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _native


def base_frequencies(dim: int = 2048, theta: float = 10000.0) -> torch.Tensor:
    """``theta ** linspace(log_theta(1), log_theta(theta), dim // 6) * pi / 2`` (fp32)."""
    freqs = theta ** torch.linspace(math.log(1.0, theta), math.log(theta, theta), dim // 6,
                                    dtype=torch.float32)
    return freqs * math.pi / 2.0


@dataclass
class RopeAxisTable:
    """Device table of (cos, sin) per (axis, coordinate, frequency)."""

    table: torch.Tensor  # float32 [(F + H + W) * nfreq * 2]
    frames: int
    height: int
    width: int
    nfreq: int
    # Optional device int32 [F*H*W]: grid position (f*H*W + h*W + w) of the
    # token at each sequence position, when tokens are not in raster order.
    grid_index: torch.Tensor | None = None

    @property
    def tokens(self) -> int:
        return self.frames * self.height * self.width

    def in_order(self, grid_index: torch.Tensor) -> "RopeAxisTable":
        """The same table for a sequence laid out in another token order."""
        index = grid_index.to(device=self.table.device, dtype=torch.int32).contiguous()
        if index.numel() != self.tokens:
            raise ValueError("grid_index needs one entry per token")
        return RopeAxisTable(self.table, self.frames, self.height, self.width, self.nfreq, index)

    def full(self, batch: int = 1, dim: int = 2048) -> tuple[torch.Tensor, torch.Tensor]:
        """Expand to the reference's [B, F*H*W, dim] cos/sin tables (for tests and
        for callers of the table-based fusion interface)."""
        t = self.table.view(-1, 2)
        nf, dev = self.nfreq, self.table.device
        f = torch.arange(self.frames, device=dev).repeat_interleave(self.height * self.width)
        h = torch.arange(self.height, device=dev).repeat_interleave(self.width).repeat(self.frames)
        w = torch.arange(self.width, device=dev).repeat(self.frames * self.height)
        k = torch.arange(nf, device=dev)
        base = torch.tensor([0, self.frames * nf, (self.frames + self.height) * nf], device=dev)
        coords = torch.stack([f, h, w], dim=-1)  # [S, 3]
        idx = base.view(1, 1, 3) + coords.view(-1, 1, 3) * nf + k.view(1, nf, 1)  # [S, nf, 3]
        vals = t[idx.flatten(1)]  # [S, nf*3, 2]
        cos = vals[..., 0].repeat_interleave(2, dim=-1)
        sin = vals[..., 1].repeat_interleave(2, dim=-1)
        pad = dim % 6
        if pad:
            cos = torch.cat([torch.ones_like(cos[:, :pad]), cos], dim=-1)
            sin = torch.cat([torch.zeros_like(sin[:, :pad]), sin], dim=-1)
        if self.grid_index is not None:
            idx = self.grid_index.long().to(cos.device)
            cos, sin = cos[idx], sin[idx]
        return (cos.unsqueeze(0).expand(batch, -1, -1).contiguous(),
                sin.unsqueeze(0).expand(batch, -1, -1).contiguous())


class LTXVideoRotaryPosEmbed:
    """Drop-in for the reference class's constructor; ``forward`` returns a
    :class:`RopeAxisTable` instead of the two dense tables."""

    def __init__(self, dim: int = 2048, base_num_frames: int = 20, base_height: int = 2048,
                 base_width: int = 2048, patch_size: int = 1, patch_size_t: int = 1,
                 theta: float = 10000.0) -> None:
        if dim != 2048:
            raise ValueError("the fused QK-norm/RoPE kernel supports dim 2048 (32 x 64 heads)")
        self.dim = dim
        self.base_num_frames = base_num_frames
        self.base_height = base_height
        self.base_width = base_width
        self.patch_size = patch_size
        self.patch_size_t = patch_size_t
        self.theta = theta
        self._freqs: dict[torch.device, torch.Tensor] = {}

    def freqs(self, device: torch.device) -> torch.Tensor:
        cached = self._freqs.get(device)
        if cached is None:
            cached = base_frequencies(self.dim, self.theta).to(device)
            self._freqs[device] = cached
        return cached

    def forward(self, num_frames: int, height: int, width: int,
                rope_interpolation_scale=None, device: torch.device | str = "cuda") -> RopeAxisTable:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the RoPE axis table is built on a CUDA device")
        lib = _native.load()
        freqs = self.freqs(device)
        nfreq = freqs.numel()
        table = torch.empty((num_frames + height + width) * nfreq * 2, dtype=torch.float32,
                            device=device)
        if rope_interpolation_scale is None:
            scale = (1.0, 1.0, 1.0)
            use_scale = 0
        else:
            scale = tuple(float(s) for s in rope_interpolation_scale)
            use_scale = 1
        with torch.cuda.device(device):
            rc = lib.erd_rope_axis_table(
                freqs.data_ptr(), nfreq, num_frames, height, width, use_scale, scale[0], scale[1],
                scale[2], float(self.patch_size_t), float(self.patch_size),
                float(self.base_num_frames), float(self.base_height), float(self.base_width),
                table.data_ptr(), _native.stream_handle(device))
        _native.check(rc, "erd_rope_axis_table")
        return RopeAxisTable(table, num_frames, height, width, nfreq)

    __call__ = forward


SCALINGS = ("linear", "ntk", "yarn")


def rotary_frequencies(dim: int, theta: float = 10000.0, scaling: dict | None = None
                       ) -> tuple[torch.Tensor, float]:
    """Angle per position step of the ``dim / 2`` pairs (float64) and the factor
    on cosine and sine.

    ``theta ** (-2 i / dim)``, scaled for longer contexts by ``scaling["type"]``:

    - ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    - ``"ntk"``: the base becomes ``theta * factor ** (dim / (dim - 2))``, so the
      fastest pair stays and the slowest is divided by ``factor``;
    - ``"yarn"``: pairs that turn more than ``beta_fast`` (32) times within
      ``original_length`` stay, those below ``beta_slow`` (1) turns are divided by
      ``factor``, a linear ramp over the pair index between; cosine and sine are
      multiplied by ``attention_factor`` (default ``0.1 ln(factor) + 1``).
    """
    if dim <= 0 or dim % 2:
        raise ValueError("the rotated width must be positive and even")
    if not theta > 1.0:
        raise ValueError("theta must be above 1")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling is None:
        return theta ** (-i / dim), 1.0
    kind = scaling.get("type")
    if kind not in SCALINGS:
        raise ValueError(f"scaling type must be one of {SCALINGS}")
    known = {"type", "factor"} | ({"original_length", "beta_fast", "beta_slow", "attention_factor"}
                                  if kind == "yarn" else set())
    if set(scaling) - known:
        raise ValueError(f"unknown {kind} scaling arguments: {sorted(set(scaling) - known)}")
    factor = float(scaling.get("factor", 0.0))
    if not 1.0 <= factor < math.inf:
        raise ValueError("scaling needs a finite factor >= 1")
    if kind == "linear":
        return theta ** (-i / dim) / factor, 1.0
    if kind == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs a rotated width above 2")
        return (theta * factor ** (dim / (dim - 2))) ** (-i / dim), 1.0
    length = scaling.get("original_length", 0)
    if length <= 0:
        raise ValueError("yarn scaling needs original_length > 0")

    def pair_of(turns: float) -> float:  # pair index that makes `turns` turns in `length`
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))

    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not fast > slow > 0:
        raise ValueError("yarn scaling needs beta_fast > beta_slow > 0")
    low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), dim - 1)
    ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
    freqs = theta ** (-i / dim)
    amplitude = scaling.get("attention_factor")
    if amplitude is None:
        amplitude = 0.1 * math.log(factor) + 1.0
    return freqs / factor * ramp + freqs * (1.0 - ramp), float(amplitude)


class RotaryPositions:
    """How positions turn the channels of a head: built once, used by
    :func:`apply_rotary` and ``operator_fusion.apply_fused_qk_head_rmsnorm_rotary``.

    ``rotary_dim`` (default: all of ``head_dim``) leading channels are turned.
    ``layout``: ``"half"`` pairs channel i with i + rotary_dim / 2,
    ``"interleaved"`` 2 i with 2 i + 1.  ``scaling``: see :func:`rotary_frequencies`.
    ``axes_dim``: for positions on two or three axes (frame, row, column), the
    even channel count of each axis, ``sum(axes_dim) == rotary_dim``; the pairs
    are then split over the axes in that order and every axis has the
    frequencies of its own width.
    """

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, theta: float = 10000.0,
                 layout: str = "half", scaling: dict | None = None,
                 axes_dim: tuple[int, ...] | None = None,
                 device: torch.device | str = "cuda") -> None:
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if not 0 < rotary_dim <= head_dim <= 1024 or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and within head_dim, head_dim at most 1024")
        if layout not in ("half", "interleaved"):
            raise ValueError("layout must be half or interleaved")
        widths = (rotary_dim,) if axes_dim is None else tuple(axes_dim)
        if not 1 <= len(widths) <= 3 or sum(widths) != rotary_dim:
            raise ValueError("axes_dim needs one to three widths that add up to rotary_dim")
        parts = [rotary_frequencies(w, theta, scaling) for w in widths]
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.axes = len(widths)
        self.amplitude = parts[0][1]
        self.frequencies = torch.cat([f for f, _ in parts])  # float64, on the host
        ends = [sum(widths[:i + 1]) // 2 for i in range(3)]
        self.second_axis, self.third_axis = ends[0], ends[1]
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("rotary positions live on a CUDA device")
        # complete when this returns (a copy from pageable host memory), so any
        # stream may read it
        self.turns = (self.frequencies / (2 * math.pi)).to(device)
        self.device = self.turns.device
        self._stream = _native.stream_handle(self.device)


def _positions_args(rotary: RotaryPositions, positions, batch: int, tokens: int) -> tuple:
    """(pointer, int64 flag, axis / batch / token stride, start) of the positions."""
    if isinstance(positions, int):
        if rotary.axes != 1:
            raise ValueError("positions on several axes are a tensor")
        return 0, 0, 0, 0, 0, positions
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be an int or an int32 / int64 tensor")
    if positions.device != rotary.device:
        raise ValueError("positions and the rotary frequencies are on different devices")
    shape, strides, axis = positions.shape, positions.stride(), 0
    if rotary.axes > 1:
        if len(shape) < 2 or shape[0] != rotary.axes:
            raise ValueError(f"positions must be [{rotary.axes}, S] or [{rotary.axes}, B, S]")
        axis, shape, strides = strides[0], shape[1:], strides[1:]
    if shape == (tokens,):
        per_batch, per_token = 0, strides[0]
    elif shape == (batch, tokens) or shape == (1, tokens):
        per_batch, per_token = (strides[0] if shape[0] == batch else 0), strides[1]
    else:
        raise ValueError(f"positions must cover [{tokens}] or [{batch}, {tokens}] tokens")
    return positions.data_ptr(), positions.dtype == torch.int64, axis, per_batch, per_token, 0


def _check_heads(what: str, x: torch.Tensor, like: torch.Tensor | None = None) -> tuple:
    """The checks of a [B, S, H, D] operand; its (token, head, batch) strides."""
    if x.dim() != 4 or not x.is_cuda or x.dtype not in _native.DTYPE_CODES:
        raise ValueError(f"{what} must be a CUDA BF16, FP16 or FP32 [B, S, H, D] tensor")
    batch, token, head, channel = x.stride()
    if channel != 1 and x.shape[3] > 1:
        raise ValueError(f"{what} must have a contiguous head_dim")
    if like is not None and (x.dtype != like.dtype or x.device != like.device
                             or x.shape[:2] != like.shape[:2] or x.shape[3] != like.shape[3]):
        raise ValueError(f"{what} must match the query's type, device, tokens and head_dim")
    return token, head, batch


def _check_out(what: str, out: torch.Tensor, x: torch.Tensor) -> tuple:
    if out.shape != x.shape:
        raise ValueError(f"{what} must have its input's shape")
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{what} must not be an expanded view")
    return _check_heads(what, out, x)


def _new_out(x: torch.Tensor) -> tuple[torch.Tensor, tuple]:
    """An empty contiguous tensor of x's shape and its (token, head, batch) strides."""
    _, tokens, heads, dim = x.shape
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    return out, (heads * dim, dim, tokens * heads * dim)


def head_rotary_call(what: str, query, key, rotary, positions, q_weight, k_weight, norm: bool,
                     q_eps: float, k_eps: float, inverse: bool, query_out, key_out) -> tuple:
    """Checks and launch shared by the rotation with and without the norm."""
    q_strides, k_strides = _check_heads("query", query), (0, 0, 0)
    batch, tokens, heads, dim = query.shape
    kv_heads, k_out, k_ptr, ko_ptr, ko_strides = 0, None, 0, 0, (0, 0, 0)
    if key is not None:
        k_strides = _check_heads("key", key, query)
        kv_heads, k_ptr = key.shape[2], key.data_ptr()
    _native.refuse_gradients(what, query, key, q_weight, k_weight, query_out, key_out)
    if rotary is not None or not norm:
        if not isinstance(rotary, RotaryPositions):
            raise ValueError("rotary must be a RotaryPositions")
        if rotary.head_dim != dim:
            raise ValueError(f"rotary was built for head_dim {rotary.head_dim}, not {dim}")
        if rotary.device != query.device:
            raise ValueError("rotary lives on another device than the query")
        where = _positions_args(rotary, positions, batch, tokens)
        turns, amplitude = rotary.turns.data_ptr(), rotary.amplitude
        axis1, axis2 = rotary.second_axis, rotary.third_axis
        rotary_dim, interleaved = rotary.rotary_dim, rotary.layout == "interleaved"
    else:
        where, amplitude = (0, 0, 0, 0, 0, 0), 1.0
        turns = axis1 = axis2 = rotary_dim = interleaved = 0
    if query_out is None:
        q_out, qo_strides = _new_out(query)
    else:
        q_out, qo_strides = query_out, _check_out("query_out", query_out, query)
        _native.refuse_overlap("query_out", q_out, (key, q_weight, k_weight), query)
        _native.written(q_out)
    if key is not None:
        if key_out is None:
            k_out, ko_strides = _new_out(key)
        else:
            k_out, ko_strides = key_out, _check_out("key_out", key_out, key)
            _native.refuse_overlap("key_out", k_out, (query, q_out, q_weight, k_weight), key)
            _native.written(k_out)
        ko_ptr = k_out.data_ptr()
    elif key_out is not None:
        raise ValueError("key_out needs a key")
    if batch * tokens * (heads + kv_heads) * dim == 0:
        return q_out, k_out
    if heads == 0:
        raise ValueError("the query needs at least one head")
    weight = q_weight if q_weight is not None else k_weight
    device = query.device
    _native.call("erd_head_norm_rotary", device, _native.pack(
        "erd_head_norm_rotary", query.data_ptr(), k_ptr,
        0 if q_weight is None else q_weight.data_ptr(),
        0 if k_weight is None else k_weight.data_ptr(), turns, where[0], q_out.data_ptr(), ko_ptr,
        *q_strides, *k_strides, *qo_strides, *ko_strides, *where[2:],
        _native.DTYPE_CODES[query.dtype], batch, tokens, heads, kv_heads, dim, rotary_dim,
        interleaved, norm, weight is not None and weight.dtype == torch.float32, inverse, axis1,
        axis2, where[1], q_eps, k_eps, amplitude))
    if rotary is not None and _native.raw_stream(device.index) != rotary._stream:
        rotary.turns.record_stream(torch.cuda.current_stream(device))
    return q_out, k_out


def apply_rotary(query: torch.Tensor, key: torch.Tensor | None, rotary: RotaryPositions,
                 positions: torch.Tensor | int, *, inverse: bool = False,
                 query_out: torch.Tensor | None = None, key_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Turn the heads of query [B, S, H, D] and key [B, S, Hkv, D] (or None) by
    their tokens' positions.

    ``positions``: int32 / int64 [S] or [B, S] (with ``rotary.axes`` > 1 behind a
    leading axis dimension), or an int: the position of the first token.
    ``inverse`` turns back (the transposed rotation, and so the gradient's).
    ``query_out`` / ``key_out`` may be the inputs themselves (in place).
    """
    return head_rotary_call("apply_rotary", query, key, rotary, positions, None, None, False, 1.0,
                            1.0, inverse, query_out, key_out)
