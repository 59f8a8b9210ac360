"""ctypes binding of ``liberaserdit_b200.so`` (declared in ``include/eraserdit_b200.h``).

The library is the only compute path: if it is missing or cannot be loaded,
every entry point raises.  There is no CPU or PyTorch fallback.

Tensors are passed as raw device pointers with element strides, on the
caller's current CUDA stream, in the style of the reference's mask-STA ctypes
binding (``layers/attention/backends/mask_sta.py:108-131``): a nonzero return
code raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading
from pathlib import Path

import torch
from torch.autograd import forward_ad

LIBRARY_PATH = Path(__file__).resolve().parent / "liberaserdit_b200.so"
ABI_VERSION = 6

_c_int, _c_i64, _c_float, _vp = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

# name -> argument types, in header order.
SIGNATURES = {
    "erd_abi_version": [],
    "erd_error_string": [_c_int],
    "erd_rope_axis_table": [_vp, _c_int, _c_int, _c_int, _c_int, _c_int, _c_float, _c_float,
                            _c_float, _c_float, _c_float, _c_float, _c_float, _c_float, _vp, _vp],
    "erd_qk_norm_rope": [_vp, _vp, _vp, _c_i64, _c_i64, _c_int, _c_int, _c_int, _vp, _vp,
                         _c_float, _c_int, _vp, _vp, _c_i64, _c_i64, _vp, _c_int, _c_int, _c_int,
                         _c_int, _c_int, _vp, _vp, _vp, _vp, _c_i64, _c_i64, _c_i64, _c_int,
                         _c_i64, _vp],
    "erd_attn_fwd_bf16": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4 + [_vp, _c_int, _c_float,
                                                                            _vp] + [_c_i64] * 4
                         + [_vp, _vp],
    "erd_attn_fwd_sparse_bf16": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4
                                + [_vp, _c_int, _c_float, _vp] + [_c_i64] * 4
                                + [_vp, _c_int, _vp, _c_i64, _vp, _vp, _vp],
    "erd_gather_tokens": [_vp, _c_i64, _c_i64, _c_int, _vp, _c_i64, _c_i64, _vp, _c_int, _c_int,
                          _c_int, _vp],
    "erd_qk_norm_rope_peer": [_vp, _vp, _vp, _c_i64, _c_i64, _c_int, _c_int, _c_int, _vp, _vp,
                              _c_float, _c_int, _vp, _vp, _c_i64, _c_i64, _vp, _c_int, _c_int,
                              _c_int, _c_int, _c_int, _vp, _vp, _c_int, _c_i64, _c_i64, _c_i64,
                              _c_i64, _c_i64, _c_int, _vp],
    "erd_attn_fwd_bf16_peer": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4
                              + [_vp, _c_int, _c_float, _vp] + [_c_i64] * 3 + [_vp, _vp],
    "erd_attn_fwd_sparse_bf16_peer": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4
                                     + [_vp, _c_int, _c_float, _vp] + [_c_i64] * 3
                                     + [_vp, _c_int, _vp, _c_i64, _vp, _vp],
    "erd_attn_fwd_fp8_peer": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4
                             + [_vp, _c_int, _c_float, _vp] + [_c_i64] * 3
                             + [_vp, ctypes.c_size_t, _vp, _vp],
    "erd_quantize_e4m3": [_vp, _vp, _c_i64, _c_float, _vp],
    "erd_linear_bf16": [_vp, _c_i64, _vp, _c_i64, _vp, _vp, _c_i64, _c_int, _c_int, _c_int, _vp,
                        _vp],
    "erd_linear_bf16_scatter": [_vp, _c_i64, _vp, _c_i64, _vp, _vp, _c_i64, _c_int, _c_int,
                                _c_int, _c_int, _vp, _c_int, _c_int, _c_int, _c_i64, _c_i64,
                                _vp, _vp],
    "erd_linear_fp8": [_vp, _c_i64, _vp, _c_i64, _vp, _vp, _vp, _c_i64, _c_int, _c_int, _c_int,
                       _vp, _vp],
    "erd_attn_fwd_cross_bf16": [_vp, _vp, _vp] + [_c_i64] * 9 + [_c_int] * 4
                               + [_vp, _c_int, _c_float, _vp] + [_c_i64] * 3 + [_vp, _vp],
    "erd_ring_state_bytes": [_c_int, _c_int, _c_int, _c_int],
    "erd_attn_fwd_ring_bf16": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4
                              + [_vp, _c_int, _c_int, _vp, _c_int, _c_float, _vp] + [_c_i64] * 4
                              + [_vp, _vp, ctypes.c_size_t, _c_int, _vp, _vp],
    "erd_peer_alloc": [ctypes.c_size_t, ctypes.POINTER(_vp)],
    "erd_peer_free": [_vp],
    "erd_peer_ipc_handle": [_vp, _vp],
    "erd_peer_ipc_open": [_vp, ctypes.POINTER(_vp)],
    "erd_peer_ipc_close": [_vp],
    "erd_peer_signal": [_vp, _c_int, ctypes.c_int32, _vp],
    "erd_peer_wait": [_vp, _c_int, ctypes.c_int32, _c_i64, _vp, _vp],
    "erd_attn_fp8_workspace_bytes": [_c_int, _c_int, _c_int, _c_int],
    "erd_attn_fwd_fp8": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4 + [_vp, _c_int, _c_float,
                                                                           _vp] + [_c_i64] * 4
                        + [_vp, ctypes.c_size_t, _vp, _vp],
    "erd_attn_fwd_fp8_static_scratch": [_vp, _vp, _vp] + [_c_i64] * 12 + [_c_int] * 4
                                       + [_vp, _c_int, _c_float, _vp] + [_c_i64] * 4 + [_vp, _vp],
    "erd_block_topk_workspace_bytes": [_c_int] * 8,
    "erd_block_topk_attn": [ctypes.c_char_p, _vp, _vp],
    "erd_block_key_means": [_c_int, _vp, _c_i64, _c_i64, _c_i64, _c_int, _c_int, _c_int, _c_int,
                            _vp, _vp, _vp],
    "erd_linear_act": [ctypes.c_char_p, _vp, _vp],
    "erd_head_norm_rotary": [ctypes.c_char_p, _vp],
}
# The argument structs of the header, in its field order: packing one and passing
# its address takes 0.5 us where 40 converted arguments took 4.
STRUCTS = {name: struct.Struct(fields) for name, fields in {
    "erd_block_topk_attn": "@q8P13q10if0q",
    "erd_linear_act": "@q6P4q6i0q",
    "erd_head_norm_rotary": "@q8P16q14i3f0q",
}.items()}
RESTYPES = {"erd_error_string": ctypes.c_char_p, "erd_attn_fp8_workspace_bytes": ctypes.c_size_t,
            "erd_ring_state_bytes": ctypes.c_size_t,
            "erd_block_topk_workspace_bytes": ctypes.c_size_t}

_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load the library once; raise if it is absent or of another ABI version."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = Path(os.environ.get("ERASERDIT_B200_LIBRARY", LIBRARY_PATH))
        if not path.exists():
            raise RuntimeError(
                f"eraserdit_b200 CUDA library not found at {path}; build it with "
                "`python -m eraserdit_b200.csrc.build` (no fallback path exists)")
        lib = ctypes.CDLL(str(path))
        for name, argtypes in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = argtypes
            fn.restype = RESTYPES.get(name, ctypes.c_int)
        if lib.erd_abi_version() != ABI_VERSION:
            raise RuntimeError(
                f"eraserdit_b200 ABI mismatch: library {lib.erd_abi_version()}, "
                f"binding {ABI_VERSION}")
        _lib = lib
    return _lib


def check(code: int, what: str) -> None:
    if code != 0:
        message = load().erd_error_string(code).decode()
        raise RuntimeError(f"{what} failed ({code}): {message}")


def stream_handle(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# Value type codes of the entry points that take several (ERD_BF16, ...).
DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


_entry_points: dict[str, object] = {}
# The current stream's handle without a Stream object around it (1.3 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(index: int) -> int:
    return _raw_stream(index) if _raw_stream is not None else \
        torch.cuda.current_stream(index).cuda_stream


def call(name: str, device: torch.device, *args) -> None:
    """Call an entry point whose last argument is the stream, on ``device``'s
    current stream with ``device`` current, and raise on its error code."""
    fn = _entry_points.get(name)
    if fn is None:
        fn = _entry_points[name] = getattr(load(), name)
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, raw_stream(index))
    if rc:
        check(rc, name)


def pack(name: str, *fields) -> bytes:
    """The argument struct of an entry point (0 for a null pointer)."""
    layout = STRUCTS[name]
    try:
        return layout.pack(layout.size, *fields)
    except struct.error as error:  # a size beyond its field
        raise ValueError(f"{name}: {error}") from None


def _span(dims) -> int:
    """Bytes from the first to the end of the last element over (size, byte stride) dims."""
    return sum((n - 1) * step for n, step in dims)


def may_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two strided tensors may share memory.  Tensors whose address ranges
    interleave (columns of one buffer) are told apart by a stride that both have:
    modulo it each covers one range."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    sides = []
    for t in (a, b):
        size = t.element_size()
        dims = [(n, step * size) for n, step in zip(t.shape, t.stride()) if n > 1]
        sides.append((t.data_ptr(), dims, size))
    (pa, da, sa), (pb, db, sb) = sides
    if pa + _span(da) + sa <= pb or pb + _span(db) + sb <= pa:
        return False
    for period in {step for _, step in da} & {step for _, step in db} - {0}:
        widths = []
        for _, dims, size in sides:
            inner = _span([d for d in dims if d[1] < period]) + size
            if inner > period or any(step % period for _, step in dims if step >= period):
                break
            widths.append(inner)
        if len(widths) == 2:
            gap = (pb - pa) % period  # where b's range starts behind a's
            if gap >= widths[0] and gap + widths[1] <= period:
                return False
    return True


def refuse_overlap(what: str, out: torch.Tensor, inputs, in_place: torch.Tensor | None = None) -> None:
    """A caller's destination shares no memory with the inputs; ``in_place``, an input
    that may be the destination itself (the same elements), shares all or none."""
    if in_place is not None and not (out.data_ptr() == in_place.data_ptr()
                                     and out.stride() == in_place.stride()):
        inputs = (*inputs, in_place)
    for t in inputs:
        if t is not None and may_overlap(out, t):
            raise ValueError(f"{what} overlaps an input")


def written(out: torch.Tensor) -> None:
    """A caller's destination is written in place: autograd refuses what it saved of it."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def refuse_gradients(what: str, *tensors) -> None:
    """The operators have no backward pass and no forward derivative: an input or a
    destination that wants a gradient while gradients are recorded, or that carries a
    tangent, is an error, not a silently detached result."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no backward pass: call it under torch.no_grad() or "
                                 "with detached inputs")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # within a dual level
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what} has neither a backward pass nor a forward derivative: "
                                 "call it with primal inputs")


_status: dict[int, torch.Tensor] = {}
# Words of calls that a CUDA graph recorded before their device had its own.
_captured_status: dict[int, list[torch.Tensor]] = {}


def _capturing(index: int) -> bool:
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _captured_word(index: int) -> torch.Tensor:
    """A word for one recorded call, cleared by the graph itself before that call's
    kernels: the device's word cannot be made now, as nothing may wait for its zero."""
    device = torch.device("cuda", index)
    word = torch.zeros(1, dtype=torch.int32, device=device)
    with torch.cuda.stream(torch.cuda.Stream(device)):  # not recorded: 0 until the first replay
        word.zero_()
    with _lock:
        _captured_status.setdefault(index, []).append(word)
    return word


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 word that kernels set when a bounded wait gives up."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    word = _status.get(index)
    if word is not None:
        return word
    if _capturing(index):
        return _captured_word(index)
    with _lock:  # a second word would leave the first caller's kernels a freed one
        word = _status.get(index)
        if word is None:
            word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
            # zero before any stream's kernel looks at it
            torch.cuda.current_stream(index).synchronize()
            _status[index] = word
    return word


def status_pointer(device: torch.device) -> int:
    """Address of the device's status word."""
    return status_word(device).data_ptr()


def read_status(device: torch.device, reset: bool = True) -> int:
    """Synchronise and return the device status bits (0 = no kernel timed out)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    words = [status_word(device), *_captured_status.get(index, ())]
    if len(words) > 1:
        torch.cuda.synchronize(index)  # graphs replay on any stream
    value = 0
    for word in words:
        bits = int(word.item())
        if reset and bits:
            word.zero_()
        value |= bits
    return value


_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def workspace(device: torch.device, nbytes: int) -> int:
    """Address of a caller-owned, 1024-byte aligned device buffer of at least
    ``nbytes`` for work enqueued on the current stream of ``device`` (one buffer
    per stream, grown on demand, reused in that stream's order)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    key = (index, stream_handle(torch.device("cuda", index)))
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes + 1024:
        buf = torch.empty(nbytes + 1024, dtype=torch.uint8, device=torch.device("cuda", index))
        _workspaces[key] = buf
    base = buf.data_ptr()
    return (base + 1023) // 1024 * 1024


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()
