"""Attention over the key blocks that a cheap score selects.

``mask_sta`` keeps the key blocks that a latent mask and a window name, the same
for every head; here every block of queries of every head picks its own, from
the data: the ``topk`` key blocks whose mean key has the highest product with
the summed queries (``erd_block_topk_attn``).  A query block is 128 queries (the
tokens of a clip, tensor-core attention) or a single query (one new token
against the keys kept so far).

The scores are computed in FP64, so the choice does not depend on the order of
summation; ties go to the lowest index.  ``pool_key_blocks`` gives the key
blocks' means; a program that keeps keys keeps these beside them
(``key_pool=``), and a call for single queries then reads the means and the
chosen blocks only.
"""

from __future__ import annotations

import torch

from . import _native

HEAD_DIM = 64
QUERY_BLOCKS = (1, 128)
KEY_BLOCKS = (64, 128)
MAX_TOPK = 0x7fff0000
MIN_SCALE, MAX_SCALE = 2.0 ** -149, 2.3e38  # FP32's least, and what log2(e) times is finite


def _strides(what: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(token, head, batch) strides of a BSHD tensor, 0 for a dimension of one."""
    batch, token, head, channel = t.stride()
    nb, nt, nh, _ = t.shape
    if channel != 1:
        raise ValueError(f"{what} must have a contiguous head_dim")
    batch, token, head = batch if nb > 1 else 0, token if nt > 1 else 0, head if nh > 1 else 0
    if t.data_ptr() % 16 or (batch | token | head) % 8:
        raise ValueError(f"{what} needs 16-byte aligned rows (strides multiple of 8 elements)")
    if (nb > 1 and not batch) or (nt > 1 and not token) or (nh > 1 and not head):
        raise ValueError(f"{what} must not be an expanded view (shared key heads are given once)")
    return token, head, batch


def _check_tensor(what: str, t: torch.Tensor) -> None:
    if t.dim() != 4 or not t.is_cuda or t.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what} must be a CUDA BF16 or FP16 [B, S, H, {HEAD_DIM}] tensor")
    if t.shape[3] != HEAD_DIM:
        raise ValueError(f"{what} must have head_dim {HEAD_DIM}")


def _check_lengths(key_lengths: torch.Tensor | None, key: torch.Tensor) -> None:
    if key_lengths is not None and (
            key_lengths.dtype != torch.int32 or key_lengths.shape != key.shape[:1]
            or key_lengths.device != key.device or not key_lengths.is_contiguous()):
        raise ValueError("key_lengths must be a contiguous int32 [B] tensor on the keys' device")


def _check_means(means: torch.Tensor, key: torch.Tensor, key_block: int) -> None:
    shape = (key.shape[0], key.shape[2], -(-key.shape[1] // key_block), HEAD_DIM)
    if (means.dtype != torch.float64 or means.shape != shape or means.device != key.device
            or not means.is_contiguous() or means.data_ptr() % 16):
        raise ValueError(f"key_pool must be a contiguous float64 {list(shape)} tensor")


def pool_key_blocks(key: torch.Tensor, key_block: int = 64, *,
                    key_lengths: torch.Tensor | None = None, out: torch.Tensor | None = None
                    ) -> torch.Tensor:
    """Means of every block of ``key_block`` keys [B, S, Hkv, 64] over its keys below
    ``key_lengths`` (int32 [B]; default all): float64 [B, Hkv, blocks, 64], 0 for a
    block without one."""
    _check_tensor("key", key)
    if key_block not in KEY_BLOCKS:
        raise ValueError(f"key_block must be one of {KEY_BLOCKS}")
    _check_lengths(key_lengths, key)
    _native.refuse_gradients("pool_key_blocks", key, out)
    batch, length, heads, _ = key.shape
    if out is None:
        out = torch.empty(batch, heads, -(-length // key_block), HEAD_DIM, device=key.device,
                          dtype=torch.float64)
    else:
        _check_means(out, key, key_block)
        _native.refuse_overlap("out", out, (key, key_lengths))
        _native.written(out)
    if out.numel():
        _native.call("erd_block_key_means", key.device, _native.DTYPE_CODES[key.dtype],
                     key.data_ptr(), *_strides("key", key), batch, heads, length, key_block,
                     _native.ptr(key_lengths), out.data_ptr())
    return out


def block_topk_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                         softmax_scale: float, topk: int, *, query_block: int = 128,
                         key_block: int = 64, key_lengths: torch.Tensor | None = None,
                         key_pool: torch.Tensor | None = None, out: torch.Tensor | None = None,
                         return_selection: bool = False
                         ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """softmax(Q K^T * scale) V of every query over its query block's ``topk``
    highest-scoring key blocks.

    query [B, Sq, H, 64], key / value [B, Sk, Hkv, 64] (H a multiple of Hkv), BF16
    or FP16.  ``query_block``: 128 or 1 consecutive queries that share a choice;
    ``key_block``: 64 or 128 keys.  ``key_lengths`` (int32 [B] on the device): keys
    from there on are left out, whatever they hold; a sequence without keys gives
    zeros.  ``out`` may be ``query`` itself.  ``key_pool``: what ``pool_key_blocks(key,
    key_block, key_lengths=...)`` gave, kept by the caller; else computed here.  With
    ``return_selection`` also the chosen blocks, int32 [B, H, query blocks, topk],
    ascending, -1 behind the last.
    """
    for what, t in (("query", query), ("key", key), ("value", value)):
        _check_tensor(what, t)
        if t.dtype != query.dtype or t.device != query.device or t.shape[0] != query.shape[0]:
            raise ValueError(f"{what} must match the query's type, device and batch")
    if key.shape != value.shape:
        raise ValueError("key and value must have the same shape")
    batch, q_len, heads, _ = query.shape
    kv_len, kv_heads = key.shape[1], key.shape[2]
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be a positive multiple of the key heads")
    if query_block not in QUERY_BLOCKS or key_block not in KEY_BLOCKS:
        raise ValueError(f"query_block must be one of {QUERY_BLOCKS}, key_block of {KEY_BLOCKS}")
    if not isinstance(topk, int) or not 1 <= topk <= MAX_TOPK:
        raise ValueError(f"topk must be an int from 1 to {MAX_TOPK}")
    if not MIN_SCALE <= softmax_scale <= MAX_SCALE:
        raise ValueError("softmax_scale must be positive and finite (in FP32, in base 2)")
    _check_lengths(key_lengths, key)
    _native.refuse_gradients("block_topk_attention", query, key, value, out)
    if key_pool is not None:
        _check_means(key_pool, key, key_block)
    device, dtype = query.device, query.dtype
    groups = -(-q_len // query_block)
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != query.device:
        raise ValueError("out must have the query's shape, type and device")
    else:
        _native.refuse_overlap("out", out, (key, value, key_lengths, key_pool), query)
        _native.written(out)
    if not return_selection:  # no list is wider than the blocks there are
        topk = min(topk, max(1, -(-kv_len // key_block)))
    selection = query.new_empty((batch, heads, groups, topk), dtype=torch.int32)
    if batch and q_len and kv_len:
        nbytes = 0
        workspace = None
        if key_pool is None or query_block != 1:
            nbytes = int(_native.load().erd_block_topk_workspace_bytes(
                batch, heads, kv_heads, q_len, kv_len, query_block, key_block,
                key_pool is not None))
            # from torch's allocator, call by call: it follows streams and captures
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
        _native.call("erd_block_topk_attn", device, _native.pack(
            "erd_block_topk_attn", query.data_ptr(), key.data_ptr(), value.data_ptr(),
            0 if key_lengths is None else key_lengths.data_ptr(),
            0 if key_pool is None else key_pool.data_ptr(), out.data_ptr(), selection.data_ptr(),
            0 if workspace is None else workspace.data_ptr(), *_strides("query", query),
            *_strides("key", key), *_strides("value", value), *_strides("out", out), nbytes,
            _native.DTYPE_CODES[dtype], batch, heads, kv_heads, q_len, kv_len, HEAD_DIM, topk,
            query_block, key_block, softmax_scale), _native.status_pointer(device))
    elif batch and q_len:  # no keys at all
        out.zero_()
        selection.fill_(-1)
    return (out, selection) if return_selection else out
