"""Operators of the paged 8-bit KV cache: appending with the position rotation on the way, attention, read-back.

The reference's caches hold one sequence in one slab of 2/3/4-bit codes (cache_mlx.py:40-799).  These operators serve
batches of sequences whose keys and values lie in pages of a shared pool, in 8-bit codes with one scale for each page
and head:

* ``key_pages`` int8 ``[num_pages, kv_heads, page_size, head_dim]``,
* ``value_pages`` int8 ``[num_pages, kv_heads, head_dim, page_size]`` (transposed),
* ``key_scales`` / ``value_scales`` float32 ``[num_pages, kv_heads]``.

``page_table`` int32 ``[batch, max_pages]`` lists each sequence's pages, ``context_lens`` int32 ``[batch]`` counts its
tokens *including those of the call*, and ``token_starts`` int32 ``[batch + 1]`` gives the rows of the call that are
each sequence's newest tokens (``None``: one row each).  These three stay on the device: no call waits for the GPU, so
a step can be captured into a graph and replayed with other lengths.  Places and page numbers outside the table or the
pool are passed over: their tokens are not written and not seen.

There is no backward pass: a call whose operands want gradients raises.
"""

from __future__ import annotations

from functools import lru_cache
from math import sqrt
from typing import Sequence

import torch

from torque_hip import _lib
from torque_hip._tensors import ptr, stream_handle

SUPPORTED_PAGE_SIZES: tuple[int, ...] = (16, 32, 64)

_TYPES = {torch.float32: _lib.TQ_F32, torch.float16: _lib.TQ_F16, torch.bfloat16: _lib.TQ_BF16}


def _launch(dev: torch.device, name: str, *args: object) -> None:
    """Call an entry point on ``dev``'s current stream with ``dev`` current."""
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, stream_handle(dev))


def _pool(key_pages: torch.Tensor, value_pages: torch.Tensor, key_scales: torch.Tensor,
          value_scales: torch.Tensor) -> tuple[torch.device, int, int, int, int]:
    """Check the four tensors of a pool; its device, pages, heads, slots and head_dim."""
    if key_pages.dim() != 4 or key_pages.dtype is not torch.int8:
        raise ValueError("key_pages must be int8 [num_pages, kv_heads, page_size, head_dim]")
    pages, heads, size, dim = key_pages.shape
    dev = key_pages.device
    if value_pages.dtype is not torch.int8 or value_pages.shape != (pages, heads, dim, size):
        raise ValueError(f"value_pages must be int8 {(pages, heads, dim, size)} (transposed), got {tuple(value_pages.shape)}")
    for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
        if t.dtype is not torch.float32 or t.shape != (pages, heads):
            raise ValueError(f"{name} must be float32 {(pages, heads)}, got {tuple(t.shape)}")
    for name, t in (("key_pages", key_pages), ("value_pages", value_pages), ("key_scales", key_scales), ("value_scales", value_scales)):
        if t.device != dev or dev.type != "cuda":
            raise ValueError(f"{name} must be on the pool's HIP device")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    return dev, pages, heads, size, dim


def _batch(dev: torch.device, tokens: int, page_table: torch.Tensor, context_lens: torch.Tensor,
           token_starts: torch.Tensor | None) -> tuple[int, int]:
    """Check a batch's three tensors; its sequences and the table's width."""
    if page_table.dim() != 2 or page_table.dtype is not torch.int32:
        raise ValueError("page_table must be int32 [batch, max_pages]")
    batch, width = page_table.shape
    if width > 1 and page_table.stride(1) != 1 or batch > 1 and page_table.stride(0) < width:
        raise ValueError("page_table rows must be contiguous and must not overlap")
    if context_lens.dtype is not torch.int32 or context_lens.shape != (batch,) or not context_lens.is_contiguous():
        raise ValueError(f"context_lens must be contiguous int32 {(batch,)}, got {tuple(context_lens.shape)}")
    if token_starts is None:
        if tokens != batch:
            raise ValueError(f"without token_starts there is one token per sequence: {tokens} tokens, {batch} sequences")
    elif token_starts.dtype is not torch.int32 or token_starts.shape != (batch + 1,) or not token_starts.is_contiguous():
        raise ValueError(f"token_starts must be contiguous int32 {(batch + 1,)}, got {tuple(token_starts.shape)}")
    for name, t in (("page_table", page_table), ("context_lens", context_lens), ("token_starts", token_starts)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} must be on the pool's device")
    return batch, width


def _rows(name: str, t: torch.Tensor, dev: torch.device, tokens: int | None, heads: int | None, dim: int) -> torch.Tensor:
    """Check [tokens, heads, head_dim] rows; the rows with unit stride along head_dim."""
    if t.dim() != 3 or t.shape[2] != dim or (tokens is not None and t.shape[0] != tokens) or (heads is not None and t.shape[1] != heads):
        want = ("tokens" if tokens is None else tokens, "heads" if heads is None else heads, dim)
        raise ValueError(f"{name} must have shape [{want[0]}, {want[1]}, {want[2]}], got {tuple(t.shape)}")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} must be on the pool's device")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"the paged cache has no backward pass: {name} wants a gradient (use torch.no_grad())")
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.stride(2) == 1 else t.contiguous()


@lru_cache(maxsize=256)
def _axis_bytes(pair_axes: tuple[int, ...]) -> bytes:
    if any(not 0 <= int(a) < 4 for a in pair_axes):
        raise ValueError("pair_axes names axes 0 to 3")
    return bytes(int(a) for a in pair_axes)


def paged_append(
    key: torch.Tensor,
    value: torch.Tensor,
    *,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    token_starts: torch.Tensor | None = None,
    query: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    pair_axes: Sequence[int] | None = None,
    tables_by_token: bool = False,
    signs_left: torch.Tensor | None = None,
    signs_right: torch.Tensor | None = None,
    rotate_values: bool = False,
) -> torch.Tensor | None:
    """Append ``[tokens, kv_heads, head_dim]`` keys and values to their sequences' pages, in place, in one launch.

    ``cos`` / ``sin`` ``[rows, rotary_dim]`` turn keys (and ``query`` ``[tokens, query_heads, head_dim]``) by rotary
    positions, halves paired: by the cache position, by ``positions`` ``[tokens]``, by positions of several axes
    ``[axes, tokens]`` with ``pair_axes[i]`` the axis that turns the pair ``(i, i + rotary_dim / 2)`` (time, height and
    width of an image's patches), or, with ``tables_by_token``, by the row's own table row.  ``signs_left`` /
    ``signs_right`` then take keys and queries into the rotated basis (values with ``rotate_values``).

    A page's scale is the least power of two (2^-40 or more) that holds its largest element in 127 steps.  Where new
    tokens make it grow, the sequence's earlier codes in the page are rounded anew; it does not shrink before the page
    is filled from its first slot again.  Infinities are held as the largest code, NaN as 0; a key whose position is
    outside the tables is not written, and its query becomes NaN.  A page may be written for one sequence only.

    Returns the turned queries in ``query``'s dtype (rows of no sequence zero), or None without ``query``.
    """
    dev, pages, heads, size, dim = _pool(key_pages, value_pages, key_scales, value_scales)
    key = _rows("key", key, dev, None, heads, dim)
    tokens = key.shape[0]
    value = _rows("value", value, dev, tokens, heads, dim)
    if key.dtype is not value.dtype:
        raise ValueError(f"key and value must share a dtype, got {key.dtype} and {value.dtype}")
    batch, width = _batch(dev, tokens, page_table, context_lens, token_starts)
    q_heads, q_type, q_strides, query_out = 0, 0, (0, 0), None
    if query is not None:
        query = _rows("query", query, dev, tokens, None, dim)
        q_heads, q_type, q_strides = query.shape[1], _TYPES[query.dtype], query.stride()
        query_out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    rows = rotary = table_type = 0
    strides = (0, 0)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None and sin is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not sin.dtype or cos.dtype not in _TYPES:
            raise ValueError("cos and sin must be [rows, rotary_dim] of one floating dtype")
        if cos.device != dev or sin.device != dev:
            raise ValueError("cos and sin must be on the pool's device")
        cos, sin = (t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous() for t in (cos, sin))
        rows, rotary = cos.shape
        table_type, strides = _TYPES[cos.dtype], (cos.stride(0), sin.stride(0))
    elif positions is not None or pair_axes is not None or tables_by_token:
        raise ValueError("positions, pair_axes and tables_by_token need cos and sin")
    axes, wide, pos_stride, axis_bytes = 1, 0, 0, None
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != dev:
            raise ValueError("positions must be int32 or int64 on the pool's device")
        if positions.dim() not in (1, 2) or positions.shape[-1] != tokens:
            raise ValueError(f"positions must be [{tokens}] or [axes, {tokens}], got {tuple(positions.shape)}")
        if tokens > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
        if positions.dim() == 2:
            axes, pos_stride = positions.shape[0], positions.stride(0)
        wide = int(positions.dtype is torch.int64)
    if pair_axes is not None:
        if len(pair_axes) != rotary // 2:
            raise ValueError(f"pair_axes must name {rotary // 2} axes, got {len(pair_axes)}")
        axis_bytes = _axis_bytes(tuple(pair_axes))
    for name, t in (("signs_left", signs_left), ("signs_right", signs_right)):
        if t is not None and (t.dtype is not torch.float32 or t.shape != (dim,) or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 [{dim}] on the pool's device")
    flags = (_lib.TQ_ROTATE_VALUES if rotate_values else 0) | (_lib.TQ_TABLES_BY_TOKEN if tables_by_token else 0)
    _launch(
        dev, "tq_paged_append", key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
        _TYPES[key.dtype], ptr(query), q_strides[0], q_strides[1], q_type, q_heads, ptr(query_out), tokens, heads, dim,
        key_pages.data_ptr(), value_pages.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), pages, size,
        page_table.data_ptr(), max(page_table.stride(0), width), width, context_lens.data_ptr(), ptr(token_starts), batch,
        ptr(cos), strides[0], ptr(sin), strides[1], table_type, rows, rotary, ptr(positions), wide, pos_stride, axes,
        axis_bytes, ptr(signs_left), ptr(signs_right), flags,
    )
    return query_out


def paged_dequantize(
    page_ids: torch.Tensor,
    *,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    dtype: torch.dtype = torch.float32,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[count, kv_heads, page_size, head_dim]`` that pages ``page_ids`` (int32 ``[count]``) stand for
    (the counterpart of ``export_dequantized``, cache.py:189-214); a number outside the pool gives zeros."""
    dev, pages, heads, size, dim = _pool(key_pages, value_pages, key_scales, value_scales)
    if page_ids.dtype is not torch.int32 or page_ids.dim() != 1 or page_ids.device != dev or not page_ids.is_contiguous():
        raise ValueError("page_ids must be contiguous int32 [count] on the pool's device")
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    count = page_ids.shape[0]
    keys, values = (torch.empty((count, heads, size, dim), dtype=dtype, device=dev) for _ in range(2))
    _launch(
        dev, "tq_paged_dequantize", page_ids.data_ptr(), count, key_pages.data_ptr(), value_pages.data_ptr(),
        key_scales.data_ptr(), value_scales.data_ptr(), pages, size, heads, dim, keys.data_ptr(), values.data_ptr(), _TYPES[dtype],
    )
    return keys, values


@lru_cache(maxsize=None)
def _num_cus(dev: torch.device) -> int:
    return int(torch.cuda.get_device_properties(dev).multi_processor_count)


@lru_cache(maxsize=1024)
def _workspace_bytes(*shape: int) -> int:
    return int(_lib.call("tq_paged_attention_workspace_bytes", *shape))


def paged_attention(
    query: torch.Tensor,
    *,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    token_starts: torch.Tensor | None = None,
    max_tokens: int | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of each sequence's newest tokens ``[tokens, query_heads, head_dim]`` over its pages.

    Row i of a sequence's n stands at position ``context_lens[b] - n + i`` and sees the keys up to it; a row that sees
    none gives zeros.  ``max_tokens``, the most rows any sequence has, only chooses the kernel (None: as many as there
    may be); ``scale`` is ``head_dim ** -0.5`` unless given.  The result has ``query``'s dtype; rows of no sequence are
    zero in a new tensor and left as they were in ``out``.
    """
    dev, pages, heads, size, dim = _pool(key_pages, value_pages, key_scales, value_scales)
    query = _rows("query", query, dev, None, None, dim)
    tokens, q_heads = query.shape[0], query.shape[1]
    batch, width = _batch(dev, tokens, page_table, context_lens, token_starts)
    if out is None:
        out = (torch.empty if token_starts is None else torch.zeros)(query.shape, dtype=query.dtype, device=dev)
    else:
        if out.shape != query.shape or out.dtype is not query.dtype or out.device != dev:
            raise ValueError(f"out must be {query.dtype} {tuple(query.shape)} on the pool's device")
        if out.stride(2) != 1 or out.is_neg():
            raise ValueError("out must have unit stride along head_dim")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("the paged cache has no backward pass: out wants a gradient (use torch.no_grad())")
        if out.untyped_storage().data_ptr() == query.untyped_storage().data_ptr():
            raise ValueError("out must not share memory with query")
    most = 0 if max_tokens is None else int(max_tokens)
    if max_tokens is not None and most < 1:
        raise ValueError("max_tokens must be positive")
    nbytes = _workspace_bytes(tokens, batch, int(token_starts is not None), q_heads, heads, dim, width, size, most, _num_cus(dev))
    # A tensor of the call's own, from the stream's pool or the graph's: calls on other streams and other graphs'
    # replays have theirs.
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch(
        dev, "tq_paged_attention", query.data_ptr(), query.stride(0), query.stride(1), _TYPES[query.dtype], tokens, q_heads, heads,
        dim, key_pages.data_ptr(), value_pages.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), pages, size,
        page_table.data_ptr(), max(page_table.stride(0), width), width, context_lens.data_ptr(), ptr(token_starts), batch, most,
        1.0 / sqrt(dim) if scale is None else float(scale), ptr(workspace), nbytes, out.data_ptr(), out.stride(0), out.stride(1),
    )
    return out
