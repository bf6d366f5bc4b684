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

import ctypes
from functools import lru_cache
from types import ModuleType
from typing import Sequence

import torch

from torque_hip import _lib

SUPPORTED_PAGE_SIZES: tuple[int, ...] = (16, 32, 64)


def _load() -> ModuleType:
    """The CPython module over the C ABI (csrc/paged_binding.cpp), bound to the library that the package has opened."""
    global _MODULE
    if _MODULE is None:
        lib = _lib.load()
        try:
            from torque_hip import _paged
        except ImportError as e:
            raise RuntimeError(
                "torque_hip/_paged.so is not built; run `python -c 'import __graft_entry__ as g; g.build()'` from the repository root"
            ) from e
        address = lambda name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value  # noqa: E731
        _paged.bind(address("tq_paged_append"), address("tq_paged_dequantize"), address("tq_paged_attention"),
                    address("tq_paged_attention_workspace_bytes"), _lib.check)
        _MODULE = _paged
    return _MODULE


_MODULE: ModuleType | None = None


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
    return (_MODULE or _load()).append(
        key, value, key_pages, value_pages, key_scales, value_scales, page_table, context_lens, token_starts, query, cos, sin, positions,
        None if pair_axes is None else _axis_bytes(tuple(pair_axes)), tables_by_token, signs_left, signs_right, rotate_values,
    )


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
    return (_MODULE or _load()).dequantize(page_ids, key_pages, value_pages, key_scales, value_scales, dtype)


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
    if max_tokens is not None and max_tokens < 1:
        raise ValueError("max_tokens must be positive")
    return (_MODULE or _load()).attention(
        query, key_pages, value_pages, key_scales, value_scales, page_table, context_lens, token_starts, max_tokens or 0, scale, out
    )
