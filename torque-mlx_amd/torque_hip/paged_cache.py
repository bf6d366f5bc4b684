"""``TorquePagedKVCache``: an 8-bit KV cache of several sequences in pages, for one attention layer.

The reference's caches hold one sequence (batch size 1 throughout cache_mlx.py and qwen_mlx.py:633-734).  This class
keeps the pages, page table and lengths that ``ops.paged_append`` and ``ops.paged_attention`` take: sequences come and
go, grow by prompts, single tokens or drafted tokens, and are cut back to the tokens that were accepted.
"""

from __future__ import annotations

from typing import Any, Sequence

import torch

from torque_hip._tensors import device as current_device
from torque_hip.paged import SUPPORTED_PAGE_SIZES, paged_append, paged_attention, paged_dequantize
from torque_hip.rotation import RotationSpec, validate_head_dim


class TorquePagedKVCache:
    """Pages of ``page_size`` tokens, shared by up to ``max_sequences`` sequences of up to ``max_tokens`` tokens each.

    With ``rotation``, keys (and the queries given to ``append``) go into the rotated basis, which spreads a key's large
    channels over all of them before they are held in 8 bits; ``rotate_values`` takes values there too, and ``attend``
    then leaves its result in that basis (``rotation.inverse_device`` takes it back).
    """

    def __init__(
        self,
        *,
        kv_heads: int,
        head_dim: int,
        num_pages: int,
        max_sequences: int,
        max_tokens: int,
        page_size: int = 64,
        rotation: RotationSpec | None = None,
        rotate_values: bool = False,
        device: torch.device | str | None = None,
    ) -> None:
        validate_head_dim(head_dim)
        if page_size not in SUPPORTED_PAGE_SIZES:
            raise ValueError("page_size must be one of " + ", ".join(map(str, SUPPORTED_PAGE_SIZES)))
        for name, value in (("kv_heads", kv_heads), ("num_pages", num_pages), ("max_sequences", max_sequences), ("max_tokens", max_tokens)):
            if value <= 0:
                raise ValueError(f"{name} must be positive")
        if rotation is not None and rotation.head_dim != head_dim:
            raise ValueError(f"rotation head_dim {rotation.head_dim} does not match the cache's {head_dim}")
        if rotate_values and rotation is None:
            raise ValueError("rotate_values needs a rotation")
        self.kv_heads, self.head_dim, self.page_size = kv_heads, head_dim, page_size
        self.num_pages, self.max_sequences, self.max_tokens = num_pages, max_sequences, max_tokens
        self.rotation, self.rotate_values = rotation, rotate_values
        dev = current_device() if device is None else torch.device(device)
        self.key_pages = torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=torch.int8, device=dev)
        self.value_pages = torch.zeros((num_pages, kv_heads, head_dim, page_size), dtype=torch.int8, device=dev)
        self.key_scales, self.value_scales = (torch.ones((num_pages, kv_heads), dtype=torch.float32, device=dev) for _ in range(2))
        self._table = torch.full((max_sequences, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=dev)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}  # of each sequence
        self._lengths: dict[int, int] = {}

    # ------------------------------------------------------------ sequences

    @property
    def device(self) -> torch.device:
        return self.key_pages.device

    @property
    def sequences(self) -> tuple[int, ...]:
        return tuple(sorted(self._lengths))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._lengths[self._known(sequence)]

    def _known(self, sequence: int) -> int:
        if sequence not in self._lengths:
            raise ValueError(f"no sequence {sequence}")
        return sequence

    def add_sequence(self) -> int:
        """A new, empty sequence; its number."""
        for slot in range(self.max_sequences):
            if slot not in self._lengths:
                self._lengths[slot], self._pages[slot] = 0, []
                return slot
        raise ValueError(f"the cache holds {self.max_sequences} sequences already")

    def free_sequence(self, sequence: int) -> None:
        """Forget a sequence; its pages serve others."""
        self.truncate(sequence, 0)
        del self._lengths[sequence], self._pages[sequence]

    def truncate(self, sequence: int, length: int) -> None:
        """Keep a sequence's first ``length`` tokens (after drafted tokens were refused)."""
        if not 0 <= length <= self.length(sequence):
            raise ValueError(f"sequence {sequence} has {self.length(sequence)} tokens, cannot keep {length}")
        pages, keep = self._pages[sequence], -(-length // self.page_size)
        self._free.extend(reversed(pages[keep:]))
        del pages[keep:]
        self._lengths[sequence] = length

    def _plan(self, tokens: int, sequences: Sequence[int] | None, counts: Sequence[int] | None) -> tuple[list[int], list[int]]:
        """The sequences of a call of ``tokens`` rows, and how many of the rows each has."""
        seqs = list(self.sequences) if sequences is None else [self._known(int(s)) for s in sequences]
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        if counts is None:
            if not seqs or tokens % len(seqs):
                raise ValueError(f"{tokens} tokens cannot be dealt out evenly to {len(seqs)} sequences")
            counts = [tokens // len(seqs)] * len(seqs)
        n = [int(c) for c in counts]
        if len(n) != len(seqs) or sum(n) != tokens or any(c < 0 for c in n):
            raise ValueError(f"counts must give {len(seqs)} sequences {tokens} tokens, got {n}")
        return seqs, n

    def reserve(self, sequences: Sequence[int], counts: Sequence[int]) -> None:
        """Pages for ``counts`` more tokens of each sequence; nothing changes where there are too few."""
        need = {}
        for s, n in zip(sequences, counts):
            total = self.length(s) + n
            if total > self.max_tokens:
                raise ValueError(f"sequence {s} would have {total} tokens, the cache holds {self.max_tokens} of each")
            need[s] = -(-total // self.page_size) - len(self._pages[s])
        if sum(need.values()) > len(self._free):
            raise RuntimeError(f"the cache is out of pages: {sum(need.values())} needed, {len(self._free)} free")
        for s, more in need.items():
            if more > 0:
                first = len(self._pages[s])
                self._pages[s].extend(self._free.pop() for _ in range(more))
                self._table[s, first : first + more] = torch.tensor(self._pages[s][first:], dtype=torch.int32, device=self.device)

    def _batch(self, seqs: list[int], counts: list[int]) -> dict[str, Any]:
        numbers = [self._lengths[s] for s in seqs]
        # no wider than the longest sequence: the width is what the attention's choice of kernel knows of the lengths
        table = self._table[:, : max(1, -(-max(numbers, default=0) // self.page_size))]
        table = table[: len(seqs)] if seqs == list(range(len(seqs))) else table[torch.tensor(seqs, device=self.device)]
        if counts == [1] * len(seqs):
            return dict(page_table=table, context_lens=torch.tensor(numbers, dtype=torch.int32, device=self.device), token_starts=None)
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        both = torch.tensor(numbers + starts, dtype=torch.int32, device=self.device)  # one copy
        return dict(page_table=table, context_lens=both[: len(seqs)], token_starts=both[len(seqs) :])

    @property
    def _pool(self) -> dict[str, torch.Tensor]:
        return dict(key_pages=self.key_pages, value_pages=self.value_pages, key_scales=self.key_scales, value_scales=self.value_scales)

    # ------------------------------------------------------------ the calls

    def append(
        self,
        key: torch.Tensor,
        value: torch.Tensor,
        *,
        sequences: Sequence[int] | None = None,
        counts: Sequence[int] | None = None,
        query: torch.Tensor | None = None,
        cos: torch.Tensor | None = None,
        sin: torch.Tensor | None = None,
        positions: torch.Tensor | None = None,
        pair_axes: Sequence[int] | None = None,
        tables_by_token: bool = False,
    ) -> torch.Tensor | None:
        """Append ``[tokens, kv_heads, head_dim]`` keys and values, ``counts`` rows for each of ``sequences`` (all
        sequences and equal shares unless given); the queries turned and rotated, as ``attend`` takes them."""
        if key.dim() != 3:
            raise ValueError(f"key must have shape [tokens, {self.kv_heads}, {self.head_dim}], got {tuple(key.shape)}")
        seqs, n = self._plan(int(key.shape[0]), sequences, counts)
        if cos is not None and positions is None and not tables_by_token:
            longest = max((self._lengths[s] + c for s, c in zip(seqs, n) if c), default=0)
            if longest > cos.shape[0]:
                raise ValueError(f"the rotary tables have {cos.shape[0]} rows, a sequence would have {longest} tokens")
        self.reserve(seqs, n)
        signs = (None, None) if self.rotation is None else self.rotation.device_signs(self.device)
        before = dict(self._lengths)
        for s, c in zip(seqs, n):
            self._lengths[s] += c
        try:
            return paged_append(
                key, value, query=query, cos=cos, sin=sin, positions=positions, pair_axes=pair_axes, tables_by_token=tables_by_token,
                signs_left=signs[0], signs_right=signs[1], rotate_values=self.rotate_values, **self._batch(seqs, n), **self._pool,
            )
        except BaseException:
            self._lengths = before  # the pages stay reserved
            raise

    def attend(
        self,
        query: torch.Tensor,
        *,
        sequences: Sequence[int] | None = None,
        counts: Sequence[int] | None = None,
        scale: float | None = None,
    ) -> torch.Tensor:
        """Causal attention of the newest ``counts`` tokens of each sequence, ``[tokens, query_heads, head_dim]`` rows as
        ``append`` returned them."""
        if query.dim() != 3:
            raise ValueError(f"query must have shape [tokens, heads, {self.head_dim}], got {tuple(query.shape)}")
        seqs, n = self._plan(int(query.shape[0]), sequences, counts)
        return paged_attention(query, max_tokens=max([1, *n]), scale=scale, **self._batch(seqs, n), **self._pool)

    def export_dequantized(self, sequence: int, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """A sequence's keys and values ``[kv_heads, length, head_dim]`` as attention reads them (cache.py:189-214)."""
        length, pages = self.length(sequence), self._pages[sequence]
        ids = torch.tensor(pages, dtype=torch.int32, device=self.device)
        return tuple(  # type: ignore[return-value]
            x.transpose(0, 1).reshape(self.kv_heads, -1, self.head_dim)[:, :length] for x in paged_dequantize(ids, dtype=dtype, **self._pool)
        )
