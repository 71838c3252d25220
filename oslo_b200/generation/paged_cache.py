"""Keys and values of sequences that come and go, in pages of pools that they share."""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from .. import ops


class PagedKVCache:
    """Per layer two pools ``[pages, heads, page, dim]`` (``quantised``: e4m3 values with a scale per vector), shared by ``rows``
    sequences. Where ``StaticKVCache`` reserves the longest length for every row, a row here holds the pages its tokens need.

    ``extend([n_0, n_1, ...])`` makes room for that many more tokens per row and counts them; every layer then ``append``s their keys and
    values, and reads: ``attend`` for single tokens, ``read`` and ``ops.ragged_attention`` for prompts. ``release(row)`` gives a row's
    pages back. ``lengths`` and ``table`` are the device's copies, updated in place, so a captured step that reads them keeps doing so;
    pages are handed out on the host, before the step. ``max_length``: tokens a row can hold (default: all pages). ``dtype``: the keys' and
    values' type, 16-bit on a GPU."""

    def __init__(self, layers: int, pages: int, page: int, heads: int, dim: int, rows: int, dtype: torch.dtype = torch.bfloat16,
                 device=None, quantised: bool = False, max_length: Optional[int] = None) -> None:
        if min(layers, pages, page, heads, dim, rows) <= 0 or (max_length is not None and max_length <= 0):
            raise ValueError("PagedKVCache: sizes must be positive")
        where = torch.get_default_device() if device is None else torch.device(device)
        if where.type == "cuda" and (dtype not in (torch.bfloat16, torch.float16) or dim > 256 or dim % (16 if quantised else 8)):
            raise ValueError("PagedKVCache: on a GPU keys and values are bf16 or fp16, in heads of a multiple of 8 (quantised: 16) values up to 256")
        store = torch.float8_e4m3fn if quantised else dtype
        shape = (pages, heads, page, dim)
        # zeros in bytes: not every operator exists for 8-bit floats
        make = lambda: torch.zeros(shape, dtype=torch.uint8 if quantised else store, device=device).view(store)  # noqa: E731
        scale = lambda: torch.zeros(shape[:3], dtype=torch.float32, device=device) if quantised else None  # noqa: E731
        self.k, self.v = [make() for _ in range(layers)], [make() for _ in range(layers)]
        self.k_scale, self.v_scale = [scale() for _ in range(layers)], [scale() for _ in range(layers)]
        self.page, self.dtype = page, dtype
        self.max_length = pages * page if max_length is None else min(pages * page, max_length)
        columns = self._pages(self.max_length)
        self.table = torch.full((rows, columns), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        self._table = torch.full((rows, columns), -1, dtype=torch.int32, device="cpu")
        self._lengths: List[int] = [0] * rows
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def _publish(self) -> None:
        self.table.copy_(self._table)
        self.lengths.copy_(torch.tensor(self._lengths, dtype=torch.int32, device="cpu"))

    def extend(self, new: Sequence[int]) -> None:
        """Room for ``new[r]`` more tokens of row ``r``. Refuses, and changes nothing, where pages run out or a row would be longer than
        ``max_length``."""
        if len(new) != len(self._lengths) or any(n < 0 for n in new):
            raise ValueError(f"PagedKVCache: {len(self._lengths)} rows, {len(new)} numbers of new tokens")
        then = [a + int(n) for a, n in zip(self._lengths, new)]
        need = [self._pages(t) - self._pages(a) for t, a in zip(then, self._lengths)]
        if max(then) > self.max_length:
            raise RuntimeError(f"KV cache overflow: {max(then)} tokens in a row, which holds {self.max_length}")
        if sum(need) > len(self._free):
            raise RuntimeError(f"KV cache overflow: {sum(need)} more pages, {len(self._free)} are free")
        for r, n in enumerate(need):
            at = self._pages(self._lengths[r])
            for i in range(at, at + n):
                self._table[r, i] = self._free.pop()
        self._lengths = then
        self._publish()

    def release(self, row: int) -> None:
        """Forget row ``row``."""
        self._free.extend(p for p in self._table[row].tolist() if p >= 0)
        self._table[row] = -1
        self._lengths[row] = 0
        self._publish()

    def append(self, layer: int, k: Tensor, v: Tensor, offsets: Optional[Tensor] = None) -> None:
        """Keys and values ``[T, heads, dim]`` of the tokens that ``extend`` counted last (``ops.paged_append``)."""
        ops.paged_append(k, v, self.k[layer], self.v[layer], self.table, self.lengths, offsets, self.k_scale[layer], self.v_scale[layer])

    def attend(self, layer: int, q: Tensor, window: Optional[int] = None, scale: Optional[float] = None) -> Tensor:
        """Attention of one token per row, ``q`` ``[rows, query heads, dim]`` (``ops.paged_attention``)."""
        return ops.paged_attention(q, self.k[layer], self.v[layer], self.table, self.lengths, window, scale, self.k_scale[layer], self.v_scale[layer])

    def read(self, layer: int) -> Tuple[Tensor, Tensor, Tensor]:
        """All rows' keys and values, one row behind another, and the offsets where they start (``ops.paged_read``)."""
        offsets = [0]
        for n in self._lengths:
            offsets.append(offsets[-1] + n)
        at = torch.tensor(offsets, dtype=torch.int32, device=self.table.device)
        k, v = ops.paged_read(self.k[layer], self.v[layer], self.table, at, offsets[-1], self.k_scale[layer], self.v_scale[layer], self.dtype)
        return k, v, at
