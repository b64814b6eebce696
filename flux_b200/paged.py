"""A paged key/value cache for serving many sequences of different lengths.

:class:`PagedKVCache` owns the pools, the page table, the lengths and the page
counts, and calls the paged-cache operators of :mod:`flux_b200.operators` on
them.  The reference's caches are dense and hold one sequence.

All state lives on the device and no method waits for it (a caller reads
``status`` tensors when it wants to), so a decode step made of these calls can
be captured into a CUDA graph."""

from __future__ import annotations

import torch

from flux_b200 import operators as ops


class PagedKVCache:
    """Pools of ``pages`` pages of ``page_size`` rows for ``layers`` layers, shared by ``sequences`` sequences of at
    most ``max_rows`` rows, rounded up to whole pages.

    A step: :meth:`advance` gives every listed sequence room for its new row and returns the rows' positions; per
    layer, :meth:`write` rotates and stores the packed QKV rows and :meth:`attend` attends over the cache."""

    def __init__(self, *, layers: int, pages: int, kv_heads: int, head_dim: int, sequences: int, max_rows: int,
                 page_size: int = 16, dtype: torch.dtype = torch.float32, device: torch.device | str = "cuda"):
        if min(layers, pages, kv_heads, head_dim, sequences, max_rows, page_size) < 1:
            raise ValueError("paged cache sizes must be positive")
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError("paged cache pages must be float32, bfloat16 or float16")
        if head_dim % 8 != 0 or head_dim > 256:
            raise ValueError("paged cache head_dim must be a multiple of 8 up to 256")
        columns = -(-max_rows // page_size)
        if (pages > 2 ** 20 or sequences > 2 ** 18 or kv_heads > 65535 or page_size > 65536
                or columns * page_size >= 2 ** 31):
            raise ValueError("paged cache sizes must be at most 1048576 pages, 262144 sequences, 65535 KV heads, 65536 "
                             "rows of a page and 2147483647 rows of a sequence")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.page_size = page_size
        self.key_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.value_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.page_table = torch.full((sequences, columns), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int64, device=device)
        self.page_counts = torch.zeros(pages, dtype=torch.int32, device=device)

    def reserve(self, sequences: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        """Pages for ``rows[i]`` more rows of ``sequences[i]``; statuses (0 done, 1 refused, 2 no pages left)."""
        return ops.cache_sequences_reserve_native(self.page_table, self.lengths, self.page_counts, sequences, rows,
                                                  self.page_size)

    def advance(self, sequences: torch.Tensor, rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Reserve and count ``rows[i]`` more rows of each listed sequence.  Returns their first positions and the
        statuses; a sequence whose status is not 0 keeps its length, and its position is -1 (its rows are not
        written)."""
        status = self.reserve(sequences, rows)
        granted = status == 0
        inside = sequences.clamp(0, self.lengths.shape[0] - 1)
        positions = torch.where(granted, self.lengths[inside], -1)
        self.lengths.index_add_(0, inside, torch.where(granted, rows, 0))
        return positions, status

    def write(self, layer: int, packed_qkv, cos, sin, positions, sequences=None) -> torch.Tensor:
        """Rotated queries ``[tokens, Hq, 1, D]``; keys and values go into ``layer``'s pages."""
        return ops.paged_qkv_rope_cache_native(packed_qkv, cos, sin, self.key_pages[layer], self.value_pages[layer],
                                               self.page_table, positions, sequences)

    def attend(self, layer: int, query, scale: float, sequences=None) -> torch.Tensor:
        """Attention of one query row per sequence (per listed sequence) over ``layer``'s rows; zeros for a listed
        index that is no sequence."""
        table, lengths = self.page_table, self.lengths
        if sequences is not None:
            inside = sequences.clamp(0, lengths.shape[0] - 1)
            table, lengths = table[inside], torch.where(inside == sequences, lengths[inside], 0)
        return ops.paged_gqa_decode_attention_native(query, self.key_pages[layer], self.value_pages[layer], table,
                                                     lengths, scale)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
        """Each empty ``children[i]`` becomes a copy of ``parents[i]``; statuses as for :meth:`reserve`."""
        return ops.cache_sequences_fork_native(self.key_pages, self.value_pages, self.page_table, self.lengths,
                                               self.page_counts, parents, children)

    def free(self, sequences: torch.Tensor) -> None:
        """Drop the listed sequences and release their pages."""
        ops.cache_sequences_free_native(self.page_table, self.lengths, self.page_counts, sequences)

    def compact(self) -> torch.Tensor:
        """Move the used pages to the front of the pools; returns how many there are (a device scalar)."""
        return ops.cache_pages_compact_native(self.key_pages, self.value_pages, self.page_table, self.page_counts)


__all__ = ["PagedKVCache"]
