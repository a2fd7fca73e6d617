"""The paged key-value cache that ``HipContext.kv_append`` fills and
``HipContext.attention_paged`` reads (include/headshot_hip.h)."""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class PagedKV:
    """One layer's cache over ``page_table`` and ``lens``, which the layers of
    a model share: key p of sequence s is row p % page of page
    ``page_table[s, p // page]``. ``lens`` counts a step's new tokens before
    the step's calls run; the calls change neither array."""
    k: torch.Tensor           # (n_pages, heads, page, head_dim) f32 or f16
    v: torch.Tensor           # like k
    page_table: torch.Tensor  # (sequences, max_pages) int32
    lens: torch.Tensor        # (sequences,) int32: keys of each sequence

    heads = property(lambda self: self.k.shape[1])
    page = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])

    @staticmethod
    def empty(n_pages: int, heads: int, page: int, head_dim: int, dtype, page_table,
              lens) -> "PagedKV":
        """A cache of uninitialised pages on ``page_table``'s device."""
        def pool():
            return torch.empty((n_pages, heads, page, head_dim), dtype=dtype,
                               device=page_table.device)

        return PagedKV(pool(), pool(), page_table, lens)
