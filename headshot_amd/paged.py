"""The paged key-value cache that ``HipContext.kv_append`` fills and
``HipContext.attention_paged`` reads (include/headshot_hip.h)."""
from __future__ import annotations

import torch


class PagedKV:
    """One layer's cache over ``page_table`` and ``lens``, which the layers of
    a model share: key p of sequence s is row p % page of page
    ``page_table[s, p // page]``. ``lens`` counts a step's new tokens before
    the step's calls run; the calls change neither array.

    ``k``, ``v`` (n_pages, heads, page, head_dim) f32 or f16, ``page_table``
    (sequences, max_pages) and ``lens`` (sequences,) int32, all contiguous and
    on one device. They are checked here and when one is replaced; their
    values may change at any time, their shapes not."""
    __slots__ = ("k", "v", "page_table", "lens", "shape", "dtype", "device_index")

    def __init__(self, k, v, page_table, lens):
        for name, t in zip(("k", "v", "page_table", "lens"), (k, v, page_table, lens)):
            object.__setattr__(self, name, t)
        self._check()

    def __setattr__(self, name, value):
        if getattr(self, name) is not value:
            old = getattr(self, name)
            object.__setattr__(self, name, value)
            try:
                self._check()
            except AssertionError:
                object.__setattr__(self, name, old)
                raise

    def __reduce__(self):  # copies and pickles
        return PagedKV, (self.k, self.v, self.page_table, self.lens)

    def _check(self) -> None:
        k, v, table, lens = self.k, self.v, self.page_table, self.lens
        assert k.dim() == 4 and v.shape == k.shape, "cache: k and v (n_pages, heads, page, d)"
        assert k.dtype == v.dtype and k.dtype in (torch.float32, torch.float16), "cache: k and v dtype"
        assert table.dim() == 2 and table.dtype == torch.int32, "page_table wants (sequences, max_pages) int32"
        assert lens.shape == table.shape[:1] and lens.dtype == torch.int32, "lens wants (sequences,) int32"
        assert all(t.is_contiguous() for t in (k, v, table, lens)), "cache tensors must be contiguous"
        assert len({t.get_device() for t in (k, v, table, lens)}) == 1, "cache tensors must share a device"
        # (n_pages, heads, page, head_dim, sequences, max_pages)
        object.__setattr__(self, "shape", (*k.shape, *table.shape))
        object.__setattr__(self, "dtype", k.dtype)
        object.__setattr__(self, "device_index", k.get_device())

    heads = property(lambda self: self.shape[1])
    page = property(lambda self: self.shape[2])
    head_dim = property(lambda self: self.shape[3])

    @staticmethod
    def empty(n_pages: int, heads: int, page: int, head_dim: int, dtype, page_table,
              lens) -> "PagedKV":
        """A cache of uninitialised pages on ``page_table``'s device."""
        def pool():
            return torch.empty((n_pages, heads, page, head_dim), dtype=dtype,
                               device=page_table.device)

        return PagedKV(pool(), pool(), page_table, lens)
