"""The paged key-value caches that ``HipContext.kv_append`` fills and
``HipContext.attention_paged`` reads, and the pool that
``HipContext.plan_pages`` hands their pages out of (include/headshot_hip.h)."""
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


class PagedKV8:
    """``PagedKV`` held in 8 bits: ``k``, ``v`` (n_pages, heads, page, head_dim)
    of ``torch.float8_e4m3fn`` codes, ``k_scale``, ``v_scale`` (n_pages, heads) of
    ``torch.float8_e8m0fnu``, powers of two. A value is its code times its
    page's and head's scale, as ``dtype`` holds that (f16: multiples of 2^-24 below
    2^-14, infinite past its range). ``dtype`` is the type of the rows beside it, f32
    or f16. ``page_table`` and ``lens`` are as there."""
    __slots__ = ("k", "v", "k_scale", "v_scale", "page_table", "lens", "dtype", "shape", "device_index")

    def __init__(self, k, v, k_scale, v_scale, page_table, lens, dtype):
        for name, t in zip(self.__slots__, (k, v, k_scale, v_scale, page_table, lens, dtype)):
            object.__setattr__(self, name, t)
        self._check()

    __setattr__ = PagedKV.__setattr__

    def __reduce__(self):  # copies and pickles
        return PagedKV8, (self.k, self.v, self.k_scale, self.v_scale, self.page_table, self.lens, self.dtype)

    def _check(self) -> None:
        k, v, ks, vs, table, lens = self.k, self.v, self.k_scale, self.v_scale, self.page_table, self.lens
        assert self.dtype in (torch.float32, torch.float16), "cache: dtype of its rows"
        assert k.dim() == 4 and v.shape == k.shape, "cache: k and v (n_pages, heads, page, d)"
        assert k.dtype == v.dtype == torch.float8_e4m3fn, "cache: k and v must be float8_e4m3fn"
        assert ks.shape == k.shape[:2] and vs.shape == ks.shape, "cache: scales (n_pages, heads)"
        assert ks.dtype == vs.dtype == torch.float8_e8m0fnu, "cache: scales must be float8_e8m0fnu"
        assert table.dim() == 2 and table.dtype == torch.int32, "page_table wants (sequences, max_pages) int32"
        assert lens.shape == table.shape[:1] and lens.dtype == torch.int32, "lens wants (sequences,) int32"
        every = (k, v, ks, vs, table, lens)
        assert all(t.is_contiguous() for t in every), "cache tensors must be contiguous"
        assert len({t.get_device() for t in every}) == 1, "cache tensors must share a device"
        # (n_pages, heads, page, head_dim, sequences, max_pages)
        object.__setattr__(self, "shape", (*k.shape, *table.shape))
        object.__setattr__(self, "device_index", k.get_device())

    heads = property(lambda self: self.shape[1])
    page = property(lambda self: self.shape[2])
    head_dim = property(lambda self: self.shape[3])

    @staticmethod
    def empty(n_pages: int, heads: int, page: int, head_dim: int, dtype, page_table,
              lens) -> "PagedKV8":
        """A cache of uninitialised pages on ``page_table``'s device."""
        def pool(shape, kind):
            return torch.empty(shape, dtype=kind, device=page_table.device)

        codes, scales = (n_pages, heads, page, head_dim), (n_pages, heads)
        return PagedKV8(pool(codes, torch.float8_e4m3fn), pool(codes, torch.float8_e4m3fn),
                        pool(scales, torch.float8_e8m0fnu), pool(scales, torch.float8_e8m0fnu),
                        page_table, lens, dtype)


def in_eight_bits(cache) -> bool:
    """Whether ``cache`` is a ``PagedKV8``, a class made from it included; what is neither that nor a ``PagedKV``
    is refused, since the pools' bytes alone do not say what they hold."""
    if isinstance(cache, PagedKV8):
        return True
    assert isinstance(cache, PagedKV), f"cache wants a PagedKV or a PagedKV8, not {type(cache).__name__}"
    return False


class PagePool:
    """The pages of caches that share ``page_table`` (sequences, max_pages) and
    ``lens`` (sequences,): entry i of a sequence is its page of keys [i page,
    (i + 1) page), -1 where it has none. Free pages lie in a ring, ``free``
    (n_pages,), ``state[1]`` of them from place ``state[0]`` on; ``state[2]``
    is the number of pages that the last ``plan_pages`` call did not get.
    All int32, contiguous and on one device; the tensors stay, their values
    change from call to call."""
    __slots__ = ("page_table", "lens", "free", "state", "page", "shape", "device_index")

    def __init__(self, page_table, lens, free, state, page: int):
        every = (page_table, lens, free, state)
        assert page_table.dim() == 2 and lens.shape == page_table.shape[:1], \
            "pool: page_table (sequences, max_pages) and lens (sequences,)"
        assert free.dim() == 1 and state.shape == (3,), "pool: free (n_pages,) and state (3,)"
        assert all(t.dtype == torch.int32 and t.is_contiguous() for t in every), "pool tensors must be contiguous int32"
        assert len({t.get_device() for t in every}) == 1, "pool tensors must share a device"
        assert page > 0 and page & (page - 1) == 0, f"pool: page {page} is no power of two"
        for name, t in zip(self.__slots__, (*every, page)):
            object.__setattr__(self, name, t)
        # (sequences, max_pages, n_pages)
        object.__setattr__(self, "shape", (*page_table.shape, free.shape[0]))
        object.__setattr__(self, "device_index", page_table.get_device())

    def __setattr__(self, name, value):
        raise AttributeError("a pool's tensors stay; write into them")

    def __reduce__(self):
        return PagePool, (self.page_table, self.lens, self.free, self.state, self.page)

    @staticmethod
    def empty(sequences: int, max_pages: int, n_pages: int, page: int, device) -> "PagePool":
        """Sequences without tokens, and every page free."""
        def ints(shape, value):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        state = torch.tensor([0, n_pages, 0], dtype=torch.int32, device=device)
        return PagePool(ints((sequences, max_pages), -1), ints((sequences,), 0),
                        torch.arange(n_pages, dtype=torch.int32, device=device), state, page)
