"""Which kernels a cache goes to: by what its pools hold, not by the exact class. On the CPU, with the launches
recorded instead of made."""
import pytest
import torch

from headshot_amd import _lib, aggregator, context
from headshot_amd.paged import PagedKV, PagedKV8

L = _lib.load()


class Eight(PagedKV8):
    """A caller's own class, with nothing of its own."""


class Full(PagedKV):
    """The same of a full cache."""


class Other:
    """Shaped like a cache, and neither class."""

    def __init__(self, like):
        for name in ("k", "v", "page_table", "lens", "shape", "dtype", "device_index"):
            setattr(self, name, getattr(like, name))


def caches():
    table, lens = torch.zeros((3, 4), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    eight = PagedKV8.empty(5, 2, 16, 64, torch.float16, table, lens)
    full = PagedKV.empty(5, 2, 16, 64, torch.float16, table, lens)
    parts = (full.k, full.v, table, lens)
    return (eight, Eight(eight.k, eight.v, eight.k_scale, eight.v_scale, table, lens, torch.float16)), (full, Full(*parts))


@pytest.fixture
def ctx(monkeypatch):
    """A context without a device that keeps the entry points it would call."""
    monkeypatch.setattr(context, "_device", lambda: -1)  # CPU tensors' device number
    c = context.HipContext.__new__(context.HipContext)
    c.lib, c.calls = L, []
    c._launch_held = lambda name, fn, held, *args: c.calls.append(fn.__name__)
    return c


def rows(n, w):
    return torch.zeros(n, w, dtype=torch.float16)


def test_classes_made_from_the_caches(ctx):
    offsets = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    eights, fulls = caches()
    for cache in eights:
        ctx.kv_append(cache, rows(3, 128), rows(3, 128))
        ctx.attention_paged(rows(3, 256), cache)
        ctx.attention_paged_prompts(rows(3, 256), cache, offsets)
    assert ctx.calls == ["hs_kv_append_f8", "hs_attention_paged_f8", "hs_attention_prompts_f8"] * 2
    ctx.calls.clear()
    for cache in fulls:
        ctx.kv_append(cache, rows(3, 128), rows(3, 128))
        ctx.attention_paged(rows(3, 256), cache)
        with pytest.raises(AssertionError, match="PagedKV8"):
            ctx.attention_paged_prompts(rows(3, 256), cache, offsets)
    assert ctx.calls == ["hs_kv_append", "hs_attention_paged"] * 2


def test_what_is_no_cache_is_refused(ctx):
    offsets = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    for like in (c[0] for c in caches()):
        other = Other(like)
        for call in (lambda: ctx.kv_append(other, rows(3, 128), rows(3, 128)),
                     lambda: ctx.attention_paged(rows(3, 256), other),
                     lambda: ctx.attention_paged_prompts(rows(3, 256), other, offsets),
                     lambda: aggregator.block_forward_cached(None, None, rows(3, 128), other, 2)):
            with pytest.raises(AssertionError, match="PagedKV8"):
                call()
    assert ctx.calls == []


def test_block_over_a_class_made_from_the_cache(monkeypatch):
    """A prompt over such a cache is not refused as one into held sequences: it takes the path over pages."""
    taken = []

    class Ctx:
        def layernorm(self, x, *_, **__):
            return x

        def linear(self, x, *_):
            return torch.cat([x, x, x], 1)

        def kv_append(self, cache, k, v, offsets, q=None, k_rows=False, **_):
            assert not k_rows
            return q, None

        def attention_paged_prompts(self, q, cache, offsets, causal):
            taken.append(type(cache).__name__)
            return q

        def linear_ls_residual(self, x, w, g, res, b):
            return res

        def linear_gelu(self, x, *_):
            return x

    class Weights:
        qkv_w = qkv_b = proj_w = fc1_w = fc2_w = None

        class p:
            ln1 = ln2 = (None, None)
            qn = kn = ls1 = ls2 = proj_b = fc1_b = fc2_b = None

    eight = caches()[0][1]
    eight.lens = torch.full((3,), 9, dtype=torch.int32)  # keys before the call's
    offsets = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    aggregator.block_forward_cached(Ctx(), Weights, rows(3, 128), eight, 2, offsets=offsets)
    assert taken == ["Eight"]
