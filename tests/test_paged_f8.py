"""The 8-bit cache's operators and the pages' hand-out on the CPU: refusals through the C ABI with addresses
that are never dereferenced and through the Python surface, and the references that the GPU tests use. Nothing
here launches a kernel."""
import copy
import ctypes
import math

import pytest
import torch

import f8_reference as F
from headshot_amd import _lib, context
from headshot_amd.paged import PagedKV, PagedKV8, PagePool

L = _lib.load()
F16, F32 = _lib.HS_F16, _lib.HS_F32
OK, EINVAL, EUNSUPPORTED = _lib.HS_OK, _lib.HS_EINVAL, _lib.HS_EUNSUPPORTED
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def at(i):
    """The i-th of some buffers 256 MiB apart."""
    return ctypes.c_void_p(0x10000000 * (i + 1))


def odd(i, by=8):
    return ctypes.c_void_p(0x10000000 * (i + 1) + by)


def refused(status, code, needle):
    assert status == code, _lib.status_name(status)
    assert needle in L.hs_last_error().decode(), L.hs_last_error().decode()


def append(dt=F16, q=at(0), qs=256, k=at(1), ks=128, v=at(2), vs=128, qw=None, qb=None, kw=None, kb=None, sn=None,
           cs=None, rows=0, pos=None, off=at(3), table=at(4), lens=at(5), qo=at(6), ko=at(7), kc=at(8), vc=at(9),
           kx=at(10), vx=at(11), n=10, b=2, h=4, h_kv=2, d=64, page=16, n_pages=8, max_pages=4, eps=1e-5):
    return L.hs_kv_append_f8(None, dt, q, qs, k, ks, v, vs, qw, qb, kw, kb, sn, cs, rows, pos, off, table, lens, qo, ko,
                             kc, vc, kx, vx, n, b, h, h_kv, d, page, n_pages, max_pages, eps)


def test_append_refusals():
    refused(append(dt=7), EINVAL, "dtype")
    refused(append(h=3), EINVAL, "heads")
    refused(append(h_kv=0), EINVAL, "heads")
    refused(append(d=32), EUNSUPPORTED, "head_dim")
    refused(append(page=24), EUNSUPPORTED, "power of two")
    refused(append(page=0), EINVAL, "page")
    refused(append(n=-1), EINVAL, "negative")
    refused(append(off=None), EINVAL, "one token per sequence")
    refused(append(qw=at(12)), EINVAL, "weight and bias")
    refused(append(kb=at(12)), EINVAL, "weight and bias")
    refused(append(sn=at(12)), EINVAL, "sin and cos")
    refused(append(pos=at(12)), EINVAL, "positions")
    refused(append(kw=at(12), kb=at(13), eps=0.0), EINVAL, "eps")
    refused(append(k=None), EINVAL, "null k")
    refused(append(v=None), EINVAL, "null v")
    refused(append(qo=None), EINVAL, "null q_out")
    refused(append(kc=None), EINVAL, "null cache")
    refused(append(lens=None), EINVAL, "null cache")
    refused(append(kx=None), EINVAL, "null scales")
    refused(append(vx=None), EINVAL, "null scales")
    refused(append(ks=120), EINVAL, "overlap")
    refused(append(ks=132), EUNSUPPORTED, "16-byte")
    refused(append(k=odd(1)), EUNSUPPORTED, "16-byte")
    refused(append(kc=odd(8)), EUNSUPPORTED, "16-byte")
    refused(append(qo=odd(6)), EUNSUPPORTED, "16-byte")
    refused(append(ko=at(1)), EINVAL, "overlaps an input")
    refused(append(kc=at(2)), EINVAL, "overlaps an input")
    refused(append(kx=at(0)), EINVAL, "overlaps an input")
    refused(append(vc=at(8)), EINVAL, "outputs overlap")
    refused(append(qo=at(9)), EINVAL, "outputs overlap")
    refused(append(kx=at(8)), EINVAL, "outputs overlap")
    refused(append(vx=at(10)), EINVAL, "outputs overlap")
    refused(append(n=1 << 29), EINVAL, "2^30")
    refused(append(page=1 << 20, max_pages=1 << 10), EINVAL, "2^30")
    refused(append(n_pages=1 << 30), EINVAL, "too large")
    assert append(n=0, q=None, k=None, v=None, qo=None, ko=None, kc=None, vc=None, kx=None, vx=None, lens=None) == OK
    assert append(n=0, b=0, off=None) == OK


def paged(dt=F16, q=at(0), qs=256, kc=at(1), vc=at(2), kx=at(3), vx=at(4), table=at(5), lens=at(6), out=at(7),
          ws=at(8), nbytes=1 << 27, b=2, h=4, h_kv=2, d=64, page=16, n_pages=8, max_pages=4, scale=0.125):
    return L.hs_attention_paged_f8(None, dt, q, qs, kc, vc, kx, vx, table, lens, out, ws, nbytes, b, h, h_kv, d, page,
                                   n_pages, max_pages, scale)


def test_paged_refusals():
    refused(paged(dt=2), EINVAL, "dtype")
    refused(paged(h=5), EINVAL, "heads")
    refused(paged(d=256), EUNSUPPORTED, "head_dim")
    refused(paged(b=-1), EINVAL, "negative")
    refused(paged(page=48), EUNSUPPORTED, "power of two")
    refused(paged(q=None), EINVAL, "null q")
    refused(paged(out=None), EINVAL, "null")
    refused(paged(lens=None), EINVAL, "null")
    refused(paged(table=None), EINVAL, "null")
    refused(paged(kc=None), EINVAL, "null")
    refused(paged(kx=None), EINVAL, "null scales")
    refused(paged(qs=200), EINVAL, "overlap")
    refused(paged(qs=260), EUNSUPPORTED, "16-byte")
    refused(paged(vc=odd(2)), EUNSUPPORTED, "16-byte")
    refused(paged(out=odd(7)), EUNSUPPORTED, "16-byte")
    refused(paged(ws=odd(8)), EUNSUPPORTED, "16-byte")
    refused(paged(scale=math.nan), EINVAL, "finite")
    refused(paged(scale=math.inf), EINVAL, "finite")
    refused(paged(nbytes=0), EINVAL, "workspace")
    refused(paged(ws=None), EINVAL, "workspace")
    refused(paged(ws=at(1)), EINVAL, "workspace overlaps")
    refused(paged(ws=at(7)), EINVAL, "overlaps")
    refused(paged(out=at(3)), EINVAL, "overlaps")
    refused(paged(out=at(2)), EINVAL, "overlaps")
    refused(paged(b=1 << 22), EINVAL, "2^23")
    assert L.hs_attention_paged_f8_workspace(2, 4, 2, 64) > 0
    for bad in [(0, 4, 2, 64), (2, 5, 2, 64), (2, 4, 0, 64), (2, 4, 2, 96), (1 << 22, 4, 2, 64), (1, 8192, 2, 64)]:
        assert L.hs_attention_paged_f8_workspace(*bad) == 0
    assert paged(b=0, q=None, out=None) == OK


def prompts(dt=F16, q=at(0), qs=256, kc=at(1), vc=at(2), kx=at(3), vx=at(4), table=at(5), lens=at(6), off=at(7),
            out=at(8), ws=at(9), nbytes=1 << 27, n=10, b=2, h=4, h_kv=2, d=64, page=16, n_pages=8, max_pages=4, causal=1,
            scale=0.125):
    return L.hs_attention_prompts_f8(None, dt, q, qs, kc, vc, kx, vx, table, lens, off, out, ws, nbytes, n, b, h, h_kv,
                                     d, page, n_pages, max_pages, causal, scale)


def test_prompts_refusals():
    refused(prompts(dt=2), EINVAL, "dtype")
    refused(prompts(h=5), EINVAL, "heads")
    refused(prompts(d=96), EUNSUPPORTED, "head_dim")
    refused(prompts(causal=-1), EINVAL, "causal")
    refused(prompts(n=-1), EINVAL, "negative")
    refused(prompts(b=-1), EINVAL, "negative")
    refused(prompts(off=None), EINVAL, "null offsets")
    refused(prompts(out=None), EINVAL, "null")
    refused(prompts(q=None), EINVAL, "null q")
    refused(prompts(table=None), EINVAL, "null")
    refused(prompts(vx=None), EINVAL, "null scales")
    refused(prompts(page=3), EUNSUPPORTED, "power of two")
    refused(prompts(qs=248), EINVAL, "overlap")
    refused(prompts(qs=1 << 22), EINVAL, "2^22")
    refused(prompts(scale=math.inf), EINVAL, "finite")
    refused(prompts(q=odd(0)), EUNSUPPORTED, "16-byte")
    refused(prompts(kc=odd(1)), EUNSUPPORTED, "16-byte")
    refused(prompts(out=odd(8)), EUNSUPPORTED, "16-byte")
    refused(prompts(out=at(2)), EINVAL, "overlaps")
    refused(prompts(out=at(4)), EINVAL, "overlaps")
    refused(prompts(n=1 << 29), EINVAL, "2^30")
    refused(prompts(max_pages=1 << 26), EINVAL, "2^30")
    assert prompts(n=0) == OK
    assert prompts(b=0) == OK


def plan(counts=at(0), lens=at(1), table=at(2), free=at(3), state=at(4), off=at(5), pos=at(6), slots=at(7), ws=at(8),
         nbytes=1 << 27, n=10, b=2, page=16, n_pages=8, max_pages=4):
    return L.hs_plan_pages(None, counts, lens, table, free, state, off, pos, slots, ws, nbytes, n, b, page, n_pages, max_pages)


def test_plan_refusals():
    refused(plan(n=-1), EINVAL, "negative")
    refused(plan(n_pages=-1), EINVAL, "negative")
    refused(plan(page=0), EINVAL, "page")
    refused(plan(page=24), EUNSUPPORTED, "power of two")
    refused(plan(page=1 << 20, max_pages=1 << 10), EINVAL, "2^30")
    refused(plan(n=1 << 30), EINVAL, "2^30")
    refused(plan(b=1 << 16, max_pages=1 << 16), EINVAL, "2^30")
    for name in ("counts", "lens", "table", "free", "state", "off"):
        refused(plan(**{name: None}), EINVAL, "null")
    refused(plan(lens=odd(1, 2)), EUNSUPPORTED, "aligned")
    refused(plan(slots=odd(7, 4)), EUNSUPPORTED, "aligned")
    refused(plan(lens=at(0)), EINVAL, "overlap")
    refused(plan(pos=at(7)), EINVAL, "overlap")
    refused(plan(state=at(3)), EINVAL, "overlap")
    assert L.hs_plan_pages_workspace(10, 2, 4) == 0
    assert L.hs_plan_pages_workspace(1 << 20, 2, 4) > 0
    refused(plan(n=1 << 20, nbytes=8), EINVAL, "workspace")
    refused(plan(n=1 << 20, ws=None), EINVAL, "workspace")
    refused(plan(n=1 << 20, ws=odd(8)), EUNSUPPORTED, "aligned")
    refused(plan(n=1 << 20, ws=at(6)), EINVAL, "overlap")


# ------------------------------------------------------------------ Python


def cache(pages=5, heads=2, page=16, d=64, b=3, width=4, dtype=torch.float16):
    return PagedKV8.empty(pages, heads, page, d, dtype, torch.zeros((b, width), dtype=torch.int32),
                          torch.zeros(b, dtype=torch.int32))


def test_cache_checks_itself():
    c = cache()
    assert c.shape == (5, 2, 16, 64, 3, 4) and (c.heads, c.page, c.head_dim) == (2, 16, 64)
    assert c.k.dtype == E4M3 and c.k_scale.dtype == E8M0 and c.k_scale.shape == (5, 2)
    parts = (c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lens)
    for i, wrong in [(0, c.k.view(torch.uint8)), (1, c.v[:4]), (2, c.k_scale.float()), (3, c.v_scale[:, :1]),
                     (4, c.page_table.long()), (5, c.lens[:2]), (0, c.k.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :, :])]:
        with pytest.raises(AssertionError):
            PagedKV8(*parts[:i], wrong, *parts[i + 1:], torch.float16)
    with pytest.raises(AssertionError):
        PagedKV8(*parts, torch.bfloat16)
    with pytest.raises(AssertionError):
        c.k = c.k[:3]
    assert c.k is parts[0]
    c.lens = torch.ones(3, dtype=torch.int32)
    twin = copy.copy(c)
    deep = copy.deepcopy(c)
    assert twin.k is c.k and twin.dtype == torch.float16 and deep.shape == c.shape and deep.k is not c.k


def test_pool_checks_itself():
    p = PagePool.empty(3, 4, 7, 16, "cpu")
    assert p.shape == (3, 4, 7) and p.free.tolist() == list(range(7)) and p.state.tolist() == [0, 7, 0]
    assert (p.page_table == -1).all() and (p.lens == 0).all()
    parts = (p.page_table, p.lens, p.free, p.state)
    for i, wrong in [(0, p.page_table[0]), (1, p.lens[:2]), (2, p.free.long()), (3, p.state[:2])]:
        with pytest.raises(AssertionError):
            PagePool(*parts[:i], wrong, *parts[i + 1:], 16)
    for page in (0, 24, -16):
        with pytest.raises(AssertionError):
            PagePool(*parts, page)
    with pytest.raises(AttributeError):
        p.lens = p.lens
    assert copy.copy(p).free is p.free


def bare():
    """A context without a device: the checks before a launch."""
    ctx = context.HipContext.__new__(context.HipContext)
    ctx.lib = L
    return ctx


def test_python_refusals(monkeypatch):
    monkeypatch.setattr(context, "_device", lambda: -1)  # CPU tensors' device number
    ctx, c = bare(), cache()
    rows = lambda n, w, t=torch.float16: torch.zeros(n, w, dtype=t)  # noqa: E731
    with pytest.raises(AssertionError, match="one token per sequence"):
        ctx.kv_append(c, rows(2, 128), rows(2, 128))
    with pytest.raises(AssertionError, match="k wants"):
        ctx.kv_append(c, rows(3, 128, torch.float32), rows(3, 128))
    with pytest.raises(AssertionError, match="one query row"):
        ctx.attention_paged(rows(2, 256), c)
    with pytest.raises(AssertionError, match="q wants"):
        ctx.attention_paged(rows(3, 256, torch.float32), c)
    plain = PagedKV.empty(5, 2, 16, 64, torch.float16, c.page_table, c.lens)
    off = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AssertionError, match="PagedKV8"):
        ctx.attention_paged_prompts(rows(5, 256), plain, off)
    with pytest.raises(AssertionError, match="offsets"):
        ctx.attention_paged_prompts(rows(5, 256), c, off[:3])
    with pytest.raises(AssertionError, match="offsets"):
        ctx.attention_paged_prompts(rows(5, 256), c, off.long())
    with pytest.raises(AssertionError, match="causal"):
        ctx.attention_paged_prompts(rows(5, 256), c, off, causal=-1)
    with pytest.raises(AssertionError, match="out"):
        ctx.attention_paged_prompts(rows(5, 256), c, off, out=rows(4, 256))
    pool = PagePool.empty(3, 4, 7, 16, "cpu")
    counts = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(AssertionError, match="counts"):
        ctx.plan_pages(pool, counts.long(), 4)
    with pytest.raises(AssertionError, match="counts"):
        ctx.plan_pages(pool, counts[:2], 4)
    with pytest.raises(AssertionError, match="n -1"):
        ctx.plan_pages(pool, counts, -1)
    out = (torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int64))
    for i, wrong in [(0, out[0][:3]), (1, out[1].long()), (2, out[2].int())]:
        with pytest.raises(AssertionError):
            ctx.plan_pages(pool, counts, 4, out=(*out[:i], wrong, *out[i + 1:]))
    monkeypatch.setattr(context, "_device", lambda: 0)
    for call in (lambda: ctx.kv_append(c, rows(3, 128), rows(3, 128)), lambda: ctx.attention_paged(rows(3, 256), c),
                 lambda: ctx.attention_paged_prompts(rows(5, 256), c, off), lambda: ctx.plan_pages(pool, counts, 4)):
        with pytest.raises(AssertionError, match="current device"):
            call()


# ------------------------------------------------------------------ the references


def test_codes_of_the_reference():
    """Every code stands for itself, midpoints go to the even neighbour, torch agrees."""
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    fine = every[every.isfinite()].sort().values.unique()
    assert torch.equal(F.round_e4m3(fine), fine)
    mid = (fine[1:] + fine[:-1]) / 2
    assert torch.equal(F.round_e4m3(mid), mid.float().to(E4M3).double())
    x = torch.randn(4096, generator=torch.Generator().manual_seed(1)).mul_(60).clamp_(-448, 448)
    assert torch.equal(F.round_e4m3(x.double()), x.to(E4M3).double())


def test_scales_of_the_reference():
    for e in (-117, -20, -8, 0, 8, 120):
        assert F.exponent_for(448.0 * 2.0 ** e) == e
        assert F.exponent_for(448.0 * 2.0 ** e * (1 + 2.0 ** -20)) == e + 1
    assert F.exponent_for(0.0) == F.exponent_for(1e-40) == -117
    # what a cache holds at most comes back as itself
    for dtype, e in ((torch.float16, 8), (torch.float32, 120)):
        assert F.exponent_for(F.HELD[dtype]) == e and F.HELD[dtype] <= torch.finfo(dtype).max


def test_pages_of_the_reference():
    p = F.Pages(3, 4, 5, 8)
    assert p.plan([9, 0, 8]) == ([0, 9, 9, 17], [*range(9), *range(8)], [*range(9), *range(16, 24)])
    assert p.table == [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]] and p.missing == 0 and p.free == [3, 4]
    p.plan([-9, 24, 1])  # the pages of the first go back behind; the second lacks one, and so does the third
    assert p.table == [[-1] * 4, [3, 4, -1, -1], [2, -1, -1, -1]] and p.missing == 2 and p.free == [0, 1]
    p.plan([0, 8, 8])    # behind a page that was not there: none
    assert p.missing == 2 and p.free == [0, 1] and p.lens == [0, 32, 17]
    p.plan([0, -17, -17])
    assert p.lens == [0, 15, 0] and p.table[1] == [3, 4, -1, -1] and p.free == [0, 1, 2]
