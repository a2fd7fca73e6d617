"""Values of an 8-bit cache that are no numbers in its rows' type: codes that their page's scale brings past it,
which count as infinite, and NaN, alone and among others, seen by all tokens or by some, of any weight; against
softmax in 64 bits."""
import math

import pytest
import torch

import f8_reference as F
import paged_reference as R
from headshot_amd.paged import PagedKV8

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
WIDE = {F16: 127 + 8, F32: 127 + 120}  # the least scale with which a code (448) passes the type


def i32(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


def bits(t):
    return t.view(torch.uint8)


def make_cache(gen, lens, heads, page, d, dtype):
    """Pages in no order, of ordinary codes and scales, CPU."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen).tolist()
    width = max(need) + 1
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    codes = [(torch.randn((pages, heads, page, d), generator=gen) * 90).clamp(-448, 448).to(E4M3) for _ in range(2)]
    scales = [torch.randint(118, 122, (pages, heads), generator=gen).to(torch.uint8).view(E8M0) for _ in range(2)]
    return PagedKV8(*codes, *scales, i32(table, "cpu"), i32(lens, "cpu"), dtype)


def widen(c, s, key, x, gen, which="v"):
    """Key ``key`` of sequence ``s``, head and channel -> code: its page's scale grows until the largest code is
    infinite, the page's others are small."""
    page = c.page
    at, row = int(c.page_table[s, key // page]), key % page
    codes, scale = getattr(c, which), getattr(c, which + "_scale")
    for h, channel, code in x:
        if int(bits(scale)[at, h]) < WIDE[c.dtype]:
            bits(scale)[at, h] = WIDE[c.dtype]
            codes[at, h] = (torch.randn(codes[at, h].shape, generator=gen) * 0.5).to(E4M3)
        bits(codes)[at, h, row, channel] = code


def reference(q, c, offsets, causal, scale):
    """(n, heads, d) f64 result and bound, of values as the rows' type has them."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    for s in range(len(c.lens)):
        a, b = (s, s + 1) if offsets is None else (offsets[s], offsets[s + 1])
        length = int(c.lens[s])
        k, v = (F.gathered(getattr(c, x), getattr(c, x + "_scale"), c.page_table, length, s)[0].to(c.dtype).double() for x in "kv")
        for t in range(a, b):
            seen = length if causal == 0 or offsets is None else min(((length - (b - t)) // causal + 1) * causal, length)
            o, mag = R.attention(q[t:t + 1].double(), k[:seen], v[:seen], [seen], scale)
            out[t] = o[0]
            finite = [x.nan_to_num(0.0, 0.0, 0.0) for x in (o, mag, q[t:t + 1], k[:seen], v[:seen])]
            bound[t] = R.attention_bound(*finite, [seen], scale, c.dtype)[0]
    return out, bound


def check(ctx, c, new, causal, std, scale, gen, h):
    """``new`` None: attention_paged."""
    d = c.head_dim
    n = len(c.lens) if new is None else sum(new)
    q = (torch.randn((n, h, d), generator=gen) * std).to(c.dtype)
    gpu = PagedKV8(*(t.to(DEV) for t in (c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lens)), c.dtype)
    off = None if new is None else [sum(new[:i]) for i in range(len(new) + 1)]
    if new is None:
        got = ctx.attention_paged(q.to(DEV), gpu, scale=scale)
    else:
        got = ctx.attention_paged_prompts(q.to(DEV), gpu, i32(off), causal=causal, scale=scale)
    got = got.unflatten(1, (h, d)).cpu().double()
    ref, bound = reference(q, c, off, causal, scale)
    odd = ~ref.isfinite()
    assert torch.equal(got[odd].isnan(), ref[odd].isnan()), "NaN places"
    assert torch.equal(got[odd].nan_to_num(0.0), ref[odd].nan_to_num(0.0)), "infinities"
    R.assert_within(got[~odd], ref[~odd], bound[~odd], "finite channels")
    return ref


NEW = [None, [1, 1, 1], [1, 4, 3], [1, 60, 45]]  # one token, tiles of few rows, of many
INF, LOW, NAN = 0x7E, 0xFE, 0x7F  # 448, -448, NaN


@pytest.mark.parametrize("new", NEW, ids=str)
@pytest.mark.parametrize("page", [4, 32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_values(ctx, dtype, d, page, new):
    """A key alone; one that all see beside finite ones; both signs in a channel; NaN; ones that some tokens see."""
    print(f"[odd {dtype} d={d} page={page} new={new}]", flush=True)
    gen = torch.Generator().manual_seed(1)
    c = make_cache(gen, [1, 130, 75], 2, page, d, dtype)
    widen(c, 0, 0, [(0, 3, INF), (1, 5, LOW), (1, 6, NAN)], gen)
    widen(c, 1, 5, [(0, 7, INF), (1, 8, LOW), (1, 9, INF)], gen)
    widen(c, 1, 40, [(1, 9, LOW)], gen)
    widen(c, 1, 100, [(0, 10, LOW), (1, 11, NAN)], gen)
    bits(c.v)[int(c.page_table[2, 60 // page]), 0, 60 % page, 12] = NAN  # of an ordinary scale
    widen(c, 2, 74, [(0, 13, INF)], gen)
    widen(c, 2, 2, [(1, 14, LOW)], gen)
    for causal in (1, 0) if new is not None else (0,):
        ref = check(ctx, c, new, causal, 1.0, 1 / math.sqrt(d), gen, 4)
        assert ref[0, 0, 3] == math.inf and ref[0, 2, 5] == -math.inf and ref[0, 3, 6].isnan() and ref[-1, 1, 13] == math.inf
    assert ref[1, 2, 9].isnan() and ref[1, 0, 7] == math.inf


@pytest.mark.parametrize("new", [None, [2, 1], [70, 40]], ids=str)
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_values_of_no_weight(ctx, dtype, page, new):
    """Scores far apart: infinities on keys whose weight f32, or a step's or piece's join, makes 0 come through."""
    print(f"[odd far {dtype} page={page} new={new}]", flush=True)
    gen = torch.Generator().manual_seed(2)
    c = make_cache(gen, [2900, 700], 2, page, 64, dtype)
    for s, keys in ((0, range(3, 2800, 97)), (1, range(1, 600, 50))):
        for i, key in enumerate(keys):
            widen(c, s, key, [(0, i, INF if i % 2 else LOW), (1, 63 - i, LOW)], gen)
    ref = check(ctx, c, new, 1, 40.0, 0.125, gen, 4)
    assert (~ref.isfinite()).any()


@pytest.mark.parametrize("new", NEW[:1] + NEW[2:], ids=str)
@pytest.mark.parametrize("page", [4, 16])
def test_infinite_keys(ctx, page, new):
    """f16 rows: a key past f16 scores an infinity: its token's head is NaN, or the key weighs nothing."""
    gen = torch.Generator().manual_seed(3)
    c = make_cache(gen, [1, 130, 75], 2, page, 64, F16)
    widen(c, 1, 50, [(0, 4, INF)], gen, "k")
    widen(c, 2, 70, [(1, 4, LOW)], gen, "k")
    ref = check(ctx, c, new, 1, 1.0, 0.125, gen, 4)
    assert ref[:, :2].isnan().any() or ref[:, 2:].isnan().any()


@pytest.mark.parametrize("new", [None, [1], [300]], ids=str)
@pytest.mark.parametrize("dtype", [F16, F32])
def test_largest_finite_values(ctx, dtype, new):
    """The largest that an append holds, on pages of the same scales, stay numbers."""
    gen = torch.Generator().manual_seed(4)
    c = make_cache(gen, [330], 1, 16, 64, dtype)
    bits(c.v_scale).fill_(WIDE[dtype])
    bits(c.v).fill_(0)
    bits(c.v)[int(c.page_table[0, 3]), 0, 2] = 0x77   # 240, where all see it
    bits(c.v)[int(c.page_table[0, 20]), 0, 5] = 0xF7  # -240
    ref = check(ctx, c, new, 1, 1.0, 0.125, gen, 2)
    assert ref.isfinite().all()


def test_infinite_values_of_wide_tiles(ctx):
    """Calls of 256 rows a tile, at both head dims: one channel of one early key, the others as they were."""
    for d, h, h_kv, n, past in ((64, 16, 16, 8300, 40), (128, 32, 8, 4200, 3000)):
        print(f"[odd wide d={d}]", flush=True)
        gen = torch.Generator().manual_seed(5)
        c = make_cache(gen, [past + n], h_kv, 16, d, F16)
        q = torch.randn((n, h, d), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
        gpu = lambda: PagedKV8(*(t.to(DEV) for t in (c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lens)), F16)  # noqa: E731
        at, late = int(c.page_table[0, 1]), int(c.page_table[0, (past + n - 9) // 16])
        for x in (at, late):  # infinite where a code is large, which none is yet
            bits(c.v_scale)[x, 1] = WIDE[F16]
            c.v[x, 1] = (torch.randn(c.v[x, 1].shape, generator=gen) * 0.5).to(E4M3)
        off = i32([0, n])
        plain = ctx.attention_paged_prompts(q, gpu(), off).unflatten(1, (h, d))
        bits(c.v)[at, 1, 4, 9], bits(c.v)[late, 1, (past + n - 9) % 16, 8] = INF, LOW
        odd = ctx.attention_paged_prompts(q, gpu(), off).unflatten(1, (h, d))
        g = h // h_kv
        heads = slice(g, 2 * g)
        assert (odd[:, heads, 9] == math.inf).all()
        assert (odd[-9:, heads, 8] == -math.inf).all() and odd[:-9, heads, 8].isfinite().all()
        kept = torch.ones(odd.shape, dtype=torch.bool, device=DEV)
        kept[:, heads, 9] = False
        kept[-9:, heads, 8] = False
        kept[:-9, heads, 8] = True
        assert torch.equal(odd[kept], plain[kept])


@pytest.mark.parametrize("new", NEW, ids=str)
@pytest.mark.parametrize("page", [4, 32])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_nan_of_other_pages_beside_infinities(ctx, dtype, page, new):
    """A channel with an infinity on one page and NaN on an ordinary one, in either order, is NaN; channels with one
    of them are that; queries of NaN have no finite channel."""
    gen = torch.Generator().manual_seed(8)
    c = make_cache(gen, [40, 150, 90], 2, page, 64, dtype)
    for s, length in enumerate((40, 150, 90)):
        for first, second, channel in ((3, length // 2, 20), (length // 2 + 1, 4, 21)):
            bits(c.v)[int(c.page_table[s, first // page]), 0, first % page, channel] = NAN
            widen(c, s, second + page, [(0, channel, INF)], gen)
        widen(c, s, 2 * page + 1, [(1, 30, LOW)], gen)
        bits(c.v)[int(c.page_table[s, 0]), 1, 1, 31] = NAN
    ref = check(ctx, c, new, 1, 1.0, 0.125, gen, 4)
    assert ref[-1, 0, 20].isnan() and (ref[:, 2, 30] == -math.inf).any() and ref[:, 2, 31].isnan().any()
    n = ref.shape[0]
    q = torch.randn((n, 4, 64), generator=gen).to(dtype)
    q[n - 1, 3, 9] = math.nan
    gpu = PagedKV8(*(t.to(DEV) for t in (c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lens)), dtype)
    off = None if new is None else [sum(new[:i]) for i in range(4)]
    got = ctx.attention_paged(q.to(DEV), gpu) if new is None else ctx.attention_paged_prompts(q.to(DEV), gpu, i32(off))
    assert got.unflatten(1, (4, 64))[n - 1, 3].isnan().all()
