"""The cache held in 8 bits, its attention and its pages on the GPU, against plain definitions in 64 bits
(tests/f8_reference.py and tests/paged_reference.py, which derive the tolerances), and together as a block uses
them."""
import math

import pytest
import torch

import f8_reference as F
import paged_reference as R
from headshot_amd.aggregator import BlockWeights, block_forward_cached
from headshot_amd.paged import PagedKV8, PagePool

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
DTYPES = [F16, F32]
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def normal(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen) * std + mean).to(dtype)


def i32(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


def offsets_of(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def make_cache(gen, lens, heads, page, d, dtype, spare=3, width=2, low=-9, high=-5):
    """Pages in no order, of codes and scales already there; CPU and GPU copies."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    m = max(need, default=0) + width
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (m - n))
        at += n
    codes = [normal(gen, (pages, heads, page, d), F32, 90.0).clamp(-448, 448).to(E4M3) for _ in range(2)]
    scales = [torch.randint(127 + low, 127 + high + 1, (pages, heads), generator=gen).to(torch.uint8).view(E8M0)
              for _ in range(2)]
    parts = (*codes, *scales, torch.tensor(table, dtype=torch.int32).reshape(len(lens), m), i32(lens, "cpu"))
    return PagedKV8(*parts, dtype), PagedKV8(*(t.to(DEV) for t in parts), dtype)


def parts_of(c):
    return c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lens


def bits(t):
    return t.view(torch.uint8)


def rope_tables(rows, d):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2) / (d // 2))
    # the two halves of a row are read separately: make them differ
    return (torch.cat([angle.sin(), (angle * 1.5).sin()], 1).float(),
            torch.cat([angle.cos(), (angle * 1.5).cos()], 1).float())


# ------------------------------------------------------------------ kv_append


def run_append(ctx, seed, dtype, d, h, h_kv, page, new, past, norm, rope, step=False, wide=True, positions=None,
               spoil=None, behind=0, rows=None, std=1.5, change=None, low=-9, high=-5):
    gen = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(past, new)]
    cpu, gpu = make_cache(gen, lens, h_kv, page, d, dtype, low=low, high=high)
    if spoil:
        spoil(cpu)
        for a, b in zip(parts_of(gpu), parts_of(cpu)):
            bits(a).copy_(bits(b))
    n = sum(new) + behind
    qkv = normal(gen, (n, (h + 2 * h_kv) * d + (64 if wide else 0)), dtype, std, 0.25 if std < 10 else 0.0)
    parts = [h * d, h_kv * d, h_kv * d]
    cut = lambda t: [x if wide else x.contiguous() for x in t[:, :sum(parts)].split(parts, 1)]  # noqa: E731
    heads = lambda t: t.unflatten(1, (-1, d))  # noqa: E731
    if change:
        change(*(heads(x) for x in qkv[:, :sum(parts)].split(parts, 1)))
    q, k, v = cut(qkv)
    gq, gk, gv = cut(qkv.to(DEV))
    nrm = lambda: (normal(gen, (d,), F32, 0.2, 1.0), normal(gen, (d,), F32, 0.2)) if norm else None  # noqa: E731
    qn, kn = nrm(), nrm()
    tables = rope_tables(rows or max(lens) + 1, d) if rope else None
    up = lambda p: None if p is None else tuple(t.to(DEV) for t in p)  # noqa: E731
    off = None if step else offsets_of(new)
    mark = 7.0
    out_q, out_k = (torch.full((n, x * d), mark, dtype=dtype, device=DEV) for x in (h, h_kv))
    pos = None if positions is None else i32(positions)
    got_q, got_k = ctx.kv_append(gpu, gk, gv, None if step else i32(off), q=gq, qn=up(qn), kn=up(kn), rope=up(tables),
                                 positions=pos, out_q=out_q, out_k=out_k)
    torch.cuda.synchronize()
    live = sum(new)
    for got, x, nm, what in ((got_q, q, qn, "q rows"), (got_k, k, kn, "k rows")):
        ref = F.transformed(heads(x), nm, tables, cpu.lens, off, positions, 1e-5)
        fine = ref[:live].isfinite()
        R.assert_within(heads(got)[:live].cpu()[fine], ref[:live][fine],
                        R.append_bound(ref[:live], x.nan_to_num(0, 0, 0), dtype)[fine], what)
        assert (got[live:] == mark).all(), "rows behind the last sequence"
    kx = F.transformed(heads(k), kn, tables, cpu.lens, off, positions, 1e-5)
    error = F.transform_error(kx, k) if norm or rope else 0
    F.check_append("k", (cpu.k, cpu.k_scale), (gpu.k.cpu(), gpu.k_scale.cpu()), cpu.page_table, cpu.lens, off, kx, dtype, error)
    F.check_append("v", (cpu.v, cpu.v_scale), (gpu.v.cpu(), gpu.v_scale.cpu()), cpu.page_table, cpu.lens, off, heads(v), dtype, 0)
    # nothing but the pages without q and k rows, the same bits
    again = PagedKV8(*(t.to(DEV) for t in parts_of(cpu)), dtype)
    none = ctx.kv_append(again, gk, gv, None if step else i32(off), kn=up(kn), rope=up(tables), positions=pos)
    assert none == (None, None)
    for a, b in zip(parts_of(again), parts_of(gpu)):
        assert torch.equal(bits(a), bits(b))
    return cpu, gpu


@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_prompts(ctx, dtype, d, norm, rope):
    for i, (h, h_kv, page, new, past) in enumerate([
        (4, 4, 16, [5, 0, 33, 1, 0], [0, 9, 17, 300, 0]),
        (7, 1, 1, [3, 2], [1, 0]),
        (10, 5, 64, [70, 129], [63, 0]),
        (16, 16, 8, [1], [0]),
        (3, 1, 128, [200, 3], [5, 126]),
        (2, 2, 512, [700], [100]),
    ]):
        print(f"[append f8 {dtype} d={d} norm={norm} rope={rope} case {i}]", flush=True)
        run_append(ctx, 100 + i, dtype, d, h, h_kv, page, new, past, norm, rope, wide=i % 2 == 0, behind=3 * (i % 3))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_steps(ctx, dtype, d):
    for i, (h, h_kv, page, past) in enumerate([(3, 3, 4, [0, 3, 4, 1000]), (32, 8, 32, [31, 32, 0] * 43), (8, 2, 256, [5]),
                                               (4, 4, 1, [0, 6])]):
        print(f"[append f8 step {dtype} d={d} case {i}]", flush=True)
        run_append(ctx, 200 + i, dtype, d, h, h_kv, page, [1] * len(past), past, True, True, step=True, wide=i != 1)


@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_scales_that_grow(ctx, dtype, page):
    """Pages that the call goes on with: its values are far larger than the page's, far smaller, and of its size;
    older codes become subnormal or nothing, NaN among them stay."""
    def old_nan(c):
        bits(c.k)[:, :, 0, 3] = 0x7F

    for i, (std, low, high) in enumerate([(300.0, -17, -12), (1e-3, -6, -5), (1.5, -8, -6), (3e4, -24, -20)]):
        for new, past, step in (([3, page + 1, 2], [5, 3, page - 1], False), ([1, 1, 1], [1, page - 1, page + 2], True)):
            run_append(ctx, 220 + i, dtype, 64, 2, 2, page, new, past, False, False, step=step, std=std, low=low, high=high,
                       spoil=old_nan)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_extremes(ctx, dtype, d):
    """Zeros alone, one tiny value, the type's largest, infinities and NaN beside ordinary values, ties."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps

    def change(q, k, v):
        for t in (k, v):
            t[0:4] = 0
            t[4:8, 0, 3] = tiny
            t[8, 0, 1], t[8, 1, 1], t[9, 0, 0] = top, -top, top / 2
            t[12, 0, 5], t[13, 1, 5], t[13, 0, 2] = math.inf, -math.inf, math.nan
            t[16:20] = 0
            t[16:20, :, 7] = tiny
            t[20] = torch.arange(d) * 0.03125 - 1.0   # ties and even neighbours
            t[24:28] = math.inf
            t[28:32, 1] = math.nan

    run_append(ctx, 230, dtype, d, 2, 2, 4, [40], [0], False, False, change=change)
    run_append(ctx, 231, dtype, d, 2, 2, 32, [40], [2], False, False, change=change)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_positions(ctx, dtype):
    """Rows of the tables by token; rows outside them (prefix tokens: -1) are not rotated."""
    run_append(ctx, 300, dtype, 64, 4, 2, 16, [6, 5], [0, 11], False, True, rows=9,
               positions=[-1, -1, 0, 3, 8, 9, 2 ** 31 - 1, -2 ** 31, 4, 4, 0])
    run_append(ctx, 301, dtype, 128, 4, 2, 16, [40], [0], True, True, rows=20)  # longer than the tables


@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_without_a_place(ctx, dtype, page):
    """Page numbers outside the pool and lengths outside the table: the tokens are not stored, everything else is
    as usual."""
    def spoil(c):
        c.page_table[0, 0], c.page_table[1, 1] = -1, c.k.shape[0]
        c.page_table[2, 0] = 2 ** 31 - 1

    run_append(ctx, 310, dtype, 64, 2, 2, page, [page + 4, 2 * page + 4, 9], [0, 4, 0], True, True, spoil=spoil)

    def lengths(c):
        c.lens[0], c.lens[1], c.lens[2] = 3, 2 ** 31 - 1, c.page_table.shape[1] * page + 2  # 5 keys before the first

    run_append(ctx, 311, dtype, 64, 2, 2, page, [8, 20, 9], [0, 4, 0], False, False, spoil=lengths)

    def steps(c):
        c.lens[0], c.lens[1], c.lens[2], c.lens[3] = 0, -5, 2 ** 31 - 1, c.page_table.shape[1] * page + 1
        c.page_table[4, 0] = -7

    run_append(ctx, 312, dtype, 64, 2, 2, page, [1] * 6, [0] * 6, False, False, step=True, spoil=steps)


def test_append_nothing(ctx):
    cpu, gpu = make_cache(torch.Generator().manual_seed(1), [4, 0], 2, 4, 64, F16)
    rows = torch.empty((0, 128), dtype=F16, device=DEV)
    q, k = ctx.kv_append(gpu, rows, rows, i32([0, 0, 0]), q=rows, k_rows=True)
    assert q.shape == k.shape == (0, 128) and torch.equal(bits(gpu.k.cpu()), bits(cpu.k))


def test_append_token_by_token_is_the_prompt(ctx):
    """A page filled token by token holds what it holds filled at once but for what the earlier scales, which are
    the same or smaller, rounded to subnormals: here nothing."""
    gen = torch.Generator().manual_seed(9)
    k, v = (normal(gen, (21, 128), F16).to(DEV) for _ in range(2))
    table = torch.arange(2, dtype=torch.int32, device=DEV)[None]
    one, all_ = (PagedKV8.empty(2, 2, 16, 64, F16, table, i32([21])) for _ in range(2))
    for c in (one, all_):
        for t in parts_of(c)[:4]:
            bits(t).fill_(0x55)
    ctx.kv_append(all_, k, v, i32([0, 21]))
    for i in range(21):
        one.lens.fill_(i + 1)
        ctx.kv_append(one, k[i:i + 1], v[i:i + 1])
    for x in "kv":
        a, b = (F.values(getattr(c, x).cpu(), getattr(c, x + "_scale").cpu()) for c in (one, all_))
        fine = a.abs() > 2.0 ** -6 * getattr(all_, x + "_scale").cpu().double()[..., None, None]
        assert torch.equal(getattr(one, x + "_scale").view(torch.uint8), getattr(all_, x + "_scale").view(torch.uint8))
        rows = torch.zeros_like(fine)
        rows[0], rows[1, :, :5] = True, True
        assert torch.equal(a[fine & rows], b[fine & rows])


# ------------------------------------------------------------------ attention


def run_attend(ctx, seed, dtype, d, h, h_kv, page, lens, new=None, causal=1, scale=None, std=1.0, wide=False, behind=0,
               spoil=None, low=-9, high=-5, width=2):
    """``new``: tokens per sequence; None: attention_paged's one."""
    gen = torch.Generator().manual_seed(seed)
    cpu, gpu = make_cache(gen, lens, h_kv, page, d, dtype, low=low, high=high, width=width)
    if spoil:
        spoil(cpu)
        for a, b in zip(parts_of(gpu), parts_of(cpu)):
            bits(a).copy_(bits(b))
    n = (len(lens) if new is None else sum(new)) + behind
    q = normal(gen, (n, (h + wide) * d), dtype, std)
    gq = q.to(DEV)[:, wide * d:]
    q = q[:, wide * d:].unflatten(1, (h, d))
    mark = 7.0
    out = torch.full((n, h * d), mark, dtype=dtype, device=DEV)
    off = None if new is None else offsets_of(new)
    if new is None:
        got = ctx.attention_paged(gq, gpu, scale=scale, out=out)
    else:
        got = ctx.attention_paged_prompts(gq, gpu, i32(off), causal=causal, scale=scale, out=out)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    got = got.unflatten(1, (h, d)).cpu()
    ref, bound = F.attend(q, parts_of(cpu), off, causal, 1 / math.sqrt(d) if scale is None else scale, dtype)
    live = n - behind
    odd = ~ref[:live].isfinite()
    g = got[:live].double()
    assert torch.equal(g[odd].isnan(), ref[:live][odd].isnan()), "NaN places"
    assert torch.equal(g[odd].nan_to_num(0.0), ref[:live][odd].nan_to_num(0.0)), "infinities"
    R.assert_within(g[~odd], ref[:live][~odd], bound[:live][~odd], "attention")
    assert (got[live:] == mark).all(), "rows behind the last sequence"


@pytest.mark.parametrize("page", [1, 4, 16, 64])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_lengths(ctx, dtype, d, page):
    for i, (h, h_kv, lens) in enumerate([(2, 2, [1, 0, 63, 64, 65]), (4, 1, [129, 2, 700]), (6, 2, [257, 1]), (1, 1, [33]),
                                         (34, 2, [50, 9]), (40, 5, [17])]):
        print(f"[paged f8 {dtype} d={d} page={page} case {i}]", flush=True)
        run_attend(ctx, 500 + i, dtype, d, h, h_kv, page, lens, wide=i == 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_split(ctx, dtype):
    """Long sequences beside short ones: pieces and their join."""
    for d, h, h_kv, page, lens in [(64, 2, 1, 16, [5000, 3, 900]), (128, 8, 2, 32, [3001]), (64, 16, 1, 8, [2100, 2047]),
                                   (128, 20, 1, 16, [1500, 1])]:
        print(f"[paged f8 split {dtype} d={d} page={page}]", flush=True)
        run_attend(ctx, 520, dtype, d, h, h_kv, page, lens)


@pytest.mark.parametrize("new", [None, [1, 2, 1]])
@pytest.mark.parametrize("page", [4, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_not_there(ctx, dtype, page, new):
    """Keys on pages outside the pool are not seen, lengths past the table's width are held to it, and what pages
    hold past a sequence's end is not seen: NaN there and in scales of no sequence."""
    def spoil(c):
        c.page_table[0, 1], c.page_table[0, 3], c.page_table[1, 0] = -1, 2 ** 31 - 1, c.k.shape[0]
        used = {}
        for s in range(3):
            for p in range(int(c.lens[s])):
                used.setdefault(int(c.page_table[s, p // page]), set()).add(p % page)
        for at in range(c.k.shape[0]):
            rows = [r for r in range(page) if r not in used.get(at, ())]
            bits(c.k)[at, :, rows], bits(c.v)[at, :, rows] = 0x7F, 0xFF
            if at not in used:
                bits(c.k_scale)[at], bits(c.v_scale)[at] = 0xFF, 0xFF

    run_attend(ctx, 530, dtype, 64, 4, 2, page, [5 * page + 1, page + 2, 3 * page - 1], new, spoil=spoil)

    def lengths(c):
        c.lens[0], c.lens[1], c.lens[2] = 2 ** 31 - 1, -3, c.page_table.shape[1] * page + 1

    run_attend(ctx, 531, dtype, 64, 4, 2, page, [3 * page, 5, page], new, spoil=lengths)

    def none(c):
        c.page_table.fill_(-1)

    run_attend(ctx, 532, dtype, 128, 4, 2, page, [3 * page, 5, page], new, spoil=none)


@pytest.mark.parametrize("new", [None, [1, 40, 3]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_codes(ctx, dtype, new):
    """NaN among the keys and values that are seen, by some tokens or by all; zeros alone; every code."""
    def spoil(c):
        page = 16
        at = lambda s, p: (int(c.page_table[s, p // page]), p % page)  # noqa: E731
        (a, r), (b, x) = at(1, 30), at(1, 70)
        bits(c.v)[a, 0, r, 5] = 0x7F
        bits(c.k)[b, 1, x, 2] = 0xFF
        bits(c.v)[b, :, x] = 0x7F
        every = torch.arange(256, dtype=torch.uint8)
        every[[127, 255]] = 0
        first = int(c.page_table[0, 0])
        bits(c.k)[first].view(-1)[:256], bits(c.v)[first].view(-1)[:256] = every, every
        bits(c.k)[int(c.page_table[2, 0])] = 0

    run_attend(ctx, 540, dtype, 64, 4, 2, 16, [40, 100, 20], new, spoil=spoil)


@pytest.mark.parametrize("new", [None, [20, 7]])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_far_apart(ctx, dtype, d, new):
    """Scales that differ by far from page to page, the least and the largest; scores of any size; a scale of the
    caller's, negative and zero ones."""
    run_attend(ctx, 550, dtype, d, 4, 2, 16, [130, 70], new, low=-24, high=-6)
    for low in (-117, -60):
        run_attend(ctx, 551, dtype, d, 4, 2, 8, [90, 70], new, low=low, high=low + 4)
    for scale, std in [(1.0, 1.0), (-0.125, 1.0), (0.0, 1.0), (0.125, 100.0)]:
        run_attend(ctx, 552, dtype, d, 2, 1, 16, [90, 140], new, scale=scale, std=std)

    def large(c):  # the largest that such a cache holds, among the values
        bits(c.v_scale).fill_(127 + (7 if dtype == F16 else 100))
        bits(c.v)[:] = bits(c.v.float().clamp(-240, 240).to(E4M3))

    run_attend(ctx, 553, dtype, d, 4, 2, 16, [90, 70], new, spoil=large)


@pytest.mark.parametrize("causal", [0, 1, 7, 64])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_lengths(ctx, dtype, d, causal):
    for i, (h, h_kv, page, new, past) in enumerate([
        (2, 2, 16, [1, 0, 63, 64, 65], [0, 9, 0, 100, 1]),
        (4, 1, 4, [129, 2], [3, 300]),
        (6, 2, 64, [200, 1, 1], [57, 0, 1]),
        (7, 1, 1, [31, 33], [5, 0]),
        (40, 2, 32, [9, 30], [130, 0]),
        (1, 1, 128, [5], [0]),
    ]):
        print(f"[prompts f8 {dtype} d={d} causal={causal} case {i}]", flush=True)
        run_attend(ctx, 560 + i, dtype, d, h, h_kv, page, [a + b for a, b in zip(new, past)], new, causal, wide=i == 1,
                   behind=2 * (i % 3))


@pytest.mark.parametrize("causal", [0, 1, 12])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_longer_than_their_keys(ctx, dtype, causal):
    """Fewer keys than tokens: the first ones see nothing under a mask."""
    def spoil(c):
        c.lens[0], c.lens[1] = 20, 0

    run_attend(ctx, 570, dtype, 64, 4, 2, 16, [50, 30, 9], [50, 30, 2], causal, spoil=spoil)


def gpu_values(c, x, s, length):
    page = c.page
    place = torch.arange(length, device=DEV)
    at = c.page_table[s].long()[place // page]
    codes = bits(getattr(c, x))[at, :, place % page].view(E4M3).double()
    return codes * getattr(c, x + "_scale").double()[at][..., None]


def gpu_check(got, q, c, off, new, lens, causal, dtype, what):
    """Longer calls, in f64 on the GPU, every query."""
    n, h, d = q.shape
    for s, (m, length) in enumerate(zip(new, lens)):
        if m == 0:
            continue
        k, v = (gpu_values(c, x, s, length) for x in "kv")
        seen = R.seen_keys(m, length, causal) if off is not None else torch.full((m,), length)
        a = off[s] if off is not None else s
        qs = q[a:a + m]
        ref, mag = torch.empty(m, h, d, dtype=torch.float64), torch.empty(m, h, d, dtype=torch.float64)
        hidden = torch.arange(length, device=DEV) >= seen.to(DEV)[:, None]
        for i in range(h):
            j = i // (h // k.shape[1])
            p = torch.softmax((qs[:, i].double() @ k[:, j].T / math.sqrt(d)).masked_fill(hidden, -math.inf), 1)
            ref[:, i], mag[:, i] = (p @ v[:, j]).cpu(), (p @ v[:, j].abs()).cpu()
        step = max(1, 1 << 23 // max(1, length))
        for b in range(0, m, step):
            z = slice(b, b + step)
            bound = R.attention_bound(ref[z], mag[z], qs[z].cpu(), k.cpu(), v.cpu(), seen[z], 1 / math.sqrt(d), dtype)
            R.assert_within(got[a + b:a + min(b + step, m)], ref[z], bound, f"{what}, sequence {s}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,h,h_kv,page,new,past,causal", [
    (64, 16, 16, 64, [1374], [1374], 1374),
    (128, 8, 2, 16, [700, 1, 300], [900, 1200, 0], 1),
    (64, 4, 4, 16, [3, 17], [9000, 4100], 1),
    (128, 14, 2, 32, [6, 2, 5, 1], [1500, 30, 0, 2600], 1),
    (64, 5, 1, 8, [900], [333], 137),
    (128, 2, 1, 128, [257], [6000], 0),
])
def test_prompts_longer(ctx, dtype, d, h, h_kv, page, new, past, causal):
    gen = torch.Generator().manual_seed(d + h)
    lens = [a + b for a, b in zip(new, past)]
    _, c = make_cache(gen, lens, h_kv, page, d, dtype)
    q = normal(gen, (sum(new), h, d), dtype).to(DEV)
    got = ctx.attention_paged_prompts(q, c, i32(offsets_of(new)), causal=causal).unflatten(1, (h, d))
    gpu_check(got, q, c, offsets_of(new), new, lens, causal, dtype, "prompts")


@pytest.mark.parametrize("d,h,h_kv,page,new,past,causal", [
    (64, 16, 16, 16, [8300], [0], 1),           # eight waves, head dim 64
    (128, 32, 8, 16, [4200], [3000], 1),        # and 128
    (128, 32, 8, 64, [4100], [100], 700),
    (128, 32, 8, 32, [2100, 40, 1], [0, 9000, 5], 1),  # many tiles, one sequence's much longer
])
def test_prompts_that_fill_the_chip(ctx, d, h, h_kv, page, new, past, causal):
    gen = torch.Generator().manual_seed(d + page)
    lens = [a + b for a, b in zip(new, past)]
    _, c = make_cache(gen, lens, h_kv, page, d, F16)
    q = torch.randn((sum(new), h, d), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    off = offsets_of(new)
    got = ctx.attention_paged_prompts(q, c, i32(off), causal=causal).unflatten(1, (h, d))
    # each head's first, last and some middle rows against 64 bits; the rest against the same tokens asked for in
    # pieces, whose tiles are other ones (both are off by at most their bounds)
    for s, (m, length) in enumerate(zip(new, lens)):
        pick = sorted({0, m - 1, *range(0, m, max(1, m // 60))})
        k, v = (gpu_values(c, x, s, length) for x in "kv")
        seen = R.seen_keys(m, length, causal)[pick]
        qs = q[off[s]:off[s + 1]][pick]
        ref, mag = (torch.empty(len(pick), h, d, dtype=torch.float64) for _ in range(2))
        hidden = torch.arange(length, device=DEV) >= seen.to(DEV)[:, None]
        for i in range(h):
            j = i // (h // h_kv)
            p = torch.softmax((qs[:, i].double() @ k[:, j].T / math.sqrt(d)).masked_fill(hidden, -math.inf), 1)
            ref[:, i], mag[:, i] = (p @ v[:, j]).cpu(), (p @ v[:, j].abs()).cpu()
        bound = R.attention_bound(ref, mag, qs.cpu(), k.cpu(), v.cpu(), seen, 1 / math.sqrt(d), F16)
        R.assert_within(got[off[s]:off[s + 1]][pick], ref, bound, f"sequence {s}")
    # the last 300 tokens of the first sequence alone
    tail = min(300, new[0])
    alone = PagedKV8(*parts_of(c)[:4], c.page_table[:1].contiguous(), i32([lens[0]]), F16)
    a, b = off[1] - tail, off[1]
    other = ctx.attention_paged_prompts(q[a:b], alone, i32([0, tail]), causal=causal).unflatten(1, (h, d))
    assert ((got[a:b].double() - other.double()).abs().amax() <= 2 * bound.amax().item())


@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_tiles_leave_masked_values_alone(ctx, dtype):
    """Calls of eight-wave tiles: NaN in keys and values that later tokens see, and pages that are not there."""
    gen = torch.Generator().manual_seed(5)
    h, d, n, page = 16, 64, 8192 + 300, 32
    cpu, c = make_cache(gen, [n], h, page, d, dtype)
    q = torch.randn((n, h, d), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    off = i32([0, n])
    clean = ctx.attention_paged_prompts(q, c, off, causal=1)
    at = int(cpu.page_table[0, 5000 // page])
    bits(c.v)[at, :, 5000 % page, 7] = 0x7F
    bits(c.k)[int(cpu.page_table[0, 8000 // page]), :, 8000 % page] = 0xFF
    got = ctx.attention_paged_prompts(q, c, off, causal=1)
    assert torch.equal(got[:5000], clean[:5000])
    rows = got.unflatten(1, (h, d))
    assert rows[5000:8000, :, 7].isnan().all() and rows[8000:].isnan().all()
    keep = [x for x in range(d) if x != 7]
    assert torch.equal(rows[5000:8000, :, keep], clean.unflatten(1, (h, d))[5000:8000, :, keep])
    # the pages of keys [0, 64) and [7000, 8192 + 300) not there: as if the sequence had none of them
    c.page_table[0, :2] = -1
    c.page_table[0, 7008 // page:] = -1
    got = ctx.attention_paged_prompts(q[:1000], PagedKV8(*parts_of(c)[:4], c.page_table, i32([1000]), dtype), i32([0, 1000]), causal=1)
    short = PagedKV8(*parts_of(c)[:4], c.page_table[:, 2:].contiguous(), i32([1000 - 64]), dtype)
    want = ctx.attention_paged_prompts(q[64:1000], short, i32([0, 1000 - 64]), causal=1)
    assert (got[:64] == 0).all()
    eps = torch.finfo(dtype).eps  # another order of sums, values below 448 2^-5 = 14
    assert ((got[64:].double() - want.double()).abs() <= 32 * eps * 14).all()
    whole = ctx.attention_paged_prompts(q, c, off, causal=1)
    assert (whole[:64] == 0).all()
    assert ((whole[64:1000].double() - want.double()).abs() <= 32 * eps * 14).all()


@pytest.mark.parametrize("page", [1, 8, 16, 64])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens(ctx, dtype, d, page):
    """Sequences whose rows (tokens by heads of a key head) are 1 to 16, 17 to 32 and more, beside each other, over
    keys of part of a wave's step and of several steps of all waves."""
    for i, (h, h_kv, new, past, causal) in enumerate([
        (2, 2, [1, 16, 17, 32, 33, 0], [0, 500, 63, 300, 40, 7], 1),
        (7, 1, [2, 4, 5], [700, 30, 255], 1),
        (3, 1, [5, 10, 11], [0, 1, 600], 4),
        (16, 1, [1, 2], [513, 100], 0),
        (32, 1, [1, 1, 2], [300, 0, 70], 1),
        (1, 1, [3, 20, 200], [257, 128, 90], 64),
    ]):
        print(f"[few {dtype} d={d} page={page} case {i}]", flush=True)
        run_attend(ctx, 620 + i, dtype, d, h, h_kv, page, [a + b for a, b in zip(new, past)], new, causal, wide=i == 1,
                   behind=i % 3)


@pytest.mark.parametrize("h", [1, 2])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens_odd_values(ctx, dtype, page, h):
    """NaN at keys that some of a sequence's few tokens see and that all see; pages that are not there among them."""
    def spoil(c):
        at = lambda s, p: (int(c.page_table[s, p // page]), p % page)  # noqa: E731
        for s, key, channel in [(0, 295, 5), (0, 301, 63), (0, 20, 9), (1, 600, 17), (1, 612, 0), (2, 3, 40)]:
            a, r = at(s, key)
            bits(c.v)[a, 0, r, channel] = 0x7F
        a, r = at(0, 299)
        bits(c.k)[a, 0, r] = 0xFF
        c.page_table[1, 40 // page] = -1
        c.page_table[2, 1] = c.k.shape[0]

    run_attend(ctx, 640, dtype, 64, h, 1, page, [302, 615, 2 * page + 3], [8, 15, 6], 1, spoil=spoil)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens_beside_many(ctx, dtype):
    """A long prompt, single tokens and sequences without any in one call; some of whose keys lie in pieces."""
    gen = torch.Generator().manual_seed(7)
    new, past = [300, 1, 0, 1, 6, 1, 2], [2000, 5000, 40, 0, 3100, 1, 800]
    lens = [a + b for a, b in zip(new, past)]
    for d, h, h_kv, page in [(64, 8, 4, 32), (128, 8, 2, 8)]:
        _, c = make_cache(gen, lens, h_kv, page, d, dtype)
        q = normal(gen, (sum(new), h, d), dtype).to(DEV)
        got = ctx.attention_paged_prompts(q, c, i32(offsets_of(new)), causal=1).unflatten(1, (h, d))
        gpu_check(got, q, c, offsets_of(new), new, lens, 1, dtype, f"beside {d}")


@pytest.mark.parametrize("h,h_kv,d", [(2, 1, 64), (16, 16, 64), (16, 8, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens_of_many_sequences(ctx, dtype, h, h_kv, d):
    """More sequences than a wave's lanes, one much longer than the others, in one round of pieces and in several."""
    gen = torch.Generator().manual_seed(8)
    new = [i % 4 for i in range(131)]
    past = [9000 if i == 66 else 37 * i % 700 for i in range(131)]
    lens = [a + b for a, b in zip(new, past)]
    _, c = make_cache(gen, lens, h_kv, 16, d, dtype)
    q = normal(gen, (sum(new), h, d), dtype).to(DEV)
    got = ctx.attention_paged_prompts(q, c, i32(offsets_of(new)), causal=1).unflatten(1, (h, d))
    gpu_check(got, q, c, offsets_of(new), new, lens, 1, dtype, "many")


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_longer(ctx, dtype):
    gen = torch.Generator().manual_seed(3)
    for d, h, h_kv, page, lens in [(128, 32, 8, 16, [1, 4000, 17, 8192]), (64, 16, 16, 64, [30001]), (64, 28, 4, 32, [3001, 5] * 9)]:
        _, c = make_cache(gen, lens, h_kv, page, d, dtype)
        q = normal(gen, (len(lens), h, d), dtype).to(DEV)
        got = ctx.attention_paged(q, c).unflatten(1, (h, d))
        gpu_check(got, q, c, None, [1] * len(lens), lens, 0, dtype, "paged")


def test_no_sequences_and_no_pages(ctx):
    empty = PagedKV8.empty(0, 2, 16, 64, F16, torch.zeros((3, 0), dtype=torch.int32, device=DEV), i32([5, 0, 2]))
    q = torch.ones((3, 4, 64), dtype=F16, device=DEV)
    assert (ctx.attention_paged(q, empty) == 0).all()
    assert (ctx.attention_paged_prompts(q, empty, i32([0, 1, 2, 3])) == 0).all()
    none = PagedKV8.empty(4, 2, 16, 64, F16, torch.zeros((0, 2), dtype=torch.int32, device=DEV), i32([]))
    assert ctx.attention_paged(q[:0], none).shape == (0, 256)
    assert ctx.attention_paged_prompts(q[:0], none, i32([0])).shape == (0, 256)


# ------------------------------------------------------------------ pages


def state_of(pool):
    head, count, missing = pool.state.tolist()
    n = pool.free.numel()
    return [int(pool.free[(head + i) % n]) for i in range(count)], missing


def same_pages(pool, model):
    assert pool.page_table.tolist() == model.table
    assert pool.lens.tolist() == model.lens
    free, missing = state_of(pool)
    assert free == model.free and missing == model.missing


@pytest.mark.parametrize("b,width,pages,page,most,extra", [
    (5, 6, 20, 8, 40, 0), (1, 3, 2, 16, 30, 3), (70, 4, 90, 1, 4, 0), (3, 8, 7, 4, 20, 5000), (1500, 3, 2500, 2, 5, 0),
    (40, 1000, 9000, 16, 7000, 0), (4, 0, 3, 8, 9, 1), (6, 9, 0, 8, 9, 0), (300, 2000, 5000, 4, 60, 0),
])
def test_plan_pages(ctx, b, width, pages, page, most, extra):
    """Sequences that grow, drop, end and run out of pages, call after call, against a plain simulation."""
    gen = torch.Generator().manual_seed(b + pages)
    pool, model = PagePool.empty(b, width, pages, page, DEV), F.Pages(b, width, pages, page)
    for call in range(12):
        change = torch.randint(-most, most + 1, (b,), generator=gen)
        change[torch.rand(b, generator=gen) < 0.2] = 0
        change[torch.rand(b, generator=gen) < 0.1] = -(1 << 30) - 7
        change = change.tolist()
        n = sum(max(c, 0) for c in change) + extra
        mark = -77
        out = (torch.full((b + 1,), mark, dtype=torch.int32, device=DEV), torch.full((n,), mark, dtype=torch.int32, device=DEV),
               torch.full((n,), mark, dtype=torch.int64, device=DEV))
        got = ctx.plan_pages(pool, i32(change), n, out=out)
        assert got == out
        offsets, positions, slots = model.plan(change)
        assert out[0].tolist() == offsets, f"call {call}"
        assert out[1].tolist() == positions + [mark] * extra and out[2].tolist() == slots + [mark] * extra, f"call {call}"
        same_pages(pool, model)


def test_plan_fewer_rows_than_tokens(ctx):
    """Rows past n are not written; the pages are as ever."""
    pool, model = PagePool.empty(2, 8, 9, 4, DEV), F.Pages(2, 8, 9, 4)
    wide = torch.full((20,), -77, dtype=torch.int32, device=DEV)
    offsets, positions, slots = ctx.plan_pages(pool, i32([5, 9]), 7, out=(wide[:3], wide[4:11], wide[12:].new_full((7,), -77, dtype=torch.int64)))
    want = model.plan([5, 9])
    assert offsets.tolist() == want[0] and positions.tolist() == want[1][:7] and slots.tolist() == want[2][:7]
    assert wide[3] == -77 and (wide[11:] == -77).all()
    same_pages(pool, model)
    empty = PagePool.empty(0, 3, 4, 8, DEV)
    offsets, positions, slots = ctx.plan_pages(empty, i32([]), 0)
    assert offsets.tolist() == [0] and positions.numel() == slots.numel() == 0 and state_of(empty) == ([0, 1, 2, 3], 0)


def test_plan_lengths_at_their_limits(ctx):
    """Lengths stay within 2^30 whatever counts and lens hold; counts are added without overflow."""
    pool = PagePool.empty(4, 2, 16, 8, DEV)
    pool.lens.copy_(i32([2 ** 31 - 1, -5, 1 << 30, 3]))
    off, pos, slots = ctx.plan_pages(pool, i32([2 ** 31 - 1, 4, -(2 ** 31), 2]), 6)
    assert pool.lens.tolist() == [1 << 30, 4, 0, 5]
    assert off.tolist() == [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
    assert pos.tolist() == [(1 << 30) + i for i in range(6)] and (slots == -1).all()


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_then_steps(ctx, dtype, d):
    """Pages, append, prompts over the pages in two pieces, then steps: each attention is that of the values the
    cache holds; sequences end and others begin in their pages."""
    gen = torch.Generator().manual_seed(40)
    h, h_kv, page = 4, 2, 8
    pool = PagePool.empty(3, 12, 20, page, DEV)
    cache = PagedKV8.empty(20, h_kv, page, d, dtype, pool.page_table, pool.lens)
    tables = tuple(t.to(DEV) for t in rope_tables(100, d))
    kn = (normal(gen, (d,), F32, 0.2, 1.0).to(DEV), normal(gen, (d,), F32, 0.2).to(DEV))
    for counts in ([20, 1, 33], [7, 40, 0], [1, 1, 1], [1, 1, 1], [-40, 1, -34], [12, 3, 30], [1, 1, 1]):
        fresh = [max(c, 0) for c in counts]
        n = sum(fresh)
        offsets, positions, slots = ctx.plan_pages(pool, i32(counts), n)
        assert offsets.tolist() == offsets_of(fresh) and int(pool.state[2]) == 0
        if n == 0:
            continue
        qkv = normal(gen, (n, (h + 2 * h_kv) * d), dtype).to(DEV)
        q, k, v = qkv.split([h * d, h_kv * d, h_kv * d], 1)
        steps = fresh == [1, 1, 1]
        q, _ = ctx.kv_append(cache, k, v, None if steps else offsets, q=q, qn=kn, kn=kn, rope=tables)
        got = ctx.attention_paged(q, cache) if steps else ctx.attention_paged_prompts(q, cache, offsets)
        cpu = tuple(t.cpu() for t in parts_of(cache))
        ref, bound = F.attend(q.cpu().unflatten(1, (h, d)), cpu, None if steps else offsets_of(fresh), 1, 1 / math.sqrt(d), dtype)
        R.assert_within(got.unflatten(1, (h, d)), ref, bound, f"counts {counts}")
        # the slots are where the tokens went
        flat = F.values(cpu[1], cpu[3]).transpose(1, 2).flatten(0, 1)[slots.cpu()]
        x = v.cpu().double().unflatten(1, (h_kv, d))
        step = cpu[3].double()[slots.cpu() // page][..., None]
        R.assert_within(flat, x, F.HALF_CODE * x.abs() + F.TINY_CODE * step, "values at their slots")


@pytest.mark.parametrize("causal", [1, 10])
@pytest.mark.parametrize("dtype", DTYPES)
def test_block_over_eight_bits(ctx, dtype, causal):
    """A block over a cache in 8 bits: prompts, further pieces of them and steps are its operators one after the
    other, bit for bit (each is held to 64 bits above)."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    heads, d, dim = 4, 64, 256
    w = BlockWeights.random(dim, 512, d, dtype, DEV, gen, ls_init=0.5)
    lens = i32([0, 0])
    table = torch.arange(12, dtype=torch.int32, device=DEV).reshape(2, 6)
    one, two = (PagedKV8.empty(12, heads, 16, d, dtype, table, lens) for _ in range(2))
    p = w.p
    for new in ([40, 30], [15, 20], [1, 1], [0, 13], [1, 1]):
        lens += i32(new)
        x = torch.randn((sum(new), dim), generator=gen, device=DEV).to(dtype)
        off = None if new == [1, 1] else i32(offsets_of(new))
        got = block_forward_cached(ctx, w, x, one, heads, offsets=off, causal=causal)
        q, k, v = ctx.linear(ctx.layernorm(x, *p.ln1, eps=1e-6), w.qkv_w, w.qkv_b).split(dim, 1)
        q, _ = ctx.kv_append(two, k, v, off, q=q, qn=p.qn, kn=p.kn, eps=1e-6)
        attn = ctx.attention_paged(q, two) if off is None else ctx.attention_paged_prompts(q, two, off, causal=causal)
        x1 = ctx.linear_ls_residual(attn, w.proj_w, p.ls1, x, p.proj_b)
        act = ctx.linear_gelu(ctx.layernorm(x1, *p.ln2, eps=1e-6), w.fc1_w, p.fc1_b)
        assert torch.equal(got, ctx.linear_ls_residual(act, w.fc2_w, p.ls2, x1, p.fc2_b)), f"{new}"
        assert torch.isfinite(got).all() and not torch.equal(got, x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_calls_follow_their_inputs(ctx, dtype):
    """A step (pages, append, attention) and a prompt captured with their workspaces: every replay is the eager
    call on the same state, whatever the workspaces hold, with eager work between."""
    gen = torch.Generator().manual_seed(60)
    h, h_kv, d, page, b = 4, 2, 64, 16, 3
    pool, twin = (PagePool.empty(b, 60, 200, page, DEV) for _ in range(2))
    cache, eager = (PagedKV8.empty(200, h_kv, page, d, dtype, p.page_table, p.lens) for p in (pool, twin))
    for c in (cache, eager):
        for t in parts_of(c)[:4]:
            bits(t).fill_(0x38)
    n = 40
    rows = [normal(gen, (n, x * d), dtype).to(DEV) for x in (h, h_kv, h_kv)]
    counts = i32([10, 20, 10])
    sizes = (ctx.attention_paged_workspace(b, h, h_kv, d, eight=True), ctx.attention_paged_prompts_workspace(cache, n, h),
             ctx.plan_pages_workspace(pool, n))
    ws = [torch.empty(max(s, 16), dtype=torch.uint8, device=DEV) for s in sizes]
    out = (i32([0] * (b + 1)), i32([0] * n), torch.zeros(n, dtype=torch.int64, device=DEV))
    o = [torch.zeros(n, h * d, dtype=dtype, device=DEV) for _ in range(2)]
    single = torch.zeros(b, h * d, dtype=dtype, device=DEV)
    oq = torch.zeros(n, h * d, dtype=dtype, device=DEV)

    def call(p, c, spaces, to, to_single):
        q, k, v = rows
        ctx.plan_pages(p, counts, n, out=out, workspace=spaces[2])
        ctx.kv_append(c, k, v, out[0], q=q, out_q=oq)
        ctx.attention_paged_prompts(oq, c, out[0], out=to, workspace=spaces[1])
        ctx.attention_paged(oq[:b], c, out=to_single, workspace=spaces[0])

    call(pool, cache, ws, o[0], single)
    call(twin, eager, (None, None, None), o[1], single)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(pool, cache, ws, o[0], single)
    torch.cuda.synchronize()
    for i, change in enumerate([[1, 1, 1], [-5, 33, 2], [3, -500, 37], [0, 0, 0], [12, 20, 8], [1, 1, 1]]):
        counts.copy_(i32(change))
        for t in rows:
            t.copy_(normal(gen, t.shape, dtype).to(DEV))
        for t in ws:
            t.fill_(255 if i % 2 else 0)
        for t in (o[0], o[1], single):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = single.clone()
        kept = [t.clone() for t in out]
        call(twin, eager, (None, None, None), o[1], single)
        torch.cuda.synchronize()
        assert torch.equal(got, single) and torch.equal(o[0], o[1]), f"replay {i}"
        assert all(torch.equal(x, y) for x, y in zip(kept, out)), f"replay {i}"
        for x, y in zip((*parts_of(cache), pool.free, pool.state), (*parts_of(eager), twin.free, twin.state)):
            assert torch.equal(bits(x), bits(y)), f"replay {i}"


def test_two_streams(ctx):
    """The same calls on two streams at once, each with its own cache and workspace."""
    gen = torch.Generator().manual_seed(61)
    sides = []
    for i in range(2):
        _, c = make_cache(gen, [900, 40], 2, 16, 64, F16)
        q = normal(gen, (2, 4, 64), F16).to(DEV)
        k = normal(gen, (2, 128), F16).to(DEV)
        sides.append((c, q, k))
    want = []
    for c, q, k in sides:
        copy = PagedKV8(*(t.clone() for t in parts_of(c)), F16)
        ctx.kv_append(copy, k, k)
        want.append((ctx.attention_paged(q, copy), ctx.attention_paged_prompts(q, copy, i32([0, 1, 2]))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = []
    for st, (c, q, k) in zip(streams, sides):
        off = i32([0, 1, 2])
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            ctx.kv_append(c, k, k)
            got.append((ctx.attention_paged(q, c), ctx.attention_paged_prompts(q, c, off)))
    torch.cuda.synchronize()
    for (a, b), (x, y) in zip(got, want):
        assert torch.equal(a, x) and torch.equal(b, y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_past_32_bits(ctx, dtype):
    """A pool of more than 2^32 codes: a sequence in its last pages, appended and read."""
    heads, page, d = 16, 64, 128
    pages = (1 << 32) // (heads * page * d) + 40
    table = torch.tensor([[pages - 1, pages - 3], [0, 1]], dtype=torch.int32, device=DEV)
    c = PagedKV8.empty(pages, heads, page, d, dtype, table, i32([100, 70]))
    gen = torch.Generator().manual_seed(62)
    k, v = (normal(gen, (170, heads * d), dtype).to(DEV) for _ in range(2))
    ctx.kv_append(c, k, v, i32([0, 100, 170]))
    q = normal(gen, (2, heads, d), dtype).to(DEV)
    used = table.flatten().long()
    small = PagedKV8(*(bits(t)[used].view(t.dtype).contiguous() for t in parts_of(c)[:4]), i32([[0, 1], [2, 3]]), c.lens, dtype)
    direct = PagedKV8(*(torch.zeros_like(bits(t)).view(t.dtype) for t in parts_of(small)[:4]), i32([[0, 1], [2, 3]]), c.lens, dtype)
    ctx.kv_append(direct, k, v, i32([0, 100, 170]))
    for s, rows in ((0, 100), (1, 70)):
        for x in "kv":
            assert torch.equal(gpu_values(small, x, s, rows), gpu_values(direct, x, s, rows))
    assert torch.equal(ctx.attention_paged(q, c), ctx.attention_paged(q, small))
    off = i32([0, 1, 2])
    assert torch.equal(ctx.attention_paged_prompts(q, c, off), ctx.attention_paged_prompts(q, small, off))
