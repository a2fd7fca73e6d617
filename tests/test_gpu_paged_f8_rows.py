"""Calls over the 8-bit cache that are given fewer rows than their offsets name, as a call of a fixed number of rows
after ``plan_pages`` is: the rows given are the first ones, with the key numbers, places, rotations and visible
keys that they would have beside the others."""
import math

import pytest
import torch

import f8_reference as F
import paged_reference as R
from headshot_amd.paged import PagedKV8, PagePool

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
DTYPES = [F16, F32]
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def bits(t):
    return t.view(torch.uint8)


def parts_of(c):
    return c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lens


def rope_tables(rows, d):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2) / (d // 2))
    return (torch.cat([angle.sin(), (angle * 1.5).sin()], 1).float().to(DEV),
            torch.cat([angle.cos(), (angle * 1.5).cos()], 1).float().to(DEV))


def cache_of(pool, pages, h_kv, page, d, dtype):
    c = PagedKV8.empty(pages, h_kv, page, d, dtype, pool.page_table, pool.lens)
    for t in parts_of(c)[:2]:
        bits(t).fill_(0x38)  # 1.0
    for t in parts_of(c)[2:4]:
        bits(t).fill_(120)
    return c


# past: keys held before; counts: new tokens, of which the first `n` rows are given. Steps through tiles of few
# rows, of many, cut inside a page and on its border, with sequences behind the cut; page sizes of one wave, two
# and four, and read twice
CASES = [
    (64, 4, 2, 8, [3, 0, 9], [6, 9, 4], 10),
    (64, 4, 1, 16, [0, 40], [9, 30], 7),
    (64, 2, 2, 64, [70, 5, 0], [100, 90, 3], 133),
    (128, 8, 2, 128, [0, 300], [260, 150], 390),
    (64, 2, 1, 512, [100], [900], 555),
    (128, 4, 4, 16, [17, 0], [400, 20], 200),
    (64, 6, 2, 4, [1, 2, 3, 4], [1, 1, 1, 1], 2),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_fewer_rows_than_tokens(ctx, dtype, case):
    d, h, h_kv, page, past, counts, n = CASES[case]
    print(f"[rows {dtype} {CASES[case]}]", flush=True)
    gen = torch.Generator().manual_seed(70 + case)
    b, total = len(counts), sum(counts)
    width = max(-(-(p + c) // page) for p, c in zip(past, counts)) + 1
    pages = b * width
    pool = PagePool.empty(b, width, pages, page, DEV)
    ctx.plan_pages(pool, i32(past), sum(past))
    offsets, positions, slots = ctx.plan_pages(pool, i32(counts), n)
    assert int(offsets[-1]) == total > n
    off = offsets.tolist()
    keys = [p + i for p, c in zip(past, counts) for i in range(c)]
    assert positions.tolist() == keys[:n]
    # a call of the same tokens whose sequences end where the rows do is held to the definition elsewhere
    cut = [min(o, n) for o in off]
    ended = [p + cut[s + 1] - cut[s] for s, p in enumerate(past)]

    qkv = (torch.randn((n, (h + 2 * h_kv) * d), generator=gen) * 1.5 + 0.25).to(dtype).to(DEV)
    q, k, v = qkv.split([h * d, h_kv * d, h_kv * d], 1)
    norm = (torch.randn(d, generator=gen) * 0.2 + 1).to(DEV), (torch.randn(d, generator=gen) * 0.2).to(DEV)
    tables = rope_tables(max(p + c for p, c in zip(past, counts)), d)
    one, two = (cache_of(pool, pages, h_kv, page, d, dtype) for _ in range(2))
    two.lens = i32(ended)
    q1, k1 = ctx.kv_append(one, k, v, offsets, q=q, qn=norm, kn=norm, rope=tables, k_rows=True)
    q2, k2 = ctx.kv_append(two, k, v, i32(cut), q=q, qn=norm, kn=norm, rope=tables, k_rows=True)
    # the rotated rows by the key numbers that plan_pages gave, too
    q3, k3 = ctx.kv_append(cache_of(pool, pages, h_kv, page, d, dtype), k, v, offsets, q=q, qn=norm, kn=norm, rope=tables,
                           positions=positions, k_rows=True)
    assert torch.equal(q1, q2) and torch.equal(k1, k2) and torch.equal(q1, q3) and torch.equal(k1, k3)
    for a, c in zip(parts_of(one)[:4], parts_of(two)[:4]):
        assert torch.equal(bits(a), bits(c))
    # values lie where plan_pages said (no norm, no rotation: half a code's step off)
    assert (slots >= 0).all()
    flat = F.values(one.v.cpu(), one.v_scale.cpu()).transpose(1, 2).flatten(0, 1)[slots.cpu()]
    x = v.cpu().double().unflatten(1, (h_kv, d))
    step = one.v_scale.cpu().double()[slots.cpu() // page][..., None]
    R.assert_within(flat, x, F.HALF_CODE * x.abs() + F.TINY_CODE * step, "values at their slots")

    for causal in (1, 7, 0):
        out = torch.full((n, h * d), 7.0, dtype=dtype, device=DEV)
        ctx.attention_paged_prompts(q1, one, offsets, causal=causal, out=out)
        padded = torch.zeros(total, h, d, dtype=dtype)
        padded[:n] = q1.cpu().unflatten(1, (h, d))
        ref, bound = F.attend(padded, tuple(t.cpu() for t in parts_of(one)), off, causal, 1 / math.sqrt(d), dtype)
        R.assert_within(out.unflatten(1, (h, d)), ref[:n], bound[:n], f"causal {causal}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_step_of_fixed_rows(ctx, dtype):
    """Pages, append and attention captured with a fixed number of rows: replays whose counts pass it are the
    eager calls, and what they append and rotate is by the numbers that plan_pages gives."""
    gen = torch.Generator().manual_seed(80)
    d, h, h_kv, page, b, n = 64, 4, 2, 8, 3, 12
    pool, twin = (PagePool.empty(b, 20, 60, page, DEV) for _ in range(2))
    cache, eager = (cache_of(p, 60, h_kv, page, d, dtype) for p in (pool, twin))
    tables = rope_tables(200, d)
    q, k, v = (torch.randn((n, x * d), generator=gen).to(dtype).to(DEV) for x in (h, h_kv, h_kv))
    counts = i32([4, 4, 4])
    spaces = [(i32([0] * (b + 1)), i32([0] * n), torch.zeros(n, dtype=torch.int64, device=DEV),
               *(torch.zeros(n, x * d, dtype=dtype, device=DEV) for x in (h, h))) for _ in range(2)]
    work = torch.empty(max(16, ctx.attention_paged_prompts_workspace(cache, n, h)), dtype=torch.uint8, device=DEV)

    def call(p, c, space, ws):
        offsets, positions, slots, rows, out = space
        ctx.plan_pages(p, counts, n, out=space[:3])
        ctx.kv_append(c, k, v, offsets, q=q, rope=tables, out_q=rows)
        ctx.attention_paged_prompts(rows, c, offsets, out=out, workspace=ws)

    call(pool, cache, spaces[0], work)
    call(twin, eager, spaces[1], None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(pool, cache, spaces[0], work)
    for change in ([1, 1, 1], [5, 9, 6], [0, 20, 1], [-9, 3, 30], [2, 3, 4]):
        counts.copy_(i32(change))
        for s in spaces:
            s[4].fill_(7.0)
        bits(work).fill_(0x5A)
        graph.replay()
        call(twin, eager, spaces[1], None)
        torch.cuda.synchronize()
        live = min(n, sum(max(c, 0) for c in change))
        for a, c in zip(spaces[0][:3], spaces[1][:3]):
            assert torch.equal(a[:live], c[:live])
        for i in (3, 4):
            assert torch.equal(spaces[0][i][:live], spaces[1][i][:live])
        for a, c in zip(parts_of(cache), parts_of(eager)):
            assert torch.equal(bits(a), bits(c))
        # each token's rows are rotated, and stored, by the position given
        lone = cache_of(pool, 60, h_kv, page, d, dtype)
        by_token, _ = ctx.kv_append(lone, k, v, spaces[0][0], q=q, rope=tables, positions=spaces[0][1])
        assert torch.equal(by_token[:live], spaces[0][3][:live])
        flat = F.values(cache.v.cpu(), cache.v_scale.cpu()).transpose(1, 2).flatten(0, 1)
        at = spaces[0][2][:live].cpu()
        x = v[:live].cpu().double().unflatten(1, (h_kv, d))
        R.assert_within(flat[at], x, F.HALF_CODE * x.abs() + F.TINY_CODE * cache.v_scale.cpu().double()[at // page][..., None],
                        f"{change}: values at their slots")
        assert (spaces[0][4][live:] == 7.0).all()
