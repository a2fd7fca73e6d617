"""The paged key-value cache and its attention on the GPU, against plain
definitions in 64 bits (tests/paged_reference.py, which also derives the
tolerances), and together as a block uses them."""
import math

import pytest
import torch

import paged_reference as R
from headshot_amd.aggregator import BlockWeights, block_forward, block_forward_cached
from headshot_amd.paged import PagedKV

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
DTYPES = [F16, F32]


def normal(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen) * std + mean).to(dtype)


def i32(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


def offsets_of(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def make_cache(gen, lens, heads, page, d, dtype, spare=3, width=2):
    """Pages in no order, of values already there; CPU and GPU copies."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    m = max(need, default=0) + width
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (m - n))
        at += n
    k, v = (normal(gen, (pages, heads, page, d), dtype) for _ in range(2))
    table = torch.tensor(table, dtype=torch.int32).reshape(len(lens), m)
    cpu = PagedKV(k, v, table, i32(lens, "cpu"))
    return cpu, PagedKV(*(t.to(DEV) for t in (k, v, table, cpu.lens)))


def rope_tables(rows, d):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2) / (d // 2))
    # the two halves of a row are read separately: make them differ
    return (torch.cat([angle.sin(), (angle * 1.5).sin()], 1).float(),
            torch.cat([angle.cos(), (angle * 1.5).cos()], 1).float())


# ------------------------------------------------------------------ kv_append


def run_append(ctx, seed, dtype, d, h, h_kv, page, new, past, norm, rope, step=False, wide=True, positions=None,
               spoil=None, behind=0, rows=None):
    gen = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(past, new)]
    cpu, gpu = make_cache(gen, lens, h_kv, page, d, dtype)
    if spoil:
        spoil(cpu)
        gpu.page_table.copy_(cpu.page_table)
        gpu.lens.copy_(cpu.lens)
    n = sum(new) + behind
    qkv = normal(gen, (n, (h + 2 * h_kv) * d + (64 if wide else 0)), dtype, 1.5, 0.25)
    parts = [h * d, h_kv * d, h_kv * d]
    cut = lambda t: [x if wide else x.contiguous() for x in t[:, :sum(parts)].split(parts, 1)]  # noqa: E731
    q, k, v = cut(qkv)
    gq, gk, gv = cut(qkv.to(DEV))
    nrm = lambda: (normal(gen, (d,), F32, 0.2, 1.0), normal(gen, (d,), F32, 0.2)) if norm else None  # noqa: E731
    qn, kn = nrm(), nrm()
    tables = rope_tables(rows or max(lens) + 1, d) if rope else None
    up = lambda p: None if p is None else tuple(t.to(DEV) for t in p)  # noqa: E731
    off = None if step else offsets_of(new)
    mark = 7.0
    out_q, out_k = (torch.full((n, x * d), mark, dtype=dtype, device=DEV) for x in (h, h_kv))
    got_q, got_k = ctx.kv_append(gpu, gk, gv, None if step else i32(off), q=gq, qn=up(qn), kn=up(kn),
                                 rope=up(tables), positions=None if positions is None else i32(positions),
                                 out_q=out_q, out_k=out_k)
    assert got_q.data_ptr() == out_q.data_ptr() and got_k.data_ptr() == out_k.data_ptr()
    heads = lambda t: t.unflatten(1, (-1, d))  # noqa: E731
    rq, rk, rkc, rvc = R.append(cpu.k, cpu.v, cpu.page_table, cpu.lens, heads(k), heads(v), off, heads(q), qn, kn,
                                tables, positions, 1e-5)
    live = sum(new)
    R.assert_within(heads(got_q)[:live], rq[:live], R.append_bound(rq[:live], q, dtype), "q rows")
    R.assert_within(heads(got_k)[:live], rk[:live], R.append_bound(rk[:live], k, dtype), "k rows")
    assert (got_q[live:] == mark).all() and (got_k[live:] == mark).all(), "rows behind the last sequence"
    R.assert_within(gpu.k, rkc, R.append_bound(rkc, k, dtype), "k cache")
    touched = (rkc != cpu.k.double()).any(-1)
    assert torch.equal(gpu.k.cpu()[~touched], cpu.k[~touched]), "pages of no new token"
    assert torch.equal(gpu.v.cpu().double(), rvc), "v cache"
    # nothing but the pages without q and k rows, the same bits
    again = PagedKV(cpu.k.to(DEV), cpu.v.to(DEV), gpu.page_table, gpu.lens)
    none = ctx.kv_append(again, gk, gv, None if step else i32(off), kn=up(kn), rope=up(tables),
                         positions=None if positions is None else i32(positions))
    assert none == (None, None)
    assert torch.equal(again.k, gpu.k) and torch.equal(again.v, gpu.v)


@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_prompts(ctx, dtype, d, norm, rope):
    for i, (h, h_kv, page, new, past) in enumerate([
        (4, 4, 16, [5, 0, 33, 1, 0], [0, 9, 17, 300, 0]),
        (7, 1, 1, [3, 2], [1, 0]),
        (10, 5, 64, [70, 129], [63, 0]),
        (16, 16, 8, [1], [0]),
    ]):
        print(f"[append {dtype} d={d} norm={norm} rope={rope} case {i}]", flush=True)
        run_append(ctx, 100 + i, dtype, d, h, h_kv, page, new, past, norm, rope, wide=i % 2 == 0, behind=3 * (i % 3))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_steps(ctx, dtype, d):
    for i, (h, h_kv, page, past) in enumerate([(3, 3, 4, [0, 3, 4, 1000]), (32, 8, 32, [31, 32, 0] * 43), (8, 2, 256, [5])]):
        print(f"[append step {dtype} d={d} case {i}]", flush=True)
        run_append(ctx, 200 + i, dtype, d, h, h_kv, page, [1] * len(past), past, True, True, step=True, wide=i != 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_positions(ctx, dtype):
    """Rows of the tables by token; rows outside them (prefix tokens: -1) are
    not rotated."""
    run_append(ctx, 300, dtype, 64, 4, 2, 16, [6, 5], [0, 11], False, True, rows=9,
               positions=[-1, -1, 0, 3, 8, 9, 2 ** 31 - 1, -2 ** 31, 4, 4, 0])
    run_append(ctx, 301, dtype, 128, 4, 2, 16, [40], [0], True, True, rows=20)  # longer than the tables


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_without_a_place(ctx, dtype):
    """Page numbers outside the pool and lengths outside the table: the tokens
    are not stored, everything else is as usual."""
    def spoil(c):
        c.page_table[0, 0], c.page_table[1, 1] = -1, c.k.shape[0]
        c.page_table[2, 0] = 2 ** 31 - 1

    run_append(ctx, 310, dtype, 64, 2, 2, 8, [12, 20, 9], [0, 4, 0], True, True, spoil=spoil)

    def lengths(c):
        c.lens[0], c.lens[1], c.lens[2] = 3, 2 ** 31 - 1, c.page_table.shape[1] * 8 + 2  # 5 keys before the first

    run_append(ctx, 311, dtype, 64, 2, 2, 8, [8, 20, 9], [0, 4, 0], False, False, spoil=lengths)


def test_append_nothing(ctx):
    cpu, gpu = make_cache(torch.Generator().manual_seed(1), [4, 0], 2, 4, 64, F16)
    rows = torch.empty((0, 128), dtype=F16, device=DEV)
    q, k = ctx.kv_append(gpu, rows, rows, i32([0, 0, 0]), q=rows, k_rows=True)
    assert q.shape == k.shape == (0, 128) and torch.equal(gpu.k.cpu(), cpu.k)


# ------------------------------------------------------------- attention_packed


def run_packed(ctx, seed, dtype, d, h, h_kv, nq, nk, causal, scale=None, std=1.0, wide=False, behind=0, poison=None):
    gen = torch.Generator().manual_seed(seed)
    n, m = sum(nq) + behind, sum(nk) + (behind if nk != nq else 0)
    m = n if nk == nq else m

    def rows(count, heads):
        if not wide:
            return normal(gen, (count, heads, d), dtype, std)
        return normal(gen, (count, (heads + 1) * d), dtype, std)[:, d:].unflatten(1, (heads, d))

    q, k, v = rows(n, h), rows(m, h_kv), rows(m, h_kv)
    if poison:
        poison(q, k, v)
    qo, ko = offsets_of(nq), offsets_of(nk)
    mark = 7.0
    out = torch.full((n, h * d), mark, dtype=dtype, device=DEV)
    got = ctx.attention_packed(*(x.to(DEV) if not wide else up_wide(x, d) for x in (q, k, v)), i32(qo),
                               None if nk == nq else i32(ko), causal=causal, scale=scale, out=out)
    assert got.data_ptr() == out.data_ptr()
    got = got.unflatten(1, (h, d)).cpu()
    sc = 1 / math.sqrt(d) if scale is None else scale
    for s in range(len(nq)):
        qs, ks, vs = q[qo[s]:qo[s + 1]], k[ko[s]:ko[s + 1]], v[ko[s]:ko[s + 1]]
        seen = R.seen_keys(nq[s], nk[s], causal)
        ref, mag = R.attention(qs.double(), ks.double(), vs.double(), seen, sc)
        fin = [torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (qs, ks, vs)]
        bound = R.attention_bound(ref.nan_to_num(0.0, 0.0, 0.0), mag.nan_to_num(0.0, 0.0, 0.0), *fin, seen, sc, dtype)
        g = got[qo[s]:qo[s + 1]]
        odd = ~ref.isfinite() & bound.isfinite()
        assert torch.equal(g.isnan() & odd, ref.isnan()), f"sequence {s}: NaN places"
        assert torch.equal(g[odd].nan_to_num(0.0), ref[odd].to(dtype).nan_to_num(0.0)), f"sequence {s}: infinities"
        R.assert_within(g[~odd], ref[~odd], bound[~odd], f"sequence {s}")
    assert (got[sum(nq):] == mark).all(), "rows behind the last sequence"


def up_wide(x, d):
    """The same column range of a wider row on the GPU."""
    base = torch.zeros((x.shape[0], (x.shape[1] + 1) * d), dtype=x.dtype)
    base[:, d:] = x.flatten(1)
    return base.to(DEV)[:, d:].unflatten(1, (x.shape[1], d))


@pytest.mark.parametrize("causal", [0, 1, 5, 64])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_lengths(ctx, dtype, d, causal):
    for i, (h, h_kv, n) in enumerate([(2, 2, [1, 0, 63, 64, 65]), (4, 1, [129, 2, 200]), (6, 2, [257, 1, 1]),
                                      (1, 1, [31, 33])]):
        print(f"[packed {dtype} d={d} causal={causal} case {i}]", flush=True)
        run_packed(ctx, 400 + i, dtype, d, h, h_kv, n, n, causal, wide=i == 1, behind=2 * i)


@pytest.mark.parametrize("causal", [0, 1, 7])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_other_keys(ctx, dtype, causal):
    """More keys than queries (a kept prefix), fewer (rows that see nothing),
    none on either side."""
    run_packed(ctx, 410, dtype, 64, 4, 2, [3, 70, 0, 5, 40], [100, 70, 9, 0, 23], causal, behind=3)
    run_packed(ctx, 411, dtype, 128, 2, 1, [130, 1, 66], [64, 300, 1], causal)


@pytest.mark.parametrize("causal", [0, 1, 12])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_short_shared_heads(ctx, dtype, d, causal):
    """Short sequences whose query heads share key heads, by two, four and more."""
    for i, (h, h_kv, nq, nk) in enumerate([
        (8, 2, [5, 32, 1, 0, 7], [5, 32, 1, 0, 7]),
        (12, 1, [33, 20], [33, 320]),
        (6, 1, [60, 64], [60, 64]),
        (32, 8, [1, 2, 3], [65, 64, 0]),
        (64, 4, [9], [130]),
    ]):
        print(f"[packed shared {dtype} d={d} causal={causal} case {i}]", flush=True)
        run_packed(ctx, 445 + i, dtype, d, h, h_kv, nq, nk, causal, wide=i % 2 == 0, behind=i)


@pytest.mark.parametrize("value", [math.inf, math.nan, "lowest"])
def test_packed_short_masked_values(ctx, value):
    x = torch.finfo(F16).min if value == "lowest" else value

    def poison(q, k, v):
        k[20], v[15, :, 3], v[33] = x, x, x

    run_packed(ctx, 446, F16, 64, 8, 2, [30, 6], [30, 6], 1, poison=poison)


def split(ctx, dtype, d, h, h_kv, nq, nk, causal):
    """Whether a call's keys are split."""
    return ctx.attention_packed_workspace(dtype, sum(nq), sum(nk), len(nq), h, h_kv, d, causal) > 0


@pytest.mark.parametrize("causal", [0, 1, 7, 1000])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_split_keys(ctx, dtype, d, causal):
    """Few queries over many keys, of sequences long and short; rows that see
    nothing, no key or no query; wide rows; tiles of both kinds."""
    for i, (h, h_kv, nq, nk) in enumerate([
        (2, 1, [1], [2048]),
        (3, 3, [1, 16, 17], [2500, 1, 900]),
        (8, 2, [3, 0, 40, 2], [700, 900, 20, 3000]),
        (2, 2, [1, 1, 1, 1], [0, 2100, 64, 65]),
        (2, 1, [200, 130], [3001, 1500]),
        (1, 1, [2200], [2200]),
        (1, 1, [300], [4200]),
    ]):
        print(f"[packed split {dtype} d={d} causal={causal} case {i}]", flush=True)
        assert split(ctx, dtype, d, h, h_kv, nq, nk, causal)
        run_packed(ctx, 450 + i, dtype, d, h, h_kv, nq, nk, causal, wide=i % 2 == 1, behind=i)


@pytest.mark.parametrize("nq", [5, 150])
@pytest.mark.parametrize("value", [math.inf, math.nan, "lowest"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_split_odd_values(ctx, dtype, value, nq):
    """Infinities and NaN in seen and in masked places of a split call, and
    scores that move the maximum from piece to piece."""
    x = torch.finfo(dtype).min if value == "lowest" else value

    def poison(q, k, v):
        n = k.shape[0]
        k[: n // 2] *= 1.5
        v[n // 3, :, 3], v[n - 2, :, 5], k[n - 1, :, 0] = x, x, x

    for causal in (1, 10):
        assert split(ctx, dtype, 64, 2, 1, [nq], [2700], causal)
        run_packed(ctx, 460, dtype, 64, 2, 1, [nq], [2700], causal, poison=poison)


def test_packed_split_f32_sizes(ctx):
    """f32 values that the bf16 parts do not hold, in one piece's keys, in the
    values, in some queries: those are computed another way, the rest is not."""
    def at(where, x):
        def poison(q, k, v):
            {"q": q, "k": k, "v": v}[where][17, :, 5] = x
        return poison

    for where, x in [("q", 2.0 ** 60), ("k", 2.0 ** 55), ("v", 2.0 ** 70), ("v", 2.0 ** -120), ("k", 2.0 ** -130)]:
        assert split(ctx, F32, 64, 2, 2, [300], [2500], 1)
        run_packed(ctx, 470, F32, 64, 2, 2, [300], [2500], 1, poison=at(where, x))


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_split_graph(ctx, dtype):
    """A captured split call follows its offsets, the caller's workspace holding
    anything; the call's own workspace gives the same."""
    gen = torch.Generator().manual_seed(14)
    q, k, v = (normal(gen, (n, h, 64), dtype).to(DEV) for n, h in ((60, 4), (4000, 2), (4000, 2)))
    off, koff = i32([0, 30, 60]), i32([0, 2000, 4000])
    size = ctx.attention_packed_workspace(dtype, 60, 4000, 2, 4, 2, 64, 1)
    assert size > 0
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device=DEV)
    ctx.attention_packed(q, k, v, off, koff, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ctx.attention_packed(q, k, v, off, koff, workspace=ws)
    for i, (cut, kcut) in enumerate([(30, 2000), (0, 0), (60, 4000), (1, 3999), (59, 10), (17, 2048)]):
        off.copy_(i32([0, cut, 60]))
        koff.copy_(i32([0, kcut, 4000]))
        ws.fill_(255 if i % 2 else 0)
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        assert torch.equal(got, ctx.attention_packed(q, k, v, off, koff)), f"cut {cut} {kcut}"


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_scales(ctx, dtype):
    """Peaked weights, a scale of the caller's, negative and zero ones."""
    for scale, std in [(1.0, 1.0), (0.05, 3.0), (-0.125, 1.0), (0.0, 1.0), (0.125, 400.0)]:
        run_packed(ctx, 420, dtype, 64, 2, 1, [90, 140], [90, 140], 1, scale=scale, std=std)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_growing_scores(ctx, dtype, d):
    """Scores that rise and fall by large steps along the keys, so the running
    maximum moves late and often."""
    def steps(q, k, v):
        q.copy_(torch.ones_like(q) * 0.5)
        level = torch.tensor([0, 9, -20, 14, 13, -3, 30, 2, 45, 44], dtype=torch.float32)
        k.copy_((k.float() * 0.05 + level[(torch.arange(k.shape[0]) // 37) % 10][:, None, None] / d ** 0.5 * 2).to(k.dtype))

    for causal in (0, 1):
        run_packed(ctx, 430, dtype, d, 2, 1, [370], [370], causal, poison=steps)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, "lowest"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_masked_values(ctx, dtype, d, value):
    """What a later key or value holds leaves the queries before it alone."""
    x = torch.finfo(dtype).min if value == "lowest" else value

    def poison(q, k, v):
        k[50], v[51, :, 3], v[77] = x, x, x
        k[100:103] = x

    for causal in (1, 10):
        run_packed(ctx, 440, dtype, d, 2, 1, [150], [150], causal, poison=poison)

    def last(q, k, v):  # the next sequence's keys, and rows of no sequence
        k[40:], v[40:] = x, x

    gen = torch.Generator().manual_seed(1)
    q, k, v = (normal(gen, (60, 2, d), dtype) for _ in range(3))
    clean = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v)), i32([0, 40, 55]), causal=0)
    last(q, k, v)
    got = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v)), i32([0, 40, 55]), causal=0)
    assert torch.equal(got[:40], clean[:40])


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_longer(ctx, dtype):
    """Several query tiles and many key tiles: against f64 on the GPU."""
    for d, h, h_kv, lens, causal in [(64, 16, 16, [1374, 700], 0), (128, 8, 2, [1500, 3, 611], 1), (64, 5, 5, [2000], 137),
                                     (128, 6, 1, [513, 1025], 0)]:
        print(f"[packed longer {dtype} d={d} causal={causal}]", flush=True)
        gen = torch.Generator().manual_seed(d + h)
        n = sum(lens)
        q, k, v = (normal(gen, (n, x, d), dtype).to(DEV) for x in (h, h_kv, h_kv))
        got = ctx.attention_packed(q, k, v, i32(offsets_of(lens)), causal=causal).unflatten(1, (h, d))
        for a, m in zip(offsets_of(lens), lens):
            qs, ks, vs = (x[a:a + m].double().transpose(0, 1) for x in (q, k, v))
            ks, vs = ks.repeat_interleave(h // h_kv, 0), vs.repeat_interleave(h // h_kv, 0)
            s = qs @ ks.transpose(1, 2).contiguous() / math.sqrt(d)
            s.masked_fill_(torch.arange(m, device=DEV) >= R.seen_keys(m, m, causal).to(DEV)[:, None], -math.inf)
            p = torch.softmax(s, -1)
            ref, mag = (p @ vs).transpose(0, 1).cpu(), (p @ vs.abs()).transpose(0, 1).cpu()
            bound = R.attention_bound(ref, mag, *(x[a:a + m].cpu() for x in (q, k, v)),
                                      R.seen_keys(m, m, causal), 1 / math.sqrt(d), dtype)
            R.assert_within(got[a:a + m], ref, bound, f"d={d} length {m}")


def gpu_reference(q, k, v, seen, scale):
    """(result, sum(p |v|)) of one sequence in f64 on the GPU; values that a
    query does not see count as zeros."""
    h, h_kv = q.shape[1], k.shape[1]
    qs, ks, vs = (x.double().transpose(0, 1) for x in (q, k, v))
    ks, vs = ks.repeat_interleave(h // h_kv, 0), vs.repeat_interleave(h // h_kv, 0)
    hidden = torch.arange(k.shape[0], device=DEV) >= seen.to(DEV)[:, None]
    out, mag = torch.empty_like(qs), torch.empty_like(qs)
    for i in range(h):
        s = (qs[i] @ ks[i].T * scale).masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1)
        odd = ~vs[i].isfinite()
        plain = torch.where(odd, 0.0, vs[i])
        out[i], mag[i] = p @ plain, p @ plain.abs()
        for j in odd.any(1).nonzero().flatten().tolist():
            at = ~hidden[:, j]
            out[i, at] += torch.where(odd[j], p[at, j, None] * vs[i, j], 0.0)
    return out.transpose(0, 1).cpu(), mag.transpose(0, 1).cpu()


@pytest.mark.parametrize("what", ["plain", "inf", "nan", "huge", "huge q", "tiny"])
@pytest.mark.parametrize("d,h,h_kv", [(64, 16, 8), (128, 16, 8), (128, 32, 4)])
def test_packed_f32_tiles(ctx, d, h, h_kv, what):
    """f32 over enough queries for the tiles of 32 a wave, with values that the
    three bf16 parts do not hold among them."""
    lens = [1301, 900, 130]
    gen = torch.Generator().manual_seed(d)
    q, k, v = (normal(gen, (sum(lens), x, d), F32) for x in (h, h_kv, h_kv))
    if what in ("inf", "nan"):
        x = math.inf if what == "inf" else math.nan
        v[700, 3, 7], v[1310, :, 1], v[2331 - 40, min(5, h_kv - 1)] = x, -x, x
    elif what == "huge":
        v[700] *= 2.0 ** 60
        k[1500, 2] *= 2.0 ** 55
    elif what == "huge q":
        q[800:803] *= 2.0 ** 52
        q[2000, 5] *= 2.0 ** 70
    elif what == "tiny":
        v[:1301] *= 2.0 ** -110
        k[1400:1500] *= 2.0 ** -115
        q[1600:1700] *= 2.0 ** -115
    for causal in (1, 0, 137):
        print(f"[packed f32 tiles d={d} {what} causal={causal}]", flush=True)
        got = ctx.attention_packed(*(x.to(DEV) for x in (q, k, v)), i32(offsets_of(lens)), causal=causal)
        got = got.unflatten(1, (h, d)).cpu()
        for s, (a, n) in enumerate(zip(offsets_of(lens), lens)):
            qs, ks, vs = (x[a:a + n] for x in (q, k, v))
            seen = R.seen_keys(n, n, causal)
            ref, mag = gpu_reference(*(x.to(DEV) for x in (qs, ks, vs)), seen, 1 / math.sqrt(d))
            fin = [torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (qs, ks, vs)]
            bound = R.attention_bound(ref.nan_to_num(0.0, 0.0, 0.0), mag, *fin, seen, 1 / math.sqrt(d), F32)
            g = got[a:a + n]
            odd = ~ref.isfinite()
            nans = g.isnan(), ref.isnan()
            assert torch.equal(*nans), f"sequence {s}: NaN places"
            assert torch.equal(g[odd].nan_to_num(0.0), ref[odd].float().nan_to_num(0.0)), f"sequence {s}: infinities"
            R.assert_within(g[~odd], ref[~odd], bound[~odd], f"sequence {s}")


@pytest.mark.parametrize("what", ["plain", "odd", "growing"])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_f16_long(ctx, d, what):
    """f16 over enough long sequences for tiles of eight waves."""
    lens, h, h_kv = [5203, 130], 32, 8
    gen = torch.Generator().manual_seed(d + 1)
    q, k, v = (normal(gen, (sum(lens), x, d), F16) for x in (h, h_kv, h_kv))
    if what == "odd":
        v[700, 3, 7], v[1310, :, 1], v[5100, 5], v[5210, 2, 2] = math.inf, -math.inf, math.nan, math.inf
    elif what == "growing":
        k.mul_(0.1)
        q.copy_(torch.ones_like(q) * 0.5)
        k.add_(((torch.arange(k.shape[0]) * 7919 % 61)[:, None, None] / d ** 0.5).half())
    for causal in (1, 1374, 0):
        print(f"[packed f16 long d={d} {what} causal={causal}]", flush=True)
        got = ctx.attention_packed(*(x.to(DEV) for x in (q, k, v)), i32(offsets_of(lens)), causal=causal)
        got = got.unflatten(1, (h, d)).cpu()
        for s, (a, n) in enumerate(zip(offsets_of(lens), lens)):
            qs, ks, vs = (x[a:a + n, :1 + i] for x, i in ((q, 7), (k, 1), (v, 1)))  # two key heads of the eight
            seen = R.seen_keys(n, n, causal)
            ref, mag = gpu_reference(*(x.to(DEV) for x in (qs, ks, vs)), seen, 1 / math.sqrt(d))
            fin = [torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (qs, ks, vs)]
            bound = R.attention_bound(ref.nan_to_num(0.0, 0.0, 0.0), mag, *fin, seen, 1 / math.sqrt(d), F16)
            g = got[a:a + n, :8]
            odd = ~ref.isfinite()
            nans = g.isnan(), ref.isnan()
            assert torch.equal(*nans), f"sequence {s}: NaN places"
            assert torch.equal(g[odd].nan_to_num(0.0), ref[odd].half().nan_to_num(0.0)), f"sequence {s}: infinities"
            R.assert_within(g[~odd], ref[~odd], bound[~odd], f"sequence {s}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_many_sequences(ctx, dtype):
    """More sequences than a wave has lanes, empty ones among them."""
    lens = [(i * 37) % 23 for i in range(200)]
    run_packed(ctx, 450, dtype, 64, 2, 1, lens, lens, 1, behind=2)
    run_packed(ctx, 451, dtype, 128, 8, 8, lens, [n + i % 3 for i, n in enumerate(lens)], 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_no_keys(ctx, dtype):
    """Queries of sequences without keys get zeros, also large ones."""
    q = torch.full((700, 32, 64), 1e30 if dtype == F32 else 6e4, dtype=dtype, device=DEV)
    k = torch.empty((0, 32, 64), dtype=dtype, device=DEV)
    got = ctx.attention_packed(q, k, k, i32([0, 400, 700]), i32([0, 0, 0]))
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_graph(ctx, dtype):
    """A captured prompt follows its offsets."""
    gen = torch.Generator().manual_seed(12)
    q, k, v = (normal(gen, (300, h, 64), dtype).to(DEV) for h in (4, 2, 2))
    off = i32([0, 100, 300])
    ctx.attention_packed(q, k, v, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ctx.attention_packed(q, k, v, off)
    for cut in (100, 0, 299, 300, 17):
        off.copy_(i32([0, cut, 300]))
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        assert torch.equal(got, ctx.attention_packed(q, k, v, off)), f"cut {cut}"


def test_two_streams(ctx):
    """Calls on two streams at once, a workspace each, give what they give alone."""
    gen = torch.Generator().manual_seed(13)
    sides = []
    for i in range(2):
        cpu, gpu = make_cache(gen, [3000 + i, 40, 900], 4, 16, 64, F16)
        q = normal(gen, (3, 8, 64), F16).to(DEV)
        ws = torch.empty(ctx.attention_paged_workspace(3, 8, 4, 64), dtype=torch.uint8, device=DEV)
        sides.append((torch.cuda.Stream(), q, gpu, ws, ctx.attention_paged(q, gpu)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (stream, q, gpu, ws, _alone) in enumerate(sides):
            with torch.cuda.stream(stream):
                got[i].append(ctx.attention_paged(q, gpu, workspace=ws))
    torch.cuda.synchronize()
    for i, side in enumerate(sides):
        assert all(torch.equal(x, side[4]) for x in got[i])


@pytest.mark.parametrize("n,m", [(300, 300), (40, 4000), (400, 2500)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_bad_offsets(ctx, dtype, n, m):
    """Offsets that do not ascend or leave the rows: no write outside the
    buffers, whole keys and split ones."""
    gen = torch.Generator().manual_seed(16)
    q, k, v = (normal(gen, (rows, h, 64), dtype).to(DEV) for rows, h in ((n, 2), (m, 1), (m, 1)))
    size = ctx.attention_packed_workspace(dtype, n, m, 4, 2, 1, 64, 1)
    assert (size > 0) == (m >= 1536)
    guard = 1 << 16
    ws = torch.full((size + 2 * guard,), 0xA5, dtype=torch.uint8, device=DEV)
    out = torch.full((n + 64, 128), 7.0, dtype=dtype, device=DEV)
    big = 2 ** 31 - 1
    for off, koff in [([0, n, 0, n, 0], [0, m, 0, m, 0]), ([-5, 3, big, 2, n], [big, -big, m, 1, m + 9]),
                      ([0, 5, 9, 20, n], [m, m // 2, m, 0, m]), ([n, n, 3, n, n], [0, 5, m, 5, m]),
                      ([0, n // 2, 0, n // 3, n], [0, m, 1, m, 2])]:
        for causal in (0, 1):
            print(f"[bad offsets {dtype} {off} {koff} causal={causal}]", flush=True)
            ctx.attention_packed(q, k, v, i32(off), i32(koff), causal=causal, out=out[32:32 + n],
                                 workspace=ws[guard:guard + size] if size else None)
    assert (ws[:guard] == 0xA5).all() and (ws[guard + size:] == 0xA5).all()
    assert (out[:32] == 7).all() and (out[32 + n:] == 7).all()


def test_two_streams_split(ctx):
    """Split packed calls on two streams at once, of their own workspaces."""
    gen = torch.Generator().manual_seed(15)
    sides = []
    for i in range(2):
        q, k, v = (normal(gen, (n, h, 64), F16).to(DEV) for n, h in ((20 + i, 4), (3000, 2), (3000, 2)))
        call = (q, k, v, i32([0, 20 + i]), i32([0, 3000]))
        assert split(ctx, F16, 64, 4, 2, [20 + i], [3000], 1)
        sides.append((torch.cuda.Stream(), call, ctx.attention_packed(*call)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (stream, call, _alone) in enumerate(sides):
            with torch.cuda.stream(stream):
                got[i].append(ctx.attention_packed(*call))
    torch.cuda.synchronize()
    for i, side in enumerate(sides):
        assert all(torch.equal(x, side[2]) for x in got[i])


# -------------------------------------------------------------- attention_paged


def paged_reference(cpu, q, dtype, scale):
    """(result, bound) per sequence; pages outside the pool are not seen."""
    n_pages, h_kv, page, d = cpu.k.shape
    outs, bounds = [], []
    for s in range(q.shape[0]):
        n = max(0, min(int(cpu.lens[s]), cpu.page_table.shape[1] * page))
        pos = torch.arange(n)
        at = cpu.page_table[s].long()[pos // page]
        ok = (at >= 0) & (at < n_pages)
        k, v = (c[at[ok], :, pos[ok] % page] for c in (cpu.k, cpu.v))
        ref, mag = R.attention(q[s:s + 1].double(), k.double(), v.double(), [int(ok.sum())], scale)
        outs.append(ref)
        bounds.append(R.attention_bound(ref, mag, q[s:s + 1], k, v, [int(ok.sum())], scale, dtype))
    return torch.cat(outs), torch.cat(bounds)


def run_paged(ctx, seed, dtype, d, h, h_kv, page, lens, scale=None, wide=False, spoil=None, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    cpu, gpu = make_cache(gen, lens, h_kv, page, d, dtype)
    # what no sequence reaches holds NaN
    reached = torch.zeros(cpu.k.shape[0], page, dtype=torch.bool)
    for s, n in enumerate(lens):
        pos = torch.arange(n)
        reached[cpu.page_table[s].long()[pos // page], pos % page] = True
    for c in (cpu.k, cpu.v):
        c.transpose(1, 2)[~reached] = math.nan
    if spoil:
        spoil(cpu)
    gpu = PagedKV(*(t.to(DEV) for t in (cpu.k, cpu.v, cpu.page_table, cpu.lens)))
    q = normal(gen, (len(lens), h, d), dtype, std)
    gq = up_wide(q, d) if wide else q.to(DEV)
    got = ctx.attention_paged(gq, gpu, scale=scale).unflatten(1, (h, d))
    ref, bound = paged_reference(cpu, q, dtype, 1 / math.sqrt(d) if scale is None else scale)
    R.assert_within(got, ref, bound, "paged")
    return gq, gpu, got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_lengths(ctx, dtype, d):
    for i, (h, h_kv, page, lens) in enumerate([
        (2, 2, 16, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129]),
        (16, 16, 16, [300, 1, 0, 77, 800]),
        (8, 1, 1, [40, 5]),
        (6, 2, 2, [70, 131]),
        (9, 3, 4, [1000]),
        (35, 5, 8, [3, 260]),
        (40, 2, 64, [513, 64, 200]),          # 20 query heads to a key head
        (33, 1, 128, [100, 129]),             # 33
        (4, 4, 1024, [1500, 2049]),
        (1, 1, 32, [0, 0]),
        (4, 2, 16, [5] * 130),                # more sequences than lanes
    ]):
        print(f"[paged {dtype} d={d} case {i}]", flush=True)
        run_paged(ctx, 500 + i, dtype, d, h, h_kv, page, lens, wide=i % 2 == 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_long(ctx, dtype):
    """One sequence split over its keys as far as it goes, beside short ones."""
    for h, h_kv, lens in [(1, 1, [20000]), (8, 2, [9001, 1, 0, 4500]), (2, 2, [1] * 70 + [7777] + [3] * 9)]:
        print(f"[paged long {dtype} {h}/{h_kv}]", flush=True)
        run_paged(ctx, 520, dtype, 64, h, h_kv, 32, lens)
        run_paged(ctx, 521, dtype, 128, h, h_kv, 16, lens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_shared_pages(ctx, dtype):
    """Sequences with a common prefix read the same pages, and a table may name
    a page twice."""
    def share(c):
        c.page_table[1, :2] = c.page_table[0, :2]
        c.page_table[2, :3] = c.page_table[0, :1]

    for h, h_kv in [(3, 3), (8, 2)]:
        run_paged(ctx, 535, dtype, 64, h, h_kv, 16, [100, 61, 48], spoil=share)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_scales(ctx, dtype):
    for scale, std in [(1.0, 1.0), (0.3, 3.0), (-0.125, 1.0), (0.0, 1.0), (40.0, 100.0)]:
        run_paged(ctx, 530, dtype, 64, 4, 2, 16, [500, 90], scale=scale, std=std)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_bad_pages(ctx, dtype):
    """Page numbers outside the pool are not read, lengths past the table stop
    at its end, negative ones are empty."""
    def pages(c):
        c.page_table[0, 1], c.page_table[1, 0], c.page_table[2] = -1, c.k.shape[0], 2 ** 31 - 1

    run_paged(ctx, 540, dtype, 64, 4, 2, 16, [70, 40, 33, 50], spoil=pages)

    def lengths(c):
        c.lens[0], c.lens[1] = 2 ** 31 - 1, -5
        c.page_table[0] = c.page_table[2]
        c.k[:], c.v[:] = c.k.nan_to_num(0.5), c.v.nan_to_num(0.25)

    run_paged(ctx, 541, dtype, 128, 4, 2, 16, [70, 40, 100], spoil=lengths)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_infinite_values(ctx, dtype):
    """Seen infinities and NaN come through as the definition has them."""
    def spoil(c):
        at = int(c.page_table[0, 2])
        c.v[at, 0, 3, 5], c.v[at, 1, 4, 6], c.v[at, 1, 5, 6] = math.inf, math.inf, -math.inf
        c.k[int(c.page_table[1, 0]), 1, 2, 0] = math.nan

    gen = torch.Generator().manual_seed(7)
    cpu, _ = make_cache(gen, [60, 60, 60], 2, 16, 64, dtype)
    spoil(cpu)
    gpu = PagedKV(*(t.to(DEV) for t in (cpu.k, cpu.v, cpu.page_table, cpu.lens)))
    q = normal(gen, (3, 4, 64), dtype)
    got = ctx.attention_paged(q.to(DEV), gpu).unflatten(1, (4, 64)).cpu()
    assert (got[0, :2, 5] == math.inf).all() and got[0, 2:, 6].isnan().all() and got[1, 2:].isnan().all()
    odd = torch.zeros(got.shape, dtype=torch.bool)
    odd[0, :2, 5], odd[0, 2:, 6], odd[1, 2:] = True, True, True
    assert got[~odd].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_graph(ctx, dtype):
    """A captured step follows lens and page_table; eager work between the
    replays; a side stream; a workspace of the caller's."""
    gen = torch.Generator().manual_seed(9)
    cpu, gpu = make_cache(gen, [900, 350, 64], 2, 16, 64, dtype)
    rows = normal(gen, (6, 3, (4 + 2 + 2) * 64), dtype).to(DEV)
    x = rows[0].clone()
    ws = torch.empty(ctx.attention_paged_workspace(3, 4, 2, 64), dtype=torch.uint8, device=DEV)
    tables = tuple(t.to(DEV) for t in rope_tables(1000, 64))

    def step():
        q, k, v = x.split([256, 128, 128], 1)
        q, _ = ctx.kv_append(gpu, k, v, q=q, rope=tables)
        return ctx.attention_paged(q, gpu, workspace=ws)

    gpu.lens.copy_(i32([10, 350, 3]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i, lens in enumerate([[10, 350, 3], [900, 1, 64], [1, 2, 3], [0, 0, 0], [899, 349, 63]]):
        gpu.lens.copy_(i32(lens))
        x.copy_(rows[i % 3])
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        eager = step()
        assert torch.equal(got, eager), f"replay {i}"
        (eager.float() * 2).sum().item()


def test_paged_far_pages(ctx):
    """Offsets past 2^31 elements in the pool, written and read."""
    page, h_kv, d = 1024, 8, 128
    pages = (1 << 31) // (page * h_kv * d) + 8   # 2056 pages, 4.3 GB each
    k, v = (torch.empty((pages, h_kv, page, d), dtype=F16, device=DEV) for _ in range(2))
    far = [pages - 1, 0, pages - 2]
    gen = torch.Generator().manual_seed(11)
    kk, vv, q = (normal(gen, (2100, h, d), F16).to(DEV) for h in (h_kv, h_kv, 16))
    far_c = PagedKV(k, v, i32([far]), i32([2100]))
    near = PagedKV.empty(3, h_kv, page, d, F16, i32([[1, 0, 2]]), i32([2100]))
    outs = []
    for c in (far_c, near):
        ctx.kv_append(c, kk, vv, i32([0, 2100]))
        outs.append(ctx.attention_paged(q[:1], c))
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(k[far[0]], near.k[1]) and torch.equal(v[far[2], :, :52], near.v[2, :, :52])


# --------------------------------------------------------------------- together


def block_reference(w, x, heads, seen, eps, tables=None):
    """The block over one sequence in f64 on the CPU, rotated by position."""
    p, d = w.p, x.shape[1] // heads
    f = lambda t: t.cpu().double()  # noqa: E731
    ln = lambda t, n: torch.nn.functional.layer_norm(t, t.shape[-1:], f(n[0]), f(n[1]), eps)  # noqa: E731
    qkv = ln(x, p.ln1) @ f(w.qkv_w).T + f(w.qkv_b)
    q, k, v = (t.unflatten(1, (heads, d)) for t in qkv.chunk(3, 1))
    q, k = ln(q, p.qn), ln(k, p.kn)
    if tables is not None:
        q, k = (torch.stack([torch.stack([R.norm_rope(t[i, h], None, tables, i, eps) for h in range(heads)])
                             for i in range(len(t))]) for t in (q, k))
    att, _ = R.attention(q, k, v, seen, 1 / math.sqrt(d))
    x = x + f(p.ls1) * (att.flatten(1) @ f(w.proj_w).T + f(p.proj_b))
    h = torch.nn.functional.gelu(ln(x, p.ln2) @ f(w.fc1_w).T + f(p.fc1_b))
    return x + f(p.ls2) * (h @ f(w.fc2_w).T + f(p.fc2_b))


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("dtype,dim,heads", [(F32, 256, 2), (F16, 256, 4)])
def test_prompt_then_steps(ctx, dtype, dim, heads, rope):
    """Prompts of different lengths, then single tokens, through a block: each
    row is the one of the whole sequence in 64 bits."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    w = BlockWeights.random(dim, 2 * dim, dim // heads, dtype, DEV, gen, ls_init=0.1)
    lens, steps, eps = [17, 1, 40], 4, 1e-6
    total = [n + steps for n in lens]
    x = [torch.randn((n, dim), generator=gen, device=DEV).to(dtype) for n in total]
    _, cache = make_cache(torch.Generator().manual_seed(4), total, heads, 16, dim // heads, dtype)
    cache.lens.copy_(i32(lens))
    tables = rope_tables(max(total), dim // heads) if rope else None
    up = tuple(t.to(DEV) for t in tables) if rope else None
    # the prompt's positions given, the steps' from the cache
    positions = i32([i for n in lens for i in range(n)]) if rope else None
    got = block_forward_cached(ctx, w, torch.cat([a[:n] for a, n in zip(x, lens)]), cache, heads,
                               offsets=i32(offsets_of(lens)), rope=up, positions=positions, eps=eps)
    rows = [list(t) for t in got.split(lens)]
    for i in range(steps):
        cache.lens += 1
        y = block_forward_cached(ctx, w, torch.stack([a[n + i] for a, n in zip(x, lens)]), cache, heads,
                                 rope=up, eps=eps)
        for r, t in zip(rows, y):
            r.append(t)
    # The f32 block's sums are of up to 512 terms; in f16 each of the eight
    # stored intermediates is rounded once (2^-11 of values of order 4), behind
    # factors of 0.1 (LayerScale) for all but the last two.
    tol = 512 * R.U32 * 8 if dtype == F32 else 2.0 ** -11 * 4 * (2 + 8 * 0.5)
    for a, n, r in zip(x, total, rows):
        ref = block_reference(w, a.cpu().double(), heads, R.seen_keys(n, n, 1), eps, tables)
        R.assert_within(torch.stack(r), ref, torch.full_like(ref, tol), f"length {n}")


def test_block_by_frames(ctx):
    """A prompt of frames through a block, masked by frames: the first frame is
    the plain block's over it alone."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    w = BlockWeights.random(256, 512, 64, F16, DEV, gen, ls_init=0.1)
    t, frames = 37, 3
    x = torch.randn((t * frames, 256), generator=gen, device=DEV).half()
    _, cache = make_cache(torch.Generator().manual_seed(4), [t * frames], 4, 16, 64, F16)
    got = block_forward_cached(ctx, w, x, cache, 4, offsets=i32([0, t * frames]), causal=t)
    alone = block_forward(ctx, w, x[:t], 1, t, 4)
    # both within the bound that test_prompt_then_steps derives for a block
    R.assert_within(got[:t], alone.cpu().double(), 2 * 2.0 ** -11 * 4 * (2 + 8 * 0.5), "first frame")
