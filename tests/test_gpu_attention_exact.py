"""Packed and paged attention on the GPU where each key shows: all keys weighing
the same, over piece and tile boundaries, and ordinary scores under a close
bound (attention_exact.py)."""
import math

import pytest
import torch

import attention_exact as X
import paged_reference as R
from headshot_amd.paged import PagedKV

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
DTYPES = [F16, F32]


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def offsets_of(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ------------------------------------------------------------- attention_packed


def packed_means(ctx, dtype, d, h, h_kv, nq, nk, causal):
    print(f"[packed means {dtype} d={d} {h}/{h_kv} {nq} over {nk} causal={causal}]", flush=True)
    qo, ko = offsets_of(nq), offsets_of(nk)
    gen = torch.Generator().manual_seed(d + sum(nk))
    q, k = (torch.randn(n, x, d, generator=gen).to(dtype) for n, x in ((qo[-1], h), (ko[-1], h_kv)))
    v = X.signs(ko[-1], h_kv, d, sum(nq) + causal)
    got = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v.to(dtype))), i32(qo), i32(ko), causal=causal, scale=0.0)
    got = got.unflatten(1, (h, d)).cpu()
    for s in range(len(nq)):
        seen = R.seen_keys(nq[s], nk[s], causal)
        ref = X.means(v[ko[s]:ko[s + 1]], seen, h // h_kv)
        R.assert_within(got[qo[s]:qo[s + 1]], ref, X.means_bound(ref, dtype), f"sequence {s}")


@pytest.mark.parametrize("causal", [0, 1, 137])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_means(ctx, dtype, d, causal):
    for h, h_kv, nq, nk in [
        (2, 1, [1, 0, 17, 64, 129], [1, 5, 63, 64, 131]),
        (1, 1, [2049], [2049]),                         # split
        (2, 2, [300, 7], [4200, 2111]),                 # split
        (8, 2, [3, 40], [9001, 1500]),                  # split, heads together in f16
        (1, 1, [1], [20000]), (4, 1, [16], [20001]),    # split
        (16, 4, [1300, 900, 130], [1300, 900, 130]),    # f32: tiles
        (32, 8, [4097], [4097]),                        # f16: eight waves
    ]:
        packed_means(ctx, dtype, d, h, h_kv, nq, nk, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_piece_boundaries(ctx, dtype, d):
    """Key counts around multiples of the 256 keys that a piece has at least."""
    for nk in (2047, 2048, 2049, 2303, 2304, 2305, 2560, 2815, 4097):
        size = ctx.attention_packed_workspace(dtype, 20, nk, 1, 2, 1, d, 1)
        assert size > 0
        packed_means(ctx, dtype, d, 2, 1, [20], [nk], 1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_split_close(ctx, dtype, d):
    """Pieces, joined: a wave of a piece sums up to 16 units of 64 keys one behind
    the other here, in products of up to 16 keys, and up to 100 pieces follow."""
    for h, h_kv, nq, nk in [(1, 1, 5, 20000), (4, 2, 33, 9001), (2, 1, 200, 4200), (8, 2, 1, 2048)]:
        print(f"[packed close {dtype} d={d} {h}/{h_kv} {nq} over {nk}]", flush=True)
        assert ctx.attention_packed_workspace(dtype, nq, nk, 1, h, h_kv, d, 1) > 0
        gen = torch.Generator().manual_seed(nk + d)
        q, k, v = (torch.randn(n, x, d, generator=gen).to(dtype) for n, x in ((nq, h), (nk, h_kv), (nk, h_kv)))
        got = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v)), i32([0, nq]), i32([0, nk]), causal=1)
        seen = R.seen_keys(nq, nk, 1)
        ref, mag = X.attention(q, k, v, seen, 1 / math.sqrt(d))
        bound = X.close_bound(ref, mag, q, k, seen, 1 / math.sqrt(d), dtype, 16 * 64 + 100, 2.0 ** -11)
        R.assert_within(got.unflatten(1, (h, d)), ref, bound, f"{nq} over {nk}")


# -------------------------------------------------------------- attention_paged


def pages_of(k, v, lens, page, seed):
    """A cache of the sequences' rows (one after the other), its pages in no order;
    what no sequence reaches holds NaN."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    kc, vc = (torch.full((sum(need) + 2, page, *k.shape[1:]), math.nan, dtype=k.dtype) for _ in range(2))
    table = torch.zeros(len(lens), max(need) + 1, dtype=torch.int32)
    at = row = 0
    for s, n in enumerate(lens):
        mine = order[at:at + need[s]]
        table[s, :need[s]] = torch.tensor(mine, dtype=torch.int32)
        pos = torch.arange(n)
        where = torch.tensor(mine, dtype=torch.long)[pos // page]
        kc[where, pos % page], vc[where, pos % page] = k[row:row + n], v[row:row + n]
        at, row = at + need[s], row + n
    return PagedKV(*(t.transpose(1, 2).contiguous().to(DEV) for t in (kc, vc)), table.to(DEV), i32(lens))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_means(ctx, dtype, d):
    for h, h_kv, page, lens in [
        (1, 1, 16, [1, 0, 15, 17, 63, 64, 65, 127, 128, 129, 255, 257]),
        (1, 1, 32, [20000]), (8, 2, 16, [9001, 1, 0, 4500]), (2, 2, 64, [1] * 70 + [7777] + [3] * 9),
        (16, 16, 16, [2047, 2048, 2049, 511, 513]), (20, 1, 8, [4200, 33]), (40, 2, 128, [1025, 2303]),
        (4, 1, 1, [700, 66]), (1, 1, 1024, [131071]),
    ]:
        print(f"[paged means {dtype} d={d} {h}/{h_kv} page={page} {len(lens)} to {max(lens)}]", flush=True)
        gen = torch.Generator().manual_seed(d + page)
        q, k = (torch.randn(n, x, d, generator=gen).to(dtype) for n, x in ((len(lens), h), (sum(lens), h_kv)))
        v = X.signs(sum(lens), h_kv, d, sum(lens))
        got = ctx.attention_paged(q.to(DEV), pages_of(k, v.to(dtype), lens, page, d), scale=0.0)
        ref = torch.cat([X.means(t, [len(t)], h // h_kv) for t in v.split(lens)])
        R.assert_within(got.unflatten(1, (h, d)), ref, X.means_bound(ref, dtype), "paged")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_close(ctx, dtype, d):
    """As few sequences as here are cut into pieces of one unit, in which a wave
    takes 32 keys (16 in f32); at most 40 joins follow, of 32 pieces in turn."""
    for h, h_kv, page, lens in [(1, 1, 32, [20000]), (8, 2, 16, [9001, 1, 4500]), (3, 3, 8, [2048, 77]), (20, 1, 16, [4200])]:
        print(f"[paged close {dtype} d={d} {h}/{h_kv} {lens}]", flush=True)
        gen = torch.Generator().manual_seed(d + h)
        q, k, v = (torch.randn(n, x, d, generator=gen).to(dtype) for n, x in
                   ((len(lens), h), (sum(lens), h_kv), (sum(lens), h_kv)))
        got = ctx.attention_paged(q.to(DEV), pages_of(k, v, lens, page, d)).unflatten(1, (h, d)).cpu()
        for s, (a, n) in enumerate(zip(offsets_of(lens), lens)):
            args = q[s:s + 1], k[a:a + n], v[a:a + n], [n], 1 / math.sqrt(d)
            ref, mag = X.attention(*args)
            bound = X.close_bound(ref, mag, q[s:s + 1], k[a:a + n], [n], 1 / math.sqrt(d), dtype, 200, 2.0 ** -22)
            R.assert_within(got[s:s + 1], ref, bound, f"sequence {s}")
