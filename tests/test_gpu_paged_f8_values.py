"""What a code of the 8-bit cache stands for: code times scale, as the rows' type holds it. Every code under every
scale, as a value; keys so small that f16 rounds them."""
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


def i32(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("new", [None, 1, 8, 70], ids=str)
@pytest.mark.parametrize("page", [2, 16])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_every_code_under_every_scale(ctx, dtype, page, new):
    """Sequences of one key: the result is its value, to the bit (a weight of 1 over a sum of 1)."""
    scales = list(range(10, 248))
    b, h, d = len(scales), 4, 64
    codes = torch.zeros((b, h, page, d), dtype=torch.uint8)
    codes[:, :, 0] = torch.arange(256, dtype=torch.uint8).reshape(h, d)
    kept = torch.tensor(scales, dtype=torch.uint8)[:, None].expand(b, h).contiguous()
    k = torch.zeros((b, h, page, d), dtype=torch.uint8).view(E4M3)
    cache = PagedKV8(*(t.to(DEV) for t in (k, codes.view(E4M3), torch.full((b, h), 127, dtype=torch.uint8).view(E8M0), kept.view(E8M0),
                                           torch.arange(b, dtype=torch.int32)[:, None], torch.ones(b, dtype=torch.int32))), dtype)
    want = (codes[:, :, 0].view(E4M3).double() * torch.exp2(kept.double() - 127)[..., None]).to(dtype)
    q = torch.ones((b * (new or 1), h, d), dtype=dtype, device=DEV)
    if new is None:
        got = ctx.attention_paged(q, cache)
    else:
        got = ctx.attention_paged_prompts(q, cache, i32([new * i for i in range(b + 1)]), causal=0)
    got = got.reshape(b, -1, h, d).cpu()
    for t in range(got.shape[1]):
        same = (got[:, t] == want) | (got[:, t].isnan() & want.isnan())
        assert same.all(), f"token {t}: {[(scales[i], hex(j * d + x)) for i, j, x in (~same).nonzero()[:8].tolist()]}"


@pytest.mark.parametrize("new", [None, [3, 1], [50, 70]], ids=str)
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_below_f16s_normal_range(ctx, d, page, new, monkeypatch):
    """Keys that the cache holds to 4 bits and f16 to fewer, or as 0, under a caller's scale that makes scores of
    order 1 of them: the scores are those of the f16 values, in 64 bits, and not those of the codes."""
    gen = torch.Generator().manual_seed(6)
    lens, h, h_kv = [130, 90], 4, 2
    need = [-(-n // page) for n in lens]
    pages, width = sum(need), max(need)
    table = i32([[*range(need[0])] + [0] * (width - need[0]), [*range(need[0], pages)] + [0] * (width - need[1])], "cpu")
    codes = [(torch.randn((pages, h_kv, page, d), generator=gen) * 90).clamp(-448, 448).to(E4M3) for _ in range(2)]
    tiny = torch.randint(127 - 34, 127 - 26, (pages, h_kv), generator=gen).to(torch.uint8)  # 90 2^-30: 1.4 steps of f16's
    parts = (*codes, tiny.view(E8M0), torch.full((pages, h_kv), 120, dtype=torch.uint8).view(E8M0), table, i32(lens, "cpu"))
    off = None if new is None else [0, new[0], sum(new)]
    n = len(lens) if new is None else sum(new)
    q, scale = torch.randn((n, h, d), generator=gen).half(), 2.0 ** 20
    gpu = PagedKV8(*(t.to(DEV) for t in parts), F16)
    if new is None:
        got = ctx.attention_paged(q.to(DEV), gpu, scale=scale)
    else:
        got = ctx.attention_paged_prompts(q.to(DEV), gpu, i32(off), scale=scale)
    got = got.unflatten(1, (h, d))
    codes_ref, _ = F.attend(q, parts, off, 1, scale, F16)
    gathered = F.gathered

    def as_f16(*args):
        out, there = gathered(*args)
        return out.half().double(), there

    monkeypatch.setattr(F, "gathered", as_f16)
    ref, bound = F.attend(q, parts, off, 1, scale, F16)
    R.assert_within(got, ref, bound, "f16 keys")
    assert ((codes_ref - ref).abs() > bound).any()  # (the two can be told apart)
    assert math.isfinite(float(got.float().abs().max()))
