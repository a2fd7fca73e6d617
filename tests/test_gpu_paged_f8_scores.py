"""Prompts over the 8-bit cache whose every score is -infinity: tokens that see keys, so that the definition has no
number for them, unlike those that see none."""
import pytest
import torch

from headshot_amd.paged import PagedKV8

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def i32(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("new", [2, 9, 40, 300])
@pytest.mark.parametrize("past", [0, 30, 2500])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_scores_of_minus_infinity(ctx, dtype, page, past, new):
    """Queries with an infinity where every key is negative, beside ordinary ones; the first key's page not there;
    tokens of a sequence that is shorter than its tokens."""
    gen = torch.Generator().manual_seed(7)
    h, d = 2, 64
    n = past + new
    width = -(-n // page)
    pages = 2 * width
    k, v = (torch.randn((pages, h, page, d), generator=gen) * 90 for _ in range(2))
    k[..., 5] = -1.0 - k[..., 5].abs()
    codes = [x.clamp(-448, 448).to(E4M3) for x in (k, v)]
    table = torch.arange(pages, dtype=torch.int32).reshape(2, width)
    table[0, 0] = -1
    short = new // 2  # keys of the second sequence: its first tokens see none
    scale = torch.full((pages, h), 120, dtype=torch.uint8).view(E8M0)
    cache = PagedKV8(*(t.to(DEV) for t in (*codes, scale, scale, table, i32([n, short], "cpu"))), dtype)
    q = torch.randn((2 * new, h, d), generator=gen)
    q[1::3, 1, 5] = float("inf")
    got = ctx.attention_paged_prompts(q.to(dtype).to(DEV), cache, i32([0, new, 2 * new])).unflatten(1, (h, d)).cpu()
    for s, (length, first) in enumerate(((n, page), (short, 0))):
        for i in range(new):
            row, seen = s * new + i, length - new + i + 1
            for head in range(h):
                out = got[row, head]
                what = f"sequence {s}, token {i}, head {head}"
                if seen <= first:
                    assert (out == 0).all(), what
                elif row % 3 == 1 and head == 1:
                    assert out.isnan().all(), what
                else:
                    assert out.isfinite().all(), what
    # as attention_paged has it
    single = ctx.attention_paged(q[[1, 1]].to(dtype).to(DEV), cache).unflatten(1, (h, d)).cpu()
    assert single[1, 1].isnan().all() and single[:, 0].isfinite().all()
    assert single[0, 1].isnan().all() if n > page else (single[0] == 0).all()
