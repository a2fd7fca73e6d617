"""The workspace of prompts over the 8-bit cache: what it comes to at most, and that calls that it is not for are
right without one."""
import math

import pytest
import torch

import paged_reference as R
from headshot_amd import _lib
from headshot_amd.paged import PagedKV8

L = _lib.load()
F16, F32 = _lib.HS_F16, _lib.HS_F32
MOST = 245 << 20  # the largest that the plan allows: 7 places' tiles of 256 rows of 64 channels, 512 places


def size(dt, n, b, h, h_kv, d, page=16, max_pages=4096, causal=1):
    return L.hs_attention_prompts_f8_workspace(dt, n, b, h, h_kv, d, page, max_pages, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", [F16, F32])
def test_workspace_is_bounded(dt, d):
    some = 0
    for h_kv in (1, 2, 3, 8, 16, 40, 100, 256, 257, 384, 512, 700, 1024, 4096):
        for group in (1, 2, 8):
            h = h_kv * group
            if h > 4096:
                continue
            for b in (1, 2, 7, 40, 300, 4000):
                for each in (1, 3, 32, 130, 600, 2100):
                    n = b * each
                    if n * h < 1 << 30:
                        for page in (8, 16):
                            bytes_ = size(dt, n, b, h, h_kv, d, page)
                            some += bytes_ > 0
                            assert bytes_ <= MOST, (n, b, h, h_kv, d, page, bytes_ / 2 ** 20)
    assert some > 100


def test_no_workspace_where_heads_fill_the_chip():
    """(256 CUs are what a machine without one counts as; a card has no more.)"""
    for h_kv in (512, 1024, 4096):
        for n in (1, 200, 380):
            assert size(F16, n, 1, h_kv, h_kv, 128) == 0
    assert size(F16, 200, 1, 8, 8, 128) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_many_key_heads(ctx, dtype):
    """As many key heads as fill the chip: whole keys, no workspace, the definition's result in 64 bits."""
    dev, d, page, n, past, h = "cuda:0", 128, 16, 130, 700, 520
    gen = torch.Generator(device=dev).manual_seed(1)
    pages = -(-(n + past) // page)
    codes = [(torch.randn((pages, h, page, d), generator=gen, device=dev) * 90).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.randint(119, 122, (pages, h), generator=gen, device=dev).to(torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32)[None].to(dev)
    cache = PagedKV8(*codes, *scales, table, torch.tensor([n + past], dtype=torch.int32, device=dev), dtype)
    assert ctx.attention_paged_prompts_workspace(cache, n, h) == 0
    q = torch.randn((n, h, d), generator=gen, device=dev).to(dtype)
    got = ctx.attention_paged_prompts(q, cache, torch.tensor([0, n], dtype=torch.int32, device=dev)).unflatten(1, (h, d))
    k, v = ((c.double() * s.double()[..., None, None])[table[0].long()].transpose(1, 2).flatten(0, 1)[:n + past] for c, s in zip(codes, scales))
    hidden = torch.arange(n + past, device=dev) > (torch.arange(n, device=dev) + past)[:, None]
    seen = R.seen_keys(n, n + past, 1)
    for i in range(h):
        s = (q[:, i].double() @ k[:, i].T) / math.sqrt(d)
        p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
        one = [x[:, None].cpu() for x in (p @ v[:, i], p @ v[:, i].abs(), q[:, i], k[:, i], v[:, i])]
        bound = R.attention_bound(*one, seen, 1 / math.sqrt(d), dtype)
        R.assert_within(got[:, i:i + 1], one[0], bound, f"head {i}")
