"""That the bounds of attention_exact.py show a lost, doubled or misplaced key."""
import math

import pytest
import torch

import attention_exact as X
import paged_reference as R

F16, F32 = torch.float16, torch.float32


def outside(got, ref, bound):
    with pytest.raises(AssertionError, match="outside"):
        R.assert_within(got, ref, bound, "changed")


def test_means_are_the_definition():
    gen = torch.Generator().manual_seed(0)
    q, k = (torch.randn(n, h, 64, generator=gen) for n, h in ((5, 4), (9, 2)))
    v = X.signs(9, 2, 64, 1)
    seen = [0, 3, 9, 1, 8]
    ref, _ = R.attention(q.double(), k.double(), v.double(), seen, 0.0)
    R.assert_within(X.means(v, seen, 2), ref, 1e-15, "means")
    out, mag = X.attention(q, k, v, seen, 0.3)
    ref, ref_mag = R.attention(q.double(), k.double(), v.double(), seen, 0.3)
    R.assert_within(out, ref, 1e-14, "attention")
    R.assert_within(mag, ref_mag, 1e-14, "sum(p |v|)")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 17, 2048, 20000, 131072])
def test_means_show_each_key(n, dtype):
    v = X.signs(n, 1, 64, n)
    ref = X.means(v, [n], 1)
    bound = X.means_bound(ref, dtype)
    R.assert_within(ref.to(dtype), ref, bound, "itself")
    total = v.double().sum(0)
    for j in {0, n // 3, n - 1}:
        outside((total + v[j]) / (n + 1) if n > 1 else 2 * total, ref[0], bound[0])  # doubled
        outside((total - v[j]) / max(n - 1, 1), ref[0], bound[0])                    # lost
        outside((total - v[j]) / n, ref[0], bound[0])                                # lost in the product alone
        if n > 1:
            outside((total - v[j] + v[j - 1]) / n, ref[0], bound[0])                 # another's instead


@pytest.mark.parametrize("dtype,weight", [(F32, None), (F16, 2.0 ** -11), (F16, 2.0 ** -22)])
@pytest.mark.parametrize("nk", [2048, 9001, 20000])
def test_close_bound_shows_a_block(nk, dtype, weight):
    """16 keys lost or doubled, for inputs as the GPU tests have them."""
    d, scale = 64, 1 / math.sqrt(64)
    gen = torch.Generator().manual_seed(nk)
    q, k, v = (torch.randn(n, 1, d, generator=gen).to(dtype) for n in (8, nk, nk))
    seen = torch.full((8,), nk)
    ref, mag = X.attention(q, k, v, seen, scale)
    bound = X.close_bound(ref, mag, q, k, seen, scale, dtype, 200, weight)
    for at in (0, nk // 2 // 16 * 16, nk - 16):
        for keep in (torch.cat([torch.arange(at), torch.arange(at + 16, nk)]),
                     torch.cat([torch.arange(nk), torch.arange(at, at + 16)])):
            got, _ = X.attention(q, k[keep], v[keep], torch.full((8,), len(keep)), scale)
            outside(got, ref, bound)
