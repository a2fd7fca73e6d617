"""What packed and paged attention make of their weights on the GPU: rows of
which one key takes nearly all of the weight, and sums that numerator and
denominator share."""
import math

import pytest
import torch

import paged_reference as R
from headshot_amd.paged import PagedKV

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ------------------------------------------------------- values that are all one


# (keys that score 0, the others -1; scale). Weights of one, and others of which
# f16 makes something else: 1 + e^-7.42 = 1 + 0.61 x 2^-10, which rounds up to 1 +
# 2^-10, and e^-0.69268 = 1/2 + 0.95 x 2^-12, which rounds down to 1/2.
PATTERNS = [(lambda j: j % 64 < 32, 7.42), (lambda j: j == 0, 0.69268)]


def two_levels(pattern, d, nq, nk, h, h_kv):
    """f16 rows of such scores, and values of one."""
    q, k = torch.zeros(nq, h, d), torch.zeros(nk, h_kv, d)
    q[..., 0] = 1
    k[..., 0] = torch.where(pattern(torch.arange(nk)), 0.0, -1.0)[:, None]
    return q.half(), k.half(), torch.ones(nk, h_kv, d).half()


# A row's numerator and denominator are sums of the same weights, whatever each
# was rounded to: of n terms in f32, they differ by at most 2 n 2^-24 relative,
# and the quotient by two roundings more. For n up to 2000 that is 2.4e-4, less
# than 2^-12, half the step of f16 below one (2^-11 is that above): the result
# rounds to one.
@pytest.mark.parametrize("d,h,h_kv,nq,nk", [
    (64, 2, 1, 200, 200), (128, 2, 2, 150, 1990), (64, 4, 4, 7, 1500), (128, 8, 2, 40, 2000), (64, 8, 1, 16, 64),
    (64, 1, 1, 1900, 1900),       # split over the keys
    (64, 64, 8, 2048, 2000), (128, 64, 8, 2048, 2000),  # eight waves
])
def test_packed_constant_values(ctx, d, h, h_kv, nq, nk):
    for pattern, scale in PATTERNS:
        q, k, v = two_levels(pattern, d, nq, nk, h, h_kv)
        for causal in (0, 1):
            got = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v)), i32([0, nq]), i32([0, nk]), causal=causal,
                                       scale=scale)
            got = got[(R.seen_keys(nq, nk, causal) > 0).to(DEV)].float()
            assert (got == 1).all(), f"scale {scale}, causal {causal}: {(got - 1).abs().max()} off"
