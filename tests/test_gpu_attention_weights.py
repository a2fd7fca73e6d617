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
PATTERNS = [(lambda j: j % 64 < 32, 7.42), (lambda j: j % 16 == 0, 0.69268)]


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


# ---------------------------------------------------- one key with all the weight


def sink(d, nq, nk, h, h_kv, at, above, seed):
    """f16 rows of which key ``at`` scores ``above`` more than the others, whose
    scores lie within 1/4 of each other; its value is 0, theirs 500 to 1500.
    (Channel 0 makes that score: the queries' is 4, the key's above sqrt(d) / 4.)"""
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(nq, h, d, generator=gen).clamp(-2, 2) * 0.1
    k = torch.randn(nk, h_kv, d, generator=gen).clamp(-2, 2) * 0.1
    v = torch.rand(nk, h_kv, d, generator=gen) * 1000 + 500
    q[..., 0], k[..., 0] = 4, 0
    k[at], v[at] = 0, 0
    k[at, :, 0] = above * math.sqrt(d) / 4
    return q.half(), k.half(), v.half()


def sink_bound(q, k, ref, nk, scale, lost):
    """No value is negative, so a weight's relative error is the result's, twice
    (numerator and denominator). Of a weight: the score's (a sum of d products
    and a multiplication, each partial sum within the largest sum |q k|, and the
    exponential's four roundings; see attention_bound) and the rounding for the
    product, 2^-11. The row's sums add n 2^-24 each, and the result is rounded.
    Below 2^-14 a weight's rounding is no longer relative: 2^-25 of the unit, of
    which the largest weight is 2^lost at least."""
    d, group = q.shape[2], q.shape[1] // k.shape[1]
    size = ((q.double().abs().permute(1, 0, 2) @ k.double().abs().repeat_interleave(group, 1).permute(1, 2, 0)).amax()
            * scale).item()
    weight = 2 * (d + 4) * R.U32 * size + (2 * size + 4) * R.U32
    relative = 2 * weight + 2 * R.HALF[F16] + 2 * nk * R.U32 + R.HALF[F16]
    return relative * ref.abs() + nk * 2.0 ** -(25 + lost) * 1500 + R.TINY[F16]


def sink_reference(q, k, v, seen, scale):
    """In f64 on the GPU, head by head."""
    group = q.shape[1] // k.shape[1]
    q, k, v = (t.to(DEV).double() for t in (q, k, v))
    out = torch.zeros_like(q)
    hidden = torch.arange(k.shape[0], device=DEV) >= seen.to(DEV)[:, None]
    for i in range(q.shape[1]):
        s = (q[:, i] @ k[:, i // group].T.contiguous() * scale).masked_fill(hidden, -math.inf)
        out[:, i] = torch.softmax(s, -1) @ v[:, i // group]
    return out.cpu()


# The largest weight: 2^12 in attention_packed, unless a later score raised it.
@pytest.mark.parametrize("above", [14, 16, 17, 18])
@pytest.mark.parametrize("d,h,h_kv,nq,nk", [
    (64, 2, 1, 100, 300), (128, 2, 2, 70, 1100), (128, 4, 1, 5, 700), (64, 1, 1, 1900, 1900), (64, 2, 1, 9, 3000),
    (64, 64, 8, 2048, 2048), (128, 64, 8, 2048, 2048),
])
def test_packed_sink(ctx, d, h, h_kv, nq, nk, above):
    for at in (0, 63, nk // 2, nk - 1):
        q, k, v = sink(d, nq, nk, h, h_kv, at, above, d + nk + at)
        got = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v)), i32([0, nq]), i32([0, nk]), causal=0)
        ref = sink_reference(q, k, v, torch.full((nq,), nk), 1 / math.sqrt(d))
        R.assert_within(got.unflatten(1, (h, d)), ref, sink_bound(q, k, ref, nk, 1 / math.sqrt(d), 12),
                        f"key {at}, {above} above")


@pytest.mark.parametrize("d", [64, 128])
def test_packed_rows_apart(ctx, d):
    """A row is the same beside rows whose scores rise by steps along the keys,
    so that their wave's references move, and beside even ones."""
    gen = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(n, 2, d, generator=gen).half() for n in (90, 900, 900))
    k[..., 0] = (torch.arange(900) // 50)[:, None].half()  # what the first channel of a query adds
    q[..., 0] = 0
    args = i32([0, 90]), i32([0, 900])
    even = ctx.attention_packed(*(t.to(DEV) for t in (q, k, v)), *args, causal=0)
    for at in (0, 40, 63):
        steep = q.clone()
        steep[at, :, 0] = 4 * math.sqrt(d)
        got = ctx.attention_packed(*(t.to(DEV) for t in (steep, k, v)), *args, causal=0)
        rest = torch.arange(90) != at
        assert torch.equal(got[rest.to(DEV)], even[rest.to(DEV)]) and not torch.equal(got[at], even[at])


# --------------------------------------------------------- the same over the pages


def pages_of(k, v, page=16):
    """A cache of one sequence: its pages, the last filled up with zeros."""
    n, h_kv, d = k.shape
    count = -(-n // page)
    rows = torch.zeros(2, count * page, h_kv, d, dtype=k.dtype)
    rows[0, :n], rows[1, :n] = k, v
    rows = rows.unflatten(1, (count, page)).transpose(2, 3).contiguous().to(DEV)
    return PagedKV(rows[0], rows[1], i32([list(range(count))]), i32([n]))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,h_kv,nk", [(1, 1, 100), (8, 2, 1000), (20, 1, 333), (4, 4, 2000)])
def test_paged_constant_values(ctx, d, h, h_kv, nk):
    """As test_packed_constant_values, the weights the same to 2^-22."""
    for page in (4, 16):
        for pattern, scale in PATTERNS:
            q, k, v = two_levels(pattern, d, 1, nk, h, h_kv)
            got = ctx.attention_paged(q.to(DEV), pages_of(k, v, page), scale=scale).float()
            assert (got == 1).all(), f"page {page}, scale {scale}: {(got - 1).abs().max()} off"


# The largest weight: 2^15 in attention_paged.
@pytest.mark.parametrize("above", [14, 16, 17, 18])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,h_kv,nk", [(1, 1, 100), (1, 1, 32), (8, 2, 700), (20, 1, 128), (2, 2, 3000)])
def test_paged_sink(ctx, d, h, h_kv, nk, above):
    for at in (0, nk // 2, nk - 1):
        q, k, v = sink(d, 1, nk, h, h_kv, at, above, d + nk + at)
        got = ctx.attention_paged(q.to(DEV), pages_of(k, v))
        ref = sink_reference(q, k, v, torch.full((1,), nk), 1 / math.sqrt(d))
        R.assert_within(got.unflatten(1, (h, d)), ref, sink_bound(q, k, ref, nk, 1 / math.sqrt(d), 15),
                        f"key {at}, {above} above")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,h_kv,nk", [(8, 8, 2), (8, 2, 20), (20, 1, 333), (4, 4, 3000)])
def test_paged_f16_weights(ctx, d, h, h_kv, nk):
    """f16 results are off by their own rounding and what f32 weights would be
    off: scores as in attention_bound, small ones here; 2^-22 of a weight, twice;
    and sums of chains of up to 128 keys a wave, its pieces and waves behind."""
    gen = torch.Generator().manual_seed(d + nk)
    q = (torch.randn(1, h, d, generator=gen) * 0.05).half()
    k, v = (torch.randn(nk, h_kv, d, generator=gen).half() for _ in range(2))
    scale = 1 / math.sqrt(d)
    ref, mag = R.attention(q.double(), k.double(), v.double(), [nk], scale)
    size = (q.double().abs().transpose(0, 1) @ k.double().abs().repeat_interleave(h // h_kv, 1).permute(1, 2, 0)).amax()
    weight = 2 * (d + 4) * R.U32 * size * scale + (2 * size * scale + 4) * R.U32 + 2.0 ** -22
    bound = (2 * weight + 2 * min(nk, 200) * R.U32) * mag + R.HALF[F16] * ref.abs() + R.TINY[F16]
    got = ctx.attention_paged(q.to(DEV), pages_of(k, v))
    R.assert_within(got.unflatten(1, (h, d)), ref, bound, f"{nk} keys")


@pytest.mark.parametrize("d", [64, 128])
def test_paged_infinity_beside(ctx, d):
    """An infinity among the values is its own channel's alone, whatever bits its
    key's weight has; the others stay within a weight's leading 11 bits."""
    gen = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(n, 2, d, generator=gen).half() for n in (1, 700, 700))
    plain = v.clone()
    for j, x in ((3, math.inf), (40, -math.inf), (699, math.inf)):
        v[j, :, j % 7] = x
        plain[j, :, j % 7] = 0
    ref, mag = R.attention(q.double(), k.double(), plain.double(), [700], 1 / math.sqrt(d))
    got = ctx.attention_paged(q.to(DEV), pages_of(k, v)).unflatten(1, (2, d)).cpu()
    assert (got[..., 3] == math.inf).all() and (got[..., 40 % 7] == -math.inf).all() and (got[..., 699 % 7] == math.inf).all()
    rest = [c for c in range(d) if c not in (3, 40 % 7, 699 % 7)]
    bound = R.attention_bound(ref, mag, q, k, plain, [700], 1 / math.sqrt(d), F16)
    R.assert_within(got[..., rest], ref[..., rest], bound[..., rest], "the other channels")


# ------------------------------------------------------------------ enormous scores


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("d,h,h_kv,nk", [(64, 2, 1, 300), (128, 2, 2, 300), (64, 1, 1, 2100), (128, 1, 1, 2100)])
def test_enormous_scores(ctx, d, h, h_kv, nk, sign):
    """Scores up to 2^29, at each power of two: keys 3, 100 and nk - 1 share the
    largest, others lie at half of it and at 0 (sign 1), or at the double and more
    below (-1), thousands of powers of two away in weight. The result is the mean
    of three values whatever an exponent's rounding is."""
    at = [3, 100, nk - 1]
    for bits in range(12, 30):
        a, b = bits - bits // 2, bits // 2
        q, k = torch.zeros(5, h, d), torch.zeros(nk, h_kv, d)
        q[..., 0] = 2.0 ** a
        k[..., 0] = (torch.arange(nk) % 2 / 2 if sign > 0 else -2.0 - torch.arange(nk) % 2)[:, None] * 2.0 ** b
        k[at, :, 0] = sign * 2.0 ** b
        v = torch.randn(nk, h_kv, d, generator=torch.Generator().manual_seed(bits)).half()
        ref = v[at].double().mean(0).repeat_interleave(h // h_kv, 0)
        bound = (R.HALF[F16] + 8 * R.U32) * ref.abs() + 8 * R.U32 * v[at].double().abs().mean(0).max() + R.TINY[F16]
        got = ctx.attention_packed(*(t.half().to(DEV) for t in (q, k, v)), i32([0, 5]), i32([0, nk]), causal=0, scale=1.0)
        R.assert_within(got.unflatten(1, (h, d)), ref.expand(5, h, d), bound.expand(5, h, d), f"packed, 2^{bits}")
        got = ctx.attention_paged(q[:1].half().to(DEV), pages_of(k.half(), v), scale=1.0)
        R.assert_within(got.unflatten(1, (h, d)), ref[None], bound[None], f"paged, 2^{bits}")
