"""The paged-cache operators in 64 bits on the CPU, loop by loop, and the error
that their arithmetic allows (shared by the tests; not a test itself)."""
import math

import torch

U32 = 2.0 ** -24  # half a step of f32, relative
HALF = {torch.float16: 2.0 ** -11, torch.float32: U32}   # a rounding to the type
TINY = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # the same among subnormals


def norm_rope(x, norm, table, row, eps):
    """One head vector (d,) f64; ``table`` = (sin, cos) or None."""
    if norm is not None:
        w, b = norm[0].double(), norm[1].double()
        x = (x - x.mean()) / (x.var(unbiased=False) + eps).sqrt() * w + b
    if table is not None and 0 <= row < table[0].shape[0]:
        sin, cos = table[0][row].double(), table[1][row].double()
        d = x.numel() // 2
        x = torch.cat([x[:d] * cos[:d] - x[d:] * sin[:d], x[d:] * cos[d:] + x[:d] * sin[d:]])
    return x


def append(k_cache, v_cache, page_table, lens, k, v, offsets, q, qn, kn, rope, positions, eps):
    """CPU tensors; q, k, v (n, heads, d). Returns f64 (q_out, k_out, k_cache,
    v_cache); rows of no sequence are NaN in q_out and k_out."""
    n_pages, h_kv, page, d = k_cache.shape
    kc, vc = k_cache.double().clone(), v_cache.double().clone()
    n = k.shape[0]
    k_out = torch.full((n, h_kv, d), math.nan, dtype=torch.float64)
    q_out = None if q is None else torch.full(q.shape, math.nan, dtype=torch.float64)
    for s in range(len(lens)):
        a, b = (s, s + 1) if offsets is None else (int(offsets[s]), int(offsets[s + 1]))
        for t in range(a, b):
            pos = int(lens[s]) - (b - t)
            row = pos if positions is None else int(positions[t])
            for h in range(h_kv):
                k_out[t, h] = norm_rope(k[t, h].double(), kn, rope, row, eps)
            if q is not None:
                for h in range(q.shape[1]):
                    q_out[t, h] = norm_rope(q[t, h].double(), qn, rope, row, eps)
            if 0 <= pos < page_table.shape[1] * page:
                at = int(page_table[s, pos // page])
                if 0 <= at < n_pages:
                    kc[at, :, pos % page], vc[at, :, pos % page] = k_out[t], v[t].double()
    return q_out, k_out, kc, vc


def append_bound(ref, x, dtype):
    """The f32 arithmetic of a norm and a rotation: sums over a head vector are
    at most 32 additions deep and the rest some 30 roundings, each of a value no
    larger than the largest normalised one (of x itself without a norm), then
    one rounding to the type."""
    size = ref.abs().nan_to_num().amax() + x.abs().amax().double() + 1
    return 64 * U32 * size + HALF[dtype] * ref.abs().nan_to_num() + TINY[dtype]


def attention(q, k, v, seen, scale):
    """q (nq, h, d), k, v (nk, h_kv, d) f64; query i sees keys below seen[i].
    Returns the result and sum(p |v|), both (nq, h, d)."""
    nq, h, d = q.shape
    group = h // k.shape[1]
    out, mag = torch.zeros(nq, h, d, dtype=torch.float64), torch.zeros(nq, h, d, dtype=torch.float64)
    for i in range(nq):
        m = int(seen[i])
        if m == 0:
            continue
        kk = k[:m].repeat_interleave(group, 1)
        vv = v[:m].repeat_interleave(group, 1)
        p = torch.softmax((q[i] * kk).sum(-1) * scale, 0)[..., None]
        out[i], mag[i] = (p * vv).sum(0), (p * vv.abs()).sum(0)
    return out, mag


def seen_keys(nq, nk, causal):
    at = torch.arange(nq) + (nk - nq)
    if causal == 0:
        return torch.full((nq,), nk)
    return ((torch.div(at, causal, rounding_mode="floor") + 1) * causal).clamp(0, nk)


def attention_bound(out, mag, q, k, v, seen, scale, dtype):
    """A score is a sum of d products (each off by U32 at most, and so is each
    partial sum, none above sum |q k|), then one multiplication; the exponent
    is taken of a difference of two such and is itself good to 4 roundings. So
    a weight is off by 2 (score error) + (2 |s| + 4) U32 relative, twice over
    (numerator and denominator), and the sums of nk terms by nk U32 each. In
    f16 a weight is rounded once for the product with V (2^-11 of itself, and
    2^-25 of the largest among subnormals) and the row sum may add the rounded
    ones pairwise in f16 (two levels), then the result is rounded. Query i's
    scores and values are those of its seen[i] keys. A score of which sum |q k|
    passes f32's range may be infinite, and its row is whatever that makes it:
    no bound."""
    q, k, v = q.double(), k.double(), v.double()
    nk, d = k.shape[0], k.shape[2]
    if nk == 0 or out.numel() == 0:
        return torch.full_like(out, TINY[dtype])
    kk = k.abs().repeat_interleave(q.shape[1] // k.shape[1], 1)
    visible = torch.arange(nk) < torch.as_tensor(seen)[:, None]
    size = ((q.abs().permute(1, 0, 2) @ kk.permute(1, 2, 0)) * visible).amax((0, 2))[:, None, None]
    over = size * max(1.0, abs(scale)) > torch.finfo(torch.float32).max / 2
    size = size * abs(scale)
    weight = 2 * (d + 4) * U32 * size + (2 * size + 4) * U32
    vmax = (v.abs().amax((1, 2)) * visible).amax(1)[:, None, None]
    bound = (2 * weight + 2 * nk * U32) * vmax + HALF[dtype] * out.abs() + TINY[dtype]
    if dtype == torch.float16:
        h = HALF[dtype]
        bound = bound + h * mag + 3 * h * out.abs() + nk * 2.0 ** -24 * vmax
    return torch.where(over, math.inf, bound)


def assert_within(got, ref, bound, what):
    got, ref, bound = got.detach().cpu().double(), ref.double(), torch.as_tensor(bound, dtype=torch.float64)
    bound = bound.expand_as(ref)
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} != {tuple(ref.shape)}"
    bad = ~((got - ref).abs() <= bound) & (bound != math.inf)
    if bad.any():
        worst = torch.where(bad, ((got - ref).abs() / bound).nan_to_num(math.inf), 0)
        i = int(worst.flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {worst.flatten()[i]:.3g} x "
                             f"bound, got {got.flatten()[i]} want {ref.flatten()[i]}")
