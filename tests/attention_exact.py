"""Attention that shows each key by itself, and a bound close enough to show a lost
one (shared by the tests; not a test itself)."""
import math

import torch

import paged_reference as R


def signs(n, heads, d, seed):
    """Values of 1 and -1, (n, heads, d) f32 on the CPU. Under scale 0 all keys
    weigh the same and a result is the mean of what its query sees: a key that is
    lost, doubled or another's moves every channel, or every other one, by 1 / n
    of about 1 / sqrt(n), 2^-11 of which (f16) it exceeds up to 2^20 keys."""
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, 2, (n, heads, d), generator=gen).float() * 2 - 1


def means(v, seen, group):
    """Those results in f64: (queries, heads * group, d), zeros where seen is 0.
    ``v`` (keys, heads, d); query i sees the first seen[i]."""
    sums = torch.cat([torch.zeros(1, *v.shape[1:], dtype=torch.float64), v.double().cumsum(0)])
    seen = torch.as_tensor(seen).long()
    return (sums[seen] / seen.clamp(min=1)[:, None, None]).repeat_interleave(group, 1)


def means_bound(ref, dtype):
    """Weights are a power of two, and sums of up to 2^24 ones exact in f32 in any
    order. What is left are the division, as a reciprocal and a product, and the
    result's rounding."""
    return (4 * R.U32 + R.HALF[dtype]) * ref.abs() + R.TINY[dtype]


def close_bound(out, mag, q, k, seen, scale, dtype, depth, weight=None):
    """As attention_bound, but that what is off in a weight is taken of sum(p |v|)
    (``mag``), and what is off in the sums of their ``depth``: additions one
    behind the other, in a wave and in the joins. ``weight``: the rounding of f16's
    weights (attention_packed 2^-11, attention_paged 2^-22)."""
    q, k = q.double(), k.double()
    nk, d = k.shape[0], k.shape[2]
    kk = k.abs().repeat_interleave(q.shape[1] // k.shape[1], 1)
    visible = torch.arange(nk) < torch.as_tensor(seen)[:, None]
    size = ((q.abs().permute(1, 0, 2) @ kk.permute(1, 2, 0)) * visible).amax((0, 2))[:, None, None] * abs(scale)
    off = 2 * (d + 4) * R.U32 * size + (2 * size + 4) * R.U32 + depth * R.U32
    if dtype == torch.float16:
        off = off + weight
    return 2 * off * mag + R.HALF[dtype] * out.abs() + R.TINY[dtype]


def attention(q, k, v, seen, scale):
    """R.attention of many keys: f64, head by head."""
    group = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    hidden = torch.arange(k.shape[0]) >= torch.as_tensor(seen)[:, None]
    for i in range(q.shape[1]):
        p = torch.softmax((q[:, i] @ k[:, i // group].T * scale).masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
        out[:, i], mag[:, i] = p @ v[:, i // group], p @ v[:, i // group].abs()
    return out, mag
