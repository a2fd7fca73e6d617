"""The operators over a cache held in 8 bits, in 64 bits on the CPU, loop by loop, and the pages' hand-out in
whole numbers, with the error that their arithmetic allows (shared by the tests; not a test itself)."""
import math

import torch

import paged_reference as R

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
HELD = {torch.float16: 240.0 * 2.0 ** 8, torch.float32: 240.0 * 2.0 ** 120}
LEAST = -117
HALF_CODE = 2.0 ** -4   # a rounding to 4 significant bits, relative
TINY_CODE = 2.0 ** -10  # the same among a code's subnormals, times the scale
LONGEST = 1 << 30


def round_e4m3(x):
    """f64 to 4 significant bits, fewer below 2^-6, ties to even; what is no number stays none."""
    size = x.abs().nan_to_num(posinf=1.0)
    step = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, math.nan)


def exponent_for(most: float) -> int:
    """The least e >= -117 with most <= 448 2^e."""
    if most == 0:
        return LEAST
    part, e = math.frexp(most)
    return max(LEAST, e - 9 if part <= 0.875 else e - 8)


def exponents(scale):
    return scale.view(torch.uint8).int() - 127


def values(codes, scale):
    """(n_pages, heads, page, d) f64."""
    return codes.double() * scale.double()[..., None, None]


def blocks(page_table, lens, offsets, n_pages, page):
    """(page, first row, tokens) of every page that a call's tokens reach, in order."""
    out = []
    for s in range(len(lens)):
        a, b = (s, s + 1) if offsets is None else (int(offsets[s]), int(offsets[s + 1]))
        found = {}
        for t in range(a, b):
            pos = int(lens[s]) - (b - t)
            if 0 <= pos < page_table.shape[1] * page:
                at = int(page_table[s, pos // page])
                if 0 <= at < n_pages:
                    found.setdefault(at, (pos % page, []))[1].append(t)
        out += [(at, first, tokens) for at, (first, tokens) in found.items()]
    return out


def check_append(what, before, after, page_table, lens, offsets, x, dtype, error):
    """``before``, ``after`` = (codes, scale) of the call, CPU; ``x`` (n, heads, d) the exact f64 values of its
    tokens, which the f32 arithmetic has to ``error`` (0: exactly). Codes and scales are what the definition
    says: exactly with error 0; else a scale is one that a magnitude that close gives, and a value off by the
    arithmetic's error and half a step of the code."""
    codes, scale = after
    n_pages, heads, page, d = codes.shape
    same = torch.ones(codes.shape[:3], dtype=torch.bool)
    old, new = exponents(before[1]), exponents(scale)
    touched = torch.zeros(n_pages, dtype=torch.bool)
    for at, first, tokens in blocks(page_table, lens, offsets, n_pages, page):
        touched[at] = True
        rows = slice(first, first + len(tokens))
        same[at, :, rows] = False
        for h in range(heads):
            v = x[tokens, h].double()
            finite = v[v.isfinite()].abs().clamp_max(HELD[dtype])
            most = finite.max().item() if finite.numel() else 0.0
            kept = int(old[at, h]) if first > 0 else LEAST
            allowed = {max(kept, exponent_for(min(m, HELD[dtype]))) for m in (most, max(most - error, 0.0), most + error)}
            e = int(new[at, h])
            assert e in allowed, f"{what}: scale 2^{e} of page {at}, head {h}, allowed {allowed}, most {most}"
            if first > 0:  # the older rows follow
                want = round_e4m3(before[0][at, h, :first].double() * 2.0 ** (int(old[at, h]) - e))
                got = codes[at, h, :first].double()
                assert torch.equal(got.nan_to_num(1e6), want.nan_to_num(1e6)), f"{what}: older codes of page {at}, head {h}"
                same[at, h, :first] = False
            got = codes[at, h, rows].double()
            held = torch.where(v.isfinite(), v.clamp(-HELD[dtype], HELD[dtype]), math.nan)
            if error == 0:
                want = round_e4m3(held / 2.0 ** e)
                assert torch.equal(got.nan_to_num(1e6), want.nan_to_num(1e6)), f"{what}: codes of page {at}, head {h}"
            else:
                bound = error + HALF_CODE * (held.abs() + error) + TINY_CODE * 2.0 ** e
                R.assert_within(got * 2.0 ** e, held, bound, f"{what}, page {at}, head {h}")
    assert torch.equal(codes.view(torch.uint8)[same], before[0].view(torch.uint8)[same]), f"{what}: rows of no new token"
    assert torch.equal(new[~touched], old[~touched]), f"{what}: scales of no new token"


def transform_error(ref, x):
    """What the f32 arithmetic of a norm and a rotation may be off by (paged_reference.append_bound, which
    derives it, without the rounding to a type)."""
    return 64 * R.U32 * float(ref.abs().nan_to_num(posinf=0.0).amax() + x.double().abs().nan_to_num(posinf=0.0).amax() + 1)


def transformed(x, norm, table, lens, offsets, positions, eps):
    """(n, heads, d) f64 rows after the norm and the rotation, by key number or position; rows of no sequence 0."""
    out = torch.zeros(x.shape, dtype=torch.float64)
    for s in range(len(lens)):
        a, b = (s, s + 1) if offsets is None else (int(offsets[s]), int(offsets[s + 1]))
        for t in range(a, b):
            pos = int(lens[s]) - (b - t)
            for h in range(x.shape[1]):
                out[t, h] = R.norm_rope(x[t, h].double(), norm, table, pos if positions is None else int(positions[t]), eps)
    return out


def gathered(codes, scale, page_table, length, s):
    """Sequence s's keys (length, heads, d) f64, and which of them there are."""
    n_pages, heads, page, d = codes.shape
    out, there = torch.zeros(length, heads, d, dtype=torch.float64), torch.zeros(length, dtype=torch.bool)
    for p in range(length):
        at = int(page_table[s, p // page])
        if 0 <= at < n_pages:
            out[p] = codes[at, :, p % page].double() * scale[at].double()[:, None]
            there[p] = True
    return out, there


def attend(q, cache, offsets, causal, scale, dtype):
    """``cache`` = (k, v, k_scale, v_scale, page_table, lens), CPU; q (n, heads, d) of ``dtype``. The result and
    the bound of paged_reference, (n, heads, d) each; rows of no sequence are NaN, with no bound."""
    k, v, ks, vs, table, lens = cache
    page = k.shape[2]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    bound = torch.full(q.shape, math.inf, dtype=torch.float64)
    for s in range(len(lens)):
        a, b = (s, s + 1) if offsets is None else (int(offsets[s]), int(offsets[s + 1]))
        if a == b:
            continue
        length = max(int(lens[s]), 0)
        held = min(length, table.shape[1] * page)
        kk, there = gathered(k, ks, table, held, s)
        vv, _ = gathered(v, vs, table, held, s)
        for t in range(a, b):
            at = length - (b - t)
            if causal == 0 or offsets is None:
                seen = held
            else:
                seen = 0 if at < 0 else min((at // causal + 1) * causal, held)
            use = there[:seen]
            kt, vt = kk[:seen][use], vv[:seen][use]
            o, mag = R.attention(q[t:t + 1].double(), kt, vt, [len(kt)], scale)
            out[t] = o[0]
            # NaN reaches the channels (of a value) and heads (of a key) that are NaN in the result themselves;
            # the others' bound is that of the finite values
            fin = [x.nan_to_num(0.0) for x in (o, mag, q[t:t + 1], kt, vt)]
            bound[t] = R.attention_bound(*fin, [len(kt)], scale, dtype)[0]
    return out, bound


# ------------------------------------------------------------------ pages


class Pages:
    """plan_pages in whole numbers."""

    def __init__(self, sequences, max_pages, n_pages, page):
        self.table = [[-1] * max_pages for _ in range(sequences)]
        self.lens = [0] * sequences
        self.free = list(range(n_pages))
        self.width, self.page, self.n_pages = max_pages, page, n_pages
        self.missing = 0

    def plan(self, counts):
        """Returns offsets, positions, slots."""
        ready, back, offsets, positions, slots = list(self.free), [], [0], [], []
        taken = self.missing = 0
        for s, c in enumerate(counts):
            row, old = self.table[s], self.lens[s]
            new = min(max(old + c, 0), LONGEST)
            have, want = -(-old // self.page), -(-new // self.page)
            whole = have == 0 or have > self.width or self.width == 0 or row[have - 1] >= 0
            for e in range(have, want):
                if e < self.width and whole and taken < len(ready):
                    row[e] = ready[taken]
                    taken += 1
                else:
                    self.missing += 1
                    whole = False
            for e in range(want, min(have, self.width)):
                if row[e] >= 0:
                    back.append(row[e])
                row[e] = -1
            for i in range(max(c, 0)):
                p = old + i
                positions.append(p)
                at = row[p // self.page] if p // self.page < self.width else -1
                slots.append(at * self.page + p % self.page if at >= 0 else -1)
            offsets.append(offsets[-1] + max(c, 0))
            self.lens[s] = new
        self.free = ready[taken:] + back
        return offsets, positions, slots
