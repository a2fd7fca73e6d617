"""A paged key-value cache and the attention around it, as cases that can be timed and checked.

Three operators, used together when sequences grow: ``kv_append`` writes a
call's new keys and values into the pages of their sequences (QK-norm and the
position rotation on the way), ``attention_packed`` is the attention of whole
prompts of different lengths in one call, ``attention_paged`` that of one new
token per sequence over the pages.

Where ``own`` is false, ``run`` computes them from elementary torch operations
in 32 bits, rounded once at the end.

Sizes come from this repository's configurations (16 heads of 64 over frames
of 1374 tokens, the camera head's 16 f32 heads of 128 over one token per
frame) and, for shared key heads, from ordinary ones (32 query heads over 8 of
128).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------
# the cases
#
# lens: tokens per sequence. append: the call's new tokens, behind "past" ones
#   already in the cache. packed: queries per sequence, "past" keys more than
#   that before them. paged: keys per sequence, the new token's among them.
# causal: 0 = every key, c = a token sees all up to the end of its own group
#   of c tokens (1: the usual mask, 1374: by frames).


def _append(name, dtype, lens, past, heads, kv_heads, dim, page, norm, rope, rows):
    """``rows``: a prompt, whose rotated keys are read as rows as well."""
    return dict(name=name, op="append", dtype=dtype, lens=lens, past=past, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, norm=norm, rope=rope, rows=rows)


def _packed(name, dtype, lens, past, heads, kv_heads, dim, causal):
    return dict(name=name, op="packed", dtype=dtype, lens=lens, past=past, heads=heads,
                kv_heads=kv_heads, dim=dim, causal=causal)


def _paged(name, dtype, lens, heads, kv_heads, dim, page):
    return dict(name=name, op="paged", dtype=dtype, lens=lens, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page)


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _ragged(count, low, high, step):
    """``count`` lengths from ``low`` to ``high``, out of order and uneven."""
    return [low + (i * step) % (high - low + 1) for i in range(count)]


def listed():
    return [
        # the camera head's step: one token of each of eight sessions
        _append("append_step_f32", "f32", _text([1] * 8), _text(_ragged(8, 0, 400, 157)), 16, 16,
                128, 16, False, True, False),
        # three clips of 4, 3 and 1 frames into a trunk block's cache, QK-norm, no rotation there
        _append("append_frames_f16", "f16", _text([4 * 1374, 3 * 1374, 1374]), _text([0, 1374, 0]),
                16, 16, 64, 64, True, False, True),
        # prompts of very different lengths, shared key heads, rotated
        _append("append_prompts_f16", "f16", _text([4099, 1, 7013, 130, 5138]),
                _text([0, 0, 517, 33, 0]), 32, 8, 128, 16, False, True, True),
        # 200 sessions' steps at once
        _append("append_steps_f16", "f16", _text([1] * 200), _text(_ragged(200, 0, 3999, 1237)), 32,
                8, 128, 32, True, True, False),
        # the camera head over eight sessions' frames so far
        _packed("packed_camera_f32", "f32", _text([1, 200, 37, 100, 8, 64, 151, 96]),
                _text([0] * 8), 16, 16, 128, 1),
        # two clips through an f32 trunk block, masked by frames
        _packed("packed_frames_f32", "f32", _text([2 * 1374, 1374]), _text([0, 0]), 16, 16, 64, 1374),
        # two clips through an f16 trunk block, masked by frames
        _packed("packed_frames_f16", "f16", _text([5 * 1374, 3 * 1374]), _text([0, 0]), 16, 16, 64,
                1374),
        # prompts of very different lengths, shared key heads, one behind a kept prefix
        _packed("packed_prompts_f16", "f16", _text([4099, 1, 6001, 777, 2048]),
                _text([0, 0, 0, 1000, 0]), 32, 8, 128, 1),
        # the camera head's step
        _paged("paged_step_f32", "f32", _text(_ragged(8, 1, 800, 331)), 16, 16, 128, 16),
        # 64 sequences of up to 8192 keys, shared key heads
        _paged("paged_steps_f16", "f16", _text(_ragged(64, 1, 8192, 3571)), 32, 8, 128, 16),
        # one token over the 95 frames before it
        _paged("paged_long_f16", "f16", _text([95 * 1374 + 1]), 16, 16, 64, 64),
        # a middling batch with seven queries per key head
        _paged("paged_odd_f16", "f16", _text(_ragged(19, 5, 3001, 1171)), 28, 4, 64, 32),
    ]


def draw(rng):
    def between(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kv = rng.choice([1, 2, 4, 5, 8, 16])
    heads = kv if kv == 16 else kv * rng.choice([g for g in (1, 2, 3, 4, 7, 8) if kv * g <= 40])
    dim = rng.choice([64, 128])
    op = rng.choice(["append", "packed", "paged"])
    dtype = rng.choice(["f16", "f16", "f32"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "append":
        step = rng.random() < 0.4
        count = between(1, 256) if step else between(1, 12)
        lens = [1 if step else between(1, 7000) for _ in range(count)]
        past = [rng.choice([0, between(1, 3000)]) for _ in range(count)]
        norm, rope = rng.random() < 0.5, rng.random() < 0.7
    elif op == "packed":
        count = between(1, 8)
        lens = [between(1, 7000) for _ in range(count)]
        past = [rng.choice([0, 0, between(1, 1400)]) for _ in range(count)]
        causal = rng.choice([0, 1, 1, 1, 17, 1374])
    else:
        count = between(1, 64)
        lens = [between(1, 130000 // count) for _ in range(count)]
    # no larger than the largest listed case of the operator and type
    top = [work(c) for c in listed() if c["op"] == op and c["dtype"] == dtype]
    top = {"bytes": max(w["bytes"] for w in top), "flops": max(w["flops"] for w in top)}
    if op == "append" and dtype == "f32":
        top = {k: 200 * v for k, v in top.items()}  # the listed one is a step
    if op == "paged" and dtype == "f32":
        top = {k: 4 * v for k, v in top.items()}
    while True:
        if op == "append":
            case = _append("", dtype, _text(lens), _text(past), heads, kv, dim, page, norm, rope, not step)
        elif op == "packed":
            case = _packed("", dtype, _text(lens), _text(past), heads, kv, dim, causal)
            past = [p * 2 // 3 for p in past]
        else:
            case = _paged("", dtype, _text(lens), heads, kv, dim, page)
        cost = work(case)
        if cost["bytes"] <= top["bytes"] and cost["flops"] <= top["flops"] or max(lens) == 1:
            return case
        lens = [max(1, n * 2 // 3) for n in lens]


# ---------------------------------------------------------------------------
# inputs


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _normal(gen, shape, dtype, mean=0.0, std=1.0):
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)
    return x.mul_(std).add_(mean).to(dtype)


def _tables(rows, dim):
    """sin and cos of the positions' angles, rows of [first half | the same again]."""
    half = torch.arange(dim // 2, dtype=torch.float64, device=DEVICE)
    angle = torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (-half / (dim // 2))
    angle = torch.cat([angle, angle], 1)
    return angle.sin().float(), angle.cos().float()


def _cache(gen, case, totals, dtype):
    """Pages of all sequences, in no order, among a few that belong to none."""
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in totals]
    width = max(need) + 2
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(gen.initial_seed())).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    return dict(k=_normal(gen, (pages, kv, page, dim), dtype), v=_normal(gen, (pages, kv, page, dim), dtype),
                table=_i32(table), lens=_i32(totals))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    lens = _ints(case["lens"])
    h, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case, dtype=dtype)
    if case["op"] == "append":
        past = _ints(case["past"])
        n = sum(lens)
        totals = [a + b for a, b in zip(past, lens)]
        # q, k and v as a projection leaves them: column ranges of one product
        if case["rope"]:
            qkv = _normal(gen, (n, (h + 2 * kv) * dim), dtype)
            s["q"], s["k"], s["v"] = qkv.split([h * dim, kv * dim, kv * dim], 1)
            s["rope"] = _tables(max(totals), dim)
        else:
            s["q"], s["k"], s["v"] = (_normal(gen, (n, c * dim), dtype) for c in (h, kv, kv))
            s["rope"] = None
        for name in ("qn", "kn"):
            s[name] = (_normal(gen, (dim,), torch.float32, 1.0, 0.1),
                       _normal(gen, (dim,), torch.float32, 0.0, 0.1)) if case["norm"] else None
        s["offsets"] = _i32(_offsets(lens)) if case["rows"] else None
        s["cache"] = _cache(gen, case, totals, dtype)
    elif case["op"] == "packed":
        past = _ints(case["past"])
        keys = [a + b for a, b in zip(past, lens)]
        s["q"] = _normal(gen, (sum(lens), h, dim), dtype)
        s["k"] = _normal(gen, (sum(keys), kv, dim), dtype)
        s["v"] = _normal(gen, (sum(keys), kv, dim), dtype)
        s["offsets"] = _i32(_offsets(lens))
        s["k_offsets"] = _i32(_offsets(keys)) if any(past) else None
    else:
        s["q"] = _normal(gen, (len(lens), h, dim), dtype)
        s["cache"] = _cache(gen, case, lens, dtype)
    if own:
        from headshot_amd.context import HipContext
        from headshot_amd.paged import PagedKV

        s["ctx"] = HipContext(DEVICE)
        if "cache" in s:
            c = s["cache"]
            s["paged"] = PagedKV(c["k"], c["v"], c["table"], c["lens"])
    return s


# ---------------------------------------------------------------------------
# one pass


def _rotate_plain(x, norm, rope, row):
    x = x.float()
    if norm is not None:
        mean = x.mean(-1, keepdim=True)
        var = ((x - mean) ** 2).mean(-1, keepdim=True)
        x = (x - mean) * (var + EPS).rsqrt() * norm[0] + norm[1]
    if rope is not None:
        sin, cos = rope[0][row][:, None], rope[1][row][:, None]
        half = x.shape[-1] // 2
        x = x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin
    return x


def _append_plain(s):
    case, c = s["case"], s["cache"]
    dim, page = case["dim"], case["page"]
    n = s["k"].shape[0]
    token = torch.arange(n, device=DEVICE)
    if s["offsets"] is None:
        seq, pos = token, c["lens"].long() - 1
    else:
        ends = s["offsets"][1:].long()
        seq = (token[:, None] >= ends).sum(1)
        pos = c["lens"].long()[seq] - ends[seq] + token
    q = _rotate_plain(s["q"].reshape(n, -1, dim), s["qn"], s["rope"], pos).to(s["dtype"]).flatten(1)
    k = _rotate_plain(s["k"].reshape(n, -1, dim), s["kn"], s["rope"], pos).to(s["dtype"])
    at = c["table"].long()[seq, pos // page]
    c["k"][at, :, pos % page] = k
    c["v"][at, :, pos % page] = s["v"].reshape(n, -1, dim)
    return [q, k.flatten(1), c["k"], c["v"]] if case["rows"] else [q, c["k"], c["v"]]


def _softmax_plain(scores):
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _attend_plain(q, k, v, seen):
    """q (nq, h, d), k and v (nk, kv, d) in 32 bits; seen (nq, nk) or None."""
    nq, h, d = q.shape
    kv = k.shape[1]
    qh = q.reshape(nq, kv, h // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
    scores = torch.bmm(qh, k.permute(1, 2, 0).contiguous()) * (1.0 / math.sqrt(d))
    if seen is not None:
        scores = scores.reshape(kv, -1, nq, k.shape[0]).masked_fill(~seen, -math.inf)
        scores = scores.reshape(kv, -1, k.shape[0])
    out = torch.bmm(_softmax_plain(scores), v.permute(1, 0, 2).contiguous())
    return out.reshape(kv, h // kv, nq, d).permute(2, 0, 1, 3).reshape(nq, h * d)


def _packed_plain(s):
    case = s["case"]
    lens = _ints(case["lens"])
    keys = [a + b for a, b in zip(_ints(case["past"]), lens)]
    qs, ks, vs = s["q"].split(lens), s["k"].split(keys), s["v"].split(keys)
    out = []
    for q, k, v in zip(qs, ks, vs):
        nq, nk, c = q.shape[0], k.shape[0], case["causal"]
        seen = None
        if c:
            at = torch.arange(nq, device=DEVICE) + (nk - nq)
            seen = torch.arange(nk, device=DEVICE) < ((at // c + 1) * c)[:, None]
        out.append(_attend_plain(q.float(), k.float(), v.float(), seen))
    return torch.cat(out).to(s["dtype"])


def _paged_plain(s):
    case, c = s["case"], s["cache"]
    page, dim = case["page"], case["dim"]
    out = []
    for i, n in enumerate(_ints(case["lens"])):
        at = c["table"][i, :-(-n // page)].long()
        k, v = (c[x][at].transpose(1, 2).reshape(-1, case["kv_heads"], dim)[:n].float() for x in "kv")
        out.append(_attend_plain(s["q"][i:i + 1].float(), k, v, None))
    return torch.cat(out).to(s["dtype"])


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"append": _append_plain, "packed": _packed_plain, "paged": _paged_plain}[op](s)
    ctx = s["ctx"]
    if op == "append":
        q, k = ctx.kv_append(s["paged"], s["k"], s["v"], offsets=s["offsets"], q=s["q"], qn=s["qn"],
                             kn=s["kn"], rope=s["rope"], eps=EPS, k_rows=s["case"]["rows"])
        return [q, k, s["paged"].k, s["paged"].v] if s["case"]["rows"] else [q, s["paged"].k, s["paged"].v]
    if op == "packed":
        return ctx.attention_packed(s["q"], s["k"], s["v"], s["offsets"], k_offsets=s["k_offsets"],
                                    causal=s["case"]["causal"])
    return ctx.attention_paged(s["q"], s["paged"])


# ---------------------------------------------------------------------------
# what a pass cannot do without


def _pairs(nq, nk, c):
    """Query-key pairs that the mask leaves."""
    if c == 0:
        return nq * nk
    total, i = 0, 0
    while i < nq:  # a group's queries see the same keys
        at = i + nk - nq
        group_end = min((at // c + 1) * c, nk)
        count = min(group_end - at, nq - i)
        if c == 1:
            return sum(range(nk - nq + 1, nk + 1))
        total += count * group_end
        i += count
    return total


def work(case):
    size = 2 if case["dtype"] == "f16" else 4
    lens = _ints(case["lens"])
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        n = sum(lens)
        moved = n * (h + 2 * kv) * d * size * 2 + (n * kv * d * size if case["rows"] else 0)
        if case["rope"]:
            moved += 2 * 4 * d * min(n, max(a + b for a, b in zip(lens, _ints(case["past"]))))
        return {"bytes": moved, "flops": n * (h + kv) * d * ((8 if case["norm"] else 0) + (3 if case["rope"] else 0))}
    if case["op"] == "packed":
        keys = [a + b for a, b in zip(_ints(case["past"]), lens)]
        pairs = sum(_pairs(a, b, case["causal"]) for a, b in zip(lens, keys))
        return {"bytes": (2 * sum(lens) * h + 2 * sum(keys) * kv) * d * size, "flops": 4 * pairs * h * d}
    return {"bytes": (2 * sum(lens) * kv + 2 * len(lens) * h) * d * size, "flops": 4 * sum(lens) * h * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_heads(x, dim, norm, rope, rows):
    """Every head vector normalised, then turned pair by pair."""
    x = x.double().unflatten(1, (-1, dim))
    if norm is not None:
        w, b = norm[0].double(), norm[1].double()
        x = (x - x.mean(2, True)) / (x.var(2, unbiased=False, keepdim=True) + EPS).sqrt() * w + b
    if rope is not None:
        half = dim // 2
        sin, cos = (t.double()[rows].unsqueeze(1) for t in rope)
        lo, hi = x[:, :, :half], x[:, :, half:]
        x = torch.cat([lo * cos[:, :, :half] - hi * sin[:, :, :half],
                       hi * cos[:, :, half:] + lo * sin[:, :, half:]], 2)
    return x


def _exact_rows(q, k, v, first):
    """One head: q (n, d), k and v (m, d); query i sees keys below first[i]."""
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // max(1, k.shape[0]))
    column = torch.arange(k.shape[0], device=q.device)
    for a in range(0, q.shape[0], step):
        logits = q[a:a + step] @ k.T / math.sqrt(q.shape[1])
        logits[column >= first[a:a + step, None]] = -math.inf
        out[a:a + step] = torch.softmax(logits, 1) @ v
    return out


def exact(case, seed):
    lens = _ints(case["lens"])
    if case["op"] == "packed" and work(case)["flops"] > 4e13:
        return None
    s = prepare(case, seed)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        past, c, page = _ints(case["past"]), s["cache"], case["page"]
        rows = torch.tensor([p + i for p, n in zip(past, lens) for i in range(n)], device=DEVICE)
        q = _exact_heads(s["q"], d, s["qn"], s["rope"], rows)
        k = _exact_heads(s["k"], d, s["kn"], s["rope"], rows)
        v = s["v"].double().unflatten(1, (-1, d))
        k_all, v_all = c["k"].double(), c["v"].double()
        table = c["table"].tolist()
        slots = torch.tensor([[table[i][p // page], p % page] for i, (a, n) in enumerate(zip(past, lens))
                              for p in range(a, a + n)], device=DEVICE)
        k_all[slots[:, 0], :, slots[:, 1]] = k
        v_all[slots[:, 0], :, slots[:, 1]] = v
        return [q.flatten(1), k.flatten(1), k_all, v_all] if case["rows"] else [q.flatten(1), k_all, v_all]
    if case["op"] == "packed":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        qa = ka = 0
        for n, p in zip(lens, _ints(case["past"])):
            m = n + p
            place = torch.arange(p, m, device=DEVICE)
            c = case["causal"]
            first = torch.full_like(place, m) if c == 0 else torch.div(place, c, rounding_mode="floor") * c + c
            for i in range(h):
                j = i // (h // kv)
                out[qa:qa + n, i] = _exact_rows(s["q"][qa:qa + n, i].double(), s["k"][ka:ka + m, j].double(),
                                                s["v"][ka:ka + m, j].double(), first)
            qa, ka = qa + n, ka + m
        return out.flatten(1)
    c, page = s["cache"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(lens):
        place = torch.arange(n, device=DEVICE)
        at = c["table"][i].long()[place // page]
        k, v = c["k"][at, :, place % page].double(), c["v"][at, :, place % page].double()
        weight = torch.softmax((s["q"][i].double().reshape(kv, 1, -1, d) * k.transpose(0, 1)[:, :, None]).sum(3)
                               / math.sqrt(d), 1)
        out[i] = (weight[..., None] * v.transpose(0, 1)[:, :, None]).sum(1).reshape(h, d)
    return out.flatten(1)
