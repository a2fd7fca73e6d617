"""A paged key-value cache held in 8 bits, its attention, and the hand-out of its pages, as cases that can
be timed and checked.

Four operators, used together when sequences grow: ``plan_pages`` gives sequences their pages from their
lengths, ``kv_append`` writes a call's new keys and values into them as e4m3 codes with a power-of-two scale
for each page and head, ``attention_paged`` is the attention of one new token per sequence over them and
``attention_paged_prompts`` that of several.

Where ``own`` is false, ``run`` computes them from elementary torch operations in 32 bits, rounded once at the
end.

Sizes come from this repository's configurations (16 heads of 64 over frames of 1374 tokens, the camera
head's 16 f32 heads of 128 over one token per frame) and, for shared key heads, from ordinary ones (32 query
heads over 8 of 128).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "f32": torch.float32}
EPS = 1e-5
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LARGEST = {"f16": 240.0 * 2.0 ** 8, "f32": 240.0 * 2.0 ** 120}  # what a cache of the type holds
LEAST = -117  # a scale's exponent
LONGEST = 1 << 30  # tokens of a sequence


# ---------------------------------------------------------------------------
# the cases
#
# lens: new tokens per sequence. past: the keys that the cache holds before them. causal: 0 = every key, c = a
# token sees all up to the end of its own group of c tokens (1: the usual mask, 1374: by frames).


def _append(name, dtype, lens, past, heads, kv_heads, dim, page, norm, rope, step):
    """``step``: one token a sequence, without offsets."""
    return dict(name=name, op="append", dtype=dtype, lens=lens, past=past, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, norm=norm, rope=rope, step=step)


def _paged(name, dtype, lens, heads, kv_heads, dim, page):
    """``lens``: keys per sequence, the new token's among them."""
    return dict(name=name, op="paged", dtype=dtype, lens=lens, heads=heads, kv_heads=kv_heads, dim=dim, page=page)


def _prompts(name, dtype, lens, past, heads, kv_heads, dim, page, causal):
    return dict(name=name, op="prompts", dtype=dtype, lens=lens, past=past, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, causal=causal)


def _pages(name, past, change, page):
    """``past``: tokens that the sequences hold. Every other sequence gets ``change`` more while the ones
    between drop as many; in the next call the other way round."""
    return dict(name=name, op="pages", past=past, change=change, page=page)


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
        _append("append8_step_f32", "f32", _text([1] * 8), _text(_ragged(8, 0, 400, 157)), 16, 16, 128, 16,
                False, True, True),
        # three clips of 4, 3 and 1 frames into a trunk block's cache, QK-norm, no rotation there
        _append("append8_frames_f16", "f16", _text([4 * 1374, 3 * 1374, 1374]), _text([0, 1374, 0]), 16, 16,
                64, 64, True, False, False),
        # prompts of very different lengths, shared key heads, rotated
        _append("append8_prompts_f16", "f16", _text([4099, 1, 7013, 130, 5138]), _text([0, 0, 517, 33, 0]), 32,
                8, 128, 16, False, True, False),
        # the camera head's step over its sessions' frames so far
        _paged("paged8_step_f32", "f32", _text(_ragged(8, 1, 800, 331)), 16, 16, 128, 16),
        # 64 sequences of up to 8192 keys, shared key heads
        _paged("paged8_steps_f16", "f16", _text(_ragged(64, 1, 8192, 3571)), 32, 8, 128, 16),
        # one token over the 95 frames before it
        _paged("paged8_long_f16", "f16", _text([95 * 1374 + 1]), 16, 16, 64, 64),
        # a frame that arrives, over the 21 before it
        _prompts("prompts8_frame_f16", "f16", _text([1374]), _text([21 * 1374]), 16, 16, 64, 64, 1374),
        # pieces of prompts of very different lengths, shared key heads
        _prompts("prompts8_pieces_f16", "f16", _text([512, 1, 2048, 77, 1024]), _text([3000, 700, 0, 5003, 8192]),
                 32, 8, 128, 16, 1),
        # a few drafted tokens of each of 32 sequences, seven queries per key head
        _prompts("prompts8_drafts_f16", "f16", _text(_ragged(32, 2, 6, 3)), _text(_ragged(32, 3, 4000, 1171)), 28,
                 4, 64, 32, 1),
        # an f32 trunk block: a frame over the two before it, beside a first one
        _prompts("prompts8_frames_f32", "f32", _text([1374, 1374]), _text([2 * 1374, 0]), 16, 16, 64, 64, 1374),
        # 256 sequences, a few tokens each: drafts rejected here, made there
        _pages("pages_steps", _text(_ragged(256, 5, 4000, 1237)), _text(_ragged(256, 1, 5, 3)), 16),
        # requests that end while others are admitted
        _pages("pages_prompts", _text(_ragged(64, 0, 300, 67)), _text(_ragged(64, 1, 8192, 3571)), 16),
    ]


def draw(rng):
    def between(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["append", "paged", "prompts", "pages"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "pages":
        count = between(1, 512)
        most = max(1, 260000 // count)
        return _pages("", _text([rng.choice([0, between(1, 2000)]) for _ in range(count)]),
                      _text([between(1, min(8192, most)) for _ in range(count)]), page)
    kv = rng.choice([1, 2, 4, 5, 8, 16])
    heads = kv if kv == 16 else kv * rng.choice([g for g in (1, 2, 3, 4, 7, 8) if kv * g <= 40])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["f16", "f16", "f32"])
    past, causal = [], 0
    if op == "append":
        step = rng.random() < 0.4
        count = between(1, 256) if step else between(1, 12)
        lens = [1 if step else between(1, 7000) for _ in range(count)]
        past = [rng.choice([0, between(1, 2900)]) for _ in range(count)]
        norm, rope = rng.random() < 0.5, rng.random() < 0.7
    elif op == "paged":
        count = between(1, 64)
        lens = [between(1, 130000 // count) for _ in range(count)]
    else:
        count = between(1, 16)
        most = rng.choice([8, 300, 2100])
        lens = [between(1, most) for _ in range(count)]
        past = [rng.choice([0, between(1, 30000 // count)]) for _ in range(count)]
        causal = rng.choice([0, 1, 1, 1, 17, 1374])
    # no larger than the largest listed case of the operator
    top = [work(c) for c in listed() if c["op"] == op]
    top = {"bytes": max(w["bytes"] for w in top), "flops": max(w["flops"] for w in top) / (8 if dtype == "f32" else 1)}
    while True:
        if op == "append":
            case = _append("", dtype, _text(lens), _text(past), heads, kv, dim, page, norm, rope, step)
        elif op == "paged":
            case = _paged("", dtype, _text(lens), heads, kv, dim, page)
        else:
            case = _prompts("", dtype, _text(lens), _text(past), heads, kv, dim, page, causal)
            past = [p * 2 // 3 for p in past]
        cost = work(case)
        if cost["bytes"] <= top["bytes"] and (op != "prompts" or cost["flops"] <= top["flops"]) or max(lens) == 1:
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


def _table(seed, totals, page):
    """Pages of all sequences, in no order, among a few that belong to none."""
    need = [-(-n // page) for n in totals]
    width = max(need) + 2
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    return table, pages


def _codes(gen, shape):
    """Codes and scales of values whose size differs from page to page and head to head."""
    scale = torch.randint(-8, -5, shape[:2], generator=gen, device=DEVICE, dtype=torch.int32)
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).mul_(90.0).clamp_(-448.0, 448.0)
    return x.to(E4M3), torch.exp2(scale.float()).to(E8M0)


def _cache(gen, case, totals):
    table, pages = _table(gen.initial_seed(), totals, case["page"])
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    (k, ks), (v, vs) = _codes(gen, shape), _codes(gen, shape)
    return dict(k=k, v=v, k_scale=ks, v_scale=vs, table=_i32(table), lens=_i32(totals))


def _prepare_pages(case, seed):
    past, change, page = _ints(case["past"]), _ints(case["change"]), case["page"]
    b = len(past)
    up = [i % 2 == 0 for i in range(b)]
    held = [p + (0 if u else c) for p, c, u in zip(past, change, up)]  # the odd ones drop first
    most = [-(-(p + c) // page) for p, c in zip(past, change)]
    width = max(most) + 1
    pages = sum(most) + 5
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in held:
        need = -(-n // page)
        table.append(order[at:at + need] + [-1] * (width - need))
        at += need
    sign = torch.tensor([1 if u else -1 for u in up], dtype=torch.int32, device=DEVICE)
    counts = _i32(change) * sign
    rows = max(sum(c for c, u in zip(change, up) if u == w) for w in (True, False))
    # the free pages lie in a ring, from its 3rd place on
    ring = [0] * pages
    for i, p in enumerate(order[at:]):
        ring[(3 + i) % pages] = p
    return dict(case=case, table=_i32(table), lens=_i32(held), free=_i32(ring), state=_i32([3 % pages, pages - at, 0]),
                counts=(counts, -counts), turn=0, rows=rows, offsets=torch.zeros(b + 1, dtype=torch.int32, device=DEVICE),
                positions=torch.full((rows,), -1, dtype=torch.int32, device=DEVICE),
                slots=torch.full((rows,), -1, dtype=torch.int64, device=DEVICE))


def prepare(case, seed):
    if case["op"] == "pages":
        s = _prepare_pages(case, seed)
        if own:
            from headshot_amd.context import HipContext
            from headshot_amd.paged import PagePool

            s["ctx"] = HipContext(DEVICE)
            s["pool"] = PagePool(s["table"], s["lens"], s["free"], s["state"], case["page"])
        return s
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    lens = _ints(case["lens"])
    h, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case, dtype=dtype)
    totals = lens if case["op"] == "paged" else [a + b for a, b in zip(_ints(case["past"]), lens)]
    n = sum(lens)
    if case["op"] == "append":
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
        s["offsets"] = None if case["step"] else _i32(_offsets(lens))
    elif case["op"] == "paged":
        s["q"] = _normal(gen, (len(lens), h, dim), dtype)
    else:
        s["q"] = _normal(gen, (n, h, dim), dtype)
        s["offsets"] = _i32(_offsets(lens))
    c = s["cache"] = _cache(gen, case, totals)
    if own:
        from headshot_amd.context import HipContext
        from headshot_amd.paged import PagedKV8

        s["ctx"] = HipContext(DEVICE)
        s["paged"] = PagedKV8(c["k"], c["v"], c["k_scale"], c["v_scale"], c["table"], c["lens"], dtype)
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


def _scale_exponent(scale):
    return torch.frexp(scale.float())[1] - 1


def _store_plain(codes, scale, x, at, row, heads_of, largest):
    """x (n, heads, d) into row ``row`` of page ``at``; heads_of: the first token of each sequence."""
    x = x.clamp(-largest, largest)
    most = torch.zeros(scale.shape, device=DEVICE)
    most.scatter_reduce_(0, at[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    part, exponent = torch.frexp(most)
    need = torch.where(most > 0, exponent - torch.where(part <= 0.875, 9, 8), LEAST).clamp_min(LEAST)
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEVICE)
    touched[at] = True
    old = _scale_exponent(scale)
    new = torch.where(touched[:, None], need, old)
    # pages that the call goes on with: the ones of the sequences' first tokens
    begun, first = at[heads_of], row[heads_of]
    goes_on = first > 0
    new[begun] = torch.where(goes_on[:, None], torch.maximum(old[begun], need[begun]), new[begun])
    raw = codes.view(torch.uint8)
    older = raw[begun].view(E4M3).float()
    held = torch.arange(codes.shape[2], device=DEVICE) < first[:, None]
    shrunk = (older * torch.exp2((old - new)[begun].float())[:, :, None, None]).to(E4M3)
    raw[begun] = torch.where(held[:, None, :, None], shrunk.view(torch.uint8), raw[begun])
    raw[at, :, row] = (x * torch.exp2(-new[at].float())[..., None]).to(E4M3).view(torch.uint8)
    scale.copy_(torch.exp2(new.float()))


def _append_plain(s):
    case, c = s["case"], s["cache"]
    dim, page = case["dim"], case["page"]
    n = s["k"].shape[0]
    token = torch.arange(n, device=DEVICE)
    if s["offsets"] is None:
        seq, pos, begins = token, c["lens"].long() - 1, token
    else:
        ends = s["offsets"][1:].long()
        seq = (token[:, None] >= ends).sum(1)
        pos = c["lens"].long()[seq] - ends[seq] + token
        begins = s["offsets"][:-1].long()
    q = _rotate_plain(s["q"].reshape(n, -1, dim), s["qn"], s["rope"], pos).to(s["dtype"]).flatten(1)
    k = _rotate_plain(s["k"].reshape(n, -1, dim), s["kn"], s["rope"], pos)
    at = c["table"].long()[seq, pos // page]
    largest = LARGEST[case["dtype"]]
    _store_plain(c["k"], c["k_scale"], k, at, pos % page, begins, largest)
    _store_plain(c["v"], c["v_scale"], s["v"].reshape(n, -1, dim).float(), at, pos % page, begins, largest)
    return [q, c["k"], c["v"], c["k_scale"], c["v_scale"]]


def _softmax_plain(scores):
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _values_plain(c, x, at):
    """The values of the pages ``at`` (.., pages), as (.., heads, keys, d) in 32 bits."""
    codes = c[x].view(torch.uint8)[at].view(E4M3).float() * c[x + "_scale"].float()[at][..., None, None]
    codes = codes.transpose(-4, -3)
    return codes.reshape(*codes.shape[:-3], -1, codes.shape[-1])


def _paged_plain(s):
    """All sequences at once, as long as the longest."""
    case, c = s["case"], s["cache"]
    b, h, d = s["q"].shape
    kv = case["kv_heads"]
    at = c["table"][:, :-(-max(_ints(case["lens"])) // case["page"])].long()
    k, v = _values_plain(c, "k", at), _values_plain(c, "v", at)
    q = s["q"].float().reshape(b * kv, h // kv, d)
    scores = torch.bmm(q, k.flatten(0, 1).transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
    seen = torch.arange(k.shape[2], device=DEVICE) < c["lens"][:, None]
    scores = scores.reshape(b, h, -1).masked_fill(~seen[:, None], -math.inf)
    return torch.bmm(_softmax_plain(scores).reshape(b * kv, h // kv, -1), v.flatten(0, 1)).reshape(b, h * d).to(s["dtype"])


def _prompts_plain(s):
    case, c = s["case"], s["cache"]
    kv, d, group = case["kv_heads"], case["dim"], case["causal"]
    lens = _ints(case["lens"])
    out = []
    for i, (q, m, p) in enumerate(zip(s["q"].split(lens), lens, _ints(case["past"]))):
        n = p + m
        at = c["table"][i, :-(-n // case["page"])].long()
        k, v = (_values_plain(c, x, at)[:, :n] for x in "kv")
        qh = q.float().reshape(m, kv, -1, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
        scores = (torch.bmm(qh, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))).reshape(kv, -1, m, n)
        if group:
            place = torch.arange(m, device=DEVICE) + p
            seen = torch.arange(n, device=DEVICE) < ((place // group + 1) * group)[:, None]
            scores = scores.masked_fill(~seen, -math.inf)
        o = torch.bmm(_softmax_plain(scores).reshape(kv, -1, n), v.contiguous())
        out.append(o.reshape(kv, -1, m, d).permute(2, 0, 1, 3).reshape(m, -1))
    return torch.cat(out).to(s["dtype"])


def _pages_plain(s, counts):
    page, table, lens, free, state = s["case"]["page"], s["table"], s["lens"], s["free"], s["state"]
    width, pages = table.shape[1], free.shape[0]
    old = lens.long()
    new = (old + counts).clamp(0, LONGEST)
    all_have, all_want = (old + page - 1) // page, (new + page - 1) // page
    have, want = all_have.clamp_max(width), all_want.clamp_max(width)
    grow = (want - have).clamp_min(0)
    # a sequence behind a page that it did not get gets no more
    end = table.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0]
    ask = torch.where((have > 0) & ((end < 0) | (end >= pages)), 0, grow)
    first = ask.cumsum(0) - ask
    head, count = state[0].long(), state[1].long()
    column = torch.arange(width, device=DEVICE)
    index = first[:, None] + column - have[:, None]
    added = (column >= have[:, None]) & (column < want[:, None])
    served = added & (index < count) & (ask > 0)[:, None]
    got = torch.where(served, free[(head + index.clamp_min(0)) % pages], -1)
    dropped = (column >= want[:, None]) & (column < have[:, None])
    back = dropped & (table >= 0) & (table < pages)
    rank = (back.flatten().cumsum(0) - 1).reshape(back.shape)
    back &= count + rank < pages
    # pages that come back go behind the ring's last
    spare = torch.cat([free, free.new_zeros(1)])
    spare[torch.where(back, (head + count + rank) % pages, pages)] = table
    free.copy_(spare[:-1])
    table.copy_(torch.where(added, got.to(table.dtype), torch.where(dropped, -1, table)))
    taken, given = served.sum(), back.sum()
    more = (all_want - all_have).clamp_min(0).sum()
    state.copy_(torch.stack([(head + taken) % pages, count - taken + given, more - taken]))
    lens.copy_(new)
    fresh = counts.long().clamp_min(0)
    s["offsets"][1:] = fresh.cumsum(0)
    row = torch.arange(s["rows"], device=DEVICE)
    seq = (row[:, None] >= s["offsets"][1:]).sum(1)
    live = seq < fresh.shape[0]
    seq = seq.clamp_max(fresh.shape[0] - 1)
    place = old[seq] + row - s["offsets"][seq]
    held = table[seq, (place // page).clamp_max(width - 1)].long()
    there = (place // page < width) & (held >= 0) & (held < pages)
    s["positions"].copy_(torch.where(live, place, s["positions"]))
    s["slots"].copy_(torch.where(live, torch.where(there, held * page + place % page, -1), s["slots"]))


def _run_pages(s):
    counts = s["counts"][s["turn"]]
    s["turn"] ^= 1
    if own:
        s["ctx"].plan_pages(s["pool"], counts, s["rows"], out=(s["offsets"], s["positions"], s["slots"]))
    else:
        _pages_plain(s, counts)
    return [s[x] for x in ("offsets", "positions", "slots", "table", "lens", "free", "state")]


def run(state):
    s = state
    op = s["case"]["op"]
    if op == "pages":
        return _run_pages(s)
    if not own:
        return {"append": _append_plain, "paged": _paged_plain, "prompts": _prompts_plain}[op](s)
    ctx, cache = s["ctx"], s["paged"]
    if op == "append":
        q, _ = ctx.kv_append(cache, s["k"], s["v"], offsets=s["offsets"], q=s["q"], qn=s["qn"], kn=s["kn"],
                             rope=s["rope"], eps=EPS)
        return [q, cache.k, cache.v, cache.k_scale, cache.v_scale]
    if op == "paged":
        return ctx.attention_paged(s["q"], cache)
    return ctx.attention_paged_prompts(s["q"], cache, s["offsets"], causal=s["case"]["causal"])


# ---------------------------------------------------------------------------
# what a pass cannot do without


def _pairs(m, n, c):
    """Query-key pairs that the mask leaves of the last m of n tokens."""
    if c == 0:
        return m * n
    if c == 1:
        return m * n - m * (m - 1) // 2
    total, at = 0, n - m
    while at < n:  # a group's queries see the same keys
        end = min((at // c + 1) * c, n)
        total += (end - at) * end
        at = end
    return total


def work(case):
    if case["op"] == "pages":
        change, page = _ints(case["change"]), case["page"]
        b, rows = len(change), sum(change[::2])
        return {"bytes": 4 * (4 * b + 1) + 12 * rows + 8 * (sum(change) // page), "flops": 4 * b + 6 * rows}
    size = 2 if case["dtype"] == "f16" else 4
    lens = _ints(case["lens"])
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    n = sum(lens)
    if case["op"] == "append":
        totals = [a + b for a, b in zip(lens, _ints(case["past"]))]
        moved = n * (h + 2 * kv) * d * size + n * h * d * size + 2 * n * kv * d + 2 * kv * (n // page)
        if case["rope"]:
            moved += 2 * 4 * d * min(n, max(totals))
        return {"bytes": moved, "flops": n * (h + kv) * d * ((8 if case["norm"] else 0) + (3 if case["rope"] else 0)) + 4 * n * kv * d}
    if case["op"] == "paged":
        return {"bytes": 2 * n * kv * d + 2 * len(lens) * h * d * size, "flops": 4 * n * h * d}
    totals = [a + b for a, b in zip(lens, _ints(case["past"]))]
    pairs = sum(_pairs(m, t, case["causal"]) for m, t in zip(lens, totals))
    return {"bytes": 2 * sum(totals) * kv * d + 2 * n * h * d * size, "flops": 4 * pairs * h * d}


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


def _exact_e4m3(x):
    """x to 4 significant bits, fewer below 2^-6, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_store(codes, scale, x, table, past, lens, page, largest):
    codes, scale = codes.double(), scale.double()
    x = x.clamp(-largest, largest)
    begin = 0
    for i, (p, m) in enumerate(zip(past, lens)):
        end = p + m
        spans = [(a // page, max(a, p), min(a + page, end)) for a in range(p // page * page, end, page)]
        for where, a, z in spans[:1] + spans[-1:] if len(spans) > 1 else spans:
            _exact_block(codes, scale, x[begin + a - p:begin + z - p], table[i][where], a % page)
        middle = spans[1:-1]  # whole pages, all at once
        if middle:
            at = torch.tensor([table[i][w] for w, _, _ in middle], device=DEVICE)
            rows = x[begin + middle[0][1] - p:begin + middle[-1][2] - p].unflatten(0, (-1, page)).transpose(1, 2)
            new = _exact_scale(rows.abs().amax((2, 3)))
            codes[at] = _exact_e4m3(rows / new[:, :, None, None])
            scale[at] = new
        begin += m
    return codes, scale


def _exact_scale(most):
    """The least power of two that brings it to 448 at most."""
    e = torch.floor(torch.log2(most.clamp_min(1e-300))) - 8
    e = e + (most > 448 * torch.exp2(e)).double()
    return torch.exp2(e.clamp_min(LEAST))


def _exact_block(codes, scale, rows, at, first):
    new = _exact_scale(rows.abs().amax((0, 2)))
    if first > 0:
        new = torch.maximum(new, scale[at])
        codes[at, :, :first] = _exact_e4m3(codes[at, :, :first] * (scale[at] / new)[:, None, None])
    codes[at, :, first:first + rows.shape[0]] = _exact_e4m3(rows.transpose(0, 1) / new[:, None, None])
    scale[at] = new


def exact(case, seed):
    if case["op"] == "pages":
        return None
    lens = _ints(case["lens"])
    s = prepare(case, seed)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    c = s["cache"]
    if case["op"] == "append":
        past = _ints(case["past"])
        rows = torch.tensor([p + i for p, n in zip(past, lens) for i in range(n)], device=DEVICE)
        q = _exact_heads(s["q"], d, s["qn"], s["rope"], rows)
        k = _exact_heads(s["k"], d, s["kn"], s["rope"], rows)
        v = s["v"].double().unflatten(1, (-1, d))
        table, largest = c["table"].tolist(), LARGEST[case["dtype"]]
        kc, ks = _exact_store(c["k"], c["k_scale"], k, table, past, lens, page, largest)
        vc, vs = _exact_store(c["v"], c["v_scale"], v, table, past, lens, page, largest)
        return [q.flatten(1), kc, vc, ks, vs]
    single = case["op"] == "paged"
    past = [n - 1 for n in lens] if single else _ints(case["past"])
    fresh = [1] * len(lens) if single else lens
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    begin = 0
    for i, (m, p) in enumerate(zip(fresh, past)):
        place = torch.arange(p + m, device=DEVICE)
        at = c["table"][i].long()[place // page]
        raw = {x: c[x].view(torch.uint8)[at, :, place % page].view(E4M3).double() for x in "kv"}
        k, v = (raw[x] * c[x + "_scale"].double()[at][..., None] for x in "kv")
        group = 0 if single else case["causal"]
        mine = place[p:]
        end = torch.full_like(mine, p + m) if group == 0 else (torch.div(mine, group, rounding_mode="floor") + 1) * group
        for j in range(h):
            g = j // (h // kv)
            logits = s["q"][begin:begin + m, j].double() @ k[:, g].T / math.sqrt(d)
            logits[place >= end[:, None]] = -math.inf
            out[begin:begin + m, j] = torch.softmax(logits, 1) @ v[:, g]
        begin += m
    return out.flatten(1)
