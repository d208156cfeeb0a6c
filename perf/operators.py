"""The operators of the paged 8-bit key/value cache as measurable cases: each in its plain form and as the framework's calls.

The cache holds keys and values in 8 bits (e4m3 or int8), cut into pages of P tokens, with one scale for each page and key head.  A page's
keys lie row by row, its values column by column; scales are powers of two.  Four operators work on it:

* ``tables``: block tables, slot maps and attention tiles of a step, from the requests' lengths and a ring of free pages,
* ``append``: new key and value rows into their slots (a page's scale grows when it has to, its older codes with it),
* ``read``: rows back as 16- or 32-bit numbers, for paths that want them dense,
* ``attend``: causal attention of the step's rows over the pages, single tokens, short questions and long prompts.

All lengths are drawn from the case alone (``mix``); values come from the seed.
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
EXP_MIN, EXP_MAX = -40, 40                     # the exponents that a scale may have


def _blocks():
    path = os.path.join(ROOT, "prompt-cache_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from promptcache_amd import _blocks as blocks
    return blocks


# ---- the cases ------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a small batch: its tables are on the path of every token
        dict(name="tables step", kind="tables", n=64, cached_lo=1, cached_hi=8192, new_lo=1, new_hi=1, ends=0.05, P=64, tile_rows=1, spare=0, mix=11),
        # a crowded server: some hundred requests, most with prompts of their own, some of them over, the free pages not quite enough
        dict(name="tables ragged", kind="tables", n=517, cached_lo=0, cached_hi=2048, new_lo=0, new_hi=400, ends=0.1, P=16, tile_rows=128, spare=-40, mix=12),
        # a decoding step writes one row a request into pages that are partly full
        dict(name="append step", kind="append", n=64, past_lo=1, past_hi=4096, new_lo=1, new_hi=1, Hkv=8, dim=128, P=64, code="e4m3", dtype="bf16", mix=21),
        # prompts and long documents of several requests are written at once
        dict(name="append prompts", kind="append", n=9, past_lo=0, past_hi=700, new_lo=500, new_hi=4096, Hkv=8, dim=128, P=64, code="int8", dtype="bf16", mix=22),
        # a cached document of 8 k tokens, 32 key heads as in the 7b models, handed on as dense rows
        dict(name="read document", kind="read", n=1, past_lo=8247, past_hi=8247, Hkv=32, dim=128, P=64, code="e4m3", dtype="bf16", mix=31),
        # ragged short passages in 32 bits
        dict(name="read passages", kind="read", n=23, past_lo=1, past_hi=600, Hkv=5, dim=80, P=16, code="int8", dtype="f32", mix=32),
        # the smallest: two requests decode behind a few hundred tokens, in 32 bits
        dict(name="attend small", kind="attend", n=2, past_lo=150, past_hi=300, new_lo=1, new_hi=1, H=16, Hkv=4, dim=64, P=16, code="int8", dtype="f32", window=0,
             sink=False, mix=41),
        # 64 requests of very different lengths decode together
        dict(name="attend step", kind="attend", n=64, past_lo=64, past_hi=8192, new_lo=1, new_hi=1, H=32, Hkv=8, dim=128, P=64, code="e4m3", dtype="bf16", window=0,
             sink=False, mix=42),
        # one request decodes behind a very long document
        dict(name="attend long", kind="attend", n=1, past_lo=131071, past_hi=131071, new_lo=1, new_hi=1, H=32, Hkv=8, dim=128, P=64, code="e4m3", dtype="bf16",
             window=0, sink=False, mix=43),
        # a question of 27 tokens over a staged document, every query head with keys of its own (the 7b models' layout)
        dict(name="attend question", kind="attend", n=1, past_lo=8247, past_hi=8247, new_lo=27, new_hi=27, H=32, Hkv=32, dim=128, P=32, code="int8", dtype="bf16",
             window=0, sink=False, mix=44),
        # long prompts behind cached prefixes, four query heads to a key head
        dict(name="attend prompt", kind="attend", n=2, past_lo=4096, past_hi=6200, new_lo=1900, new_hi=2048, H=32, Hkv=8, dim=128, P=64, code="e4m3", dtype="bf16",
             window=0, sink=False, mix=45),
        # ragged prompts in 32 bits with a window and a sink, odd sizes
        dict(name="attend ragged f32", kind="attend", n=5, past_lo=0, past_hi=900, new_lo=3, new_hi=700, H=15, Hkv=5, dim=96, P=16, code="e4m3", dtype="f32",
             window=333, sink=True, mix=46),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {"tables": 1.5e6, "append": 2.0e8, "read": 2.0e8, "attend": 2.6e8}
    while True:
        kind = rng.choice(["tables", "append", "read", "attend", "attend", "attend"])
        mix, P = rng.randrange(1 << 30), rng.choice([16, 32, 64, 128])
        if kind == "tables":
            step = rng.random() < 0.5
            case = dict(kind=kind, n=_log(rng, 1, 600), cached_lo=0, cached_hi=_log(rng, 10, 8192), new_lo=1 if step else 0,
                        new_hi=1 if step else _log(rng, 2, 500), ends=rng.choice([0.0, 0.1]), P=P, tile_rows=1 if step else rng.choice([16, 64, 128]),
                        spare=rng.choice([-9, 0, 0, 50]), mix=mix)
        else:
            Hkv, dim = rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32]), rng.choice([32, 64, 80, 96, 128, 128, 128, 192, 256])
            rest = dict(Hkv=Hkv, dim=dim, P=P, code=rng.choice(["e4m3", "int8"]), dtype=rng.choice(["bf16", "bf16", "f32"]), mix=mix)
            past = _log(rng, 16, 32768)
            low = rng.choice([0, past // 8, past // 2])                        # ragged or nearly alike
            if kind == "read":
                case = dict(kind=kind, n=_log(rng, 1, 40), past_lo=max(low, 1), past_hi=past, **rest)
            else:
                new = rng.choice([1, 1, rng.randint(2, 32), _log(rng, 33, 4000)])
                case = dict(kind=kind, n=_log(rng, 1, 64), past_lo=low, past_hi=past, new_lo=rng.choice([1, new]), new_hi=new, **rest)
            if kind == "attend":
                case.update(H=Hkv * rng.choice([1, 1, 2, 3, 4, 4, 5, 8]), window=rng.choice([0, 0, 0, _log(rng, 2, 2000)]), sink=rng.random() < 0.25)
                if case["H"] > 64:
                    continue
        w = work(case)
        if kind == "attend":
            past, new = _lengths(case)
            longest = max(past) + max(new)
            scores = case["n"] * case["H"] * max(new) * longest               # what the plain form lays out
            rows = case["n"] * case["Hkv"] * case["dim"] * longest
            if w["flops"] > 4.0e11 or scores > 1.0e9 or rows > 1.4e8:
                continue
        if w["bytes"] <= most[kind]:
            return case


def _lengths(case):
    """Tokens that each request has in the cache and tokens that it brings."""
    r = random.Random(case["mix"])
    n = case["n"]

    def some(lo, hi):
        return lo if lo >= hi else min(hi, max(lo, _log(r, max(lo, 1), hi) - (1 if lo == 0 else 0))) if hi > 8 * max(lo, 1) else r.randint(lo, hi)
    if case["kind"] == "tables":
        past = [some(case["cached_lo"], case["cached_hi"]) for _ in range(n)]
        new = [-1 if r.random() < case["ends"] else r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
        return past, new
    past = [some(case["past_lo"], case["past_hi"]) for _ in range(n)]
    new = [r.randint(case["new_lo"], case["new_hi"]) if "new_lo" in case else 0 for _ in range(n)]
    return past, new


def _up(a, b):
    return -(-a // b)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e in 32 bits, exactly, from the exponent's bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _pow2_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _values(gen, shape, dtype):
    """Keys or values as layers make them: normal numbers, channels of different size, some rows larger than others."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    x *= torch.exp2(torch.rand(shape[-1], generator=gen, device=DEV) * 3 - 2)
    x *= torch.exp2(torch.randint(-1, 3, (shape[0],) + (1,) * (len(shape) - 1), generator=gen, device=DEV).float())
    return x.to(dtype)


def _fill(gen, pages, Hkv, P, dim, code):
    """Full pages of quantised values: codes [pages, Hkv, P, dim] and scales [pages, Hkv]."""
    kind, top = CODES[code]
    codes = torch.empty((pages, Hkv, P, dim), dtype=torch.uint8, device=DEV)
    scales = torch.empty((pages, Hkv), device=DEV)
    at, some = 0, max(1, (1 << 26) // (Hkv * P * dim))
    while at < pages:
        x = _values(gen, (min(some, pages - at), Hkv, P, dim), torch.float32)
        m, e = torch.frexp(x.abs().amax((2, 3)) / top)
        s = _pow2(e)
        y = x / s[:, :, None, None]
        codes[at:at + some] = (y.to(kind) if code == "e4m3" else y.round().clamp(-top, top).to(kind)).view(torch.uint8)
        scales[at:at + some] = s
        at += some
    return codes.view(kind), scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) + 1)
    past, new = _lengths(case)
    n, P = case["n"], case["P"]
    host = random.Random("%d %d" % (case["mix"], seed))
    if case["kind"] == "tables":
        # (lengths move a little with the seed; their sums, and so every size, stay near the case's)
        past = [max(case["cached_lo"], p - host.randint(0, 7)) for p in past]
        have = [_up(p, P) for p in past]
        need = sum(_up(p + m, P) - h for p, m, h in zip(past, new, have) if m > 0)
        free = max(0, need + case["spare"])
        pool = sum(_up(p, P) + _up(p + max(m, 0), P) + 1 for p, m in zip(*_lengths(case))) + max(0, case["spare"])
        ids = list(range(pool))
        host.shuffle(ids)
        ids = ids[:sum(have) + free]
        wide = max(1, _up(case["cached_hi"] + max(case["new_hi"], 0), P))
        table = torch.full((n, wide), -1, dtype=torch.int32)
        at = 0
        for s, h in enumerate(have):
            table[s, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
            at += h
        head = host.randrange(pool)
        ring = torch.full((pool,), -1, dtype=torch.int32)
        for j, page in enumerate(ids[at:]):
            ring[(head + j) % pool] = page
        rows = n * max(case["new_hi"], 1)
        rows = sum(max(m, 0) for m in new) + 5 if case["new_hi"] > 1 else rows
        tiles = n + rows // case["tile_rows"]
        state = dict(cached=_i32(past), new=_i32(new), keep=_i32([host.choice([0, 0, min(1, h)]) for h in have]), table=table.to(DEV), ring=ring.to(DEV),
                     ring_state=_i32([head, free, 0, 0]), ring_out=_i32([0, 0, 0, 0]), status=_i32([0, 0]))
        state.update(row_start=_i32([0] * (n + 1)), kv_len=_i32([0] * n), row_seq=_i32([0] * rows), row_pos=_i32([0] * rows),
                     row_slot=torch.zeros(rows, dtype=torch.int64, device=DEV), tiles=_i32([[0] * 4] * tiles))
        return {"case": dict(case), **state}

    Hkv, dim, dtype = case["Hkv"], case["dim"], DTYPES[case["dtype"]]
    total = [p + m for p, m in zip(past, new)]
    have = [_up(t, P) for t in total]
    pages = sum(have) + 3
    ids = list(range(pages))
    host.shuffle(ids)
    table = torch.full((n, max(have + [1])), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(have):
        table[s, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
        at += h
    kc, ks = _fill(gen, pages, Hkv, P, dim, case["code"])
    vc, vs = _fill(gen, pages, Hkv, P, dim, case["code"])
    vc = vc.view(torch.uint8).transpose(2, 3).contiguous().view(vc.dtype)
    state = dict(case=dict(case), table=table.to(DEV), kc=kc, ks=ks, vc=vc, vs=vs)
    counts = past if case["kind"] == "read" else new
    rows = sum(counts)
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(counts))
    first = [0] if case["kind"] == "read" else past
    pos = torch.cat([torch.arange(c) + (0 if case["kind"] == "read" else past[s]) for s, c in enumerate(counts)]) if rows else first
    slot = table[seq, pos // P].long() * P + pos % P
    if case["kind"] in ("append", "read"):
        state["slot"] = slot.to(DEV)
    if case["kind"] == "append":
        state.update(k=_values(gen, (rows, Hkv, dim), dtype), v=_values(gen, (rows, Hkv, dim), dtype))
    if case["kind"] != "attend":
        state.update(k_out=torch.zeros((rows, Hkv, dim), dtype=dtype, device=DEV), v_out=torch.zeros((rows, Hkv, dim), dtype=dtype, device=DEV))
        return state
    T, H = min(128, max(new)), case["H"]
    tiles, at = [], 0
    for s, m in enumerate(new):
        tiles += [[s, past[s] + i, min(T, m - i), at + i] for i in range(0, m, T)]
        at += m
    q = torch.randn((rows, H, dim), generator=gen, device=DEV) * (1.5 / case["dim"] ** 0.5)
    q *= torch.exp2(torch.randint(-1, 2, (rows, H, 1), generator=gen, device=DEV).float())
    state.update(q=q.to(dtype), out=torch.zeros((rows, H, dim), dtype=dtype, device=DEV), tiles=_i32(tiles), tile_rows=T, kv_len=_i32(total), longest=max(total),
                 seq=seq.to(DEV), pos=pos.to(DEV), at=torch.cat([torch.arange(m) for m in new]).to(DEV), widest=max(new), scale=1.0, part=None,
                 sink=torch.randn(H, generator=gen, device=DEV) if case["sink"] else None)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def run(state):
    with torch.inference_mode():
        if own:
            return _run_own(state)
        return {"tables": _plain_tables, "append": _plain_append, "read": _plain_read, "attend": _plain_attend}[state["case"]["kind"]](state)


def _run_own(s):
    B, c = _blocks(), s["case"]
    if c["kind"] == "tables":
        B.page_tables(s["cached"], s["new"], s["table"], c["P"], kv_len=s["kv_len"], row_start=s["row_start"], row_seq=s["row_seq"], row_pos=s["row_pos"],
                      row_slot=s["row_slot"], tiles=s["tiles"], tile_rows=c["tile_rows"], status=s["status"], ring=s["ring"], ring_state=s["ring_state"],
                      ring_out=s["ring_out"], keep=s["keep"])
        return _tables_out(s)
    if c["kind"] == "append":
        B.pages_append(s["k"], s["v"], s["slot"], s["kc"], s["ks"], s["vc"], s["vs"])
    if c["kind"] != "attend":
        B.pages_read(s["slot"], s["kc"], s["ks"], s["vc"], s["vs"], s["k_out"], s["v_out"])
        return _rows_out(s)
    if s["part"] is None:                                                      # a workspace that a program keeps
        floats = B.attn_pages_part(s["q"].shape[0], c["H"], c["Hkv"], c["dim"], s["tiles"].shape[0], s["tile_rows"], s["longest"])
        s["part"] = torch.empty(max(floats, 1), dtype=torch.float32, device=DEV)
    B.attn_pages(s["q"], s["tiles"], s["tile_rows"], s["kv_len"], s["table"], s["kc"], s["ks"], s["vc"], s["vs"], s["out"], scale=s["scale"], window=c["window"],
                 sink=s["sink"], longest=s["longest"], part=s["part"])
    return s["out"]


def _tables_out(s):
    return {k: s[k] for k in ("table", "ring", "row_start", "kv_len", "row_seq", "row_pos", "row_slot", "tiles", "status")} | {"ring_state": s["ring_out"][:2]}


def _rows_out(s):
    """The rows as the values they stand for; of an append also the cache itself, codes and scales."""
    out = {"k": s["k_out"], "v": s["v_out"]}
    return out | {"kc": s["kc"], "ks": s["ks"], "vc": s["vc"], "vs": s["vs"]} if s["case"]["kind"] == "append" else out


# ---- plain forms ----------------------------------------------------------------------------------------------------------------------
def _plain_tables(s):
    c = s["case"]
    P, T, n, wide, cap = c["P"], c["tile_rows"], s["cached"].shape[0], s["table"].shape[1], s["ring"].shape[0]
    cached, new = s["cached"].long().clamp_min(0), s["new"].long()
    ends, count = new < 0, new.clamp_min(0)
    have = (cached + P - 1) // P
    total = (cached + count + P - 1) // P
    rows = s["row_slot"].shape[0]
    stop = count.cumsum(0)
    start = stop - count
    fits = (total <= wide) & (stop <= rows)
    need = torch.where(fits & ~ends, total - have, torch.zeros_like(have))
    upto = need.cumsum(0)
    head, free = s["ring_state"][0].long(), s["ring_state"][1].long()
    granted = ~ends & fits & ((need == 0) | (upto <= free))
    take = torch.where(granted, need, torch.zeros_like(need))
    before = upto - need
    # the tables' new entries
    col = torch.arange(wide, device=DEV)[None]
    fresh = granted[:, None] & (col >= have[:, None]) & (col < total[:, None])
    pages = s["ring"][(head + before[:, None] + col - have[:, None]).clamp_min(0) % cap]
    # the pages of requests that are over go to the ring's end
    keep = s["keep"].long().clamp_min(0)
    gone = ends[:, None] & (col >= keep[:, None]) & (col < have[:, None])
    back = (gone.sum(1).cumsum(0) - gone.sum(1))[:, None] + col - keep[:, None]
    place = torch.where(gone, (head + free + back) % cap, torch.full_like(back, cap))
    ring = torch.cat([s["ring"], s["ring"][:1]])
    ring.scatter_(0, place.reshape(-1), s["table"].reshape(-1))
    s["table"].copy_(torch.where(fresh, pages, s["table"]))
    s["ring"].copy_(ring[:cap])
    taken, given = take.sum(), gone.sum()
    s["ring_out"].copy_(torch.stack([(head + taken) % cap, free - taken + given, torch.zeros_like(taken), torch.zeros_like(taken)]))
    s["kv_len"].copy_(torch.where(ends, torch.zeros_like(cached), torch.where(granted, cached + count, cached)))
    s["row_start"].copy_(torch.cat([torch.zeros_like(stop[:1]), stop]))
    s["status"].copy_(torch.stack([(~granted & ~ends).sum(), torch.where(granted, count, torch.zeros_like(count)).sum()]))
    # rows
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(stop, r, right=True)
    live, at = seq < n, seq.clamp_max(n - 1)
    pos = cached[at] + r - start[at]
    page = s["table"][at, (pos // P).clamp(0, wide - 1)].long()
    none = torch.full_like(r, -1)
    s["row_seq"].copy_(torch.where(live, seq, none))
    s["row_pos"].copy_(torch.where(live, pos, none))
    s["row_slot"].copy_(torch.where(live & granted[at], page * P + pos % P, none))
    # tiles
    cut = torch.where(granted, (count + T - 1) // T, torch.zeros_like(count))
    last = cut.cumsum(0)
    t = torch.arange(s["tiles"].shape[0], device=DEV)
    seq = torch.searchsorted(last, t, right=True)
    live, at = seq < n, seq.clamp_max(n - 1)
    off = (t - (last - cut)[at]) * T
    tiles = torch.stack([at, cached[at] + off, torch.minimum(count[at] - off, torch.full_like(off, T)), start[at] + off], 1)
    empty = torch.tensor([[-1, 0, 0, 0]], device=DEV)
    s["tiles"].copy_(torch.where(live[:, None], tiles, empty))
    return _tables_out(s)


def _step_of(x, top):
    """The smallest power of two with x <= top * step: top = m 2^e, so 2^(f - e), or twice that where x's mantissa is above m."""
    m, e = math.frexp(top)
    y, f = torch.frexp(x)
    return _pow2(torch.where(x > 0, (f - e + (y > m).int()).clamp(EXP_MIN, EXP_MAX), torch.full_like(f, EXP_MIN)))


def _coded(x, code):
    kind, top = CODES[code]
    x = torch.nan_to_num(x, nan=0.0, posinf=top, neginf=-top).clamp(-top, top)
    return x.to(kind) if code == "e4m3" else x.round().to(kind)


def _plain_append(s):
    c = s["case"]
    _plain_write(s["k"], s["slot"], s["kc"], s["ks"], c["P"], c["code"])
    vc = s["vc"].view(torch.uint8).transpose(2, 3).contiguous().view(s["vc"].dtype)
    _plain_write(s["v"], s["slot"], vc, s["vs"], c["P"], c["code"])
    s["vc"].view(torch.uint8).copy_(vc.view(torch.uint8).transpose(2, 3))
    return _plain_read(s)


def _plain_write(x, slot, codes, scales, P, code):
    x = x.float()
    pages, Hkv, _, dim = codes.shape
    page, off = slot // P, slot % P
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    most = torch.zeros((pages, Hkv), device=DEV).scatter_reduce_(0, page[:, None].expand(-1, Hkv), size, "amax")
    old = torch.full((pages,), P, device=DEV).scatter_reduce_(0, page, off, "amin")                  # rows in front of the new ones
    touched = torch.zeros(pages, dtype=torch.bool, device=DEV).index_fill_(0, page, True)
    step = _step_of(most, CODES[code][1])
    step = torch.where((old > 0)[:, None], torch.maximum(step, scales), step)
    ratio = torch.where(touched[:, None], scales / step, torch.ones_like(scales))
    held = torch.arange(P, device=DEV)[None] < old[:, None]
    again = _coded(codes.float() * ratio[:, :, None, None], code).view(torch.uint8)
    grown = (touched[:, None] & (ratio != 1))[:, :, None, None] & held[:, None, :, None]
    raw = codes.view(torch.uint8)
    raw.copy_(torch.where(grown, again, raw))
    scales.copy_(torch.where(touched[:, None], step, scales))
    raw[page, :, off] = _coded(x / scales[page][:, :, None], code).view(torch.uint8)


def _plain_read(s):
    c = s["case"]
    page, off = s["slot"] // c["P"], s["slot"] % c["P"]
    k = s["kc"].view(torch.uint8)[page, :, off].view(s["kc"].dtype)
    v = s["vc"].view(torch.uint8)[page, :, :, off].view(s["vc"].dtype)
    s["k_out"].copy_(k.float() * s["ks"][page][:, :, None])
    s["v_out"].copy_(v.float() * s["vs"][page][:, :, None])
    return _rows_out(s)


def _plain_attend(s):
    c = s["case"]
    n, H, Hkv, dim, P = c["n"], c["H"], c["Hkv"], c["dim"], c["P"]
    G, rows, wide = H // Hkv, s["widest"], s["table"].shape[1]
    table = s["table"].long().clamp_min(0)
    k = s["kc"].view(torch.uint8)[table].view(s["kc"].dtype).float() * s["ks"][table][..., None, None]            # [n, wide, Hkv, P, dim]
    k = k.permute(0, 2, 4, 1, 3).reshape(n, Hkv, dim, wide * P)
    v = s["vc"].view(torch.uint8)[table].view(s["vc"].dtype).float() * s["vs"][table][..., None, None]            # [n, wide, Hkv, dim, P]
    v = v.permute(0, 2, 1, 4, 3).reshape(n, Hkv, wide * P, dim)
    q = torch.zeros((n, rows, H, dim), device=DEV)
    q[s["seq"], s["at"]] = s["q"].float()
    q = q.view(n, rows, Hkv, G, dim).permute(0, 2, 3, 1, 4).reshape(n, Hkv, G * rows, dim)
    score = torch.matmul(q, k).view(n, Hkv, G, rows, wide * P)
    score *= s["scale"]
    pos = torch.full((n, rows), -1, dtype=torch.int64, device=DEV)
    pos[s["seq"], s["at"]] = s["pos"]
    key = torch.arange(wide * P, device=DEV)
    seen = (key <= pos[..., None]) & (key < s["kv_len"].long()[:, None, None])
    if c["window"] > 0:
        seen &= pos[..., None] - key < c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    sink = s["sink"].view(1, Hkv, G, 1, 1) if s["sink"] is not None else None
    if sink is not None:
        top = torch.maximum(top, sink)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(score.view(n, Hkv, G * rows, wide * P), v).view(n, Hkv, G, rows, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(n, rows, H, dim)
    s["out"].copy_(out[s["seq"], s["at"]])
    return s["out"]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------
def work(case):
    past, new = _lengths(case)
    P = case["P"]
    if case["kind"] == "tables":
        rows, live = sum(max(m, 0) for m in new), sum(m >= 0 for m in new)
        pages = sum(_up(p + max(m, 0), P) - _up(p, P) for p, m in zip(past, new)) + sum(_up(p, P) for p, m in zip(past, new) if m < 0)
        tiles = sum(_up(max(m, 0), case["tile_rows"]) for m in new)
        return {"bytes": 20 * len(new) + 4 * live + 8 * pages + 16 * rows + 16 * tiles, "flops": 0}
    Hkv, dim, es = case["Hkv"], case["dim"], 2 if case["dtype"] == "bf16" else 4
    one = 2 * Hkv * dim
    if case["kind"] == "append":
        return {"bytes": sum(new) * (one * (es + 1 + 1 + es) + 16), "flops": 0}                       # rows in, codes out; codes in, rows out
    if case["kind"] == "read":
        return {"bytes": sum(past) * (one * (1 + es) + 8), "flops": 0}
    H, w = case["H"], case["window"]
    seen = keys = 0
    for p, m in zip(past, new):
        if w > 0:
            seen += sum(min(w, p + i + 1) for i in range(m))
            keys += min(p + m, w + m - 1)
        else:
            seen += m * p + m * (m + 1) // 2
            keys += p + m
    return {"bytes": keys * one + 2 * sum(new) * H * dim * es, "flops": 4 * H * dim * seen}


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------------------
def _number(codes, kind):
    """What a code stands for in units of its scale, from its bits: e4m3 has 4 exponent bits (bias 7) and 3 bits behind the point."""
    b = codes.contiguous().view(torch.uint8).long()
    if kind == "int8":
        return torch.where(b > 127, b - 256, b).double()
    e, m = (b >> 3) & 15, (b & 7).double()
    size = torch.where(e > 0, (1 + m / 8) * _pow2_64(e - 7), m / 8 * 2.0 ** -6)
    return torch.where(b > 127, -size, size)


def _nearest(x, kind):
    """The code's number nearest to x, ties to even, |x| within range."""
    if kind == "int8":
        return torch.round(x)
    ulp = _pow2_64(torch.frexp(x.abs().clamp_min(2.0 ** -6))[1].clamp(-5, 9) - 4)
    return torch.round(x / ulp) * ulp


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    past, new = _lengths(case)
    P, Hkv, dim, kind = case["P"], case["Hkv"], case["dim"], case["code"]
    with torch.inference_mode():
        if case["kind"] == "append":
            return _exact_append(s, past, new)
        pages = [s["table"][i, :_up(p + m, P)].long() for i, (p, m) in enumerate(zip(past, new))]
        if case["kind"] == "read":
            ks, vs = [], []
            for i, p in enumerate(past):
                ks.append((_number(s["kc"].view(torch.uint8)[pages[i]], kind) * s["ks"].double()[pages[i]][..., None, None]).transpose(1, 2).reshape(-1, Hkv, dim)[:p])
                vs.append((_number(s["vc"].view(torch.uint8)[pages[i]], kind) * s["vs"].double()[pages[i]][..., None, None]).permute(0, 3, 1, 2).reshape(-1, Hkv, dim)[:p])
            return {"k": torch.cat(ks), "v": torch.cat(vs)}
        G, out, at = case["H"] // Hkv, torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0
        for i, (p, m) in enumerate(zip(past, new)):
            key = torch.arange(p + m, device=DEV)
            row = torch.arange(p, p + m, device=DEV)
            hidden = key[None] > row[:, None]
            if case["window"] > 0:
                hidden |= row[:, None] - key[None] >= case["window"]
            for g in range(Hkv):
                k = _number(s["kc"].view(torch.uint8)[pages[i], g], kind) * s["ks"].double()[pages[i], g][:, None, None]
                k = k.reshape(-1, dim)[:p + m]
                v = _number(s["vc"].view(torch.uint8)[pages[i], g], kind) * s["vs"].double()[pages[i], g][:, None, None]
                v = v.transpose(1, 2).reshape(-1, dim)[:p + m]
                for h in range(g * G, g * G + G):
                    z = s["q"][at:at + m, h].double() @ k.T * s["scale"]
                    z = z.masked_fill(hidden, -math.inf)
                    if s["sink"] is not None:
                        z = torch.cat([z, s["sink"][h].double().expand(m, 1)], 1)
                    out[at:at + m, h] = torch.softmax(z, 1)[:, :p + m] @ v
            at += m
        return out


def _exact_append(s, past, new):
    case = s["case"]
    P, Hkv, dim, kind = case["P"], case["Hkv"], case["dim"], case["code"]
    top, got = CODES[kind][1], {}
    for name, x, codes, scales in (("k", s["k"], s["kc"], s["ks"]), ("v", s["v"], s["vc"], s["vs"])):
        num = _number(codes, kind)
        num = num.transpose(2, 3).contiguous() if name == "v" else num
        sc, x, back, at = scales.double().clone(), x.double(), [], 0
        for i, (p, m) in enumerate(zip(past, new)):
            done = 0
            while done < m:
                page, off = int(s["table"][i, (p + done) // P]), (p + done) % P
                k = min(P - off, m - done)
                rows = x[at + done:at + done + k]
                big = rows.abs().amax((0, 2))
                e = torch.frexp(big / top)[1].clamp(EXP_MIN, EXP_MAX)
                e = torch.where(top * _pow2_64(e - 1) >= big, e - 1, e)
                step = _pow2_64(e.clamp(EXP_MIN, EXP_MAX))
                if off:
                    step = torch.maximum(step, sc[page])
                    num[page, :, :off] = _nearest(num[page, :, :off] * (sc[page] / step)[:, None, None], kind)
                num[page, :, off:off + k] = _nearest(rows / step[None, :, None], kind).transpose(0, 1)
                sc[page] = step
                back.append((num[page, :, off:off + k] * step[:, None, None]).transpose(0, 1))
                done += k
            at += m
        num = num.transpose(2, 3).contiguous() if name == "v" else num
        got[name], got[name + "c"], got[name + "s"] = torch.cat(back), num if kind == "e4m3" else None, sc
    return got
