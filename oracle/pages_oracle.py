"""The paged 8-bit cache in plain numpy, in 64 bits, one element, row or sequence after the other: what the kernels behind ``pcb_page_tables``,
``pcb_pages_append``, ``pcb_pages_read`` and ``pcb_attn_pages`` are held to."""
import numpy as np

TOP = {"e4m3": 448.0, "int8": 127.0}


def e4m3_value(code):
    """Sign, four exponent bits (bias 7), three bits behind the point; 0x7f and 0xff are no numbers."""
    b = np.asarray(code).view(np.uint8).astype(np.int64)
    e, m = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(e > 0, np.ldexp(1 + m / 8, e - 7), np.ldexp(m / 8, -6))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b > 127, -v, v)


def value(code, kind):
    return e4m3_value(code) if kind == "e4m3" else np.asarray(code).view(np.int8).astype(np.float64)


_E4M3 = e4m3_value(np.arange(127, dtype=np.uint8))                  # 0 .. 448, ascending


def encode(x, kind):
    """Numbers in units of the scale -> codes (uint8): clamped, to the nearest, ties to the even code; what is not a number is 0."""
    x = np.asarray(x, dtype=np.float64)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -TOP[kind], TOP[kind])
    if kind == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    size = np.abs(x)
    hi = np.searchsorted(_E4M3, size, side="left").clip(0, 126)
    lo = (hi - 1).clip(0)
    low, high = size - _E4M3[lo], _E4M3[hi] - size
    code = np.where((low < high) | ((low == high) & (lo % 2 == 0)), lo, hi)
    return (code + np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_for(most, kind):
    e = -40
    while e < 40 and most > TOP[kind] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(x, slots, codes, scales, P, kind):
    """Rows ``x`` [rows, H, dim] into ``codes`` uint8 [pages, H, P, dim] (row by row) and ``scales`` [pages, H]: new copies of both."""
    codes, scales, x = codes.copy(), np.array(scales, dtype=np.float64), np.asarray(x, dtype=np.float64)
    r = 0
    while r < len(slots):
        if not 0 <= slots[r] < codes.shape[0] * P:
            r += 1
            continue
        page, n = slots[r] // P, 1
        while r + n < len(slots) and slots[r + n] // P == page and slots[r + n] >= 0:
            n += 1
        offs = [int(s % P) for s in slots[r:r + n]]
        for h in range(codes.shape[1]):
            new = x[r:r + n, h]
            s = scale_for(np.abs(new[np.isfinite(new)]).max(initial=0.0), kind)
            first = min(offs)
            if first > 0:
                old = scales[page, h]
                s = max(s, old)
                if s > old:
                    codes[page, h, :first] = encode(value(codes[page, h, :first], kind) * (old / s), kind)
            scales[page, h] = s
            for i, off in enumerate(offs):
                codes[page, h, off] = encode(new[i] / s, kind)
        r += n
    return codes, scales


def read(slots, codes, scales, P, kind, dim):
    out = np.zeros((len(slots), codes.shape[1], dim))
    for r, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * P:
            out[r] = value(codes[s // P, :, s % P], kind) * np.asarray(scales, dtype=np.float64)[s // P][:, None]
    return out


def tables(cached, brings, table, P, rows, *, tile_rows=1, n_tiles=0, ring=None, head=0, free=0, keep=None):
    """A step's tables, sequence by sequence; -> a dict of what ``pcb_page_tables`` writes."""
    table = np.array(table, dtype=np.int64)
    n, wide = table.shape
    ring = None if ring is None else np.array(ring, dtype=np.int64)
    front = None if ring is None else ring.copy()
    upto = taken = given = at = refused = granted_rows = 0
    out = dict(kv_len=[], row_start=[0], row_seq=[-1] * rows, row_pos=[-1] * rows, row_slot=[-1] * rows, tiles=[])
    for s in range(n):
        c, b = max(int(cached[s]), 0), int(brings[s])
        have = -(-c // P)
        if b < 0:
            k = 0 if keep is None else max(int(keep[s]), 0)
            if ring is not None and have <= wide:
                for j in range(k, have):
                    ring[(head + free + given) % len(ring)] = table[s, j]
                    given += 1
            out["kv_len"].append(0)
            out["row_start"].append(at)
            continue
        total = -(-(c + b) // P)
        fits = total <= wide and at + b <= rows
        need = total - have if ring is not None and fits else 0
        upto += need
        ok = fits and (need == 0 or upto <= free)
        if ok:
            for j in range(need):
                table[s, have + j] = front[(head + taken) % len(ring)]
                taken += 1
            granted_rows += b
            for i in range(0, b, tile_rows):
                out["tiles"].append([s, c + i, min(tile_rows, b - i), at + i])
        else:
            refused += 1
        for i in range(b):
            if at + i < rows:
                out["row_seq"][at + i], out["row_pos"][at + i] = s, c + i
                if ok and table[s, (c + i) // P] >= 0:
                    out["row_slot"][at + i] = int(table[s, (c + i) // P]) * P + (c + i) % P
        out["kv_len"].append(c + b if ok else c)
        at += b
        out["row_start"].append(at)
    out["tiles"] += [[-1, 0, 0, 0]] * (n_tiles - len(out["tiles"]))
    out.update(table=table, status=[refused, granted_rows])
    if ring is not None:
        out.update(ring=ring, ring_state=[(head + taken) % len(ring), free - taken + given])
    return {k: np.array(v) for k, v in out.items()}


def kept(cached, brings, table, P):
    """Of each sequence that is over, how many of its first pages one that goes on, or one before it that is over, has too (0: it goes on)."""
    table = np.asarray(table)
    pages = [[int(p) for p in table[s, :min(-(-max(int(c), 0) // P), table.shape[1])]] for s, c in enumerate(cached)]
    out = []
    for s, mine in enumerate(pages):
        most = 0
        for t, other in enumerate(pages):
            if brings[s] < 0 and t != s and (brings[t] >= 0 or t < s):
                n = 0
                while n < min(len(mine), len(other)) and mine[n] == other[n]:
                    n += 1
                most = max(most, n)
        out.append(most)
    return np.array(out)


def attend(q, seqs, positions, kv_len, table, kcodes, kscale, vcodes, vscale, P, kind, scale, window=0, sink=None):
    """Rows ``q`` [rows, H, dim] at ``positions`` of ``seqs`` (below zero: the row is left out, zeros); codes uint8, values' [pages, Hkv, dim, P]."""
    q = np.asarray(q, dtype=np.float64)
    rows, H, dim = q.shape
    pages, Hkv = kcodes.shape[:2]
    out = np.zeros((rows, H, dim))
    held = {}
    for r in range(rows):
        s = int(seqs[r])
        if s < 0:
            continue
        if s not in held:
            n = min(int(kv_len[s]), table.shape[1] * P)
            n = max(n, 0)
            pg = np.asarray(table[s, :-(-n // P)], dtype=np.int64)
            good = (pg >= 0) & (pg < pages)
            use = np.where(good, pg, 0)
            k = (value(kcodes[use], kind) * np.asarray(kscale, np.float64)[use][..., None, None]).transpose(1, 0, 2, 3).reshape(Hkv, -1, dim)[:, :n]
            v = (value(vcodes[use], kind) * np.asarray(vscale, np.float64)[use][..., None, None]).transpose(1, 0, 3, 2).reshape(Hkv, -1, dim)[:, :n]
            held[s] = k, v, np.repeat(good, P)[:n]
        k, v, good = held[s]
        j = np.arange(k.shape[1])
        see = good & (j <= positions[r]) & ((window <= 0) | (positions[r] - j < window))
        for h in range(H):
            g = h // (H // Hkv)
            if not see.any():
                continue
            z = scale * (k[g][see] @ q[r, h])
            top = z.max() if sink is None else max(z.max(), float(sink[h]))
            e = np.exp(z - top)
            den = e.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - top))
            out[r, h] = e @ v[g][see] / den
    return out
