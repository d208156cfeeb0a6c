"""The paged 8-bit cache on the GPU: tables, rows into pages and back and attention over them, each against the numpy oracle in 64 bits, and a run of them together."""
import numpy as np
import pytest
import torch

from oracle import pages_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---- tables -------------------------------------------------------------------------------------------------------------------------------
def batch(rng, n, P, cached_hi, new_hi, ends, spare, wide=None):
    cached = [int(v) for v in rng.integers(0, cached_hi + 1, n)]
    brings = [-1 if rng.random() < ends else int(v) for v in rng.integers(0, new_hi + 1, n)]
    have = [-(-c // P) for c in cached]
    need = sum(-(-(c + max(b, 0)) // P) - h for c, b, h in zip(cached, brings, have))
    free = max(0, need + spare)
    wide = wide or -(-(cached_hi + new_hi) // P) + 1
    ids = rng.permutation(sum(have) + free + 3)
    table = np.full((n, wide), -1)
    at = 0
    for s, h in enumerate(have):
        table[s, :h] = ids[at:at + h]
        at += h
    cap = len(ids)
    head = int(rng.integers(0, cap))
    ring = np.full(cap, -7)
    for j in range(free):
        ring[(head + j) % cap] = ids[at + j]
    keep = [int(rng.integers(0, 2)) if h else 0 for h in have]
    return cached, brings, table, ring, head, free, keep


def run_tables(cached, brings, table, P, rows, *, tile_rows=1, ring=None, head=0, free=0, keep=None, in_place=False, pad_table=0):
    from promptcache_amd import _blocks as B
    n, wide = table.shape
    tab = torch.full((n, wide + pad_table), -5, dtype=torch.int32, device=DEV)[:, :wide]
    tab.copy_(torch.from_numpy(table))
    got = dict(kv_len=i32([9] * n), row_start=i32([9] * (n + 1)), row_seq=i32([9] * rows), row_pos=i32([9] * rows), row_slot=torch.full((rows,), 9, dtype=torch.int64, device=DEV),
               tiles=torch.full((n + rows // tile_rows, 4), 9, dtype=torch.int32, device=DEV), status=i32([9, 9]))
    c = i32(cached)
    if in_place:
        got["kv_len"] = c
    kw = {}
    if ring is not None:
        st = i32([head, free, 0, 0])
        kw = dict(ring=i32(ring), ring_state=st, ring_out=st if in_place else i32([0, 0, 0, 0]), keep=None if keep is None else i32(keep))
    B.page_tables(c, i32(brings), tab, P, tile_rows=tile_rows, **got, **kw)
    got["table"] = tab
    if ring is not None:
        got.update(ring=kw["ring"], ring_state=kw["ring_out"][:2])
        assert kw["ring_out"][2:].tolist() == [0, 0]
    return {k: v.cpu().numpy() for k, v in got.items()}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n, P, cached_hi, new_hi, ends, spare, tile_rows, extra", [
    (1, 16, 0, 1, 0.0, 0, 1, 0), (1, 64, 300, 1, 0.0, -1, 1, 0), (3, 16, 40, 33, 0.0, 2, 16, 7), (64, 64, 8192, 1, 0.1, 0, 1, 9), (200, 32, 90, 3, 0.3, -20, 2, 0),
    (257, 16, 50, 1, 0.0, -3, 1, 4), (517, 16, 2048, 400, 0.1, -40, 128, 5), (1500, 128, 700, 9, 0.2, 3, 4, 11), (2, 128, 0, 9000, 0.0, 0, 64, 100), (40, 16, 0, 0, 0.5, 0, 1, 6)])
def test_tables(n, P, cached_hi, new_hi, ends, spare, tile_rows, extra, in_place):
    rng = np.random.default_rng(n * 1000 + P)
    cached, brings, table, ring, head, free, keep = batch(rng, n, P, cached_hi, new_hi, ends, spare)
    rows = sum(max(b, 0) for b in brings) + extra
    want = O.tables(cached, brings, table, P, rows, tile_rows=tile_rows, n_tiles=n + rows // tile_rows, ring=ring, head=head, free=free, keep=keep)
    got = run_tables(cached, brings, table, P, rows, tile_rows=tile_rows, ring=ring, head=head, free=free, keep=keep, in_place=in_place, pad_table=n % 3)
    for k, v in want.items():
        assert np.array_equal(got[k].reshape(v.shape), v), k


@pytest.mark.parametrize("rows_less, wide", [(1, None), (30, None), (0, 2), (5, 3)])
def test_tables_of_sequences_that_do_not_fit(rows_less, wide):
    """Rows behind the buffer's end, and more pages than a table has: the sequence is refused and keeps what it had."""
    rng = np.random.default_rng(5)
    cached, brings, table, ring, head, free, keep = batch(rng, 20, 16, 20, 30, 0.1, 0, wide=wide or 5)
    rows = sum(max(b, 0) for b in brings) - rows_less
    want = O.tables(cached, brings, table, 16, rows, tile_rows=8, n_tiles=20 + rows // 8, ring=ring, head=head, free=free, keep=keep)
    assert want["status"][0] > 0
    got = run_tables(cached, brings, table, 16, rows, tile_rows=8, ring=ring, head=head, free=free, keep=keep)
    for k, v in want.items():
        assert np.array_equal(got[k].reshape(v.shape), v), k


def test_tables_without_a_ring():
    """Slots of rows whose pages are there already (a cached sequence read back)."""
    rng = np.random.default_rng(6)
    table = rng.permutation(60).reshape(4, 15)
    table[2, 3] = -1                                                  # a hole: its rows have no slot
    want = O.tables([0, 16, 0, 7], [240, 3, 100, 0], table, 16, 350)
    got = run_tables([0, 16, 0, 7], [240, 3, 100, 0], table, 16, 350)
    for k in ("row_slot", "row_pos", "row_seq", "kv_len", "table"):
        assert np.array_equal(got[k], want[k]), k


def test_a_ring_state_out_of_its_range_stays_inside():
    table = np.full((2, 4), -1)
    for head, free in ((-3, 4), (1000, 1000), (2, -5)):
        got = run_tables([0, 0], [20, 20], table, 16, 40, ring=np.arange(6), head=head, free=free)
        assert got["table"].max() < 6 and got["row_slot"].max() < 96


# ---- rows into pages, and back ------------------------------------------------------------------------------------------------------------
class Pool:
    """Pages on the device and the oracle's copy of them."""

    def __init__(self, pages, Hkv, P, dim, kind, seed=0):
        rng = np.random.default_rng(seed)
        self.P, self.kind, self.dim = P, kind, dim
        self.kc = rng.integers(0, 256, (pages, Hkv, P, dim), dtype=np.uint8)      # what memory held before: any code
        self.vc = rng.integers(0, 256, (pages, Hkv, P, dim), dtype=np.uint8)      # (the oracle keeps both row by row)
        self.ks, self.vs = (np.exp2(rng.integers(-9, 3, (pages, Hkv))).astype(np.float32) for _ in range(2))
        t = KINDS[kind]
        self.dev = [torch.from_numpy(self.kc).to(DEV).view(t), torch.from_numpy(self.ks).to(DEV),
                    torch.from_numpy(np.ascontiguousarray(self.vc.transpose(0, 1, 3, 2))).to(DEV).view(t), torch.from_numpy(self.vs).to(DEV)]

    def append(self, k, v, slots):
        from promptcache_amd import _blocks as B
        B.pages_append(k, v, torch.tensor(slots, dtype=torch.int64, device=DEV), *self.dev)
        self.kc, self.ks = O.append(k.double().cpu().numpy(), slots, self.kc, self.ks, self.P, self.kind)
        self.vc, self.vs = O.append(v.double().cpu().numpy(), slots, self.vc, self.vs, self.P, self.kind)

    def check(self):
        kc, ks, vc, vs = (t.view(torch.uint8).cpu().numpy() if t.dtype in KINDS.values() else t.cpu().numpy() for t in self.dev)
        assert np.array_equal(ks, self.ks) and np.array_equal(vs, self.vs)
        same = lambda a, b: np.array_equal(np.where(a == 128, 0, a) if self.kind == "e4m3" else a, np.where(b == 128, 0, b) if self.kind == "e4m3" else b)  # noqa: E731  (-0 is 0)
        assert same(kc, self.kc) and same(vc, self.vc.transpose(0, 1, 3, 2))


def rows_of(gen, shape, dtype, wide=3):
    x = torch.randn(shape, generator=gen, device=DEV) * torch.exp2(torch.randint(-wide, wide + 1, (shape[0],) + (1,) * (len(shape) - 1), generator=gen, device=DEV).float())
    return x.to(dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("P, Hkv, dim", [(16, 1, 16), (16, 3, 80), (32, 2, 64), (64, 8, 128), (128, 2, 256), (128, 1, 48)])
def test_append_and_read(P, Hkv, dim, kind, dtype):
    """Steps of one row, of pieces of pages and of many pages; scales that grow; rows without a slot; what lies behind stays as it was."""
    gen = torch.Generator(device=DEV).manual_seed(P + dim)
    pool = Pool(12, Hkv, P, dim, kind, seed=dim)
    pages = [7, 2, 9, 0, 11, 4]
    slot = lambda i: pages[i // P] * P + i % P  # noqa: E731
    at, steps = 0, [1, 1, 3, P // 2 + 1, 1, P, 2 * P + 5, 1, 2]
    for i, n in enumerate(steps):
        n = min(n, 6 * P - at)
        slots = [slot(at + j) for j in range(n)] + [-1, -1]                       # a padded batch
        if i == 4:
            slots = [-1, 12 * P, 10 ** 12] + slots                                # places that no pool has
        k, v = rows_of(gen, (len(slots), Hkv, dim), DT[dtype]), rows_of(gen, (len(slots), Hkv, dim), DT[dtype])
        pool.append(k, v, slots)
        pool.check()
        at += n
    from promptcache_amd import _blocks as B
    slots = [slot(i) for i in range(at)]
    slots = slots[5:] + [-1] + slots[:5] + [12 * P] + slots[::-1][:7]             # rotated, a gap, some backwards
    k, v = (torch.full((len(slots), Hkv, dim), 77.0, dtype=DT[dtype], device=DEV) for _ in range(2))
    B.pages_read(torch.tensor(slots, dtype=torch.int64, device=DEV), *pool.dev, k, v)
    none = np.array([not 0 <= s < 12 * P for s in slots])
    for got, codes, scales in ((k, pool.kc, pool.ks), (v, pool.vc, pool.vs)):
        want = O.read(slots, codes, scales, P, kind, dim)
        want[none] = 77.0
        assert np.array_equal(got.double().cpu().numpy(), want)                   # a code times a power of two is a bf16 number


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [1, 37, 700])
def test_append_many_sequences_at_once(n, kind):
    """Rows of many sequences in one call, a page of each; windows of one row and of sixteen."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    rng = np.random.default_rng(n)
    P, Hkv, dim = 16, 24, 32
    pool = Pool(n + 40, Hkv, P, dim, kind)
    pages = rng.permutation(n + 40)
    slots = []
    for s in range(n):
        off = int(rng.integers(0, P))
        slots += [int(pages[s]) * P + off + j for j in range(int(rng.integers(1, P - off + 1)))]
    x = rows_of(gen, (len(slots), 2, Hkv, dim), torch.bfloat16)
    pool.append(x[:, 0], x[:, 1], slots)                                          # strided rows
    pool.check()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_of_numbers_at_the_edges(kind):
    """Zeros, numbers that are not finite, the largest and smallest, scales at both ends, ties."""
    P, dim = 16, 32
    top = O.TOP[kind]
    pool = Pool(14, 1, P, dim, kind)
    gen = torch.Generator(device=DEV).manual_seed(1)
    rows = [torch.zeros(dim), torch.full((dim,), float("inf")), torch.full((dim,), float("nan")), torch.full((dim,), 3e38), torch.full((dim,), 1e-38), torch.full((dim,), 2.0 ** -49),
            torch.full((dim,), top), torch.full((dim,), float(np.nextafter(np.float32(top), np.float32(1e9)))), torch.arange(dim) * 0.5, torch.arange(dim) + 96.5,
            torch.full((dim,), -1e-30), torch.tensor([float("nan"), 1.0, float("-inf"), -2.0] * (dim // 4))]
    for page, r in enumerate(rows):                                               # as a page's first row, then in front of ordinary ones
        pool.append(r[None, None].to(DEV), (-r)[None, None].to(DEV), [page * P])
        pool.check()
    for page in range(len(rows)):
        k = rows_of(gen, (2, 1, dim), torch.float32)
        pool.append(k, k * 2.0 ** -20, [page * P + 1, page * P + 2])
        pool.check()
    for page, r in enumerate(rows):
        pool.append(r[None, None].to(DEV), (-r)[None, None].to(DEV), [page * P + 3])
        pool.check()


def test_append_with_heads_outside_and_another_stream():
    """Rows that lie head by head, on a stream of their own."""
    P, Hkv, dim = 32, 4, 64
    gen = torch.Generator(device=DEV).manual_seed(2)
    pool = Pool(6, Hkv, P, dim, "e4m3")
    x = rows_of(gen, (50, 2 * Hkv, dim), torch.float32).transpose(0, 1).contiguous().transpose(0, 1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        pool.append(x[:, :Hkv], x[:, Hkv:], [3 * P + i if i < P else 5 * P + i - P for i in range(50)])
    torch.cuda.current_stream().wait_stream(st)
    pool.check()


@pytest.mark.parametrize("kind, dtype", [("e4m3", "bf16"), ("int8", "f32")])
def test_rows_beyond_the_caches(kind, dtype):
    """Calls of so many rows that these go past the caches store and read what calls of few rows do."""
    from promptcache_amd import _blocks as B
    P, Hkv, dim, n = 64, 16, 128, 4300
    gen = torch.Generator(device=DEV).manual_seed(3)
    assert n * Hkv * dim * (4 if dtype == "bf16" else 8) > 32 << 20
    pools = [Pool(n // P + 3, Hkv, P, dim, kind).dev for _ in range(2)]
    slots = torch.arange(7, 7 + n, dtype=torch.int64, device=DEV)
    k, v = (rows_of(gen, (n, Hkv, dim), DT[dtype]) for _ in range(2))
    B.pages_append(k, v, slots, *pools[0])
    at = 0
    for m in (57, 1024, 1600, 1619):                                 # (cut where pages end)
        B.pages_append(k[at:at + m], v[at:at + m], slots[at:at + m], *pools[1])
        at += m
    assert at == n and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*pools))
    whole, parts = ([torch.zeros_like(k), torch.zeros_like(v)] for _ in range(2))
    B.pages_read(slots, *pools[0], *whole)
    for i in range(0, n, 500):
        B.pages_read(slots[i:i + 500], *pools[0], *(t[i:i + 500] for t in parts))
    assert torch.equal(whole[0], parts[0]) and torch.equal(whole[1], parts[1])
    some = np.arange(n - 40, n)
    for got, codes, scales in ((whole[0], pools[0][0].view(torch.uint8), pools[0][1]), (whole[1], pools[0][2].view(torch.uint8).transpose(2, 3), pools[0][3])):
        want = O.read(7 + some, codes.cpu().numpy(), scales.cpu().numpy(), P, kind, dim)
        assert np.array_equal(got[n - 40:].double().cpu().numpy(), want)


# ---- attention ----------------------------------------------------------------------------------------------------------------------------
class Requests:
    """Sequences of given lengths in a pool of written pages (garbage behind them), and queries of their last rows."""

    def __init__(self, past, new, H, Hkv, dim, P, kind, dtype, seed=0, spread=1.0, scales=(-6, 1)):
        self.past, self.new, self.H, self.P, self.kind, self.dtype = past, new, H, P, kind, DT[dtype]
        rng = np.random.default_rng(seed)
        total = [p + m for p, m in zip(past, new)]
        need = [-(-t // P) for t in total]
        pages = sum(need) + 2
        ids = rng.permutation(pages)
        self.table = np.full((len(past), max(need + [1]) + 1), -1)
        at = 0
        for s, h in enumerate(need):
            self.table[s, :h] = ids[at:at + h]
            at += h
        self.kc, self.vc = (rng.integers(0, 256, (pages, Hkv, P, dim), dtype=np.uint8) for _ in range(2))
        draw = lambda shape: O.encode(rng.normal(0, 100 if kind == "e4m3" else 35, shape), kind)  # noqa: E731
        for s, t in enumerate(total):
            for i in range(need[s]):
                n = min(P, t - i * P)
                self.kc[self.table[s, i], :, :n], self.vc[self.table[s, i], :, :n] = draw((Hkv, n, dim)), draw((Hkv, n, dim))
        self.ks, self.vs = (np.exp2(rng.integers(*scales, (pages, Hkv))).astype(np.float32) for _ in range(2))
        self.vc = np.ascontiguousarray(self.vc.transpose(0, 1, 3, 2))
        self.kv = total
        self.seqs = np.repeat(np.arange(len(past)), new)
        self.pos = np.concatenate([np.arange(p, p + m) for p, m in zip(past, new)] or [[]]).astype(np.int64)
        rms = (100 if kind == "e4m3" else 35) * 2.0 ** (scales[1] - 2)
        q = rng.normal(0, spread / rms / dim ** 0.5, (sum(new), H, dim)) * np.exp2(rng.integers(-1, 2, (sum(new), H, 1)))
        self.q = torch.from_numpy(q).to(DEV, self.dtype)

    def tiles(self, T):
        out, at = [], 0
        for s, m in enumerate(self.new):
            out += [[s, self.past[s] + i, min(T, m - i), at + i] for i in range(0, m, T)]
            at += m
        return out

    def device(self):
        t = KINDS[self.kind]
        return [torch.from_numpy(self.table).to(DEV, torch.int32), torch.from_numpy(self.kc).to(DEV).view(t), torch.from_numpy(self.ks).to(DEV),
                torch.from_numpy(self.vc).to(DEV).view(t), torch.from_numpy(self.vs).to(DEV)]

    def run(self, T, *, scale=1.0, window=0, sink=None, q=None, out=None, tiles=None, longest=0, part=None, kv=None):
        from promptcache_amd import _blocks as B
        q = self.q if q is None else q
        out = torch.full((self.q.shape[0], self.H, q.shape[2]), 55.0, dtype=self.dtype, device=DEV) if out is None else out
        table, kc, ks, vc, vs = self.device()
        tiles = torch.tensor(self.tiles(T) if tiles is None else tiles, dtype=torch.int32, device=DEV).reshape(-1, 4)
        B.attn_pages(q, tiles, T, i32(self.kv if kv is None else kv), table, kc, ks, vc, vs, out, scale=scale, window=window, longest=longest, part=part,
                     sink=None if sink is None else torch.tensor(sink, dtype=torch.float32, device=DEV))
        return out

    def want(self, *, scale=1.0, window=0, sink=None, kv=None):
        """(result, how far a kernel may be from it).

        With p_j the weights and A = sum_j p_j |v_j|: a score is a sum of dim products of exact halves (fp32: sums of two, off by 2^-23 of the product) in fp32, off by at
        most (dim + 8) 2^-24 of scale sum_d |q_d k_jd| =: S_j, and its exponential by that and 2^-21 more; weights are rounded to 2^-11 (fp32: 2^-22) of themselves, or 2^-39 of the
        largest product of a weight and a scale; sums over n keys in fp32 by n 2^-24 of A at most.  A relative error e of every p_j moves the quotient by at most 2 e A."""
        q = self.q.double().cpu().numpy()
        kv = self.kv if kv is None else kv
        args = (self.seqs, self.pos, kv, self.table, self.kc, self.ks, self.vc, self.vs, self.P, self.kind, scale, window, sink)
        out = O.attend(q, *args)
        flip = np.uint8(127) if self.kind == "e4m3" else None
        vabs = self.vc & flip if flip is not None else np.abs(self.vc.view(np.int8).astype(np.int16)).clip(0, 127).astype(np.int8).view(np.uint8)
        A = O.attend(q, self.seqs, self.pos, kv, self.table, self.kc, self.ks, vabs, self.vs, self.P, self.kind, scale, window, sink)
        kmax = O.TOP[self.kind] * float(self.ks.max())
        n, dim = max(list(kv) + [1]), q.shape[2]
        S = scale * np.minimum(np.abs(q).sum(-1) * kmax, np.linalg.norm(q, axis=-1) * kmax * dim ** 0.5)[..., None]
        one = 2.0 ** -11 if self.dtype == torch.bfloat16 else 2.0 ** -22
        half = torch.finfo(self.dtype).eps / 2
        tol = half * np.abs(out) + A * (2 * ((dim + 8) * 2.0 ** -24 * S + 2.0 ** -21 * (1 if self.dtype == torch.bfloat16 else 0.25) + one) + n * 2.0 ** -24) + n * 2.0 ** -38 * A.max(initial=0.0)
        return out, tol * (1 + half)

    def check(self, got, **kw):
        want, tol = self.want(**kw)
        got = got.double().cpu().numpy()
        off = np.abs(got - want)
        assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), np.argwhere(~(off <= tol))[:5])


SIZES = [  # past, new, H, Hkv, dim, P, tile rows
    ([0], [1], 1, 1, 16, 16, 1), ([300, 7, 0, 63, 64, 1000], [1] * 6, 8, 2, 64, 16, 1), ([129, 4, 400], [1, 1, 1], 16, 1, 128, 64, 1), ([70, 1], [1, 1], 20, 1, 80, 32, 1),
    ([500], [1], 6, 2, 256, 128, 1), ([90, 0, 33], [5, 17, 3], 4, 4, 32, 32, 4), ([0, 200], [40, 31], 6, 3, 96, 64, 16), ([0], [130], 5, 5, 128, 128, 128),
    ([1500], [27], 4, 4, 128, 32, 27), ([10, 60, 0, 5], [100, 1, 65, 0], 8, 2, 192, 16, 64), ([3], [70], 10, 2, 48, 16, 128), ([2200, 100], [2, 1], 3, 3, 128, 64, 2),
    ([0, 77], [9, 260], 7, 1, 64, 16, 100), ([640], [33], 16, 8, 128, 64, 64),
    # results of many workgroups put together: by the last of them, in a launch of their own, of blocks of 128 columns
    ([9000], [1], 2, 1, 64, 64, 1), ([5000], [9], 3, 1, 32, 16, 9), ([3000, 2100], [50, 3], 2, 1, 128, 32, 64), ([700], [1], 70, 1, 32, 16, 1), ([2000], [6], 12, 2, 96, 128, 6),
    ([1800, 30], [1, 1], 5, 5, 192, 16, 1), ([2500], [40], 4, 1, 192, 64, 40), ([1300], [3], 4, 2, 256, 32, 3), ([900], [45], 3, 1, 256, 128, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("past, new, H, Hkv, dim, P, T", SIZES)
def test_attention(past, new, H, Hkv, dim, P, T, kind, dtype):
    r = Requests(past, new, H, Hkv, dim, P, kind, dtype, seed=dim + P)
    r.check(r.run(T))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("past, new, H, Hkv, dim, P, T", [x for x in SIZES if x[-1] > 1])
def test_attention_in_blocks_of_128(past, new, H, Hkv, dim, P, T, kind, dtype):
    """A bound of the lengths that has short work look like much: blocks of 128 columns where there are more than 32."""
    r = Requests(past, new, H, Hkv, dim, P, kind, dtype, seed=len(new) + dim)
    r.check(r.run(T, longest=1 << 22))


LONG = [  # work enough for blocks of 128, in key runs or not, of four waves and of eight; the last two: window, sink
    ([4000], [128], 16, 2, 64, 32, 128, 0, 0), ([9000, 300], [100, 700], 12, 2, 96, 16, 64, 0, 0), ([5000], [900], 16, 4, 128, 64, 128, 0, 1), ([5000], [900], 16, 4, 128, 64, 128, 700, 1),
    ([2000], [1500], 32, 8, 48, 128, 128, 0, 0), ([3000], [700], 16, 4, 192, 64, 128, 0, 0), ([3000], [300], 8, 2, 256, 32, 100, 0, 0), ([0], [1300], 8, 2, 128, 16, 64, 0, 1),
    ([700, 5000, 0], [600, 1, 450], 20, 4, 80, 64, 128, 900, 0)]


@pytest.mark.parametrize("dtype, kind", [("bf16", "e4m3"), ("f32", "int8"), ("f32", "e4m3")])
@pytest.mark.parametrize("past, new, H, Hkv, dim, P, T, window, sink", LONG)
def test_attention_of_much(past, new, H, Hkv, dim, P, T, window, sink, dtype, kind):
    """Long prompts and questions; two dozen of their rows against the oracle."""
    r = Requests(past, new, H, Hkv, dim, P, kind, dtype, seed=dim + window)
    kw = dict(window=window, sink=[0.5 * h - 3 for h in range(H)] if sink else None)
    got = r.run(T, **kw)
    n = sum(new)
    rows = np.unique(np.concatenate([[0, 1, 31, 32, n - 2, n - 1], np.random.default_rng(n).integers(0, n, 18)]))
    at = torch.from_numpy(rows).to(DEV)
    r.q, r.seqs, r.pos = r.q[at], r.seqs[rows], r.pos[rows]
    r.check(got[at], **kw)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("window, sink, T", [(1, False, 1), (5, True, 1), (64, True, 16), (65, False, 64), (200, True, 128), (0, True, 128), (100000, False, 33)])
def test_attention_with_windows_and_sinks(window, sink, T, kind, dtype):
    new = [1, 1, 1] if T == 1 else [3, 130, 40]
    r = Requests([333, 0, 120], new, 6, 2, 64, 16, kind, dtype, seed=window)
    sink = np.random.default_rng(1).normal(0, 2, 6).tolist() if sink else None
    r.check(r.run(T, window=window, sink=sink, scale=0.7), window=window, sink=sink, scale=0.7)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 4, 64])
def test_attention_of_rows_that_see_nothing(T, dtype):
    """Sequences of no written token, pages that no pool has, a window that only covers such a page: zeros, and nothing outside is read."""
    r = Requests([100, 100, 100, 100], [4, 4, 4, 4], 4, 2, 32, 16, "e4m3", dtype, seed=9)
    kv = [0, 104, 50, -3]
    r.table[1, 2], r.table[1, 5] = -1, 10 ** 6                        # holes
    r.table[2, :] = [-1, 99999, -5, 1 << 30] + [2 ** 31 - 1] * (r.table.shape[1] - 4)
    got = r.run(T, kv=kv)
    r.check(got, kv=kv)
    assert (got[:4] == 0).all() and (got[8:] == 0).all() and bool((got[4:8] != 0).any())
    r.check(r.run(T, kv=kv, window=3), kv=kv, window=3)
    r.check(r.run(T, kv=kv, sink=[1.0, 2.0, -3.0, 0.0]), kv=kv, sink=[1.0, 2.0, -3.0, 0.0])


@pytest.mark.parametrize("T", [1, 8, 64])
def test_attention_leaves_other_rows(T):
    """Padded batches: tiles without rows, of no sequence or outside the rows change nothing; rows behind the last tile stay as they were."""
    r = Requests([50, 9], [T, T], 4, 2, 32, 16, "int8", "bf16", seed=3)
    tiles = r.tiles(T)
    q = torch.cat([r.q, torch.full((5, 4, 32), float("nan"), dtype=r.q.dtype, device=DEV)])
    out = torch.full((2 * T + 5, 4, 32), 55.0, dtype=torch.bfloat16, device=DEV)
    tiles = [[-1, 0, 0, 0], tiles[0], [7, 3, T, 2 * T], [0, 5, 0, 2 * T], [1, 5, T, 2 * T + 5], [1, 3, T, -1], [0, -4, T, 2 * T], tiles[1], [-1, 0, 0, 0]]
    got = r.run(T, q=q, out=out, tiles=tiles)
    r.check(got[:2 * T])
    assert (got[2 * T:] == 55).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 64])
def test_attention_with_strides(T, dtype):
    """Queries inside wider rows, results head by head, a table of wider rows."""
    r = Requests([80, 300], [T, T], 6, 3, 64, 32, "e4m3", dtype, seed=4)
    q = torch.zeros((2 * T, 20, 64), dtype=r.dtype, device=DEV)
    q[:, 3:15:2] = r.q
    out = torch.zeros((6, 2 * T, 64), dtype=r.dtype, device=DEV).transpose(0, 1)
    r.check(r.run(T, q=q[:, 3:15:2], out=out))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("T", [1, 64])
def test_attention_over_scales_far_apart(T, kind):
    """Pages whose scales are 2^60 apart, pages of zeros at the smallest scale: weights and denominators keep their digits."""
    r = Requests([200, 500], [T, T], 4, 2, 64, 16, kind, "f32", seed=5, scales=(-2, 1))
    r.vs[:] = np.exp2(np.random.default_rng(1).integers(-30, 31, r.vs.shape))
    r.vs[::3] = 2.0 ** -40
    r.vc[::3] = 0
    want, tol = r.want()
    got = r.run(T).double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
    r.vs[:] = 2.0 ** -40                                              # everything at the smallest
    r.check(r.run(T))
    r.vs[:] = 2.0 ** 40
    r.check(r.run(T))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 16])
def test_attention_of_odd_queries(T, dtype):
    """Rows of zeros, far too large and far too small ones; rows with numbers that are none spoil nobody else's."""
    r = Requests([130], [16], 4, 2, 64, 16, "e4m3", dtype, seed=6)
    r.q[1] = 0
    r.q[2] *= 1e-30
    r.q[3] *= 300.0
    r.q[4] *= 1e4                                                     # one key takes it all
    bad = r.q.clone()
    bad[7, 1, 5], bad[9, 0] = float("nan"), float("nan")
    got = r.run(T, q=bad)
    none = torch.isnan(got)
    assert none[7, 1].all() and none[9, 0].all() and int(none.sum()) == 128
    r.check(torch.where(none, r.run(T), got))


@pytest.mark.parametrize("T", [1, 4, 32])
def test_attention_passes_over_tiles_that_are_none(T):
    """Tiles of no sequence, before the first position, of no rows, out of the rows or behind the last position that there can be."""
    r = Requests([700, 40], [33, 2], 4, 2, 64, 32, "e4m3", "bf16", seed=9)
    top = 2 ** 31 - 1
    none = [[-1, 0, 1, 0], [2, 0, 1, 0], [0, -1, 1, 0], [0, 5, 0, 0], [0, 5, -3, 0], [0, 5, 1, 35], [0, 5, 1, -1], [0, 5, 1, top], [top, top, top, top], [0, top, 1, 0], [1, top - T + 1, T, 0]]
    for window in (0, 30):
        got = r.run(T, window=window, tiles=none)
        assert bool((got == 55).all())
        # (more tiles are cut into other key runs: other orders of the same sums)
        r.check(r.run(T, window=window, tiles=none[:5] + r.tiles(T) + none[5:]), window=window)


@pytest.mark.parametrize("T", [1, 9, 64])
def test_attention_in_place(T):
    """Results may take their queries' place."""
    r = Requests([4000, 77, 900], [T, T, T], 8, 2, 128, 64, "e4m3", "bf16", seed=3)
    want, q = r.run(T), r.q.clone()
    assert torch.equal(r.run(T, q=q, out=q), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 20])
def test_attention_of_zeros_over_small_keys(T, dtype):
    """A row of zeros sees all its keys alike, however small their scales, and none of those it does not see."""
    r = Requests([70], [20], 4, 2, 64, 16, "int8", dtype, seed=8, scales=(-2, 1))
    r.q[3:7] = 0
    r.q[7] *= 1e-35
    r.ks[:] = 2.0 ** -40
    for scale in (1.0, 1e-3, 1e-20):
        r.check(r.run(T, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 8, 64])
@pytest.mark.parametrize("dim", [16, 48, 80, 112, 128, 144, 176, 192, 208, 256])
def test_attention_of_uneven_queries(T, dtype, dim):
    """The elements of a row are far apart in size, the largest in any sixteen of them."""
    r = Requests([300, 40], [9, 7], 6, 3, dim, 32, "int8", dtype, seed=dim)
    rng = np.random.default_rng(dim)
    up = np.exp2(rng.integers(-9, 1, (r.q.shape[0], 6, dim // 16)))
    for i in range(r.q.shape[0]):
        up[i, np.arange(6), rng.integers(0, dim // 16, 6)] = 4
    r.q = (r.q.double() * torch.from_numpy(np.repeat(up, 16, axis=2)).to(DEV)).to(r.q.dtype)
    r.check(r.run(T))


@pytest.mark.parametrize("T", [1, 9, 64])
def test_attention_many_times_alike(T):
    """The same call again and again, among others, on two streams at once: the same bits each time."""
    a, b = (Requests([4000, 77, 900], [T, T, T], 8, 2, 128, 64, "e4m3", "bf16", seed=s) for s in (1, 2))
    want = [r.run(T) for r in (a, b)]
    a.check(want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    from promptcache_amd import _blocks as B
    args = []
    for r in (a, b):
        args.append((r.q, torch.tensor(r.tiles(T), dtype=torch.int32, device=DEV), T, i32(r.kv), *r.device()))
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(r.q) for _ in range(40)] for r in (a, b)]
    for i in range(40):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                B.attn_pages(*args[k], outs[k][i], scale=1.0)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in outs[k])


@pytest.mark.parametrize("T", [1, 9, 64])
def test_two_graphs_of_attention_at_once(T):
    """Two captured calls, replayed at the same time among eager ones: scratch of their own each."""
    from promptcache_amd import _blocks as B
    rs = [Requests([4000, 77, 900], [T, T, T], 8, 2, 128, 64, "e4m3", "bf16", seed=s) for s in (1, 2)]
    made = []
    for r in rs:
        args = (r.q, torch.tensor(r.tiles(T), dtype=torch.int32, device=DEV), T, i32(r.kv), *r.device())
        out = torch.zeros_like(r.q)
        torch.cuda.synchronize()
        g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=st):
            B.attn_pages(*args, out, scale=1.0)
        made.append((g, st, out, args))
    first = []
    for i in range(10):
        for g, st, out, _ in made:
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
        rs[i % 2].run(T)
        torch.cuda.synchronize()
        if i == 0:
            first = [out.clone() for _, _, out, _ in made]
            for r, out in zip(rs, first):
                r.check(out)
        assert all(torch.equal(out, want) for (_, _, out, _), want in zip(made, first))


def test_attention_in_a_graph_is_the_eager_one_but_for_its_merge():
    """A captured call merges in a launch of its own: the same sums in the same order of runs, off by roundings of fp32."""
    r = Requests([4000, 700], [1, 1], 8, 2, 128, 64, "e4m3", "f32", seed=3)
    from promptcache_amd import _blocks as B
    eager = r.run(1)
    r.check(eager)
    tiles, kv, dev = torch.tensor(r.tiles(1), dtype=torch.int32, device=DEV), i32(r.kv), r.device()
    floats = B.attn_pages_part(2, 8, 2, 128, 2, 1, 4001)
    part, out = torch.zeros(floats, device=DEV), torch.zeros_like(r.q)
    torch.cuda.synchronize()
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=st):
        B.attn_pages(r.q, tiles, 1, kv, *dev, out, scale=1.0, longest=4001, part=part)
    for _ in range(4):
        out.zero_()
        g.replay()
        r.run(1)
        torch.cuda.synchronize()
        r.check(out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim, kind", [(48, "e4m3"), (80, "int8"), (128, "e4m3")])
def test_attention_of_more_blocks_than_the_chip_has_cus(dim, kind, dtype):
    rng = np.random.default_rng(dim)
    n = 70
    r = Requests([int(v) for v in rng.integers(0, 300, n)], [int(v) for v in rng.integers(30, 41, n)], 8, 4, dim, 32, kind, dtype, seed=dim)
    r.check(r.run(40))
    r.check(r.run(40, window=50), window=50)


def test_attention_of_more_tiles_than_are_shared_out():
    """Over 512 tiles: a workgroup a unit."""
    n = 600
    rng = np.random.default_rng(4)
    r = Requests([int(v) for v in rng.integers(0, 40, n)], [1] * n, 4, 2, 32, 16, "int8", "bf16", seed=5)
    r.check(r.run(1))
    r.check(r.run(1, longest=5000))


def test_attention_with_a_head_of_a_wrong_bound():
    """`longest` is a bound for the work's partition: a host that is wrong about it still gets every key."""
    r = Requests([5000, 40], [1, 1], 4, 2, 64, 64, "e4m3", "bf16", seed=7)
    r.check(r.run(1, longest=700))
    r.check(r.run(1, longest=100000))
    r.check(r.run(1))


def test_attention_beyond_32_bit_offsets():
    """A pool of more than 2^32 bytes of key codes: the last pages are the ones used."""
    from promptcache_amd import _blocks as B
    P, Hkv, dim, pages = 128, 32, 128, 8500
    assert pages * P * Hkv * dim > 2 ** 32
    kc, vc = (torch.zeros((pages, Hkv, P, dim), dtype=torch.uint8, device=DEV) for _ in range(2))
    vc = vc.view(pages, Hkv, dim, P)
    sc = [torch.ones((pages, Hkv), device=DEV) for _ in range(2)]
    pool = [kc.view(torch.int8), sc[0], vc.view(torch.int8), sc[1]]
    gen = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((300, Hkv, dim), generator=gen, device=DEV) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2, pages - 3]], dtype=torch.int32, device=DEV)
    slot = torch.tensor([(pages - 1 - i // P) * P + i % P for i in range(300)], dtype=torch.int64, device=DEV)
    B.pages_append(k, v, slot, *pool)
    kk, vv = torch.zeros_like(k), torch.zeros_like(v)
    B.pages_read(slot, *pool, kk, vv)
    assert float((kk - k).abs().max()) <= 2.0 ** -5 and float((vv - v).abs().max()) <= 2.0 ** -5       # |x| < 8: scales up to 2^-4, half a step
    for T, rows in ((1, 1), (64, 64)):
        q = torch.randn((rows, Hkv, dim), generator=gen, device=DEV)
        out = torch.zeros_like(q)
        B.attn_pages(q, i32([[0, 300 - rows, rows, 0]]), T, i32([300]), table, *pool, out, scale=dim ** -0.5)
        z = torch.einsum("rhd,khd->hrk", q.double(), kk.double()) * dim ** -0.5
        z = z.masked_fill(torch.arange(300, device=DEV)[None, None] > torch.arange(300 - rows, 300, device=DEV)[None, :, None], float("-inf"))
        want = torch.einsum("hrk,khd->rhd", torch.softmax(z, -1), vv.double())
        # |v| < 8 and sums over 300 keys: as in Requests.want with A <= 8
        assert float((out.double() - want).abs().max()) <= 8 * (2 * (136 * 2.0 ** -24 * 40 + 2.0 ** -21) + 300 * 2.0 ** -24)


# ---- together -----------------------------------------------------------------------------------------------------------------------------
def dense(ks, vs, q, scale):
    """Last-rows causal attention of one sequence in 64 bits; [tokens, Hkv, dim], q [rows, H, dim]."""
    k, v, q = ks.double(), vs.double(), q.double()
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    z = torch.einsum("rhd,khd->hrk", q, k) * scale
    n, m = k.shape[0], q.shape[0]
    z = z.masked_fill(torch.arange(n, device=q.device)[None, None] > torch.arange(n - m, n, device=q.device)[None, :, None], float("-inf"))
    return torch.einsum("hrk,khd->rhd", torch.softmax(z, -1), v)


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
def test_a_cache_through_prompts_steps_and_ends(codes):
    """Prompts, decoding, a sequence that ends and gives its pages to another, a shared prefix, a refusal: attention is that over the rows the cache reads back, which are the
    rows that went in but for their rounding."""
    from promptcache_amd.model.kv_arena import PageCache
    gen = torch.Generator(device=DEV).manual_seed(11)
    dims = [(2, 64), (1, 128)]
    cache = PageCache(dims, 4, 20, DEV, page_size=16, codes=codes)
    held = [[torch.zeros((0, 2, g, d), device=DEV) for g, d in dims] for _ in range(4)]
    lengths = [0] * 4

    def step(brings, tile_rows, refused=()):
        rows = sum(max(b, 0) for b in brings)
        st = cache.begin(brings, rows + 2, tile_rows=tile_rows, longest=max(n + max(b, 0) for n, b in zip(lengths, brings)))
        at = [0]
        for b in brings:
            at.append(at[-1] + max(b, 0))
        outs = []
        for layer, (g, d) in enumerate(dims):
            kv = torch.randn((rows + 2, 2, g, d), generator=gen, device=DEV).bfloat16()
            q = torch.randn((rows + 2, 4, d), generator=gen, device=DEV).bfloat16()
            cache.append(layer, kv[:, 0], kv[:, 1], st)
            outs.append((q, cache.attend(layer, q, st)))
            for s, b in enumerate(brings):
                if b < 0:
                    held[s][layer] = held[s][layer][:0]
                elif s not in refused:
                    held[s][layer] = torch.cat([held[s][layer], kv[at[s]:at[s + 1]].float()])
        for s, b in enumerate(brings):
            lengths[s] = 0 if b < 0 else lengths[s] + (0 if s in refused else b)
        assert cache.cached.tolist() == lengths and st.status.tolist()[0] == len(refused)
        for layer, (g, d) in enumerate(dims):
            q, out = outs[layer]
            assert bool((out[rows:] == 0).all())
            for s, b in enumerate(brings):
                if b <= 0 or s in refused:
                    assert b <= 0 or bool((out[at[s]:at[s + 1]] == 0).all())
                    continue
                k, v = cache.rows(layer, s, lengths[s], torch.float32)
                for got, was in ((k, held[s][layer][:, 0]), (v, held[s][layer][:, 1])):
                    # a code is off by half its step: e4m3 2^-4 of the number or 2^-10 of the scale, int8 half the scale; scales are at most 2 |x| / top, and a page that grew rounded twice
                    big = was.abs().amax((0, 2))[None, :, None]
                    lim = was.abs() * 2.0 ** -4 + big * 2.0 ** -16 if codes == torch.float8_e4m3fn else big * (2 / 127)
                    assert bool(((got - was).abs() <= lim).all())
                want = dense(k, v, q[at[s]:at[s + 1]], d ** -0.5)
                A = dense(k, v.abs(), q[at[s]:at[s + 1]], d ** -0.5)
                tol = 2.0 ** -8 * want.abs() + A * (2 * ((d + 8) * 2.0 ** -24 * 6 * d ** 0.5 + 2.0 ** -21 + 2.0 ** -11) + 320 * 2.0 ** -24) + 2.0 ** -30
                assert bool(((out[at[s]:at[s + 1]].double() - want).abs() <= tol * (1 + 2.0 ** -8)).all())

    step([40, 0, 17, 1], 32)
    for _ in range(18):
        step([1, 0, 1, 1], 1)
    step([-1, 70, 1, 0], 64)
    step([100, 1, 1, 1], 100)
    assert cache.ring_state.tolist()[:2] == [cache.ring_state.tolist()[0], 20 - sum(-(-n // 16) for n in lengths)]
    step([1, 300, 1, 1], 64, refused=(1,))                            # not enough pages: that one keeps what it had
    step([1, -1, -1, -1], 1)
    cache.share(0, 2, 96)                                             # 0 holds 102 tokens: six whole pages
    lengths[2] = 96
    for layer in range(2):
        held[2][layer] = held[0][layer][:96].clone()
    step([1, 5, 9, 0], 4)
    step([1, 0, -1, 0], 1)
    step([0, 0, 33, 0], 64)
    step([-1, -1, -1, -1], 1)
    assert cache.ring_state.tolist()[1] == 20 and sorted(cache.ring.tolist()) == list(range(20))


def test_a_captured_step_moves_on_by_itself():
    """One graph of tables, append and attention, replayed: every replay is the eager step of the same inputs, page borders and growing scales among them."""
    from promptcache_amd.model.kv_arena import PageCache
    gen = torch.Generator(device=DEV).manual_seed(12)
    n, g, d, H = 5, 2, 64, 8
    caches = [PageCache([(g, d)], n, 60, DEV, page_size=16) for _ in range(2)]
    k0, v0 = (torch.randn((90, g, d), generator=gen, device=DEV).bfloat16() for _ in range(2))
    for c in caches:
        st = c.begin([30, 15, 1, 40, 4], 90, tile_rows=16)
        c.append(0, k0, v0, st)
    ones = torch.ones(n, dtype=torch.int32, device=DEV)
    x = torch.zeros((n, 2 * g + H, d), dtype=torch.bfloat16, device=DEV)
    outs = [torch.zeros((n, H, d), dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def run(c, out):
        st = c.begin(ones, n, longest=200)
        c.append(0, x[:, :g], x[:, g:2 * g], st)
        c.attend(0, x[:, 2 * g:], st, out=out)

    def fresh():
        x.copy_(torch.randn(x.shape, generator=gen, device=DEV) * 2.0 ** float(torch.randint(-2, 4, (1,)).item()))

    fresh()
    for c, out in zip(caches, outs):                                  # (eager: makes the buffers)
        run(c, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=st):
        run(caches[0], outs[0])
    for i in range(40):
        fresh()
        graph.replay()
        run(caches[1], outs[1])
        if i % 7 == 0:
            torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(caches[0].cached, caches[1].cached) and torch.equal(caches[0].table, caches[1].table)
    assert caches[0].cached.tolist() == [71, 56, 42, 81, 45]
    for a, b in zip((caches[0].kcodes[0], caches[0].vcodes[0], caches[0].kscale[0]), (caches[1].kcodes[0], caches[1].vcodes[0], caches[1].kscale[0])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_captured_step_gives_back_what_a_later_share_left_it():
    """A graph captured before the first shared prefix: a sequence that is over keeps the shared pages out of the ring once, and its place's next one gives back all of its own."""
    from promptcache_amd.model.kv_arena import PageCache
    cache = PageCache([(1, 16)], 2, 10, DEV, page_size=16)
    brings = torch.zeros(2, dtype=torch.int32, device=DEV)
    cache.begin(brings, 40)
    torch.cuda.synchronize()
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        cache.begin(brings, 40)

    def step(*b):
        brings.copy_(torch.tensor(b, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        return cache.ring_state.tolist()[1]

    assert step(40, 0) == 7
    cache.share(0, 1, 32)
    assert step(0, 20) == 5
    assert step(0, -1) == 7
    assert step(0, 40) == 4
    assert step(0, -1) == 7
    assert step(-1, 0) == 10 and sorted(cache.ring.tolist()) == list(range(10))
