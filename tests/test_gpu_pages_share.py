"""Pages that several sequences of a paged cache begin with: whoever is over first, they stay until nobody has them, and then go back once."""
import numpy as np
import pytest
import torch

from oracle import pages_oracle as O
from tests.test_gpu_pages import DEV, dense, i32

pytestmark = pytest.mark.gpu


def family(rng, n, P, wide):
    """Lengths and tables of n sequences, many of which begin as an earlier one does."""
    cached = [int(v) for v in rng.integers(0, wide * P + 1, n)]
    table = rng.permutation(n * wide + 5)[:n * wide].reshape(n, wide)
    for s in range(1, n):
        if rng.random() < 0.6:
            t = int(rng.integers(0, s))
            k = int(rng.integers(0, min(cached[t], cached[s]) // P + 1))
            table[s, :k] = table[t, :k]
    return cached, table


@pytest.mark.parametrize("n, P, wide, ends", [(1, 16, 3, 1.0), (2, 16, 1, 0.5), (5, 32, 9, 0.5), (64, 64, 40, 0.2), (67, 16, 130, 1.0), (600, 128, 7, 0.4)])
def test_pages_that_are_kept(n, P, wide, ends):
    from promptcache_amd import _blocks as B
    for seed in range(4):
        rng = np.random.default_rng(100 * n + seed)
        cached, table = family(rng, n, P, wide)
        brings = [-1 if rng.random() < ends else int(rng.integers(0, 3)) for _ in range(n)]
        keep = i32([77] * n)
        tab = torch.full((n, wide + seed), -5, dtype=torch.int32, device=DEV)[:, :wide]
        tab.copy_(torch.from_numpy(table))
        B.pages_kept(i32(cached), i32(brings), tab, P, keep)
        assert np.array_equal(keep.cpu().numpy(), O.kept(cached, brings, table, P))


class Story:
    """A cache, what its sequences should hold, and the pages that should be free."""

    def __init__(self, seqs, pages, P=16, seed=0):
        from promptcache_amd.model.kv_arena import PageCache
        self.g, self.d, self.P = 2, 32, P
        self.cache = PageCache([(self.g, self.d)], seqs, pages, DEV, page_size=P)
        self.held = [torch.zeros((0, 2, self.g, self.d), device=DEV) for _ in range(seqs)]
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def step(self, brings):
        rows = sum(max(b, 0) for b in brings)
        st = self.cache.begin(brings, rows, tile_rows=8)
        kv = torch.randn((rows, 2, self.g, self.d), generator=self.gen, device=DEV)
        q = torch.randn((rows, 4, self.d), generator=self.gen, device=DEV)
        self.cache.append(0, kv[:, 0], kv[:, 1], st)
        out, at = self.cache.attend(0, q, st), 0
        for s, b in enumerate(brings):
            n = max(b, 0)
            self.held[s] = self.held[s][:0] if b < 0 else torch.cat([self.held[s], kv[at:at + n]])
            at += n
        assert st.status.tolist() == [0, rows] and self.cache.cached.tolist() == [h.shape[0] for h in self.held]
        at = 0
        for s, b in enumerate(brings):
            n = max(b, 0)
            if not self.held[s].shape[0]:
                continue
            k, v = self.cache.rows(0, s, self.held[s].shape[0], torch.float32)
            for got, was in ((k, self.held[s][:, 0]), (v, self.held[s][:, 1])):
                # a code is off by half its step, 2^-4 of the number or 2^-10 of the scale, which is at most 2 |x| / 448; a page that grew rounded twice
                big = was.abs().amax((0, 2))[None, :, None]
                assert bool(((got - was).abs() <= was.abs() * 2.0 ** -4 + big * 2.0 ** -16).all()), s
            if n:
                want, A = (dense(k, x, q[at:at + n], self.d ** -0.5) for x in (v, v.abs()))
                tol = 2.0 ** -24 * want.abs() + A * (2 * ((self.d + 8) * 2.0 ** -24 * 6 * self.d ** 0.5 + 2.0 ** -21) + 320 * 2.0 ** -24) + 2.0 ** -30
                assert bool(((out[at:at + n].double() - want).abs() <= tol).all()), s
            at += n
        self.free()

    def share(self, source, target, tokens):
        self.cache.share(source, target, tokens)
        n = min(tokens, self.held[source].shape[0] // self.P * self.P)
        self.held[target] = self.held[source][:n].clone()

    def free(self):
        c = self.cache
        head, n = c.ring_state.tolist()[:2]
        ring, table = c.ring.tolist(), c.table.tolist()
        free = [ring[(head + i) % c.pages] for i in range(n)]
        used = {p for s, h in enumerate(self.held) for p in table[s][:-(-h.shape[0] // self.P)]}
        assert sorted(free + sorted(used)) == list(range(c.pages))               # every page is free or in use, and free once


def test_the_source_is_over_first():
    a = Story(4, 12)
    a.step([40, 0, 0, 0])
    a.share(0, 1, 32)
    a.step([0, 5, 0, 0])
    a.step([-1, 1, 0, 0])
    a.step([100, 1, 0, 0])                                            # takes whatever is free
    a.step([0, -1, 0, 0])
    a.step([-1, 0, 0, 0])


def test_many_that_begin_alike_end_in_any_order():
    """A page of one sequence, more of it in a second one, a third from the second, two from the first; some end together, some go on, others take their pages."""
    a = Story(6, 30, seed=1)
    a.step([70, 0, 0, 0, 0, 9])
    a.share(0, 1, 48)
    a.step([1, 30, 0, 0, 0, 1])                                       # 1: three pages of 0's, two of its own
    a.share(1, 2, 64)
    a.share(0, 3, 64)
    a.share(3, 4, 16)
    a.step([1, 1, 20, 3, 1, 0])
    a.step([-1, -1, 1, 0, 2, 30])
    a.step([33, 60, 1, 1, 1, 0])
    a.step([1, 1, 1, -1, -1, 1])
    a.share(2, 3, 64)
    a.step([1, 1, -1, 40, 50, -1])
    a.share(3, 5, 32)
    a.step([-1, 1, 80, -1, -1, 1])
    a.step([0, -1, -1, 0, 0, -1])
    assert a.cache.ring_state.tolist()[1] == 30


def test_a_share_of_more_than_there_is():
    """The whole pages that the source holds: what its table has behind them are pages of others."""
    a = Story(3, 12, seed=2)
    a.step([0, 60, 0])
    a.step([20, -1, 0])
    a.step([1, 40, 0])                                                # (1's table still names a fourth page, from before)
    a.step([-1, 1, 0])
    a.share(1, 2, 64)                                                 # 41 tokens: two pages
    a.step([30, 1, 1])
    a.step([-1, 1, 1])
    a.step([0, -1, 30])
    a.step([0, 0, -1])


def test_a_captured_step_whose_source_is_over_first():
    from promptcache_amd.model.kv_arena import PageCache
    cache = PageCache([(1, 16)], 3, 12, DEV, page_size=16)
    brings = torch.zeros(3, dtype=torch.int32, device=DEV)
    cache.begin(brings, 60)
    torch.cuda.synchronize()
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        cache.begin(brings, 60)

    def step(*b):
        brings.copy_(torch.tensor(b, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        return cache.ring_state.tolist()[1]

    assert step(60, 0, 0) == 8
    cache.share(0, 1, 48)
    cache.share(0, 2, 32)
    assert step(0, 0, 20) == 6
    assert step(-1, 1, 0) == 6                                        # its fourth page comes back, 1 takes one
    first = cache.table[:, :3].tolist()
    assert first[1] == first[0] and first[2][:2] == first[0][:2]
    assert step(60, -1, 0) == 6 - 4 + 2                               # 1's own one, and the third that only it had left
    assert step(0, 0, -1) == 8 and step(-1, 0, 0) == 12 and sorted(cache.ring.tolist()) == list(range(12))


def test_rows_behind_what_a_sequence_holds():
    """Zeros: the table's entries there are pages that others have by now."""
    a = Story(2, 5, seed=3)
    a.step([40, 0])
    a.step([-1, 30])
    a.step([3, 30])                                                   # (1 has 0's former pages)
    for n in (1, 3, 4, 16, 17, 48, 100):
        k, v = a.cache.rows(0, 0, n, torch.float32)
        assert k.shape == v.shape == (n, 2, 32)
        assert bool((k[:3] != 0).any()) and not bool((k[3:] != 0).any()) and not bool((v[3:] != 0).any()), n
