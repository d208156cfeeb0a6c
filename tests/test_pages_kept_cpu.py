"""Pages that sequences share, without a GPU: the oracle, and what the entry point and the cache refuse."""
import ctypes as C

import pytest
import torch

from oracle import pages_oracle as O
from promptcache_amd import _blocks as B

PTR = 1 << 20                     # an address that nothing reads: every call below is refused before a launch


def test_the_oracle_of_kept_pages():
    table = [[0, 1, 2, 3], [0, 1, 5, 6], [0, 1, 5, 7], [9, 1, 5, 7]]
    cached = [60, 64, 33, 64]
    assert O.kept(cached, [-1, 0, 0, -1], table, 16).tolist() == [2, 0, 0, 0]
    assert O.kept(cached, [-1, -1, 0, -1], table, 16).tolist() == [2, 3, 0, 0]
    assert O.kept(cached, [-1, -1, -1, 5], table, 16).tolist() == [0, 2, 3, 0]      # each page with the first that has it
    assert O.kept([16, 64, 0, 64], [-1, -1, -1, -1], table, 16).tolist() == [0, 1, 0, 0]


@pytest.mark.parametrize("bad", [dict(n=0), dict(wide=0), dict(ld=4), dict(P=24), dict(cached=None), dict(brings=None), dict(table=None), dict(keep=None), dict(n=1 << 20, wide=1 << 12, ld=1 << 12)])
def test_what_pages_kept_refuses(bad):
    a = dict(n=3, cached=PTR, brings=PTR, table=PTR, ld=5, wide=5, P=16, keep=PTR) | bad
    lib = B.load()
    assert lib.pcb_pages_kept(a["n"], a["cached"], a["brings"], a["table"], C.c_int64(a["ld"]), a["wide"], a["P"], a["keep"], None) == -2001
    assert b"pcb_pages_kept" in lib.pcb_last_error_string()


def test_a_captured_step_takes_no_host_numbers(monkeypatch):
    """Its copy would run again with every replay, out of memory that is another's by then."""
    from promptcache_amd.model import kv_arena
    cache = kv_arena.PageCache([(1, 16)], 2, 4, "cpu", page_size=16)
    cache.device = torch.device("cuda")
    copied = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(kv_arena, "uploaded", lambda *a: copied.append(a))
    with pytest.raises(Exception) as e:
        cache.begin([1, 1], 2)
    assert not copied and e.type is RuntimeError, e.value
