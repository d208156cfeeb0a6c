"""The paged 8-bit cache without a GPU: the oracle against other ways to the same numbers, the struct mirrors, and what the entry points refuse."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from oracle import pages_oracle as O
from promptcache_amd import _blocks as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_oracles_e4m3_is_the_formats():
    codes = np.arange(256, dtype=np.uint8)
    torchs = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.e4m3_value(codes), torchs, equal_nan=True)
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(100000, generator=gen) * torch.exp2(torch.rand(100000, generator=gen) * 24 - 14)).clamp(-448, 448)
    x[:256] = torch.from_numpy(np.nan_to_num(torchs)).float()
    mid = np.sort(O.e4m3_value(np.arange(127, dtype=np.uint8)))
    x[300:426] = torch.from_numpy((mid[1:] + mid[:-1]) / 2).float()               # ties
    assert np.array_equal(O.encode(x.double().numpy(), "e4m3"), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_scales_are_the_smallest_that_hold(kind):
    top = O.TOP[kind]
    for m in (0.0, 1e-30, top * 2.0 ** -40, top * 2.0 ** -7, np.nextafter(np.float32(top), np.float32(1e9)), 1.0, 127.0, 448.0, 3e4, 3e38):
        s = O.scale_for(float(m), kind)
        assert s == 2.0 ** 40 or m <= top * s
        assert s == 2.0 ** -40 or m > top * s / 2


def test_struct_layouts_match_the_header(tmp_path):
    structs = (("pcb_page_tables_args", B.PageTablesArgs), ("pcb_pages_rows_args", B.PagesRowsArgs), ("pcb_attn_pages_args", B.AttnPagesArgs))
    body = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{ROOT}/include/promptcache_blocks.h"', 'int main(void) {']
    for st, cls in structs:
        body.append(f'  printf("{st} %zu\\n", sizeof({st}));')
        body += [f'  printf("{st}.{f} %zu\\n", offsetof({st}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(body + ["  return 0;", "}"]))
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")])
    got = dict(line.rsplit(" ", 1) for line in subprocess.check_output([str(tmp_path / "layout")], text=True).strip().splitlines())
    for st, cls in structs:
        assert int(got[st]) == C.sizeof(cls), st
        for name, _ in cls._fields_:
            assert int(got[f"{st}.{name}"]) == getattr(cls, name).offset, (st, name)


PTR = 1 << 20                     # an address on 16 bytes that nothing reads: every call below is refused before a launch


def tables_args(**kw):
    a = B.PageTablesArgs()
    for k, v in (dict(struct_bytes=C.sizeof(a), n_seqs=3, max_pages=5, ld_table=5, page_size=16, cached=PTR, brings=PTR, table=PTR, ring=PTR, ring_cap=9, ring_state=PTR, ring_out=PTR,
                      row_slot=PTR, n_rows=12, tiles=PTR, n_tiles=6, tile_rows=4) | kw).items():
        setattr(a, k, v)
    return a


def rows_args(**kw):
    a = B.PagesRowsArgs()
    for k, v in (dict(struct_bytes=C.sizeof(a), dtype=0, code=0, k=PTR, ldk=64, k_head_stride=32, v=PTR, ldv=64, v_head_stride=32, row_slot=PTR, n_rows=3, kcodes=PTR, kscale=PTR,
                      vcodes=PTR, vscale=PTR, n_pages=4, page_size=16, Hkv=2, dim=32) | kw).items():
        setattr(a, k, v)
    return a


def attn_args(**kw):
    a = B.AttnPagesArgs()
    for k, v in (dict(struct_bytes=C.sizeof(a), dtype=0, code=0, q=PTR, ldq=128, q_head_stride=32, tiles=PTR, n_tiles=2, tile_rows=1, n_rows=2, kv_len=PTR, table=PTR, ld_table=5, n_seqs=2,
                      max_pages=5, kcodes=PTR, kscale=PTR, vcodes=PTR, vscale=PTR, n_pages=9, page_size=16, H=4, Hkv=2, dim=32, scale=0.2, out=PTR, ldo=128, out_head_stride=32,
                      longest=80) | kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry, make, bad", [
    ("pcb_page_tables", tables_args, b) for b in (
        dict(struct_bytes=8), dict(n_seqs=0), dict(max_pages=0), dict(ld_table=4), dict(page_size=48), dict(page_size=8), dict(page_size=256), dict(n_rows=-1), dict(cached=None),
        dict(brings=None), dict(table=None), dict(row_slot=None), dict(ring_cap=0), dict(ring_state=None), dict(ring_out=None), dict(tile_rows=0), dict(tiles=PTR + 4),
        dict(n_rows=(1 << 30) + 1, n_tiles=1 << 29), dict(n_tiles=5), dict(n_seqs=1 << 20, max_pages=1 << 12, ld_table=1 << 12), dict(n_seqs=1, max_pages=1 << 27, ld_table=1 << 27))
] + [
    (entry, rows_args, b) for entry in ("pcb_pages_append", "pcb_pages_read") for b in (
        dict(struct_bytes=8), dict(dtype=2), dict(code=2), dict(n_rows=-1), dict(n_pages=0), dict(page_size=24), dict(Hkv=0), dict(dim=0), dict(dim=24), dict(dim=272), dict(k=None),
        dict(v=None), dict(row_slot=None), dict(kcodes=None), dict(vscale=None), dict(k=PTR + 2), dict(vcodes=PTR + 8), dict(ldk=65), dict(v_head_stride=36), dict(row_slot=PTR + 4),
        dict(n_rows=1 << 30, Hkv=64))
] + [
    ("pcb_attn_pages", attn_args, b) for b in (
        dict(struct_bytes=8), dict(dtype=2), dict(code=-1), dict(n_tiles=-1), dict(tile_rows=0), dict(n_rows=-1), dict(n_seqs=0), dict(max_pages=0), dict(ld_table=4), dict(n_pages=0),
        dict(page_size=17), dict(H=5), dict(Hkv=0), dict(dim=40), dict(dim=512), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(longest=-1),
        dict(q=None), dict(tiles=None), dict(kv_len=None), dict(table=None), dict(kcodes=None), dict(vscale=None), dict(out=None), dict(q=PTR + 2), dict(out=PTR + 8), dict(tiles=PTR + 4),
        dict(ldq=129), dict(out_head_stride=33), dict(longest=1 << 20), dict(longest=1 << 20, part=PTR, part_floats=100), dict(longest=1 << 20, part=PTR + 4, part_floats=1 << 40),
        dict(tile_rows=1 << 22), dict(max_pages=1 << 27, ld_table=1 << 27), dict(ldo=0), dict(out_head_stride=0), dict(n_tiles=1 << 23),
        dict(n_tiles=1 << 30, H=1 << 30, Hkv=1 << 30), dict(H=4098, Hkv=2), dict(H=65536, Hkv=2048),
        dict(n_tiles=512, tile_rows=8, H=65535, Hkv=65535, longest=1000, part=PTR, part_floats=1 << 50))
] + [
    ("pcb_pages_read", rows_args, b) for b in (dict(ldk=0), dict(ldv=0), dict(k_head_stride=0), dict(v_head_stride=0))
])
def test_what_is_refused(entry, make, bad):
    lib = B.load()
    assert getattr(lib, entry)(C.byref(make(**bad)), None) == -2001
    assert entry.encode() in lib.pcb_last_error_string()


def test_nothing_to_do_launches_nothing():
    lib = B.load()
    assert lib.pcb_pages_append(C.byref(rows_args(n_rows=0, k=None)), None) == 0
    assert lib.pcb_attn_pages(C.byref(attn_args(n_tiles=0, q=None)), None) == 0
    assert lib.pcb_attn_pages(C.byref(attn_args(n_rows=0, q=None)), None) == 0


def test_scratch_of_key_runs():
    assert B.attn_pages_part(64, 32, 8, 128, 64, 1, 64) == 0                       # one step of keys: nothing to cut
    one = B.attn_pages_part(1, 32, 8, 128, 1, 1, 100000)
    assert one > 0
    assert B.attn_pages_part(0, 32, 8, 128, 0, 1, 100000) == 0
    for bad in ((1, 32, 7, 128, 1, 1, 100), (1, 1 << 30, 1 << 30, 128, 1 << 30, 1, 1 << 20), (1, 32, 8, 272, 1, 1, 100), (1, 32, 8, 128, 1, 0, 100), (1, 32, 8, 128, 1 << 23, 1, 100)):
        with pytest.raises(RuntimeError):
            B.attn_pages_part(*bad)


def test_compiled_looks_are_the_python_ones():
    """What the compiled helpers accept, return and refuse is what the Python functions of the same names do (on host tensors, device -1)."""
    tensors = pytest.importorskip("promptcache_amd._tensors")
    assert tensors.torch_version == torch.__version__.split("+")[0]
    flat, heads, table, pool = B._looks
    i32, f32 = torch.arange(60, dtype=torch.int32), torch.ones(60)
    kc, vc, ks = torch.zeros((3, 2, 16, 32), dtype=torch.int8), torch.zeros((3, 2, 32, 16), dtype=torch.int8), torch.ones((3, 2))
    e4 = torch.float8_e4m3fn
    rows = torch.zeros((5, 4, 32), dtype=torch.bfloat16)
    some = [
        ("flat", flat, [(t, d, n, dev, "x") for t in (None, i32, i32[7:], i32[::2], i32.view(6, 10).t(), i32[:0], f32, i32.long(), torch.zeros(3, dtype=torch.int32).to_sparse())
                        for d in (torch.int32, torch.float32) for n in (0, 30, 60, 61) for dev in (-1, 0)]),
        ("heads", heads, [(t, h, d, dev, "x") for t in (rows, rows[:1], rows[:, :1], rows[::2], rows[:, :, ::2], rows.transpose(0, 1), rows[:0], rows[0], rows.expand(5, 4, 32), f32)
                          for h in (1, 4, 5) for d in (16, 32) for dev in (-1, 0)]),
        ("table", table, [(t, n, dev, "x") for t in (i32.view(6, 10), i32.view(6, 10)[:1], i32.view(6, 10)[:, 3:], i32.view(6, 10).t(), i32.view(6, 10)[:0], i32, f32.view(6, 10))
                          for n in (0, 1, 6, 7) for dev in (-1, 0)]),
        ("pool", pool, [(a, s, b, s2, dev, "x") for a in (kc, kc.view(e4), kc.float(), kc[:2], kc.transpose(0, 1)) for b in (vc, vc.view(e4), vc[:2], kc)
                        for s, s2 in ((ks, ks), (ks[:2], ks), (ks, ks.double()), (ks.t(), ks)) for dev in (-1, 0)]),
    ]
    taken = 0
    for name, python, calls in some:
        for args in calls:
            got = []
            for f in (python, getattr(tensors, name)):
                try:
                    got.append(f(*args))
                except Exception as e:                                             # (the same refusal, in the same words)
                    got.append((type(e), str(e)))
            assert got[0] == got[1], (name, args, got)
            taken += not isinstance(got[0], tuple) or not isinstance(got[0][0], type)
    assert taken > 40
    for bad in ((), (i32,), (i32, torch.int32, 1, -1, "x", 5), (i32, torch.int32, 1 << 70, -1, "x"), (i32, "int32", 1, -1, "x"), ("x", torch.int32, 1, -1, "x")):
        with pytest.raises(Exception):
            tensors.flat(*bad)


def test_wrappers_name_what_is_wrong():
    x = torch.zeros((2, 2, 32))
    kc = torch.zeros((4, 2, 16, 32), dtype=torch.int8)
    vc, sc = torch.zeros((4, 2, 32, 16), dtype=torch.int8), torch.ones((4, 2))
    slot = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError):
        B.pages_append(x, x, slot, kc.float(), sc, vc, sc)                         # codes of another type
    with pytest.raises(ValueError):
        B.pages_append(x, x, slot, kc, sc, kc, sc)                                 # value codes lie column by column
    with pytest.raises(TypeError):
        B.pages_append(x, x, slot, kc, sc, vc, sc)                                 # not on a device
    from promptcache_amd.model.kv_arena import PageCache
    for kw in (dict(page_size=24), dict(codes=torch.uint8), dict(max_pages=0)):
        with pytest.raises(ValueError):
            PageCache([(2, 32)], 2, 4, "cpu", **kw)
    with pytest.raises(ValueError):
        PageCache([(2, 40)], 2, 4, "cpu")
    c = PageCache([(2, 32), (1, 64)], 3, 4, "cpu", page_size=16)
    assert c.bytes_per_token() == 2 * (2 * 32 + 2 / 4) + 2 * (64 + 1 / 4)
    for bad in ((0, 1, 15), (0, 0, 16), (0, 1, 80), (0, 5, 16), (-1, 0, 16)):
        with pytest.raises(ValueError):
            c.share(*bad)
