"""Attention over the paged 8-bit cache where scores are so large that neighbouring fp32 numbers are further than e apart: rows stay finite, and the key that wins is read."""
import numpy as np
import pytest
import torch

from oracle import pages_oracle as O
from tests.test_gpu_pages import DEV, Requests

pytestmark = pytest.mark.gpu
FORMS = [(1, 0), (9, 0), (64, 0), (64, 1 << 22)]                    # tile rows; a bound of the lengths that has short work take the blocks of 128 columns


def absolute(r):
    return r.vc & 127 if r.kind == "e4m3" else np.abs(r.vc.view(np.int8).astype(np.int16)).clip(0, 127).astype(np.int8).view(np.uint8)


def compare(r, got, **kw):
    """Weights of the row's largest score are one power of two alike and all others 0 (scores are further apart than exponentials reach), so a result is a sum of codes, exact, over
    the number of winners; where one is no power of two after all (scores below 2^20), the second product has it as a half (2^-11), fp32 as two (2^-22), and the denominator whole.  A
    quotient, two products and its rounding."""
    args = (r.q.double().cpu().numpy(), r.seqs, r.pos, r.kv, r.table, r.kc, r.ks)
    want = O.attend(*args, r.vc, r.vs, r.P, r.kind, kw.get("scale", 1.0), kw.get("window", 0))
    A = O.attend(*args, absolute(r), r.vs, r.P, r.kind, kw.get("scale", 1.0), kw.get("window", 0))
    off = np.abs(got.double().cpu().numpy() - want)
    tol = torch.finfo(r.dtype).eps / 2 * np.abs(want) + (2.0 ** -11 if r.dtype == torch.bfloat16 else 2.0 ** -21) * A * (1 + 2.0 ** -8)
    assert (off <= tol).all(), (np.nanmax(off / np.maximum(tol, 1e-300)), int((~(off <= tol)).sum()), np.argwhere(~(off <= tol))[:5])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("T, longest", FORMS)
@pytest.mark.parametrize("low, high", [(10, 21), (20, 41)])
def test_rows_that_see_one_key(low, high, T, longest, kind, dtype):
    """A window of one: whatever the score, the result is that key's value."""
    r = Requests([300, 77, 1500], [T, T, T], 6, 3, 64, 32, kind, dtype, seed=T + low, scales=(low, high))
    r.vs[:] = np.exp2(np.random.default_rng(T).integers(-40, 41, r.vs.shape))
    r.q = torch.randn(r.q.shape, generator=torch.Generator(device=DEV).manual_seed(low), device=DEV).to(r.dtype)
    compare(r, r.run(T, window=1, longest=longest), window=1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("T, longest", FORMS)
@pytest.mark.parametrize("dim", [32, 128, 192])
def test_the_largest_score_wins(dim, T, longest, kind, dtype):
    """Products of small whole numbers, odd ones, under a key scale of each page's own (2^20 .. 2^40): two scores are equal only within a page, and otherwise 2^-11 of them or more apart."""
    P = 16
    r = Requests([250, 90], [T, T], 6, 3, dim, P, kind, dtype, seed=dim + T)
    rng = np.random.default_rng(dim + T)
    k = 2 * rng.integers(-1, 2, r.kc.shape)
    k[..., 0] = 2 * rng.integers(-2, 2, k.shape[:-1]) + 1
    r.kc = O.encode(k, kind)
    q = 2 * rng.integers(-1, 2, r.q.shape)
    q[..., 0] = 2 * rng.integers(-2, 2, q.shape[:-1]) + 1
    q[3:5] *= -1
    r.q = torch.from_numpy(q.astype(np.float64)).to(DEV, r.dtype)
    for s, row in enumerate(r.table):
        n = -(-r.kv[s] // P)
        assert n <= 21
        for h in range(r.ks.shape[1]):
            r.ks[row[:n], h] = np.exp2(20 + rng.permutation(21)[:n])
            r.vs[row[:n], h] = np.exp2(rng.integers(-20, 21, n))
    compare(r, r.run(T, longest=longest))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T, longest", FORMS)
def test_far_scores_of_any_kind_stay_between_the_values(T, longest, dtype):
    """Long rows of random numbers under every key scale: results are numbers, no larger than the largest value; what is no number stays where it was."""
    r = Requests([5000, 40], [T, T], 8, 2, 128, 64, "e4m3", dtype, seed=T)
    gen = torch.Generator(device=DEV).manual_seed(T)
    top = 448 * float(r.vs.max()) * (1 + 2.0 ** -7)
    for e in (4, 8, 12, 14, 16, 17, 18, 20, 24, 32, 40):
        r.ks[:] = 2.0 ** e
        r.q = torch.randn(r.q.shape, generator=gen, device=DEV).to(r.dtype)
        got = r.run(T, longest=longest)
        assert bool((got.float().abs() <= top).all()), e
    bad = r.q.clone()
    bad[T, 3, 7] = float("nan")
    none = torch.isnan(r.run(T, q=bad, longest=longest))
    assert bool(none[T, 3].all()) and int(none.sum()) == 128


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T, longest", FORMS)
def test_far_scores_beside_a_sink(T, longest, dtype):
    """One key a row, its score far above the sink or far below: its value, or 0."""
    r = Requests([3000, 77], [T, T], 8, 2, 64, 32, "int8", dtype, seed=T + 3, scales=(24, 41))
    r.q = torch.randn(r.q.shape, generator=torch.Generator(device=DEV).manual_seed(T), device=DEV).to(r.dtype)
    got = r.run(T, window=1, longest=longest, sink=[2.5, -7.0, 0.0, 30.0] * 2)
    z = O.attend(r.q.double().cpu().numpy(), r.seqs, r.pos, r.kv, r.table, r.kc, r.ks, r.vc, r.vs, r.P, r.kind, 1.0, 1, [2.5, -7.0, 0.0, 30.0] * 2)
    alone = O.attend(r.q.double().cpu().numpy(), r.seqs, r.pos, r.kv, r.table, r.kc, r.ks, r.vc, r.vs, r.P, r.kind, 1.0, 1)
    assert ((z == 0).all(-1) | (np.abs(z - alone) <= 2.0 ** -40 * np.abs(alone)).all(-1)).all()      # (so far are they: nothing in between)
    assert 0 < (z == 0).all(-1).sum() < z[..., 0].size
    assert (np.abs(got.double().cpu().numpy() - z) <= (torch.finfo(r.dtype).eps / 2 + 2.0 ** -21) * np.abs(z)).all()
