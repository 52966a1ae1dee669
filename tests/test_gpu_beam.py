"""Beam search's selection on the GPU against the same in 64 bits (tests/pagedkv_ref.py: beam)."""
import numpy as np
import pytest

from pagedkv_ref import Ws, beam

pytestmark = pytest.mark.gpu


def select(pkg, L, logits, score, done, groups, beams, eos, ld=None, shift=0):
    """`shift`: logits begin that many halves past a 16-byte boundary; rows are ld apart, NaN between them."""
    rows, V = logits.shape
    ld = ld or V
    buf = np.full(shift + rows * ld, np.nan, np.float16)
    for r in range(rows):
        buf[shift + r * ld:shift + r * ld + V] = logits[r]
    d_x = pkg.Dev.from_numpy(buf)
    d_score, d_done = pkg.Dev.from_numpy(np.asarray(score, np.float32)), pkg.Dev.from_numpy(np.asarray(done, np.int32))
    tok, par = pkg.Dev(4 * rows), pkg.Dev(4 * rows)
    ws = Ws(pkg, L.gpt2_beam_select_ws(groups, beams, V))
    L.gpt2_beam_select(tok.ptr, par.ptr, d_score.ptr, d_done.ptr, d_x.at(2 * shift), ld, d_score.ptr, d_done.ptr, groups, beams, V, eos,
                       *ws.args)   # scores and marks in place
    L.gpt2_sync()
    pkg.check("gpt2_beam_select")
    return tok.numpy(np.int32, rows), par.numpy(np.int32, rows), d_score.numpy(np.float32, rows), d_done.numpy(np.int32, rows)


def check(pkg, L, logits, score, done, groups, beams, eos, **kw):
    got = select(pkg, L, logits, score, done, groups, beams, eos, **kw)
    token, parent, want, mark, gap = beam(logits, np.asarray(score, np.float32), done, groups, beams, eos)
    # The log of the sum: each exponential's argument is off by half a step 2^-24 of at most 60, the result by one step
    # 2^-23 more, a thread's sum of 33 of them at most in fp32: below 2^-24 (60 + 2 + 33) of the sum.  The score's rounding:
    # 2^-24 of it.
    tol = 2.0 ** -24 * 95
    assert gap > 4 * tol, "two candidates too close to tell apart: not a case of this test"
    np.testing.assert_array_equal(got[0], token)
    np.testing.assert_array_equal(got[1], parent)
    np.testing.assert_array_equal(got[3], mark)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[2][~fin], want[~fin])
    assert (np.abs(got[2][fin] - want[fin]) <= tol + 2.0 ** -24 * np.abs(want[fin])).all()


def some(rng, rows, V, scale=2.0):
    x = (rng.standard_normal((rows, V)) * scale - 3).astype(np.float16)
    return x, -rng.uniform(0, 5, rows), (rng.random(rows) < 0.2).astype(np.int32)


@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (3, 5), (2, 16), (7, 2)])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 33, 1000, 8191, 8192, 8209, 50257, 65536])
def test_select(pkg, L, groups, beams, V):
    rng = np.random.default_rng(1000 * beams + V)
    x, score, done = some(rng, groups * beams, V)
    check(pkg, L, x, score, done, groups, beams, V - 1)


@pytest.mark.parametrize("V,shift", [(50257, 0), (50255, 3)])
def test_many_rows(pkg, L, V, shift):
    """As many rows as take the larger parts."""
    rng = np.random.default_rng(V)
    x, score, done = some(rng, 256, V)
    x[7] = -np.inf
    x[9, 5000:] = -np.inf
    x[11] = 0
    check(pkg, L, x, score, done, 32, 8, V - 1, shift=shift)


@pytest.mark.parametrize("shift", range(8))
def test_rows_anywhere(pkg, L, shift):
    rng = np.random.default_rng(shift)
    x, score, done = some(rng, 6, 301 + shift)
    check(pkg, L, x, score, done, 2, 3, 5, ld=333, shift=shift)
    x, score, done = some(rng, 4, 5)
    check(pkg, L, x, score, done, 1, 4, -1, ld=6, shift=shift)


def test_ties_and_extremes(pkg, L):
    """All equal; sorted both ways (one lane holds the best); +0 and -0; a single token above the rest."""
    V, beams = 9000, 8
    up = np.linspace(-4, 4, V).astype(np.float16)
    zeros = np.zeros(V, np.float16)
    zeros[::2] = -0.0
    spike = np.full(V, -10, np.float16)
    spike[8999] = 30
    for x in (np.zeros(V, np.float16), up, up[::-1], zeros, spike, np.full(V, 65504, np.float16), np.full(V, -65504, np.float16)):
        rows = np.stack([x] * beams)
        check(pkg, L, rows, -np.arange(beams) * 0.37, np.zeros(beams, np.int32), 1, beams, -1)
        got = select(pkg, L, rows, np.zeros(beams), np.zeros(beams, np.int32), 1, beams, -1)   # rows that are the same, too
        first = sorted(range(V), key=lambda t: (-float(x[t]), t))[0]
        assert got[0][0] == first and got[1][0] == 0


def test_masked_rows_and_scores(pkg, L):
    """-inf and NaN logits, rows with nothing left, +inf, beams that are not there (-inf), scores that are NaN."""
    rng = np.random.default_rng(5)
    V, beams = 500, 4
    x, _, _ = some(rng, 8, V)
    x[0, :] = -np.inf
    x[1, 3:] = -np.inf
    x[2, ::2] = np.nan
    x[3, 7] = np.inf
    x[4, :] = np.nan
    score = np.array([-1.0, -2.25, -np.inf, -0.5, -1, -np.inf, -np.inf, np.nan], np.float32)
    check(pkg, L, x, score, np.zeros(8, np.int32), 2, beams, -1)
    done = np.array([1, 0, 0, 1, 1, 1, 1, 1], np.int32)
    check(pkg, L, x, score, done, 2, beams, 9)
    # the first step of a search: only the first beam of a group counts
    y = np.concatenate([np.repeat(x[5:6], 4, 0), np.repeat(x[6:7], 4, 0)])
    check(pkg, L, y, np.array([0, -np.inf, -np.inf, -np.inf] * 2, np.float32), np.zeros(8, np.int32), 2, 4, 9)


def test_every_beam_done(pkg, L):
    rng = np.random.default_rng(6)
    x, score, _ = some(rng, 5, 100)
    check(pkg, L, x, score, np.ones(5, np.int32), 1, 5, 42)


def test_same_bits_every_time(pkg, L):
    rng = np.random.default_rng(7)
    x, score, done = some(rng, 32, 50257)
    a = select(pkg, L, x, score, done, 4, 8, 50256)
    for _ in range(3):
        b = select(pkg, L, x, score, done, 4, 8, 50256)
        for u, v in zip(a, b):
            np.testing.assert_array_equal(u, v)
