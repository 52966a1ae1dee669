"""Beam search's selection: equal scores go by the documented order wherever the rows lie, and a row gives the same bits anywhere."""
import numpy as np
import pytest

from pagedkv_ref import beam
from test_gpu_beam import select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams", [2, 4, 8, 16])
@pytest.mark.parametrize("V", [37, 1003, 9001, 50255, 50257])
def test_equal_rows_tie(pkg, L, V, beams):
    """Rows that are the same, with V odd at eight distances from a 16-byte boundary: the lower row first; groups that are the same choose
    the same, to the bit."""
    rng = np.random.default_rng(V + beams)
    groups = 3
    for spread in (0.5, 3.0):
        row = (rng.standard_normal(V) * spread - 20).astype(np.float16)
        x = np.stack([row] * (groups * beams))
        for score in (np.zeros(beams), -rng.choice([0.5, 0.75, 3.0], beams)):   # some are equal
            s = np.tile(score, groups).astype(np.float32)
            done = np.zeros(groups * beams, np.int32)
            token, parent, want, _, _ = beam(x, s, done, groups, beams, -1)
            got = select(pkg, L, x, s, done, groups, beams, -1)
            np.testing.assert_array_equal(got[0], token)
            np.testing.assert_array_equal(got[1], parent)
            bits = got[2].view(np.uint32).reshape(groups, beams)
            np.testing.assert_array_equal(bits, bits[:1].repeat(groups, 0))
            assert (np.abs(got[2] - want) <= 2.0 ** -24 * (95 + np.abs(want))).all()   # as in test_gpu_beam.check


@pytest.mark.parametrize("V,ld", [(50257, 50257), (50000, 50003), (313, 320), (9, 17), (1, 2)])
def test_a_row_anywhere(pkg, L, V, ld):
    """The same rows beginning at each even address of 16 bytes: the same scores to the bit."""
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((4, V)) * 2).astype(np.float16)
    x[1, rng.random(V) < 0.3] = -np.inf
    x[3] = x[0]
    first = None
    for shift in range(8):
        got = select(pkg, L, x, np.array([-1, -2, -1, -1], np.float32), np.zeros(4, np.int32), 1, 4, -1, ld=ld, shift=shift)
        first = first or got
        for a, b in zip(got, first):
            np.testing.assert_array_equal(a.view(np.uint32), b.view(np.uint32))
