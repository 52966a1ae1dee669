"""4-bit products whose sums are exact in fp32 in any order, so that the result is the exact one rounded to fp16 once, to the bit, at any K: no term
may be lost, and nothing may be rounded on the way.

x is +-1, a code is not 0, a scale is an odd whole number of units below 2^b: every partial sum is a whole number of units, at most
8 (2^b - 1) K of them, and bias and residual add less than 2^14.  With b = 6 that is below 2^24 up to K = 33000, with b = 11, where a scale has all of its bits, up to K = 1022.
A term is more than 1 (scales are at least 1), so leaving one out moves a result below 2048, whose steps are 1 at most, to another number of 16 bits."""
import numpy as np
import pytest

from int4_ref import TINY, U16, U32, cdiv, dequantized, gelu
from test_gpu_int4 import run
from test_gpu_int4_forms import FEW, MANY, ODD

SIZES = FEW + MANY + ODD + [(1, 300, 8192), (7, 48, 8200), (48, 48, 8200), (90, 48, 8200), (16, 600, 8190), (33, 200, 8190), (300, 130, 8191), (1, 17, 5), (20, 40, 3), (70, 33, 1000), (5, 70, 1022),
                            (129, 257, 1022), (400, 300, 1016), (2, 3100, 896), (300, 9001, 130), (600, 4099, 261), (867, 7343, 144),
                            (444, 4669, 776), (801, 1283, 1728)]


class Exact:
    def __init__(self, m, n, k, group, bits, epi=0):
        rng = np.random.default_rng([m, n, k, group, bits])
        self.m, self.n, self.k, self.group, self.epi = m, n, k, group, epi
        self.unit = 2.0 ** (1 - bits)
        assert 8 * (2 ** bits - 1) * k + 2 ** 14 <= 2 ** 24
        self.codes = rng.choice([q for q in range(-8, 8) if q], (n, k)).astype(np.int8)
        self.scales = ((rng.integers(2 ** (bits - 2), 2 ** (bits - 1), (n, cdiv(k, group))) * 2 + 1) * self.unit).astype(np.float16)   # 1 < s < 2
        self.x = rng.choice([-1, 1], (m, k)).astype(np.float16)
        self.bias = rng.integers(-4, 5, n).astype(np.float16)
        self.resid = rng.integers(-4, 5, (m, n)).astype(np.float16) if epi == 2 else None

    def want(self, x=None):
        """The exact result (whole numbers of units, in 64 bits)."""
        y = (self.x if x is None else x).astype(np.float64) @ dequantized(self.codes, self.scales, self.group).T + self.bias.astype(np.float64)
        return y if self.resid is None else y + self.resid


def sizes():
    return [(m, n, k, group, bits) for m, n, k in SIZES for group in (32, 64, 128) for bits in (6, 11) if bits == 6 or k <= 1022]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group,bits", sizes())
def test_rounded_once(pkg, L, m, n, k, group, bits):
    for epi in (0, 2):
        c = Exact(m, n, k, group, bits, epi)
        np.testing.assert_array_equal(run(pkg, L, c), c.want().astype(np.float16))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group,bits", [s for s in sizes() if s[4] == 6])
def test_gelu_of_exact_sums(pkg, L, m, n, k, group, bits):
    """Scales and biases 2^-6 of those, so that results are a few units and gelu bends them.  What it adds to the rounding is as int4_ref.product has it,
    with sums that are off by nothing: an exponent of at most 2^7 where the result is neither 0 nor v, off by a few steps of fp32, and steps of the result."""
    c = Exact(m, n, k, group, bits, epi=1)
    c.scales, c.bias = c.scales * np.float16(2.0 ** -6), c.bias * np.float16(2.0 ** -6)
    y = gelu(c.want())
    off = np.abs(run(pkg, L, c) - y)
    tol = 2.0 ** -14 * np.abs(y) * (np.abs(y) < 8) + 16 * U32 * np.abs(y)
    assert (off <= tol + U16 * (np.abs(y) + tol) + TINY).all()


@pytest.mark.parametrize("k", [3, 130, 1022, 8200])
@pytest.mark.parametrize("group", [32, 128])
def test_a_lost_term_is_seen(k, group):
    """The oracle with any one input left out, among them the last eight: other bits wherever a result is below 2048, which nearly all are."""
    c = Exact(3, 40, k, group, 6)
    full = c.want()
    low = np.abs(full) < 2046
    assert low.mean() > 0.98
    for lost in sorted(set(range(max(0, k - 8), k)) | set(range(0, k, 97))):
        x = c.x.copy()
        x[:, lost] = 0
        assert (c.want(x).astype(np.float16) != full.astype(np.float16))[low].all()


def test_a_rounding_on_the_way_is_seen():
    """The oracle with scaled weights rounded to fp16, and with groups' sums rounded to fp16: other bits in a good part of the results."""
    c = Exact(8, 64, 1000, 64, 11)
    right = c.want().astype(np.float16)
    w = dequantized(c.codes, c.scales, 64)
    x, bias = c.x.astype(np.float64), c.bias.astype(np.float64)
    rounded = x @ w.astype(np.float16).astype(np.float64).T + bias
    assert (rounded.astype(np.float16) != right).mean() > 0.1
    y = bias + sum((x[:, k:k + 64] @ w[:, k:k + 64].T).astype(np.float16).astype(np.float64) for k in range(0, 1000, 64))
    assert (y.astype(np.float16) != right).mean() > 0.1
