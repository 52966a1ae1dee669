"""4-bit weights on the GPU: the quantiser and its inverse to the bit, the products against 64 bits (tests/int4_ref.py)."""
import ctypes as C

import numpy as np
import pytest

from int4_ref import Weights, dequantized, pack, product, quantize, unpack

pytestmark = pytest.mark.gpu


def matrix(rng, n, k, scale=0.05):
    w = rng.standard_normal((n, k)) * scale * rng.uniform(0.3, 3, (n, 1))
    w[rng.random((n, k)) < 0.01] *= 6
    return w.astype(np.float16)


def quantized(pkg, L, w, group, shift=0):
    """What the library makes of w, which begins `shift` halves past a 16-byte boundary: the struct's owner."""
    n, k = w.shape
    q = pkg.Int4(n, k, group)
    buf = np.zeros(shift + w.size, np.float16)
    buf[shift:] = w.ravel()
    d = pkg.Dev.from_numpy(buf)
    L.gpt2_quantize_int4(C.byref(q.w), d.at(2 * shift))
    L.gpt2_sync()
    pkg.check("gpt2_quantize_int4")
    return q


def held(pkg, L, q):
    nt, kb, per = -(-q.w.N // 16), -(-q.w.K // 128), 128 // q.w.group
    words, scales = np.empty((nt, kb, 4, 16, 4), np.uint32), np.empty((nt, kb, 4, per, 4), np.float16)
    assert words.nbytes == L.gpt2_int4_code_bytes(q.w.N, q.w.K) and scales.size == L.gpt2_int4_scale_count(q.w.N, q.w.K, q.w.group)
    assert L.gpt2_d2h(words.ctypes.data, q.w.codes, words.nbytes) == 0 and L.gpt2_d2h(scales.ctypes.data, q.w.scales, scales.nbytes) == 0
    return words, scales


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,shift", [(1, 1, 0), (16, 128, 0), (17, 130, 0), (5, 37, 1), (48, 768, 0), (33, 200, 0), (33, 200, 4), (768, 768, 0), (2305, 96, 0)])
def test_quantize(pkg, L, n, k, shift, group):
    w = matrix(np.random.default_rng(n + k), n, k)
    q = quantized(pkg, L, w, group, shift)
    codes, scales = quantize(w, group)
    words, s = held(pkg, L, q)
    want, _ = pack(codes, scales, group)
    np.testing.assert_array_equal(words, want)   # rows past N and k past K are 0 too
    np.testing.assert_array_equal(unpack(words, s, n, k, group)[1].view(np.uint16), scales.view(np.uint16))
    buf = np.full(shift + n * k + 8, 77, np.float16)
    d = pkg.Dev.from_numpy(buf)
    L.gpt2_dequantize_int4(d.at(2 * shift), C.byref(q.w))
    L.gpt2_sync()
    pkg.check("gpt2_dequantize_int4")
    got = d.numpy(np.float16, buf.size)
    assert (got[:shift] == 77).all() and (got[shift + n * k:] == 77).all()
    np.testing.assert_array_equal(got[shift:shift + n * k].reshape(n, k), dequantized(codes, scales, group).astype(np.float16))
    q.free()


def test_quantize_odd_values(pkg, L):
    """Zeros, NaN, infinities, the smallest numbers, groups of one large value, ties between codes."""
    rng = np.random.default_rng(3)
    w = matrix(rng, 64, 256)
    w[0] = 0
    w[1, 3], w[1, 40], w[2, 5] = np.nan, np.inf, -np.inf
    w[3] = rng.integers(-40, 40, 256) * np.float16(2.0 ** -24)   # scales below the smallest number, and of few bits
    w[4] = np.float16(2.0 ** -24)
    w[5], w[5, 0] = 0.001, 60000
    w[6] = np.float16(0.5) * rng.integers(-14, 15, 256)          # s = 1: halves between codes
    w[6, ::32] = 7
    w[7] = np.float16(65504)
    w[8] = -w[6]
    for group in (32, 64, 128):
        q = quantized(pkg, L, w, group)
        codes, scales = quantize(w, group)
        got = unpack(*held(pkg, L, q), 64, 256, group)
        np.testing.assert_array_equal(got[0], codes)
        np.testing.assert_array_equal(got[1], scales)
        q.free()


class Case:
    def __init__(self, m, n, k, group, seed=0, epi=0, bias=True):
        rng = np.random.default_rng([m, n, k, group, seed])
        self.m, self.n, self.k, self.group, self.epi = m, n, k, group, epi
        self.codes = rng.integers(-8, 8, (n, k)).astype(np.int8)
        self.scales = (rng.uniform(0.3, 1.5, (n, -(-k // group))) * 0.3 / np.sqrt(k) * rng.choice([-1, 1], (n, 1), p=[0.1, 0.9])).astype(np.float16)
        self.x = rng.standard_normal((m, k)).astype(np.float16)
        self.x[:, ::31] *= 6
        self.bias = (rng.standard_normal(n) * 0.5).astype(np.float16) if bias else None
        self.resid = rng.standard_normal((m, n)).astype(np.float16) if epi == 2 else None


def run(pkg, L, c, x_shift=0, c_shift=0, in_place=False, weights=None, **kw):
    """C of case c; A and C begin so many halves past a 16-byte boundary.  What lies around C has to stay."""
    w = weights or Weights(pkg, c.codes, c.scales, c.group, **kw)
    a = np.full(x_shift + c.x.size + 8, np.nan, np.float16)
    a[x_shift:x_shift + c.x.size] = c.x.ravel()
    d_a = pkg.Dev.from_numpy(a)
    out = np.full(c_shift + c.m * c.n + 8, 77, np.float16)
    if in_place:
        out[c_shift:c_shift + c.m * c.n] = c.resid.ravel()
    d_c = pkg.Dev.from_numpy(out)
    d_b = pkg.Dev.from_numpy(c.bias) if c.bias is not None else None
    d_r = pkg.Dev.from_numpy(c.resid) if c.epi == 2 and not in_place else None
    resid = d_c.at(2 * c_shift) if in_place else d_r.ptr if d_r else None
    L.gpt2_matmul_int4(d_c.at(2 * c_shift), d_a.at(2 * x_shift), w.ref, d_b.ptr if d_b else None, c.m, c.epi, resid)
    L.gpt2_sync()
    pkg.check("gpt2_matmul_int4")
    got = d_c.numpy(np.float16, out.size)
    assert (got[:c_shift] == 77).all() and (got[c_shift + c.m * c.n:] == 77).all()
    return got[c_shift:c_shift + c.m * c.n].reshape(c.m, c.n)


def check(pkg, L, c, **kw):
    got = run(pkg, L, c, **kw)
    want, tol = product(c.x, c.codes, c.scales, c.group, c.bias, c.epi, c.resid)
    off = np.abs(got - want)
    assert (off <= tol).all(), (float((off - tol).max()), np.argwhere(off > tol)[:4])
    return got


ROWS = [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 257]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", ROWS)
def test_rows(pkg, L, m, group):
    check(pkg, L, Case(m, 2304 if m % 2 else 768, 768, group))


@pytest.mark.parametrize("m", [1, 7, 16, 40, 64, 90, 300])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (1, 128, 64), (15, 32, 32), (17, 8, 128), (33, 129, 64), (50, 250, 32), (129, 1000, 128), (257, 264, 64),
                                       (100, 3000, 32), (65, 4104, 128), (1030, 136, 64), (48, 8200, 32)])
def test_odd_sizes(pkg, L, m, n, k, group):
    check(pkg, L, Case(m, n, k, group, bias=n % 2 == 0))


@pytest.mark.parametrize("epi", [0, 1, 2])
@pytest.mark.parametrize("m,n,k,group", [(1, 768, 3072, 64), (1, 301, 200, 32), (6, 3072, 768, 32), (48, 3072, 768, 128), (64, 769, 768, 64), (333, 768, 3072, 64), (130, 255, 896, 32)])
def test_epilogues(pkg, L, m, n, k, group, epi):
    for bias in (False, True):
        c = Case(m, n, k, group, epi=epi, bias=bias)
        got = check(pkg, L, c)
        if epi == 2:
            np.testing.assert_array_equal(run(pkg, L, c, in_place=True), got)


@pytest.mark.parametrize("x_shift,c_shift", [(1, 0), (4, 1), (0, 3), (8, 2)])
@pytest.mark.parametrize("m,n,k", [(1, 96, 256), (1, 97, 256), (20, 96, 256), (20, 97, 256), (150, 96, 256), (150, 97, 256)])
def test_alignment(pkg, L, m, n, k, x_shift, c_shift):
    """The same values wherever the rows begin, to the bit where the same form runs."""
    c = Case(m, n, k, 64, epi=2)
    got = check(pkg, L, c, x_shift=x_shift, c_shift=c_shift)
    if x_shift % 8 == 0:
        np.testing.assert_array_equal(got, run(pkg, L, c))


@pytest.mark.parametrize("m", [1, 8, 30, 64, 140])
def test_vocabulary(pkg, L, m):
    check(pkg, L, Case(m, 50257, 768, 128, bias=False))


@pytest.mark.parametrize("m", [1, 16, 33, 64, 200])
def test_what_means_nothing(pkg, L, m):
    """Codes and scales of rows past N do not count, whatever they are; codes of k past K are 0, and what A has behind a row is not read as
    part of it; rows of A with NaN or infinities leave the others alone."""
    c = Case(m, 37, 200, 32)
    plain = check(pkg, L, c)
    np.testing.assert_array_equal(run(pkg, L, c, rest=3, rest_scale=np.nan), plain)
    if m > 1:
        c.x[m // 2, 5], c.x[0, 7] = np.nan, np.inf
        c.codes[:, 7] = np.where(c.codes[:, 7] == 0, 1, c.codes[:, 7])
        got = run(pkg, L, c)
        assert np.isnan(got[m // 2]).all() and not np.isfinite(got[0]).any()
        others = [r for r in range(m) if r not in (0, m // 2)]
        clean = Case(m, 37, 200, 32)
        clean.codes = c.codes
        np.testing.assert_array_equal(got[others], run(pkg, L, clean)[others])


def test_range(pkg, L):
    """Outputs past fp16 become infinities, the smallest scales and activations count."""
    for m in (1, 20, 150):
        c = Case(m, 64, 256, 64, bias=False)
        c.scales[0], c.scales[1] = 60000, 2.0 ** -24
        c.codes[0], c.x[0] = 7, 100
        got = run(pkg, L, c)
        assert np.isposinf(got[0, 0])
        c.scales[:] = np.float16(2.0 ** -24) * np.arange(1, 65)[:, None]
        c.x = (np.sign(c.x) * 1000).astype(np.float16)
        check(pkg, L, c)
        c.scales[:] = 4
        c.x = (np.float16(2.0 ** -24) * np.random.default_rng(m).integers(-900, 900, c.x.shape)).astype(np.float16)
        check(pkg, L, c)


@pytest.mark.parametrize("m,n,k", [(1, 8192, 8192), (50, 4096, 4096), (500, 2048, 4096)])
def test_large(pkg, L, m, n, k):
    check(pkg, L, Case(m, n, k, 128))


def test_same_bits_again(pkg, L):
    """Calls repeat themselves to the bit, and a row's result does not depend on the other rows' values."""
    for m in (1, 9, 40, 64, 200):
        c = Case(m, 768, 3072, 64)
        w = Weights(pkg, c.codes, c.scales, c.group)
        a = run(pkg, L, c, weights=w)
        np.testing.assert_array_equal(a, run(pkg, L, c, weights=w))
        c.x[:m - 1] = 3
        np.testing.assert_array_equal(a[m - 1], run(pkg, L, c, weights=w)[m - 1])


def test_outputs_past_4_gib(pkg, L):
    """More than 2^32 bytes of results, from rows at 16 bytes and from others: the first and the last rows."""
    for k in (32, 30):
        m, n = 43000, 50257
        c = Case(4, n, k, 32, bias=False)
        rows = np.zeros((m, k), np.float16)
        rows[:2], rows[-2:] = c.x[:2], c.x[2:]
        w = Weights(pkg, c.codes, c.scales, 32)
        d_a, d_c = pkg.Dev.from_numpy(rows), pkg.Dev(m * n * 2)
        L.gpt2_matmul_int4(d_c.ptr, d_a.ptr, w.ref, None, m, 0, None)
        L.gpt2_sync()
        pkg.check("gpt2_matmul_int4")
        got = np.empty((4, n), np.float16)
        assert L.gpt2_d2h(got.ctypes.data, d_c.ptr, 4 * n) == 0 and L.gpt2_d2h(got[2:].ctypes.data, d_c.at((m - 2) * n * 2), 4 * n) == 0
        want, tol = product(c.x, c.codes, c.scales, 32, None, 0, None)
        assert (np.abs(got - want) <= tol).all()
        d_c.free()
