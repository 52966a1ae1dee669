"""The paged attention within a bound that a lost page does not meet: every form, on both sides of the edges of its loops over
pages, and with weights that two nearly equal keys tell apart."""
import numpy as np
import pytest

from pagedkv_ref import D, P, ref
from test_gpu_pagedkv import Pair, qkv_of, rows_of

pytestmark = pytest.mark.gpu
FINE, FP16 = 22, 11   # bits of a weight: half a step is 2^-bits of it


class Keys:
    """Keys and values of one sequence and head in 64 bits, [len, 64] each."""

    def __init__(self, r, s, h):
        n, full = int(r.len[s]), int(r.len[s]) // P
        k, v = np.empty((n, D)), np.empty((n, D))
        for j in range(-(-n // P)):
            if j < full:
                page = r.table[s, j]
                a, b = (r.codes[0, page, i, h].astype(np.float64) * float(r.scales[0, page, i, h]) for i in (0, 1))
            else:
                a, b = (r.open[0, r.slot[s], i, h].astype(np.float64) for i in (0, 1))
            m = min(P, n - j * P)
            k[j * P:j * P + m] = a.reshape(P, D)[:m]
            v[j * P:j * P + m] = b.reshape(P // 8, D, 8).transpose(0, 2, 1).reshape(P, D)[:m]
        self.k, self.v = k, v

    def row(self, q, vis, bits):
        """The row's attention over its first `vis` keys, and how far a kernel may be off.

        The output is sum w v / sum w.  A weight that is off by e of itself moves it by w e (v - out) / sum w.  e: the score's sum of 64 fp32
        products, half a step 2^-24 of the running sum each, at most S = sum |q k| / 8 of them; its factors (6), the rounding of its
        distance to the maximum and of the maximum M with the 2^15 that weights are held at (4 M + 48), in half steps; 2^-23 for an
        exponential, of which there are up to 16 for moves of the maximum and joins; and the weight's own bits.  What is below fp16's range
        is off by 2^-40 of the largest weight.  Sums: a page's 32 products, then three steps a page and 64 for joins, for values and weights.
        The output's rounding: 2^-11 of it, or 2^-25."""
        k, v = self.k[:vis], self.v[:vis]
        x = k @ q / 8
        w = np.exp(x - x.max())
        tot = w.sum()
        out = w @ v / tot
        S, M = np.abs(k) @ np.abs(q) / 8, np.abs(x).max()
        e = 2.0 ** -24 * (64 * S + 6 * np.abs(x) + 4 * M + 48) + 16 * 2.0 ** -23 + 2.0 ** -bits
        away = np.abs(v - out)
        sums = 2.0 ** -24 * (32 + 3 * -(-vis // P) + 64)
        tol = (w * e) @ away + sums * (w @ np.abs(v)) * 2 + vis * 2.0 ** -40 * away.max(axis=0)
        tol = tol / tot * (1 + 2.0 ** -8) + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
        return out, tol, w

    def lost(self, out, tol, w):
        """For each page, how far past twice the bound the row without it is, at its largest (a last page of few tokens aside)."""
        n = -(-len(w) // P)
        wv, ws = np.zeros((n * P, D)), np.zeros(n * P)
        wv[:len(w)], ws[:len(w)] = w[:, None] * self.v[:len(w)], w
        wv, ws = wv.reshape(n, P, D).sum(axis=1), ws.reshape(n, P).sum(axis=1)
        left = ws.sum() - ws
        with np.errstate(invalid="ignore", divide="ignore"):
            without = (wv.sum(axis=0) - wv) / left[:, None]
        far = np.where(left > 0, (np.abs(without - out) / (2 * tol)).max(axis=1), np.inf)
        return far if len(w) % P == 0 or len(w) % P >= 8 else far[:-1]


def filled(pkg, L, rng, heads, lens, new, max_len, share=0):
    """A cache of those lengths whose last `new` tokens are the call's rows; pages anywhere in the pool (the second sequence has the first
    one's first `share`), the values of every page about a vector of its own, so that none can go unnoticed."""
    pages = sum(n // P for n in lens)
    p = Pair(pkg, L, layers=1, heads=heads, pages=pages + 2, seqs=len(lens), max_len=max_len)
    r, place, at = p.r, rng.permutation(pages + 2), 0
    for s, n in enumerate(lens):
        r.table[s, :n // P] = place[at:at + n // P]
        at += n // P
    r.table[1, :share] = r.table[0, :share]
    r.codes[:] = rng.integers(-60, 61, r.codes.shape, dtype=np.int8)
    v = r.codes[0, :, 1].reshape(-1, heads, P // 8, D, 8)
    v[:] = v // 3 + rng.choice(np.array([-50, 50], np.int8), (len(v), heads, 1, D, 1))
    r.codes[0, :, 1] = v.reshape(len(v), heads, -1)
    r.scales[:] = rng.uniform(0.006, 0.01, r.scales.shape)
    r.open[:] = rng.standard_normal(r.open.shape) * 0.2
    v = r.open[0, :, 1].reshape(-1, heads, P // 8, D, 8)
    r.open[0, :, 1] = (v + rng.choice([-0.4, 0.4], (len(v), heads, 1, D, 1))).reshape(len(v), heads, -1)
    r.len[:], r.start[:], r.slot[:] = lens, np.asarray(lens) - new, rng.permutation(len(lens))
    p.rows, p.n = rows_of(new), int(np.sum(new))
    p.d_rows = pkg.Dev.from_numpy(p.rows)
    return p


def check(p, x, got, bits, heads, rows=None, pages=None):
    """`got` within the bound, for some heads and rows (None: all); and all pages of those, or some, would be missed."""
    r, seen = p.r, 0
    got = got.astype(np.float64).reshape(len(x), -1, D)
    for s in range(r.seqs):
        mine = [i for i in range(p.rows[s], p.rows[s + 1]) if rows is None or i in rows]
        for h in heads if mine else []:
            kv = Keys(r, s, h)
            for i in mine:
                vis = int(r.start[s]) + i - int(p.rows[s]) + 1
                out, tol, w = kv.row(x[i, h * D:(h + 1) * D].astype(np.float64), vis, bits)
                err = np.abs(got[i, h] - out)
                assert (err <= tol).all(), f"sequence {s} row {i} head {h}: {(err / tol).max():.2f} of the bound ({err.max():.2e})"
                far = kv.lost(out, tol, w)
                far = far if pages is None else far[[j for j in pages if j < len(far)]]
                assert (far > 1).all(), f"sequence {s} row {i} head {h}: page {far.argmin()} would not be missed ({far.min():.2f})"
                seen += len(far)
    return seen


@pytest.mark.parametrize("seqs,rows,group,bits", [
    (4, 1, 1, FINE), (4, 1, 2, FINE), (16, 1, 8, FINE), (4, 2, 1, FINE), (16, 8, 1, FINE), (16, 8, 4, FINE),
    (16, 1, 16, FP16), (16, 9, 1, FP16), (4, 30, 1, FP16), (2, 70, 1, FP16),
])
@pytest.mark.parametrize("at,apart", [(40, 0.02), (46, 0.1), (50, 0.005), (127, 0.2)])
def test_two_nearly_equal_keys(pkg, L, seqs, rows, group, bits, at, apart):
    """Two keys of one page share nearly all of the weight and their values cancel, so that the output is how much they differ: weights of
    fp16 show there.  The others are 2^-10 and less of them."""
    heads = 2
    p, rng = Pair(pkg, L, layers=1, heads=heads, pages=seqs * 7, seqs=seqs, max_len=320), np.random.default_rng(50 + at)
    counts = [rows] + [1] * min(seqs - 1, max(seqs - rows, 1 if rows > seqs else 0)) + [0] * (rows - 1 if rows <= seqs else seqs - 2)
    assert len(counts) == seqs and (sum(counts) <= seqs) == (bits == FINE or rows in (1, 9))
    for step in ([at] * seqs, counts):
        assert p.grow(step)
        x = np.zeros((p.n, 3, heads, D), np.float16)
        x[:, 0, :, 0] = 8          # q . k / 8 is the key's first dim
        x[:, 1, :, 0] = -7 - rng.random((p.n, heads))
        x[:, 2] = rng.standard_normal((p.n, heads, D))
        on = np.flatnonzero(step)
        if step is not counts:
            v = rng.standard_normal((seqs, heads, D))
            x[p.rows[on] + at - 4, 1, :, 0], x[p.rows[on] + at - 4, 2] = 0, v[on]
        else:                      # each sequence's first new row: all of its rows see it
            x[p.rows[on], 1, :, 0], x[p.rows[on], 2] = -apart * (0.5 + rng.random((len(on), heads))), -v[on]
        x = x.reshape(p.n, -1)
        p.append(0, x)
    check(p, x, p.attend(0, x, group=group), bits, range(heads), pages=())


@pytest.mark.parametrize("length", [33, 64, 500, 2047, 2500, 5000])
@pytest.mark.parametrize("new,group,bits", [(1, 1, FINE), (3, 1, FINE), (1, 2, FINE), (9, 1, FP16)])
def test_no_page_is_lost(pkg, L, length, new, group, bits):
    """A work-group a sequence or group of beams, and 16 rows a work-group; split and not."""
    rng = np.random.default_rng(length + new)
    for max_len in (2048, 5120):
        if length <= max_len:
            lens = [length, max(length - 17, 1), 70, 5]
            p = filled(pkg, L, rng, 2, lens, [1] * 4 if group > 1 else [new, 0, 0, 0], max_len, share=lens[1] // P // 2 if group > 1 else 0)
            p.r.upload(pkg, p.c)
            x = qkv_of(rng, p.n, 2)
            assert check(p, x, p.attend(0, x, group=group), bits, (0, 1)) >= 2 * (length // P)


@pytest.mark.parametrize("heads,lens,new,rows", [
    (66, [8700, 9100, 300], [40, 19, 1], (0, 15, 16, 39, 40, 58, 59)),            # 16 rows a work-group, no splits
    (66, [8230, 8600], [35, 65], (0, 31, 34, 35, 66, 99)),                        # 32
    (121, [4190, 2112, 40], [700, 389, 11], (0, 63, 64, 699, 700, 1088, 1099)),   # 64, pages shared through LDS
    (121, [2048, 2080, 6200], [500, 300, 300], (0, 499, 500, 799, 800, 1099)),
])
def test_long_contexts_unsplit(pkg, L, heads, lens, new, rows):
    """More pages than a form looks up at once: 64 for 64 rows a work-group, 256 for the four waves of the others."""
    rng = np.random.default_rng(heads + lens[0])
    p = filled(pkg, L, rng, heads, lens, new, max(lens) + 200)
    p.r.upload(pkg, p.c)
    assert L.gpt2_pkv_attn_ws(ref(p.c), p.n) == 16, "not a case of this test: the call is split"
    x = qkv_of(rng, p.n, heads)
    x[:, :heads * D] *= np.float16(0.5)
    assert check(p, x, p.attend(0, x), FP16, (0, heads // 2, heads - 1), rows) > 1000


def test_half_a_million_tokens(pkg, L):
    """More pages than the 64 splits of one row's call look up at once, 16384: eleven pages that have most of the weight between them,
    on both sides of that edge and at the ends."""
    rng = np.random.default_rng(60)
    p, x = filled(pkg, L, rng, 1, [540010, 3], [1, 1], 540100), qkv_of(rng, 2, 1)
    r, pages = p.r, [0, 1, 255, 256, 8191, 16383, 16384, 16385, 16639, 16640, 16874]
    r.codes[0, :, 0, :, ::D] = 0
    r.codes[0, r.table[0, pages], 0, :, ::D] = 127
    r.scales[0, r.table[0, pages], 0] = 0.01
    r.upload(pkg, p.c)
    x[:, :D] *= np.float16(0.25)
    x[0, 0] = 57   # scores 9 above the others
    assert check(p, x, p.attend(0, x), FINE, (0,), rows=(0,), pages=pages) == 11
    check(p, x, p.attend(0, x), FINE, (0,), rows=(1,))
