"""Logits' rules and token histories on the GPU against plain numpy (tests/int4_ref.py)."""
import ctypes as C

import numpy as np
import pytest

from int4_ref import Histories, adjust, mask_words

pytestmark = pytest.mark.gpu


class Rules:
    """Rows of random rules, on the host and on the device."""

    def __init__(self, pkg, rng, rows, V, past, ngram=0, biases=0, masks=0, room=None, words=None, mask_row=True, penalties=True):
        self.pkg, self.V, self.ngram = pkg, V, ngram
        self.keep = []
        r = self.r = pkg.GPT2LogitsRules()
        dev = lambda a, t: self.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or self.keep[-1].ptr  # noqa: E731
        self.seqs = self.starts = None
        if past is not None:
            words = words or max(2, V // 7)
            self.seqs = [(rng.integers(0, words, n) * 7 % V).tolist() for n in past]
            self.starts = [int(rng.integers(0, n + 1)) for n in past]
            room = room or max(1, max(past))
            self.history(dev, room)
        self.rep, self.pres, self.freq = np.ones(rows, np.float32), np.zeros(rows, np.float32), np.zeros(rows, np.float32)
        if penalties:
            self.rep = rng.uniform(0.8, 1.6, rows).astype(np.float32)
            self.pres, self.freq = (rng.uniform(-0.5, 1.5, rows).astype(np.float32) for _ in range(2))
            r.repetition, r.presence, r.frequency = dev(self.rep, np.float32), dev(self.pres, np.float32), dev(self.freq, np.float32)
        r.ngram = ngram
        self.biases = [[] for _ in range(rows)]
        if biases:
            for b in self.biases:
                n = int(rng.integers(0, biases + 1))
                t = rng.integers(-3, V + 3, n)
                v = rng.standard_normal(n).astype(np.float32) * 5
                if n > 2:
                    t[n // 2], t[n - 1] = t[0], t[0]   # a token three times
                    v[1] = -np.inf
                b += list(zip(t.tolist(), v.tolist()))
            flat = sum(self.biases, [])
            r.n_bias = len(flat)
            r.bias_start = dev(np.cumsum([0] + [len(b) for b in self.biases]), np.int32)
            r.bias_token, r.bias_value = dev([t for t, _ in flat] or [0], np.int32), dev([v for _, v in flat] or [0], np.float32)
        self.masks = [None] * rows
        if masks:
            allowed = rng.random((masks, V)) < rng.random((masks, 1)) ** 2
            allowed[-1] = True
            allowed[0] = False
            self.keep.append(allowed)
            r.mask, r.n_masks = dev(mask_words(allowed), np.uint32), masks
            pick = rng.integers(-1, masks + 1, rows) if mask_row else np.arange(rows)
            if mask_row:
                r.mask_row = dev(pick, np.int32)
            self.masks = [allowed[p] if 0 <= p < masks else None for p in pick]

    def history(self, dev, room):
        h = self.h = self.pkg.GPT2History()
        tokens = np.full((len(self.seqs), room), 5, np.int32)
        for row, s in zip(tokens, self.seqs):
            row[:len(s)] = s
        h.tokens, h.len, h.start, h.arrived = dev(tokens, np.int32), dev([len(s) for s in self.seqs], np.int32), dev(self.starts, np.int32), dev([0], np.int32)
        h.nSeq, h.room = tokens.shape
        self.r.history = C.pointer(h)

    def want(self, logits):
        return adjust(logits, self.seqs, self.starts, self.rep, self.pres, self.freq, self.ngram, self.biases, self.masks)


def some_logits(rng, rows, V):
    x = (rng.standard_normal((rows, V)) * 4).astype(np.float16)
    x[rng.random((rows, V)) < 0.01] = -np.inf
    x[rng.random((rows, V)) < 0.01] = 0
    return x


def run(pkg, L, x, rules, ld=None, shift=0, out_shift=None):
    """Logits after the rules; out_shift None: in place.  What lies between the rows has to stay."""
    rows, V = x.shape
    ld = ld or V

    def rows_at(at, fill):
        buf = np.full(at + rows * ld + 8, fill, np.float16)
        inside = np.zeros(buf.size, bool)
        for r in range(rows):
            inside[at + r * ld:at + r * ld + V] = True
        return buf, inside
    buf, inside = rows_at(shift, 55)
    buf[inside] = x.ravel()
    d = pkg.Dev.from_numpy(buf)
    if out_shift is None:
        o, o_inside, at = d, inside, d.at(2 * shift)
    else:
        obuf, o_inside = rows_at(out_shift, 55)
        o = pkg.Dev.from_numpy(obuf)
        at = o.at(2 * out_shift)
    L.gpt2_logits_adjust(at, d.at(2 * shift), ld, rows, V, C.byref(rules.r))
    L.gpt2_sync()
    pkg.check("gpt2_logits_adjust")
    got = o.numpy(np.float16, o_inside.size)
    assert (got[~o_inside] == 55).all()
    if out_shift is not None:
        np.testing.assert_array_equal(d.numpy(np.uint16, buf.size), buf.view(np.uint16))
    return got[o_inside].reshape(rows, V)


def same(got, want, tol):
    fin = np.isfinite(want)
    with np.errstate(over="ignore"):
        big = np.abs(want) > 65504   # rounded to an infinity, or to the last number below
    np.testing.assert_array_equal(got[~fin], want[~fin])
    fin &= ~big
    assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all()


def check(pkg, L, x, rules, **kw):
    want, tol = rules.want(x)
    got = run(pkg, L, x, rules, **kw)
    same(got, want, tol)
    return got


PAST = [0, 1, 2, 3, 40, 300, 1000]


@pytest.mark.parametrize("V", [1, 2, 7, 8, 31, 32, 33, 1000, 4095, 4096, 4104, 8193, 50257])
@pytest.mark.parametrize("ngram,biases,masks", [(0, 0, 0), (2, 0, 0), (0, 20, 0), (0, 0, 3), (3, 300, 5)])
def test_rules(pkg, L, V, ngram, biases, masks):
    rng = np.random.default_rng([V, ngram, masks])
    rules = Rules(pkg, rng, 7, V, PAST, ngram, biases, masks, words=min(V, 60))
    x = some_logits(rng, 7, V)
    a = check(pkg, L, x, rules)
    np.testing.assert_array_equal(check(pkg, L, x, rules, out_shift=0).view(np.uint16), a.view(np.uint16))


@pytest.mark.parametrize("ld,shift,out_shift", [(1005, 0, 0), (1001, 1, 1), (1008, 3, 2), (1001, 2, 5), (1003, 7, None), (1001, 1, None)])
def test_alignment(pkg, L, ld, shift, out_shift):
    rng = np.random.default_rng(ld + shift)
    for masks in (0, 4):
        rules = Rules(pkg, rng, 7, 1000, PAST, 2, 30, masks)
        check(pkg, L, some_logits(rng, 7, 1000), rules, ld=ld, shift=shift, out_shift=out_shift)


@pytest.mark.parametrize("ngram", [1, 2, 3, 4, 7, 40, 41, 1000, 5000])
def test_ngrams(pkg, L, ngram):
    """Histories of few words, so that n-grams come again; one that repeats itself wholly; those shorter than the n-gram ban nothing."""
    rng = np.random.default_rng(ngram)
    rules = Rules(pkg, rng, 7, 700, PAST, ngram, words=2)
    rules.seqs[4] = [5] * 40
    rules.history(lambda a, t: rules.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or rules.keep[-1].ptr, 1003)
    x = some_logits(rng, 7, 700)
    got = check(pkg, L, x, rules)
    if ngram in (1, 2, 7, 40):
        assert np.isneginf(got[4, 5])


def test_no_rules_leave_all_as_it_is(pkg, L):
    rng = np.random.default_rng(9)
    x = some_logits(rng, 3, 999)
    x[0, 5], x[1, 6], x[2, 0] = np.nan, np.inf, 65504
    rules = Rules(pkg, rng, 3, 999, None, penalties=False)
    for kw in ({}, {"out_shift": 0}, {"out_shift": 1}):
        np.testing.assert_array_equal(run(pkg, L, x, rules, **kw).view(np.uint16), x.view(np.uint16))
    # a history without penalties changes nothing either
    rules = Rules(pkg, rng, 3, 999, [500, 0, 1], penalties=False)
    np.testing.assert_array_equal(run(pkg, L, x, rules)[~np.isnan(x)], x[~np.isnan(x)])


def test_nan_and_infinities(pkg, L):
    """A NaN stays one unless it is masked; infinities keep their sign; +inf and -inf make NaN, as anywhere."""
    V = 64
    x = np.zeros((2, V), np.float16)
    x[:, :6] = [np.nan, np.inf, -np.inf, np.nan, np.inf, -np.inf]
    rules = Rules(pkg, np.random.default_rng(1), 2, V, None, penalties=False)
    allowed = np.ones((1, V), bool)
    allowed[0, 3:6] = False
    dev = lambda a, t: rules.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or rules.keep[-1].ptr  # noqa: E731
    rules.seqs, rules.starts = [list(range(8)), list(range(8))], [0, 8]
    rules.history(dev, 8)
    rules.r.repetition, rules.r.presence = dev([1.5, 1.5], np.float32), dev([1, 1], np.float32)
    rules.r.mask, rules.r.n_masks, rules.r.mask_row = dev(mask_words(allowed), np.uint32), 1, dev([0, -1], np.int32)
    for out_shift in (None, 0):
        got = run(pkg, L, x, rules, out_shift=out_shift)
        assert np.isnan(got[0, 0]) and np.isposinf(got[0, 1]) and np.isneginf(got[0, 2:6]).all()
        assert np.isnan(got[1, [0, 3]]).all() and np.isposinf(got[1, [1, 4]]).all() and np.isneginf(got[1, [2, 5]]).all()
        assert got[0, 7] == -1 and got[1, 7] == 0 and (got[:, 8:] == 0).all()


def test_a_mask_of_nothing(pkg, L):
    rng = np.random.default_rng(4)
    x = some_logits(rng, 3, 5000)
    rules = Rules(pkg, rng, 3, 5000, [10, 20, 30], masks=1)   # mask 0 allows nothing
    rules.r.mask_row = None
    rules.masks = [np.zeros(5000, bool), None, None]          # rows past the masks have none
    for kw in ({}, {"out_shift": 0}):
        got = check(pkg, L, x, rules, **kw)
        assert np.isneginf(got[0]).all()


def test_books_out_of_range(pkg, L):
    """Lengths, starts, offsets and tokens that cannot be are cut to what can."""
    rng = np.random.default_rng(6)
    V, rows = 300, 4
    rules = Rules(pkg, rng, rows, V, [50] * rows, 2, 10)
    dev = lambda a, t: rules.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or rules.keep[-1].ptr  # noqa: E731
    rules.seqs[0][7], rules.seqs[0][8] = -5, 1 << 30
    rules.seqs[3] = []
    rules.starts = [-7, 1 << 30, 20, 3]
    rules.history(dev, 50)
    rules.h.len = dev([50, 1 << 20, 50, -4], np.int32)
    n = rules.r.n_bias
    flat = sum(rules.biases, [])
    rules.r.bias_start = dev([-9, 2, n + 100, 1, n], np.int32)
    rules.biases = [flat[:2], flat[2:], [], flat[1:]]
    x = some_logits(rng, rows, V)
    for kw in ({}, {"out_shift": 0}):
        check(pkg, L, x, rules, **kw)


@pytest.mark.parametrize("rows,past", [(256, 200), (5, 20000), (700, 30)])
def test_many(pkg, L, rows, past):
    rng = np.random.default_rng(rows)
    rules = Rules(pkg, rng, rows, 5000, [int(v) for v in rng.integers(0, past + 1, rows)], 2, 40, rows // 2, words=300)
    check(pkg, L, some_logits(rng, rows, 5000), rules, out_shift=0)
    check(pkg, L, some_logits(rng, rows, 5000), rules)


def test_counts_past_16_bits(pkg, L):
    rules = Rules(pkg, np.random.default_rng(2), 1, 50, [70000], words=1)
    rules.freq[0] = 0.01
    rules.r.frequency = (rules.keep.append(pkg.Dev.from_numpy(rules.freq)) or rules.keep[-1]).ptr
    rules.starts = [0]
    rules.history(lambda a, t: rules.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or rules.keep[-1].ptr, 70000)
    got = check(pkg, L, np.zeros((1, 50), np.float16), rules)
    assert got[0, 0] < -690


@pytest.mark.parametrize("V,biases", [(900, 513), (9000, 1500), (9000, 9000), (20, 3000)])
@pytest.mark.parametrize("rows", [3, 200])
def test_long_bias_lists(pkg, L, V, biases, rows):
    """Lists of more entries than a work-group has threads, of the whole vocabulary, of many entries for each token."""
    rng = np.random.default_rng([V, biases, rows])
    rules = Rules(pkg, rng, rows, V, [int(v) for v in rng.integers(0, 400, rows)], 2, biases if rows < 10 else biases // 5, rows // 2)
    check(pkg, L, some_logits(rng, rows, V), rules, out_shift=0)
    check(pkg, L, some_logits(rng, rows, V), rules)
    rules.r.mask = None
    rules.masks = [None] * rows
    check(pkg, L, some_logits(rng, rows, V), rules)


@pytest.mark.parametrize("rows", [2, 300])
def test_each_token_once(pkg, L, rows):
    """Bias lists without a token twice, some of its tokens in the history and some not, as programs make them."""
    rng = np.random.default_rng(rows)
    V = 20000
    rules = Rules(pkg, rng, rows, V, [150] * rows, 3, 0, 3, words=600)
    dev = lambda a, t: rules.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or rules.keep[-1].ptr  # noqa: E731
    rules.biases = [list(zip([int(t) for t in np.concatenate([rng.permutation(V)[:250], sorted(set(s))[::3]])], rng.standard_normal(400).astype(np.float32).tolist())) for s in rules.seqs]
    rules.biases = [list({t: v for t, v in b}.items()) for b in rules.biases]
    flat = sum(rules.biases, [])
    rules.r.n_bias, rules.r.bias_start = len(flat), dev(np.cumsum([0] + [len(b) for b in rules.biases]), np.int32)
    rules.r.bias_token, rules.r.bias_value = dev([t for t, _ in flat], np.int32), dev([v for _, v in flat], np.float32)
    check(pkg, L, some_logits(rng, rows, V), rules, out_shift=1)
    check(pkg, L, some_logits(rng, rows, V), rules)


def test_logits_past_4_gib(pkg, L):
    """Rows so far apart that the last begins past 2^32 bytes."""
    rng = np.random.default_rng(3)
    V, ld = 5000, 1 << 29
    for masks in (0, 2):
        rules = Rules(pkg, rng, 6, V, [30, 200, 0, 7, 90, 400], 2, 30, masks)
        x = some_logits(rng, 6, V)
        d = pkg.Dev((5 * ld + V) * 2)
        for r in range(6):
            assert L.gpt2_h2d(d.at(r * ld * 2), x[r].ctypes.data, V * 2) == 0
        L.gpt2_logits_adjust(d.ptr, d.ptr, ld, 6, V, C.byref(rules.r))
        L.gpt2_sync()
        pkg.check("gpt2_logits_adjust")
        got = np.empty((6, V), np.float16)
        for r in range(6):
            assert L.gpt2_d2h(got[r].ctypes.data, d.at(r * ld * 2), V * 2) == 0
        same(got, *rules.want(x))
        d.free()


# ----------------------------------------------------------------------------- histories
class Pair:
    """Histories on the host and on the device."""

    def __init__(self, pkg, L, n, room):
        self.pkg, self.L, self.n, self.room = pkg, L, n, room
        self.ref, self.dev = Histories(n, room), pkg.History(n, room)
        self.mem = np.full((n, room), -7, np.int32)   # what lies past the lengths
        assert L.gpt2_h2d(self.dev.h.tokens, self.mem.ctypes.data, self.mem.nbytes) == 0

    def step(self, parent, rows, ids, prompt=0, n_rows=None):
        d = [None if a is None else self.pkg.Dev.from_numpy(np.asarray(a, np.int32)) for a in (parent, rows, ids)]
        self.L.gpt2_history_step(C.byref(self.dev.h), *[v.ptr if v else None for v in d], len(ids) if ids is not None else 0, prompt)
        self.ref.step(parent, rows, [] if ids is None else ids, prompt)
        self.L.gpt2_sync()
        self.pkg.check("gpt2_history_step")

    def check(self):
        tokens, length, start = np.empty((self.n, self.room), np.int32), np.empty(self.n, np.int32), np.empty(self.n, np.int32)
        for a, p in ((tokens, self.dev.h.tokens), (length, self.dev.h.len), (start, self.dev.h.start)):
            assert self.L.gpt2_d2h(a.ctypes.data, p, a.nbytes) == 0
        assert length.tolist() == [len(s) for s in self.ref.seq] and start.tolist() == self.ref.start
        for s in range(self.n):   # tokens past a length stay as they were
            self.mem[s, :length[s]] = self.ref.seq[s]
        np.testing.assert_array_equal(tokens, self.mem)


@pytest.mark.parametrize("n,room", [(5, 300000), (300, 20000), (100, 50001), (1, 1), (1, 64), (8, 1024), (7, 333), (64, 100), (255, 70), (257, 129), (1000, 17), (1025, 80), (4096, 33)])
def test_history(pkg, L, n, room):
    rng = np.random.default_rng(n)
    p = Pair(pkg, L, n, room)
    p.check()
    for t in range(7):
        counts = rng.integers(0, max(2, min(room // 2, 1500)), n) * (rng.random(n) < 0.7) if t in (0, 3) else np.ones(n, int)
        rows = np.cumsum([0] + counts.tolist())
        ids = rng.integers(0, 50257, rows[-1])
        parent = None if t in (0, 4) else rng.integers(0, n, n)
        if t == 2:
            parent = (np.arange(n) + 1) % n      # all move
        if t == 5:
            parent[::3] = -1                     # some begin anew
            parent[1:2] = n
        p.step(parent, rows, ids, prompt=int(t in (0, 3)))
        p.check()
    p.step(np.zeros(n, int), None, None)
    p.check()
    p.step(None, None, None)
    p.check()
    L.gpt2_history_reset(C.byref(p.dev.h))
    p.ref = Histories(n, room)
    p.check()
    p.dev.free()


def test_history_past_4_gib(pkg, L):
    """Rows past 2^32 bytes, by blocks and by columns, from others so far."""
    rng = np.random.default_rng(12)
    n, room = 80, 1 << 24
    p = pkg.History(n, room)
    oracle = Histories(n, room)
    for t, parent in enumerate((None, np.arange(n) // 8 * 8, rng.permutation(n), None)):
        counts = rng.integers(0, 300, n)
        rows = np.cumsum([0] + counts.tolist())
        ids = rng.integers(0, 50257, rows[-1])
        d = [None if a is None else pkg.Dev.from_numpy(np.asarray(a, np.int32)) for a in (parent, rows, ids)]
        L.gpt2_history_step(C.byref(p.h), *[v.ptr if v else None for v in d], len(ids), 0)
        L.gpt2_sync()
        pkg.check("gpt2_history_step")
        oracle.step(parent, rows, ids, 0)
        for s in range(n):
            got = np.empty(len(oracle.seq[s]), np.int32)
            assert L.gpt2_d2h(got.ctypes.data, p.h.tokens + 4 * s * room, got.nbytes) == 0
            assert got.tolist() == oracle.seq[s]
    p.free()


def test_history_bad_offsets(pkg, L):
    """Offsets out of order, negative or past nRows append nothing to that sequence; the others go on."""
    p = Pair(pkg, L, 6, 40)
    p.step(None, [0, 5, 9, 9, 12, 20, 21], np.arange(21) + 100, prompt=1)
    p.check()
    p.step([1, 0, 3, 2, 4, 5], [0, 3, 2, -1, 4, 9, 6], np.arange(7))   # 3 tokens, order, negative, negative, past, order
    p.check()
    assert [len(s) for s in p.ref.seq] == [4 + 3, 5, 3, 0, 8, 1]


def test_history_same_stream_chain(pkg, L):
    """Steps follow one another without a wait between."""
    rng = np.random.default_rng(8)
    p = Pair(pkg, L, 32, 512)
    rows = pkg.Dev.from_numpy(np.arange(33, dtype=np.int32))
    parents, ids = rng.integers(0, 32, (200, 32)).astype(np.int32), rng.integers(0, 50257, (200, 32)).astype(np.int32)
    d_p, d_i = pkg.Dev.from_numpy(parents), pkg.Dev.from_numpy(ids)
    for t in range(200):
        L.gpt2_history_step(C.byref(p.dev.h), d_p.at(128 * t), rows.ptr, d_i.at(128 * t), 32, 0)
        p.ref.step(parents[t], np.arange(33), ids[t], 0)
    L.gpt2_sync()
    pkg.check("steps")
    p.check()
