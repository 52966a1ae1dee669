"""The paged INT8 K/V cache on the GPU: growing, appending, attention, reading back, forking and compacting against the
numpy cache of tests/pagedkv_ref.py, and a run of them together."""
import numpy as np
import pytest

from pagedkv_ref import D, P, Ref, Ws, ref

pytestmark = pytest.mark.gpu


def rows_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def qkv_of(rng, n, heads, wild=False):
    x = rng.standard_normal((n, 3 * heads * D)).astype(np.float32)
    x[:, ::D] *= 4
    x = x.astype(np.float16)
    if wild and n:
        kv = x[:, heads * D:]
        kv[rng.random(kv.shape) < 0.01] = 0
        kv[0, :5] = [np.nan, np.inf, -np.inf, 65504, 6e-8]
        kv[n // 2, D:2 * D] = 0
    return x


class Pair:
    """The library's cache and the numpy one, driven together."""

    def __init__(self, pkg, L, layers=2, heads=3, pages=40, seqs=5, max_len=320):
        self.pkg, self.L = pkg, L
        self.c = pkg.PagedKV(pages, seqs, max_len, layers, heads)
        self.r = Ref(layers, heads, pages, seqs, max_len)
        self.r.upload(pkg, self.c)   # buffers that nothing has written yet hold zeros in both

    def grow(self, counts):
        self.rows = rows_of(counts)
        self.d_rows = self.pkg.Dev.from_numpy(self.rows)
        self.n = int(self.rows[-1])
        self.L.gpt2_pkv_grow(ref(self.c), self.d_rows.ptr, self.n)
        return self.r.grow(self.rows)

    def append(self, layer, qkv):
        self.d_qkv = self.pkg.Dev.from_numpy(qkv)
        self.L.gpt2_pkv_append(ref(self.c), layer, self.d_qkv.ptr, self.d_rows.ptr, self.n)
        self.r.append(layer, qkv, self.rows)

    def attend(self, layer, qkv, group=1, extra=0):
        """Runs the attention; `extra` rows past the last sequence's are checked to stay."""
        n, E = self.n + extra, self.r.heads * D
        d_q = self.pkg.Dev.from_numpy(np.concatenate([qkv, np.full((extra, 3 * E), np.nan, np.float16)]))
        d_att = self.pkg.Dev.from_numpy(np.full((n, E), 7.0, np.float16))
        ws = Ws(self.pkg, self.L.gpt2_pkv_attn_ws(ref(self.c), n))
        self.L.gpt2_pkv_attn(d_att.ptr, d_q.ptr, ref(self.c), layer, self.d_rows.ptr, n, group, *ws.args)
        self.L.gpt2_sync()
        self.pkg.check("gpt2_pkv_attn")
        return d_att.numpy(np.float16, (n, E))

    def check_attention(self, layer, qkv, group=1, extra=0):
        got = self.attend(layer, qkv, group, extra).astype(np.float64)
        want, tol, on = self.r.attend(layer, qkv, self.rows)
        on = np.concatenate([on, np.zeros(extra, bool)])
        assert (got[~on] == 7).all(), "rows of no sequence were written"
        err = np.abs(got[on] - want[on[:self.n]])
        worst = (err / tol[on[:self.n]]).max(initial=0)
        assert worst <= 1, f"off by {worst:.2f} of the bound (largest error {err.max():.3e})"

    def fork(self, parent):
        parent = np.asarray(parent, np.int32)
        self.L.gpt2_pkv_fork(ref(self.c), self.pkg.Dev.from_numpy(parent).ptr)
        self.L.gpt2_sync()
        self.r.fork(parent)

    def same(self):
        self.L.gpt2_sync()
        self.pkg.check("same")
        self.r.same_books(self.pkg, self.c)
        self.r.same_data(self.pkg, self.c)

    def step(self, rng, counts, wild=False):
        assert self.grow(counts)
        x = [qkv_of(rng, self.n, self.r.heads, wild) for _ in range(self.r.layers)]
        for layer in range(self.r.layers):
            self.append(layer, x[layer])
        return x


@pytest.mark.parametrize("counts", [
    [[1, 1, 1, 1, 1]] * 3,
    [[5, 0, 31, 32, 33], [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [27, 64, 1, 0, 100]],
    [[100, 0, 0, 3, 65], [0, 0, 200, 0, 0]],
    [[31, 31, 31, 31, 31], [1, 2, 33, 34, 65]],
])
def test_append_bit_exact(pkg, L, counts):
    p, rng = Pair(pkg, L), np.random.default_rng(7)
    for c in counts:
        p.step(rng, c, wild=True)
        p.same()
    assert L.gpt2_pkv_status(ref(p.c)) == 0


def test_append_reads_only_its_rows(pkg, L):
    """Offsets need not start at 0, and rows that belong to no sequence are not looked at."""
    p, rng = Pair(pkg, L), np.random.default_rng(8)
    x = qkv_of(rng, 60, 3)
    p.rows = np.array([4, 10, 10, 50, 51, 55], np.int32)
    p.d_rows, p.n = pkg.Dev.from_numpy(p.rows), 60
    L.gpt2_pkv_grow(ref(p.c), p.d_rows.ptr, 60)
    assert p.r.grow(p.rows)
    x[:4] = x[55:] = np.nan
    p.append(0, x)
    p.append(1, x)
    p.same()
    p.check_attention(0, x)


def test_read(pkg, L):
    p, rng = Pair(pkg, L), np.random.default_rng(9)
    p.step(rng, [70, 0, 32, 31, 150])
    first, count = np.array([3, 0, 30, 0, 149], np.int32), [80, 2, 2, 31, 4]
    rows = rows_of(count)
    n = int(rows[-1]) + 3   # three rows of no sequence
    E2 = 2 * p.r.heads * D
    out = pkg.Dev.from_numpy(np.full((n, E2), 7.0, np.float16))
    d_rows, d_pos = pkg.Dev.from_numpy(rows), pkg.Dev.from_numpy(first)
    for layer in range(2):
        L.gpt2_pkv_read(out.ptr, ref(p.c), layer, d_rows.ptr, d_pos.ptr, n)
        L.gpt2_sync()
        pkg.check("read")
        got = out.numpy(np.float16, (n, E2))
        want = np.concatenate([p.r.read(layer, s, first[s], count[s]) for s in range(5)] + [np.full((3, E2), 7.0, np.float16)])
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("heads,counts", [
    (1, [[1]]),
    (3, [[1, 1, 1, 1, 1]]),
    (12, [[33, 1, 64, 17, 0], [1, 1, 1, 1, 1]]),
    (3, [[16, 17, 15, 1, 48], [1, 0, 2, 31, 33], [0, 1, 0, 1, 0]]),
    (5, [[200, 0, 0, 0, 1], [1, 0, 0, 0, 100]]),
])
def test_attention(pkg, L, heads, counts):
    p, rng = Pair(pkg, L, heads=heads, seqs=len(counts[0])), np.random.default_rng(10)
    for c in counts:
        x = p.step(rng, c)
        for layer in range(2):
            p.check_attention(layer, x[layer], extra=2)


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1024, 2047, 5000])
@pytest.mark.parametrize("new", [1, 3])
def test_attention_lengths(pkg, L, length, new):
    """One long sequence, its last rows: every number of pages and splits, pages scattered over the pool."""
    rng = np.random.default_rng(length)
    p = Pair(pkg, L, layers=1, heads=2, pages=170, seqs=2, max_len=5120)
    r = p.r
    place = rng.permutation(r.pages)
    r.table[0, :160] = place[:160]
    r.codes[:] = rng.integers(-127, 128, r.codes.shape)
    r.scales[:] = rng.uniform(0.005, 0.04, r.scales.shape)
    r.open[:] = rng.standard_normal(r.open.shape)
    new = min(new, length)
    r.len[:], r.start[:], r.slot[:] = [length, 0], [length - new, 0], [1, 0]
    r.upload(pkg, p.c)
    p.rows, p.n = rows_of([new, 0]), new
    p.d_rows = pkg.Dev.from_numpy(p.rows)
    p.check_attention(0, qkv_of(rng, new, 2))


def test_attention_many_sequences(pkg, L):
    """More sequences than a wave looks over at once, most of them with no row, some with many."""
    rng = np.random.default_rng(11)
    p = Pair(pkg, L, layers=1, heads=2, pages=260, seqs=150, max_len=128)
    p.step(rng, rng.integers(0, 60, 150))
    counts = np.where(rng.random(150) < 0.3, rng.integers(0, 40, 150), 0)
    counts[[63, 64, 65, 149]] = [17, 1, 33, 20]
    x = p.step(rng, counts)
    p.same()
    p.check_attention(0, x[0])


@pytest.mark.parametrize("heads,before,counts", [
    (12, [40, 500, 7], [300, 401, 64]),
    (12, [0, 0, 0], [704, 0, 33]),
    (16, [31, 32], [1, 640]),
    (12, [2100], [770]),
    (1024, [40, 0], [100, 33]),
    (700, [33], [200]),
    (1, [33, 1], [400, 100]),
    (2, [2100, 5], [300, 40]),
])
def test_attention_many_rows(pkg, L, heads, before, counts):
    """Batches of many rows a sequence, which take work-groups of 32 and of 64 rows, with splits and without: prompts from
    nothing, prompts on top of cached ones, ragged."""
    pages = sum(-(-(b + n) // P) for b, n in zip(before, counts))
    p, rng = Pair(pkg, L, layers=1, heads=heads, pages=pages, seqs=len(counts), max_len=3000), np.random.default_rng(20)
    p.step(rng, before)
    x = p.step(rng, counts)
    p.same()
    p.check_attention(0, x[0], extra=3)
    r = p.r   # a page that is none
    r.table[0, 0] = r.pages
    r.upload(pkg, p.c)
    p.check_attention(0, x[0])


@pytest.mark.parametrize("max_len", [320, 4000])
@pytest.mark.parametrize("group", [2, 3, 8, 16])
def test_attention_beams(pkg, L, group, max_len):
    """Beams that share a prompt's pages: the same as without the hint, to the order of sums; with beams that have no row, that
    share nothing, that have several rows."""
    seqs = 2 * group
    p, rng = Pair(pkg, L, layers=1, heads=2, pages=40 * group, seqs=seqs, max_len=max_len), np.random.default_rng(group)
    r = p.r
    p.step(rng, [200 if s == 0 else 65 if s == group else 0 for s in range(seqs)])
    p.fork([s // group * group for s in range(seqs)])
    some = np.ones(seqs, int)
    for counts in (some, some * 30, some, np.arange(seqs) % 2, np.where(np.arange(seqs) == 1, 1, 0), some):
        x = p.step(rng, counts)
        p.check_attention(0, x[0], group=group)
        plain, hinted = p.attend(0, x[0]), p.attend(0, x[0], group=group)
        assert np.abs(plain.astype(np.float32) - hinted).max(initial=0) <= 2 * p.r.attend(0, x[0], p.rows)[1].max(initial=0)
    p.fork(np.concatenate([rng.integers(0, group, group), group + rng.integers(0, group, group)]))
    r.table[0, 1] = -1   # differs from the others' from its second page on, and is none
    r.upload(pkg, p.c)
    x = p.step(rng, some)
    p.check_attention(0, x[0], group=group)


def test_stale_and_foreign_values_do_not_reach_a_row(pkg, L):
    """NaN in unused tokens of the open pages, in free pages' scales, and in other sequences' query rows."""
    rng = np.random.default_rng(12)
    p = Pair(pkg, L, layers=1, heads=2)
    p.step(rng, [40, 3, 64, 0, 17])
    r = p.r
    for s in range(r.seqs):
        buf = r.open[0, r.slot[s]].reshape(2, 2, -1).copy()
        k, v = buf[0].reshape(2, P, D), buf[1].reshape(2, P // 8, D, 8)
        k[:, r.len[s] % P:] = np.nan
        for t in range(r.len[s] % P, P):
            v[:, t // 8, :, t % 8] = np.nan
        r.open[0, r.slot[s]] = np.stack([k.reshape(2, -1), v.reshape(2, -1)])
    r.scales[0, r.refs == 0] = np.nan
    r.upload(pkg, p.c)
    x = p.step(rng, [1, 1, 1, 1, 1])[0]
    p.check_attention(0, x)
    y = x.copy()
    y[2, :] = np.nan
    got, clean = p.attend(0, y), p.attend(0, x)
    keep = [0, 1, 3, 4]
    np.testing.assert_array_equal(got[keep], clean[keep])


def test_pages_that_are_none(pkg, L):
    """A page number outside the pool stands for a page that is not there; with no page at all the row is 0."""
    rng = np.random.default_rng(13)
    p = Pair(pkg, L, layers=1, heads=2)
    p.step(rng, [70, 96, 33, 5, 64])
    r = p.r
    r.table[0, 1], r.table[1, :3], r.table[2, 0] = r.pages, [-1, 1 << 30, -2147483648], -1
    r.start[:] = np.maximum(r.len - 1, 0)
    r.upload(pkg, p.c)
    p.rows, p.n = rows_of([1] * 5), 5
    p.d_rows = pkg.Dev.from_numpy(p.rows)
    x = qkv_of(rng, 5, 2)
    p.check_attention(0, x)
    assert (p.attend(0, x)[1] == 0).all()
    out = pkg.Dev(96 * 4 * D * 2)
    d_rows, d_pos = pkg.Dev.from_numpy(np.array([0, 0, 96, 96, 96, 96], np.int32)), pkg.Dev.from_numpy(np.zeros(5, np.int32))
    L.gpt2_pkv_read(out.ptr, ref(p.c), 0, d_rows.ptr, d_pos.ptr, 96)
    L.gpt2_sync()
    assert (out.numpy(np.float16, (96, 4 * D)) == 0).all()


@pytest.mark.parametrize("parent", [
    [0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [0, 0, 0, 0, 0], [4, 4, 0, 0, 1], [-1, 2, -1, 2, 2], [-1, -1, -1, -1, -1], [1, 2, 0, -1, 3],
])
def test_fork(pkg, L, parent):
    p, rng = Pair(pkg, L, pages=60), np.random.default_rng(14)
    p.step(rng, [70, 0, 32, 31, 150])
    p.fork(parent)
    p.same()
    x = p.step(rng, [1, 1, 40, 0, 3])   # goes on after it; freed pages are taken again
    p.same()
    p.check_attention(1, x[1])
    p.fork(parent)
    p.same()


def test_fork_many(pkg, L):
    rng = np.random.default_rng(15)
    p = Pair(pkg, L, layers=1, heads=1, pages=900, seqs=300, max_len=96)
    p.step(rng, rng.integers(0, 90, 300))
    for _ in range(3):
        p.fork(rng.integers(-1, 300, 300))
        p.same()


def test_compact(pkg, L):
    p, rng = Pair(pkg, L, pages=50), np.random.default_rng(16)
    for _ in range(3):
        p.step(rng, [70, 33, 32, 31, 90])
        p.fork([0, -1, 2, 0, 3])
        L.gpt2_pkv_compact(ref(p.c))
        n = p.r.compact()
        p.same()
        status = np.empty(4, np.int32)
        L.gpt2_d2h(status.ctypes.data, p.c.c.status, 16)
        assert status[1] == n and (p.r.refs[:n] > 0).all() and (p.r.refs[n:] == 0).all()
        x = p.step(rng, [1, 1, 1, 1, 1])
        p.check_attention(0, x[0])
        p.fork([0, -1, 2, -1, -1])


def test_compact_large_and_empty(pkg, L):
    rng = np.random.default_rng(17)
    p = Pair(pkg, L, layers=1, heads=1, pages=9000, seqs=3, max_len=32 * 5000)
    L.gpt2_pkv_compact(ref(p.c))
    p.same()
    r = p.r
    where = rng.permutation(9000)[:8000]
    r.table[0, :4000], r.table[1, :4000], r.table[2, :100] = where[:4000], where[4000:], where[:100]
    r.len[:] = [32 * 4000, 32 * 4000 + 5, 3200]
    np.add.at(r.refs, where, 1)
    r.refs[where[:100]] += 1
    r.codes[:] = rng.integers(-127, 128, r.codes.shape)
    r.scales[:] = rng.uniform(0.005, 0.04, r.scales.shape)
    r.upload(pkg, p.c)
    L.gpt2_pkv_compact(ref(p.c))
    assert r.compact() == 8000
    p.same()


def test_device_side_refusals(pkg, L):
    """What only the device can see leaves the cache as it was, with no new rows, and is told once."""
    p, rng = Pair(pkg, L, pages=6, max_len=128), np.random.default_rng(18)
    p.step(rng, [40, 33, 20, 0, 0])
    p.same()

    def refused(code, what):
        p.r.start[:] = p.r.len
        p.same()
        x = qkv_of(rng, 8, 3)
        p.d_qkv = pkg.Dev.from_numpy(x)
        L.gpt2_pkv_append(ref(p.c), 0, p.d_qkv.ptr, p.d_rows.ptr, p.n)
        p.same()
        assert (p.attend(0, np.resize(x, (p.n, x.shape[1]))) == 7).all()
        assert L.gpt2_pkv_status(ref(p.c)) == code, what
        assert L.gpt2_last_error() == code
        assert L.gpt2_pkv_status(ref(p.c)) == 0

    assert not p.grow([90, 0, 80, 0, 0])
    refused(1003, "past maxPages")
    assert not p.grow([56, 63, 44, 0, 0])
    refused(1003, "no free page: 6 are needed, 4 are free")
    assert not p.grow([89, 0, 0, 0, 0])
    refused(1003, "past maxPages")
    for bad in ([0, 3, 2, 4, 5, 6], [-1, 0, 1, 2, 3, 4], [0, 1, 2, 3, 4, 9]):
        p.rows, p.n = np.array(bad, np.int32), 8
        p.d_rows = pkg.Dev.from_numpy(p.rows)
        L.gpt2_pkv_grow(ref(p.c), p.d_rows.ptr, 8)
        refused(1000, str(bad))
    p.grow([0, 0, 0, 0, 0])
    p.n = 8
    for bad in ([0, 1, 2, 3, 5], [0, 1, -2, 3, 4]):
        L.gpt2_pkv_fork(ref(p.c), pkg.Dev.from_numpy(np.array(bad, np.int32)).ptr)
        refused(1000, str(bad))
    x = p.step(rng, [24, 31, 11, 1, 1])
    p.same()
    p.check_attention(1, x[1])
    assert p.r.refs.sum() == 4   # 64 / 32 + 64 / 32 + 31 / 32


def test_embed_positions(pkg, L):
    rng = np.random.default_rng(19)
    E, V, N = pkg.N_EMBD, pkg.VOCAB, 1024
    wte, wpe = rng.standard_normal((300, E)).astype(np.float16), rng.standard_normal((N, E)).astype(np.float16)
    d_wte = pkg.Dev(V * E * 2)
    L.gpt2_h2d(d_wte.ptr, wte.ctypes.data, wte.nbytes)
    d_wpe = pkg.Dev.from_numpy(wpe)
    p = Pair(pkg, L, layers=1, heads=1, pages=60, seqs=3, max_len=1056)
    p.step(rng, [5, 0, 1022])
    p.grow([3, 1, 4])   # the last sequence's rows 2 and 3 lie past the positions
    ids = np.array([1, 299, V, 0, 7, 8, 9, -1], np.int32)
    d_x = pkg.Dev.from_numpy(np.full((10, E), 7.0, np.float16))
    d_ids = pkg.Dev.from_numpy(np.concatenate([ids, [0, 0]]).astype(np.int32))
    L.gpt2_pkv_embed(d_x.ptr, d_wte.ptr, d_wpe.ptr, d_ids.ptr, ref(p.c), p.d_rows.ptr, 10)
    L.gpt2_sync()
    pkg.check("embed")
    got = d_x.numpy(np.float16, (10, E))
    pos = [5, 6, 7, 0, 1022, 1023, 1024, 1025]
    want = [((wte[i].astype(np.float32) if 0 <= i < 300 else 0) + (wpe[q].astype(np.float32) if q < N else np.zeros(E, np.float32))).astype(np.float16)
            for i, q in zip(ids, pos)]
    np.testing.assert_array_equal(got[:8], np.stack(want))
    assert (got[8:] == 7).all()


@pytest.mark.parametrize("heads,before,counts,group", [
    (3, [96, 70, 130, 0], [1, 1, 1, 1], 1), (3, [96, 70, 130, 0], [1, 1, 1, 1], 4), (3, [96, 40], [20, 30], 1), (3, [96], [90], 1),
    (1030, [64], [130], 1),
])
def test_attention_pages_of_zeros(pkg, L, heads, before, counts, group):
    """Pages whose keys or values are all zero, whose scale says nothing of their size: keys that weigh the same exactly, values that
    add nothing to others a thousand times smaller than the queries; one head's values are all zero, and so is what it gives."""
    p, rng = Pair(pkg, L, layers=1, heads=heads, pages=30, seqs=len(counts), max_len=256), np.random.default_rng(36)
    E = heads * D
    for step in (before, counts):
        assert p.grow(step)
        x = qkv_of(rng, p.n, heads)
        x[:, :E] *= np.float16(6)
        kv = x[:, E:].reshape(-1, 2, heads, D)
        kv[:, 1] *= np.float16(2 ** -10)
        kv[:, 1, 1 % heads] = 0
        for s in range(len(counts)):   # the first 40 tokens
            rows = kv[p.rows[s]:p.rows[s + 1]]
            rows[:max(0, 40 - int(p.r.start[s])), 0, 0] = 0
            rows[:max(0, 40 - int(p.r.start[s])), 1, heads - 1] = 0
        p.append(0, x)
    p.same()
    p.check_attention(0, x, group=group)
    got = p.attend(0, x, group=group).reshape(-1, heads, D)
    assert (got[:, 1 % heads] == 0).all()


@pytest.mark.parametrize("max_len,group", [(320, 1), (4000, 1), (320, 4)])
def test_prompts_in_a_cache_of_many_sequences(pkg, L, max_len, group):
    """No more rows than sequences, but nearly all of them one sequence's: its rows and pages are shared out."""
    p, rng = Pair(pkg, L, layers=1, heads=3, pages=60, seqs=140, max_len=max_len), np.random.default_rng(37)
    counts = np.zeros(140, int)
    for before, new in ((40, 100), (3, 130)):
        counts[[3, 50, 99]] = [before, 33, 5]
        p.step(rng, counts)
        counts[[3, 50, 99]] = [new, 5, 2]
        x = p.step(rng, counts)
        p.same()
        p.check_attention(0, x[0], group=group, extra=2)


@pytest.mark.parametrize("rows,group", [(1, 1), (1, 2), (30, 1), (100, 1)])
def test_attention_many_small_weights(pkg, L, rows, group):
    """One key far ahead of thousands whose weights add up all the same: 2^-19 to 2^-23 of the largest each."""
    heads, cached = 2, 5000
    p, rng = Pair(pkg, L, layers=1, heads=heads, pages=420, seqs=2, max_len=6000), np.random.default_rng(40)
    E = heads * D
    for counts in ([cached, 70], [rows, 1]):
        assert p.grow(counts)
        x = np.zeros((p.n, 3, heads, D), np.float16)
        x[:, 0, :, 0] = 8          # q . k / 8 is the key's first dim
        x[:, 1, :, 0] = -np.log(2) * (19 + 4 * rng.random((p.n, heads)))
        x[:, 2] = 1 + rng.random((p.n, heads, D))
        if counts[0] == cached:    # the one key, with a value of its own
            x[17, 1, :, 0], x[17, 2] = 0, -1
            x[cached, 1, :, 0] = 0
        x = x.reshape(p.n, 3 * E)
        p.append(0, x)
    p.check_attention(0, x, group=group)


@pytest.mark.parametrize("size", [30, 1000, 4000])
@pytest.mark.parametrize("rows,group", [(1, 1), (1, 2), (30, 1), (100, 1)])
def test_attention_large_scores(pkg, L, rows, group, size):
    """Scores up to size^2 64 / 8, equal or a size^2 / 8 apart and more: the weight is all the largest ones'."""
    heads = 2
    p, rng = Pair(pkg, L, layers=1, heads=heads, pages=40, seqs=2, max_len=600), np.random.default_rng(41)
    for counts in ([200, 70], [rows, 1]):
        assert p.grow(counts)
        x = np.zeros((p.n, 3, heads, D), np.float16)
        x[:, 0] = size
        ones = rng.integers(1, D + 1, p.n)
        x[:, 1] = np.where(np.arange(D) < ones[:, None], size, 0)[:, None]
        x[:, 1, 1] *= -1
        x[:, 2] = rng.standard_normal((p.n, heads, D))
        x = x.reshape(p.n, 3 * heads * D)
        p.append(0, x)
    # A score is a sum of 64 products in fp32, off by up to 64 2^-24 of the sum of their sizes, S = size^2 64 / 8, however near another is:
    # 0.03 at 30, 30 at 1000, 500 at 4000.  check_attention's bound counts that (and says nothing from 1000 on).  At any size the row
    # is an average of the values: weights that are rounded alike above and below, sums of 300 fp32 terms, the output's rounding.
    p.check_attention(0, x, group=group)
    got = p.attend(0, x, group=group).astype(np.float64).reshape(-1, heads, D)
    for i in range(p.n):
        s = 0 if i < rows else 1
        v = p.r.held(0, s)[1][:, :int(p.r.start[s]) + (i - int(p.rows[s])) + 1]
        off = np.abs(v).max() * (2.0 ** -11 + 300 * 2.0 ** -24)
        assert (got[i] <= v.max(axis=1) + off).all() and (got[i] >= v.min(axis=1) - off).all()
        assert (got[i] != 0).any(axis=1).all()
