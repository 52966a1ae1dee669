"""The paged cache and the beam selection as they are used: a beam search of a two-layer model over the library's own
operators, every step checked against plain numpy on what the step itself was given; the same captured into a graph and
replayed; caches on two streams; pages past 4 GiB."""
import ctypes as C

import numpy as np
import pytest

from pagedkv_ref import D, P, Ref, Ws, beam, ref
from test_gpu_lnfold import hip_runtime
from test_gpu_pagedkv import Pair, qkv_of, rows_of

pytestmark = pytest.mark.gpu
LAYERS, GROUPS, BEAMS = 2, 2, 4
SEQS = GROUPS * BEAMS


class Search:
    """Beam search of GROUPS prompts, all state on the device: tokens, parents and scores are written where the next step
    reads them, so a step is the same calls every time."""

    def __init__(self, pkg, L, eos):
        self.pkg, self.L, self.eos = pkg, L, eos
        E, F, V = pkg.N_EMBD, 4 * pkg.N_EMBD, pkg.VOCAB
        rng = np.random.default_rng(31)

        def w(*shape, scale=0.03):
            return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(np.float16)
        self.wte, self.wpe = w(V, E, scale=0.08), w(pkg.N_CTX, E, scale=0.05)
        host = {"wte": self.wte, "wpe": self.wpe, "g": np.ones(E, np.float16), "b": np.zeros(E, np.float16)}
        for n in range(LAYERS):
            host |= {f"qkv{n}": w(3 * E, E, scale=0.06), f"ao{n}": w(E, E), f"fc{n}": w(F, E), f"pr{n}": w(E, F)}
        self.w = {k: pkg.Dev.from_numpy(v) for k, v in host.items()}
        # `extra` rows of every buffer belong to no sequence
        self.N = 80
        self.x, self.ln, self.att, self.ao = (pkg.Dev(self.N * E * 2) for _ in range(4))
        self.qkv, self.fc = [pkg.Dev(self.N * 3 * E * 2) for _ in range(LAYERS)], pkg.Dev(self.N * F * 2)
        self.atts = [pkg.Dev(self.N * E * 2) for _ in range(LAYERS)]
        self.logits = pkg.Dev(SEQS * V * 2)
        self.ids, self.parent = pkg.Dev(self.N * 4), pkg.Dev(SEQS * 4)
        self.score, self.done = pkg.Dev(SEQS * 4), pkg.Dev(SEQS * 4)
        self.c = pkg.PagedKV(40, SEQS, 256, LAYERS, pkg.N_HEAD)
        self.d_rows = pkg.Dev.from_numpy(np.arange(SEQS + 1, dtype=np.int32))
        self.ws = Ws(pkg, max(L.gpt2_pkv_attn_ws(ref(self.c), self.N), L.gpt2_pkv_attn_ws(ref(self.c), SEQS)))
        self.bws = Ws(pkg, L.gpt2_beam_select_ws(GROUPS, BEAMS, V))

    def blocks(self, rows, n, group):
        """x after the blocks; qkv and att of each layer stay for the checks."""
        L, w, E, F = self.L, self.w, self.pkg.N_EMBD, 4 * self.pkg.N_EMBD
        L.gpt2_pkv_grow(ref(self.c), rows, n)
        L.gpt2_pkv_embed(self.x.ptr, w["wte"].ptr, w["wpe"].ptr, self.ids.ptr, ref(self.c), rows, n)
        for i in range(LAYERS):
            L.gpt2_layernorm(self.ln.ptr, self.x.ptr, w["g"].ptr, w["b"].ptr, n, E)
            L.gpt2_matmul_tiled(self.qkv[i].ptr, self.ln.ptr, w[f"qkv{i}"].ptr, None, n, 3 * E, E)
            L.gpt2_pkv_append(ref(self.c), i, self.qkv[i].ptr, rows, n)
            L.gpt2_pkv_attn(self.atts[i].ptr, self.qkv[i].ptr, ref(self.c), i, rows, n, group, *self.ws.args)
            L.gpt2_matmul_tiled(self.ao.ptr, self.atts[i].ptr, w[f"ao{i}"].ptr, None, n, E, E)
            L.gpt2_add(self.x.ptr, self.ao.ptr, n * E)
            L.gpt2_layernorm(self.ln.ptr, self.x.ptr, w["g"].ptr, w["b"].ptr, n, E)
            L.gpt2_matmul_tiled(self.fc.ptr, self.ln.ptr, w[f"fc{i}"].ptr, None, n, F, E)
            L.gpt2_gelu(self.fc.ptr, n * F)
            L.gpt2_matmul_tiled(self.ao.ptr, self.fc.ptr, w[f"pr{i}"].ptr, None, n, E, F)
            L.gpt2_add(self.x.ptr, self.ao.ptr, n * E)

    def select(self):
        L, w, E, V = self.L, self.w, self.pkg.N_EMBD, self.pkg.VOCAB
        L.gpt2_layernorm(self.ln.ptr, self.x.ptr, w["g"].ptr, w["b"].ptr, SEQS, E)
        L.gpt2_matmul_tiled(self.logits.ptr, self.ln.ptr, w["wte"].ptr, None, SEQS, V, E)
        L.gpt2_beam_select(self.ids.ptr, self.parent.ptr, self.score.ptr, self.done.ptr, self.logits.ptr, V, self.score.ptr, self.done.ptr,
                           GROUPS, BEAMS, V, self.eos, *self.bws.args)

    def step(self):
        self.blocks(self.d_rows.ptr, SEQS, BEAMS)
        self.select()
        self.L.gpt2_pkv_fork(ref(self.c), self.parent.ptr)

    def prompts(self):
        """Two prompts into the first sequence of their groups, then every beam of a group from that one."""
        rng = np.random.default_rng(32)
        E, n = self.pkg.N_EMBD, [61 if s == 0 else 13 if s == BEAMS else 0 for s in range(SEQS)]
        self.rows = rows_of(n)
        self.tokens = rng.integers(0, self.pkg.VOCAB, self.rows[-1]).astype(np.int32)
        self.ids.upload(self.tokens)
        self.L.gpt2_pkv_reset(ref(self.c))
        self.d_prompt = self.pkg.Dev.from_numpy(self.rows)
        self.blocks(self.d_prompt.ptr, int(self.rows[-1]), 1)
        self.parent.upload(np.repeat(np.arange(GROUPS) * BEAMS, BEAMS).astype(np.int32))
        self.score.upload(np.where(np.arange(SEQS) % BEAMS, -np.inf, 0).astype(np.float32))
        self.done.upload(np.zeros(SEQS, np.int32))

    def first(self):
        """The prompts' last rows, one for each beam; then the first selection and the fork that it asks for."""
        E = self.pkg.N_EMBD
        for s in reversed(range(SEQS)):
            last = self.rows[s // BEAMS * BEAMS + 1] - 1
            self.L.gpt2_d2d(self.ln.at(s * E * 2), self.x.at(int(last) * E * 2), E * 2)
        self.L.gpt2_d2d(self.x.ptr, self.ln.ptr, SEQS * E * 2)
        self.L.gpt2_pkv_fork(ref(self.c), self.parent.ptr)
        self.select()

    def state(self):
        self.L.gpt2_sync()
        self.pkg.check("state")
        return [self.ids.numpy(np.int32, SEQS), self.parent.numpy(np.int32, SEQS), self.score.numpy(np.uint32, SEQS), self.done.numpy(np.int32, SEQS)]


@pytest.fixture(scope="module")
def search(pkg, L):
    return Search(pkg, L, eos=-1)


def check_selection(s, score, done, after):
    """The scores that were given out are the best ones, and those of the continuations named."""
    x = s.logits.numpy(np.float16, (SEQS, s.pkg.VOCAB))
    token, parent, got, mark = after[0], after[1], after[2].view(np.float32).astype(np.float64), after[3]
    want = beam(x, score, done, GROUPS, BEAMS, s.eos)[2]
    # as for the selection alone: the log of the sum 2^-24 * 95, the score's rounding
    tol = 2.0 ** -24 * 95 + 2.0 ** -24 * np.abs(want)
    assert (np.abs(got - want) <= tol).all()
    x = x.astype(np.float64)
    for i in range(SEQS):
        r = parent[i]
        assert r // BEAMS == i // BEAMS and mark[i] == (s.eos >= 0 and token[i] == s.eos)
        if s.eos >= 0 and done[r]:
            own = float(score[r])
            assert token[i] == s.eos
        else:
            own = float(score[r]) + x[r, token[i]] - x[r].max() - np.log(np.exp(x[r] - x[r].max()).sum())
        assert abs(got[i] - own) <= tol[i]
    assert len({(parent[i], token[i]) for i in range(SEQS)}) == SEQS


def test_beam_search_step_by_step(pkg, L, search):
    s, E = search, pkg.N_EMBD
    r = Ref(LAYERS, pkg.N_HEAD, 40, SEQS, 256)
    s.eos = -1

    def rows_seen(rows, group):
        """What the step's calls did with the rows that it had."""
        n = int(rows[-1])
        for i in range(LAYERS):
            qkv = s.qkv[i].numpy(np.float16, (n, 3 * E))
            r.append(i, qkv, rows)
            want, tol, on = r.attend(i, qkv, rows)
            err = np.abs(s.atts[i].numpy(np.float16, (n, E)).astype(np.float64) - want)
            assert on.all() and (err <= tol).all(), f"layer {i}: {(err / tol).max():.2f} of the bound"

    s.prompts()
    L.gpt2_sync()
    assert r.grow(s.rows)
    rows_seen(s.rows, 1)
    r.same_books(pkg, s.c)
    before = s.state()
    s.first()
    after = s.state()
    r.fork(before[1])
    check_selection(s, before[2].view(np.float32), before[3], after)
    L.gpt2_pkv_fork(ref(s.c), s.parent.ptr)
    r.fork(after[1])
    rows = np.arange(SEQS + 1, dtype=np.int32)
    for t in range(24):
        if t == 12:   # from here on the last beam's token ends a continuation, that beam's first
            s.eos = int(after[0][-1])
            s.done.upload((np.arange(SEQS) == SEQS - 1).astype(np.int32))
            after = s.state()
        print(f"step {t}", flush=True)
        before = after
        s.blocks(s.d_rows.ptr, SEQS, BEAMS)
        L.gpt2_sync()
        assert r.grow(rows)
        rows_seen(rows, BEAMS)
        s.select()
        after = s.state()
        check_selection(s, before[2].view(np.float32), before[3], after)
        L.gpt2_pkv_fork(ref(s.c), s.parent.ptr)
        r.fork(after[1])
        if t % 8 == 5:
            L.gpt2_pkv_compact(ref(s.c))
            r.compact()
        L.gpt2_sync()
        r.same_books(pkg, s.c)
        r.same_data(pkg, s.c)
    assert L.gpt2_pkv_status(ref(s.c)) == 0
    # the first pages are still shared: one of the longer prompt for its four beams
    assert r.refs.max() == BEAMS


def test_beam_search_captured(pkg, L, search):
    """A step captured on a stream of its own and replayed, other work between the replays: the same bits as the eager steps."""
    s, T = search, 12
    hip = hip_runtime()
    s.eos = 17

    def start():
        s.prompts()
        s.first()
        L.gpt2_pkv_fork(ref(s.c), s.parent.ptr)

    start()
    want = []
    for _ in range(T):
        s.step()
        want.append(s.state())
    other = Pair(pkg, L, layers=1, heads=2)
    rng = np.random.default_rng(33)
    start()
    L.gpt2_sync()
    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    try:
        assert hip.hipStreamCreate(C.byref(stream)) == 0
        L.gpt2_set_stream(stream)
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        s.step()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        pkg.check("capture")
        assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        for t in range(T):
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            for a, b in zip(s.state(), want[t]):
                np.testing.assert_array_equal(a, b, err_msg=f"replay {t}")
            x = other.step(rng, [1, 9, 0, 2, 17])
            other.check_attention(0, x[0])
    finally:
        L.gpt2_set_stream(None)
        if exe:
            hip.hipGraphExecDestroy(exe)
        if graph:
            hip.hipGraphDestroy(graph)
        if stream:
            hip.hipStreamDestroy(stream)
    assert L.gpt2_pkv_status(ref(s.c)) == 0


def test_two_streams(pkg, L):
    """Two caches driven in turn on a stream each, nothing waited for in between, each with its own workspace."""
    hip = hip_runtime()
    streams = [C.c_void_p(), C.c_void_p()]
    rng = np.random.default_rng(34)
    heads, seqs = 4, 6
    rows = [rows_of([33, 1, 0, 100, 64, 7]), rows_of([5, 90, 31, 32, 1, 0])]
    x = [qkv_of(rng, int(r[-1]), heads) for r in rows]
    r = [Ref(1, heads, 100, seqs, 5000) for _ in rows]
    c = [pkg.PagedKV(100, seqs, 5000, 1, heads) for _ in rows]
    for a, b in zip(r, c):
        a.upload(pkg, b)
    d_rows, d_x = [pkg.Dev.from_numpy(v) for v in rows], [pkg.Dev.from_numpy(v) for v in x]
    att = [pkg.Dev(v.shape[0] * heads * D * 2) for v in x]
    ws = [Ws(pkg, L.gpt2_pkv_attn_ws(ref(c[i]), len(x[i]))) for i in range(2)]
    parent = pkg.Dev.from_numpy(np.array([1, 1, 3, 0, 3, -1], np.int32))
    L.gpt2_sync()
    try:
        for st in streams:
            assert hip.hipStreamCreate(C.byref(st)) == 0
        for t in range(5):
            for i in range(2):
                L.gpt2_set_stream(streams[i])
                L.gpt2_pkv_grow(ref(c[i]), d_rows[i].ptr, len(x[i]))
                L.gpt2_pkv_append(ref(c[i]), 0, d_x[i].ptr, d_rows[i].ptr, len(x[i]))
                L.gpt2_pkv_attn(att[i].ptr, d_x[i].ptr, ref(c[i]), 0, d_rows[i].ptr, len(x[i]), 1, *ws[i].args)
                if t < 4:
                    L.gpt2_pkv_fork(ref(c[i]), parent.ptr)
                    L.gpt2_pkv_compact(ref(c[i]))
        for st in streams:
            assert hip.hipStreamSynchronize(st) == 0
    finally:
        L.gpt2_set_stream(None)
        for st in streams:
            if st:
                hip.hipStreamDestroy(st)
    pkg.check("two streams")
    for i in range(2):
        for t in range(5):
            assert r[i].grow(rows[i])
            r[i].append(0, x[i], rows[i])
            if t < 4:
                r[i].fork(np.array([1, 1, 3, 0, 3, -1]))
                r[i].compact()
        r[i].same_books(pkg, c[i])
        r[i].same_data(pkg, c[i])
        want, tol, on = r[i].attend(0, x[i], rows[i])
        err = np.abs(att[i].numpy(np.float16, want.shape).astype(np.float64) - want)
        assert (err[on] <= tol[on]).all()


@pytest.mark.parametrize("new", [1, 150])
def test_pages_past_4_gib(pkg, L, new):
    """The pool's last pages, 4.9 GB into the codes: appended, attended, read back, then moved to its beginning."""
    heads, pages, rng = 12, 100000, np.random.default_rng(35)
    big, small = pkg.PagedKV(pages, 2, 320, 1, heads), Ref(1, heads, 12, 2, 320)
    open_ = np.zeros_like(small.open)
    L.gpt2_h2d(big.c.open, open_.ctypes.data, open_.nbytes)
    refs = np.ones(pages, np.int32)
    refs[-12:] = 0
    L.gpt2_h2d(big.c.refs, refs.ctypes.data, refs.nbytes)
    for counts in ([130, 0], [new, new]):
        rows = rows_of(counts)
        n = int(rows[-1])
        x = qkv_of(rng, n, heads)
        d_rows, d_x, att = pkg.Dev.from_numpy(rows), pkg.Dev.from_numpy(x), pkg.Dev(n * heads * D * 2)
        L.gpt2_pkv_grow(ref(big), d_rows.ptr, n)
        L.gpt2_pkv_append(ref(big), 0, d_x.ptr, d_rows.ptr, n)
        ws = Ws(pkg, L.gpt2_pkv_attn_ws(ref(big), n))
        L.gpt2_pkv_attn(att.ptr, d_x.ptr, ref(big), 0, d_rows.ptr, n, 1, *ws.args)
        assert small.grow(rows)
        small.append(0, x, rows)
    want, tol, on = small.attend(0, x, rows)
    assert L.gpt2_pkv_status(ref(big)) == 0
    assert (np.abs(att.numpy(np.float16, want.shape).astype(np.float64) - want) <= tol).all()
    table = small.download(pkg, big, "table")
    used = small.len[0] // P
    np.testing.assert_array_equal(table[0, :used], small.table[0, :used] + pages - 12)
    assert int(table[0, 0]) * 2 * heads * P * D > 2 ** 32

    def read_back():
        out, first = pkg.Dev(100 * 2 * heads * D * 2), pkg.Dev.from_numpy(np.array([20, 0], np.int32))
        d_rows = pkg.Dev.from_numpy(np.array([0, 100, 100], np.int32))
        L.gpt2_pkv_read(out.ptr, ref(big), 0, d_rows.ptr, first.ptr, 100)
        L.gpt2_sync()
        pkg.check("read")
        np.testing.assert_array_equal(out.numpy(np.uint16, (100, 2 * heads * D)), small.read(0, 0, 20, 100).view(np.uint16))
    read_back()
    refs[:] = 0   # the pages before them were nobody's after all
    live = small.refs[:12]
    refs[-12:] = live
    L.gpt2_h2d(big.c.refs, refs.ctypes.data, refs.nbytes)
    L.gpt2_pkv_compact(ref(big))
    read_back()
    assert int(small.download(pkg, big, "table")[0, 0]) < 12
    big.free()


def test_one_cache_read_on_two_streams(pkg, L):
    """Attention and reads of one cache on two streams at once, a workspace each, a split form among them: the bits of one alone."""
    hip = hip_runtime()
    p, rng = Pair(pkg, L, layers=1, heads=4, pages=260, seqs=3, max_len=6000), np.random.default_rng(38)
    p.step(rng, [4100, 300, 2000])
    x = p.step(rng, [1, 1, 1])[0]
    p.check_attention(0, x)
    want = p.attend(0, x)
    n = len(x)
    atts, outs = [pkg.Dev(n * 4 * D * 2) for _ in range(4)], [pkg.Dev(200 * 2 * 4 * D * 2) for _ in range(4)]
    need = L.gpt2_pkv_attn_ws(ref(p.c), n)
    assert need > 16
    ws = [Ws(pkg, need) for _ in range(2)]
    d_rows, first = pkg.Dev.from_numpy(np.array([0, 150, 150, 200], np.int32)), pkg.Dev.from_numpy(np.array([3900, 0, 1960], np.int32))
    d_x = pkg.Dev.from_numpy(x)
    L.gpt2_sync()
    streams = [C.c_void_p(), C.c_void_p()]
    try:
        for st in streams:
            assert hip.hipStreamCreate(C.byref(st)) == 0
        for i in range(4):
            L.gpt2_set_stream(streams[i % 2])
            L.gpt2_pkv_attn(atts[i].ptr, d_x.ptr, ref(p.c), 0, p.d_rows.ptr, n, 1, *ws[i % 2].args)
            L.gpt2_pkv_read(outs[i].ptr, ref(p.c), 0, d_rows.ptr, first.ptr, 200)
        for st in streams:
            assert hip.hipStreamSynchronize(st) == 0
    finally:
        L.gpt2_set_stream(None)
        for st in streams:
            if st:
                hip.hipStreamDestroy(st)
    pkg.check("two streams")
    back = np.concatenate([p.r.read(0, 0, 3900, 150), p.r.read(0, 2, 1960, 50)]).view(np.uint16)
    for a, o in zip(atts, outs):
        np.testing.assert_array_equal(a.numpy(np.float16, want.shape), want)
        np.testing.assert_array_equal(o.numpy(np.uint16, back.shape), back)


def test_most_sequences(pkg, L):
    """As many sequences as there may be: pages handed out, forked, freed and packed."""
    rng = np.random.default_rng(39)
    p = Pair(pkg, L, layers=1, heads=1, pages=5000, seqs=4096, max_len=96)
    p.step(rng, rng.integers(0, 40, 4096))
    p.same()
    p.fork(rng.integers(-1, 4096, 4096))
    p.same()
    x = p.step(rng, (rng.random(4096) < 0.6).astype(int))
    L.gpt2_pkv_compact(ref(p.c))
    p.r.compact()
    p.same()
    p.check_attention(0, x[0])
    p.fork(np.where(np.arange(4096) < 4000, -1, np.arange(4096)))
    p.same()
    assert L.gpt2_pkv_status(ref(p.c)) == 0
