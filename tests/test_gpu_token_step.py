"""4-bit weights, logits' rules and token histories as they are used: a beam search of a two-layer model over the paged cache, every product with
4-bit weights, the logits shaped by penalties, n-gram bans, biases and a grammar before the selection, the histories following the beams.  Every
step is checked against plain numpy on what the step itself was given; the same captured into a graph and replayed; calls on two streams."""
import ctypes as C

import numpy as np
import pytest

from int4_ref import Histories, Weights, adjust, mask_words, product, quantize
from pagedkv_ref import beam, ref
from test_gpu_int4 import Case, run as run_product
from test_gpu_lnfold import hip_runtime
from test_gpu_logits import Pair, same
from test_gpu_paged_steps import BEAMS, GROUPS, LAYERS, SEQS, Search

pytestmark = pytest.mark.gpu
ROOM = 200


class Search4(Search):
    """Search with 4-bit weights and rules; `kept` has what the last step's products and rules were given."""

    def __init__(self, pkg, L):
        super().__init__(pkg, L, eos=-1)
        E, F, V = pkg.N_EMBD, 4 * pkg.N_EMBD, pkg.VOCAB
        self.q = {}
        for name, (n, k), group in [(f"{w}{i}", s, g) for i in range(LAYERS) for w, s, g in (("qkv", (3 * E, E), 64), ("ao", (E, E), 32), ("fc", (F, E), 64), ("pr", (E, F), 128))] + \
                                   [("head", (V, E), 128)]:
            self.q[name] = pkg.Int4(n, k, group)
            L.gpt2_quantize_int4(C.byref(self.q[name].w), self.w["wte" if name == "head" else name].ptr)
        self.bias = pkg.Dev.from_numpy((np.random.default_rng(41).standard_normal(F) * 0.1).astype(np.float16))
        self.raw = pkg.Dev(SEQS * V * 2)
        self.h = pkg.History(SEQS, ROOM)
        rng = np.random.default_rng(42)
        self.rep, self.pres, self.freq = (rng.uniform(a, b, SEQS).astype(np.float32) for a, b in ((1, 1.5), (0, 0.5), (0, 0.5)))
        self.biases = [[(int(t), float(v)) for t, v in zip(rng.integers(0, V, 20), np.float32(rng.standard_normal(20) * 3))] for _ in range(SEQS)]
        allowed = rng.random((2, V)) < np.array([[0.4], [0.01]])
        pick = np.array([-1, 0, 1, 0, 1, -1, 0, 0], np.int32)[:SEQS]
        self.masks = [allowed[p] if p >= 0 else None for p in pick]
        flat = sum(self.biases, [])
        d = self.rule_buffers = [pkg.Dev.from_numpy(np.asarray(a)) for a in (self.rep, self.pres, self.freq, np.cumsum([0] + [len(b) for b in self.biases]).astype(np.int32),
                                 np.array([t for t, _ in flat], np.int32), np.array([v for _, v in flat], np.float32), mask_words(allowed), pick)]
        r = self.rules = pkg.GPT2LogitsRules()
        r.history, r.ngram, r.n_bias, r.n_masks = C.pointer(self.h.h), 2, len(flat), 2
        r.repetition, r.presence, r.frequency, r.bias_start, r.bias_token, r.bias_value, r.mask, r.mask_row = (b.ptr for b in d)

    def product(self, out, x, name, n, bias=None, epi=0, resid=None):
        self.L.gpt2_matmul_int4(out.ptr, x.ptr, C.byref(self.q[name].w), bias.ptr if bias else None, n, epi, resid.ptr if resid else None)

    def blocks(self, rows, n, group):
        L, w, E = self.L, self.w, self.pkg.N_EMBD
        L.gpt2_pkv_grow(ref(self.c), rows, n)
        L.gpt2_pkv_embed(self.x.ptr, w["wte"].ptr, w["wpe"].ptr, self.ids.ptr, ref(self.c), rows, n)
        for i in range(LAYERS):
            L.gpt2_layernorm(self.ln.ptr, self.x.ptr, w["g"].ptr, w["b"].ptr, n, E)
            self.product(self.qkv[i], self.ln, f"qkv{i}", n)
            L.gpt2_pkv_append(ref(self.c), i, self.qkv[i].ptr, rows, n)
            L.gpt2_pkv_attn(self.atts[i].ptr, self.qkv[i].ptr, ref(self.c), i, rows, n, group, *self.ws.args)
            self.product(self.x, self.atts[i], f"ao{i}", n, epi=2, resid=self.x)
            L.gpt2_layernorm(self.ln.ptr, self.x.ptr, w["g"].ptr, w["b"].ptr, n, E)
            self.product(self.fc, self.ln, f"fc{i}", n, bias=self.bias, epi=1)
            self.product(self.x, self.fc, f"pr{i}", n, epi=2, resid=self.x)

    def select(self):
        L, w, E, V = self.L, self.w, self.pkg.N_EMBD, self.pkg.VOCAB
        L.gpt2_layernorm(self.ln.ptr, self.x.ptr, w["g"].ptr, w["b"].ptr, SEQS, E)
        self.product(self.raw, self.ln, "head", SEQS)
        L.gpt2_logits_adjust(self.logits.ptr, self.raw.ptr, V, SEQS, V, C.byref(self.rules))
        L.gpt2_beam_select(self.ids.ptr, self.parent.ptr, self.score.ptr, self.done.ptr, self.logits.ptr, V, self.score.ptr, self.done.ptr,
                           GROUPS, BEAMS, V, self.eos, *self.bws.args)

    def follow(self):
        self.L.gpt2_pkv_fork(ref(self.c), self.parent.ptr)
        self.L.gpt2_history_step(C.byref(self.h.h), self.parent.ptr, self.d_rows.ptr, self.ids.ptr, SEQS, 0)

    def step(self):
        self.blocks(self.d_rows.ptr, SEQS, BEAMS)
        self.select()
        self.follow()

    def start(self):
        """Prompts, their histories, the first selection."""
        self.L.gpt2_history_reset(C.byref(self.h.h))
        self.prompts()
        self.L.gpt2_history_step(C.byref(self.h.h), None, self.d_prompt.ptr, self.ids.ptr, int(self.rows[-1]), 1)
        self.L.gpt2_history_step(C.byref(self.h.h), self.parent.ptr, None, None, 0, 0)   # a prompt's beams from its first
        self.first()
        self.follow()

    def histories(self):
        tokens, length, start = np.empty((SEQS, ROOM), np.int32), np.empty(SEQS, np.int32), np.empty(SEQS, np.int32)
        for a, p in ((tokens, self.h.h.tokens), (length, self.h.h.len), (start, self.h.h.start)):
            assert self.L.gpt2_d2h(a.ctypes.data, p, a.nbytes) == 0
        return [t[:n].tolist() for t, n in zip(tokens, length)], start.tolist()


@pytest.fixture(scope="module")
def search(pkg, L):
    return Search4(pkg, L)


def test_search(pkg, L, search):
    s, E, V = search, pkg.N_EMBD, pkg.VOCAB
    oracle = Histories(SEQS, ROOM)
    s.start()
    after = s.state()
    oracle.step(None, s.rows, s.tokens, 1)
    oracle.step(np.repeat(np.arange(GROUPS) * BEAMS, BEAMS), None, [], 0)
    oracle.step(after[1], np.arange(SEQS + 1), after[0], 0)
    assert s.histories() == (oracle.seq, oracle.start)
    head = quantize(s.wte, 128)
    for t in range(16):
        print(f"step {t}", flush=True)
        before = after
        s.blocks(s.d_rows.ptr, SEQS, BEAMS)
        x = s.x.numpy(np.float16, (SEQS, E))
        assert np.isfinite(x).all()
        s.select()
        after = s.state()
        ln, raw, got = s.ln.numpy(np.float16, (SEQS, E)), s.raw.numpy(np.float16, (SEQS, V)), s.logits.numpy(np.float16, (SEQS, V))
        want, tol = product(ln, *head, 128, None, 0, None)
        assert (np.abs(raw - want) <= tol).all()
        same(got, *adjust(raw, oracle.seq, oracle.start, s.rep, s.pres, s.freq, 2, s.biases, s.masks))
        score = before[2].view(np.float32)
        token, parent, want, _, _ = beam(got, score, before[3], GROUPS, BEAMS, s.eos)
        assert (np.abs(after[2].view(np.float32) - want) <= 2.0 ** -24 * (95 + np.abs(want))).all()
        for r in range(SEQS):   # what was picked was allowed
            assert np.isfinite(got[after[1][r], after[0][r]])
        s.follow()
        oracle.step(after[1], np.arange(SEQS + 1), after[0], 0)
        L.gpt2_sync()
        assert s.histories() == (oracle.seq, oracle.start)
    assert L.gpt2_pkv_status(ref(s.c)) == 0
    for q in oracle.seq:   # no pair of tokens twice among those that were generated
        pairs = list(zip(q, q[1:]))[-14:]
        assert len(set(pairs)) == len(pairs)


def test_layer(pkg, L, search):
    """One layer's products in a prompt's size, from what the step had."""
    s, E, F = search, pkg.N_EMBD, 4 * pkg.N_EMBD
    rng = np.random.default_rng(5)
    x = rng.standard_normal((64, E)).astype(np.float16)
    d_x, d_f, d_o = pkg.Dev.from_numpy(x), pkg.Dev(64 * F * 2), pkg.Dev.from_numpy(x)
    s.product(d_f, d_x, "fc0", 64, bias=s.bias, epi=1)
    s.product(d_o, d_f, "pr0", 64, epi=2, resid=d_o)
    L.gpt2_sync()
    pkg.check("layer")
    f, o = d_f.numpy(np.float16, (64, F)), d_o.numpy(np.float16, (64, E))
    w_fc, w_pr = s.w["fc0"].numpy(np.float16, (F, E)), s.w["pr0"].numpy(np.float16, (E, F))
    want, tol = product(x, *quantize(w_fc, 64), 64, s.bias.numpy(np.float16, F), 1, None)
    assert (np.abs(f - want) <= tol).all()
    want, tol = product(f, *quantize(w_pr, 128), 128, None, 2, x)
    assert (np.abs(o - want) <= tol).all()


def test_search_captured(pkg, L, search):
    """A step captured on a stream of its own and replayed, other work between the replays: the same bits as the eager steps."""
    s, T = search, 10
    hip = hip_runtime()
    s.start()
    want = []
    for _ in range(T):
        s.step()
        want.append(s.state() + [s.histories()])
    rng = np.random.default_rng(9)
    other = Pair(pkg, L, 20, 64)
    s.start()
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
            assert s.histories() == want[t][4]
            c = Case(7 + 20 * t, 130, 256, 64)
            got = run_product(pkg, L, c)
            assert (np.abs(got - product(c.x, c.codes, c.scales, 64, c.bias, 0, None)[0]) <= product(c.x, c.codes, c.scales, 64, c.bias, 0, None)[1]).all()
            other.step(rng.integers(0, 20, 20), np.arange(21), rng.integers(0, 9, 20))
            other.check()
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
    """Products with one matrix and steps of two histories in turn on a stream each, nothing waited for in between."""
    hip = hip_runtime()
    cases = [Case(33, 768, 3072, 64, epi=2), Case(5, 768, 3072, 64, epi=1)]
    cases[1].codes, cases[1].scales = cases[0].codes, cases[0].scales
    w = Weights(pkg, cases[0].codes, cases[0].scales, 64)
    d = [[pkg.Dev.from_numpy(v) if v is not None else None for v in (c.x, c.bias, c.resid)] + [pkg.Dev(c.m * c.n * 2)] for c in cases]
    rng = np.random.default_rng(2)
    pairs = [Pair(pkg, L, 40, 128), Pair(pkg, L, 9, 128)]
    steps = [[(rng.integers(0, p.n, p.n), rng.integers(0, 99, p.n)) for _ in range(20)] for p in pairs]
    dev = [[[pkg.Dev.from_numpy(v.astype(np.int32)) for v in st] for st in side] for side in steps]
    rows = [pkg.Dev.from_numpy(np.arange(p.n + 1, dtype=np.int32)) for p in pairs]
    L.gpt2_sync()
    streams = [C.c_void_p(), C.c_void_p()]
    try:
        for st in streams:
            assert hip.hipStreamCreate(C.byref(st)) == 0
        for t in range(20):
            for i, c in enumerate(cases):
                L.gpt2_set_stream(streams[i])
                x, b, r, out = d[i]
                L.gpt2_matmul_int4(out.ptr, x.ptr, w.ref, b.ptr, c.m, c.epi, r.ptr if r else None)
                L.gpt2_history_step(C.byref(pairs[i].dev.h), dev[i][t][0].ptr, rows[i].ptr, dev[i][t][1].ptr, pairs[i].n, 0)
                pairs[i].ref.step(steps[i][t][0], np.arange(pairs[i].n + 1), steps[i][t][1], 0)
        for st in streams:
            assert hip.hipStreamSynchronize(st) == 0
    finally:
        L.gpt2_set_stream(None)
        for st in streams:
            if st:
                hip.hipStreamDestroy(st)
    pkg.check("two streams")
    for i, c in enumerate(cases):
        want, tol = product(c.x, c.codes, c.scales, 64, c.bias, c.epi, c.resid)
        assert (np.abs(d[i][3].numpy(np.float16, (c.m, c.n)) - want) <= tol).all()
        pairs[i].check()
