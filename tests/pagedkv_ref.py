"""A paged K/V cache in plain numpy, written from the definitions in include/gpt2_pagedkv.h: the oracle of
tests/test_gpu_pagedkv.py.  Bookkeeping and stored values are exact (the quantiser's fp32 divisions are IEEE in numpy too);
attention is in 64 bits."""
import ctypes as C

import numpy as np

P, D = 32, 64


def tiles(x):
    """[K|V, head, token, dim] as tiles [K|V, head, 2048]."""
    h = x.shape[1]
    v = x[1].reshape(h, P // 8, 8, D).transpose(0, 1, 3, 2).reshape(h, P * D)
    return np.stack([x[0].reshape(h, P * D), v])


def untile(t):
    """Tiles [K|V, head, 2048] as [K|V, head, token, dim]."""
    h = t.shape[1]
    return np.stack([t[0].reshape(h, P, D), t[1].reshape(h, P // 8, D, 8).transpose(0, 1, 3, 2).reshape(h, P, D)])


def finite(x):
    return np.clip(np.nan_to_num(x.astype(np.float32), nan=0.0, posinf=65504.0, neginf=-65504.0), -65504, 65504).astype(np.float16)


def quantize(x):
    """[K|V, head, token, dim] fp16 -> codes, scales [K|V, head]."""
    x = x.astype(np.float32)
    peak = np.abs(x).max(axis=(2, 3))
    s = np.where(peak == 0, np.float32(1), peak / np.float32(127)).astype(np.float32)
    return np.clip(np.rint(x / s[:, :, None, None]), -127, 127).astype(np.int8), s


class Ref:
    def __init__(self, layers, heads, pages, seqs, max_len):
        self.layers, self.heads, self.pages, self.seqs = layers, heads, pages, seqs
        self.max_pages = -(-max_len // P)
        self.codes = np.zeros((layers, pages, 2, heads, P * D), np.int8)
        self.scales = np.zeros((layers, pages, 2, heads), np.float32)
        self.open = np.zeros((layers, seqs, 2, heads, P * D), np.float16)
        self.table = np.zeros((seqs, self.max_pages), np.int32)
        self.len, self.start = np.zeros(seqs, np.int32), np.zeros(seqs, np.int32)
        self.slot, self.refs = np.arange(seqs, dtype=np.int32), np.zeros(pages, np.int32)

    def grow(self, rows):
        new = np.diff(rows)
        need = (self.len + new) // P - self.len // P
        free = np.flatnonzero(self.refs == 0)
        self.start[:] = self.len
        if (self.len + new > self.max_pages * P).any() or need.sum() > free.size:
            return False
        k = 0
        for s in range(self.seqs):
            for j in range(need[s]):
                self.table[s, self.len[s] // P + j] = free[k]
                self.refs[free[k]] = 1
                k += 1
        self.len += new
        return True

    def append(self, L, qkv, rows):
        E = self.heads * D
        for s in range(self.seqs):
            n = self.len[s] - self.start[s]
            if n == 0:
                continue
            x = finite(qkv[rows[s]:rows[s + 1], E:]).reshape(n, 2, self.heads, D).transpose(1, 2, 0, 3)
            buf = untile(self.open[L, self.slot[s]])
            for i in range(n):
                pos = self.start[s] + i
                buf[:, :, pos % P] = x[:, :, i]
                if pos % P == P - 1:
                    page = self.table[s, pos // P]
                    q, self.scales[L, page] = quantize(buf)
                    self.codes[L, page] = tiles(q)
                    buf = untile(self.open[L, self.slot[s]])
            # only what is left of the new rows replaces the open page's tokens
            left = untile(self.open[L, self.slot[s]])
            for i in range(n):
                pos = self.start[s] + i
                if pos >= self.len[s] // P * P:
                    left[:, :, pos % P] = x[:, :, i]
            self.open[L, self.slot[s]] = tiles(left)

    def held(self, L, s, upto=None):
        """Keys and values [K|V, head, token, dim] of a sequence, in 64 bits; keys of pages that are none are NaN."""
        n = int(self.len[s]) if upto is None else upto
        parts = [np.zeros((2, self.heads, 0, D))]
        for j in range(-(-n // P)):
            if j == self.len[s] // P:
                parts.append(untile(self.open[L, self.slot[s]]).astype(np.float64))
                continue
            page = self.table[s, j]
            if not 0 <= page < self.pages:
                parts.append(np.full((2, self.heads, P, D), np.nan))
                continue
            parts.append(untile(self.codes[L, page]).astype(np.float64) * self.scales[L, page].astype(np.float64)[:, :, None, None])
        return np.concatenate(parts, axis=2)[:, :, :n]

    def read(self, L, s, first, n):
        """fp16 rows k | v of positions first .. first + n - 1."""
        out = np.zeros((n, 2 * self.heads * D), np.float16)
        h = self.held(L, s)
        # a code times its scale is rounded to 32 bits, then to 16
        h = np.nan_to_num(h, nan=0.0).astype(np.float32).astype(np.float16)
        for i in range(n):
            if 0 <= first + i < self.len[s]:
                out[i] = h[:, :, first + i].reshape(-1)
        return out

    def attend(self, L, qkv, rows):
        """att [nRows, E] in 64 bits, how far a kernel may be off, and which rows are written."""
        E = self.heads * D
        out, tol, on = np.zeros((len(qkv), E)), np.zeros((len(qkv), E)), np.zeros(len(qkv), bool)
        for s in range(self.seqs):
            n = self.len[s] - self.start[s]
            if n == 0 or n != rows[s + 1] - rows[s]:
                continue
            k, v = self.held(L, s)
            for i in range(n):
                vis = self.start[s] + i + 1
                q = qkv[rows[s] + i, :E].astype(np.float64).reshape(self.heads, D)
                there = ~np.isnan(k[:, :vis, 0])
                sc = np.where(there, np.einsum("hd,htd->ht", q, np.nan_to_num(k[:, :vis])) / 8, -np.inf)
                mx = sc.max(axis=1, keepdims=True)
                w = np.where(there, np.exp(sc - np.where(np.isfinite(mx), mx, 0)), 0)
                tot = w.sum(axis=1, keepdims=True)
                vv = np.nan_to_num(v[:, :vis])
                out[rows[s] + i] = (np.einsum("ht,htd->hd", w, vv) / np.where(tot == 0, 1, tot)).reshape(-1)
                on[rows[s] + i] = True
                # Weights rounded to fp16, half a step 2^-11 each against the average they form (2 vmax), those below
                # 2^-29 of the largest by 2^-40 each; scores' sums of 64 fp32 products (each half a step 2^-24 of the running sum, at
                # most S = sum |q k| / 8, times 64, and the weight by as much, on both sides of the average); the output's own
                # rounding, 2^-11 of at most vmax (and 2^-25 when subnormal).
                vmax = np.abs(vv).max(axis=(1, 2))
                S = (np.abs(q)[:, None] * np.abs(np.nan_to_num(k[:, :vis]))).sum(axis=2).max(axis=1) / 8
                t = vmax * (2 * 2.0 ** -11 + vis * 2.0 ** -40 * 2 + 2 * (64 + 4) * 2.0 ** -24 * (S + 1) + 2.0 ** -11) + 2.0 ** -25
                tol[rows[s] + i] = np.repeat(t, D)
        return out, tol, on

    def fork(self, parent):
        children = [int((parent == s).sum()) for s in range(self.seqs)]
        spare = [int(self.slot[s]) for s in range(self.seqs) if children[s] == 0]
        for s in range(self.seqs):
            for j in range(self.len[s] // P):
                self.refs[self.table[s, j]] += children[s] - 1
        table, ln, slot, seen = self.table.copy(), self.len.copy(), self.slot.copy(), set()
        old_open = self.open.copy()
        for i, p in enumerate(parent):
            ln[i] = self.len[p] if p >= 0 else 0
            table[i, :ln[i] // P] = self.table[p, :ln[i] // P]
            if p >= 0 and p not in seen:
                seen.add(p)
                slot[i] = self.slot[p]
                continue
            slot[i] = spare.pop(0)
            if p >= 0:
                for L in range(self.layers):
                    src, dst = untile(old_open[L, self.slot[p]]), untile(self.open[L, slot[i]])
                    dst[:, :, :ln[i] % P] = src[:, :, :ln[i] % P]
                    self.open[L, slot[i]] = tiles(dst)
        assert not spare
        self.table, self.len, self.slot = table, ln, slot
        self.start = ln.copy()

    def compact(self):
        live = np.flatnonzero(self.refs)
        n = live.size
        movers, holes = live[live >= n], np.flatnonzero(self.refs[:n] == 0)
        to = np.arange(self.pages)
        to[movers] = holes
        self.codes[:, holes], self.scales[:, holes] = self.codes[:, movers], self.scales[:, movers]
        self.refs[holes] = self.refs[movers]
        self.refs[movers] = 0
        for s in range(self.seqs):
            for j in range(self.len[s] // P):
                self.table[s, j] = to[self.table[s, j]]
        return n

    # ------------------------------------------------------------------ against the library's cache
    FIELDS = (("codes", np.int8), ("scales", np.float32), ("open", np.float16), ("table", np.int32), ("len", np.int32),
              ("start", np.int32), ("slot", np.int32), ("refs", np.int32))

    def upload(self, pkg, cache):
        for name, t in self.FIELDS:
            a = np.ascontiguousarray(getattr(self, name), t)
            assert pkg.lib().gpt2_h2d(getattr(cache.c, name), a.ctypes.data, a.nbytes) == 0

    def download(self, pkg, cache, name):
        a = np.empty_like(np.ascontiguousarray(getattr(self, name)))
        assert pkg.lib().gpt2_d2h(a.ctypes.data, getattr(cache.c, name), a.nbytes) == 0
        return a

    def same_books(self, pkg, cache):
        for name in ("len", "start", "slot", "refs"):
            np.testing.assert_array_equal(self.download(pkg, cache, name), getattr(self, name), err_msg=name)
        got = self.download(pkg, cache, "table")
        for s in range(self.seqs):
            np.testing.assert_array_equal(got[s, :self.len[s] // P], self.table[s, :self.len[s] // P], err_msg="table")

    def same_data(self, pkg, cache):
        live = np.flatnonzero(self.refs)
        for name in ("codes", "scales"):
            np.testing.assert_array_equal(self.download(pkg, cache, name)[:, live], getattr(self, name)[:, live], err_msg=name)
        got = self.download(pkg, cache, "open")
        for s in range(self.seqs):
            n = self.len[s] % P
            for L in range(self.layers):
                np.testing.assert_array_equal(untile(got[L, self.slot[s]])[:, :, :n].view(np.uint16),
                                              untile(self.open[L, self.slot[s]])[:, :, :n].view(np.uint16), err_msg="open")


class Ws:
    """A workspace of at least n bytes."""

    def __init__(self, pkg, n):
        self.d = pkg.Dev(n)
        self.args = (self.d.ptr, n)


def beam(logits, score, done, groups, beams, eos):
    """Tokens, parents, scores in 64 bits, done; and the smallest gap between neighbours of the sorted scores that decides."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, 65504.0))
    out, gap = [], np.inf
    for g in range(groups):
        cand = []
        for r in range(g * beams, (g + 1) * beams):
            cum = float(score[r])
            if eos >= 0 and done[r]:
                cand.append((cum if cum == cum else -np.inf, r, 0, 0, eos))
                continue
            m = x[r].max()
            with np.errstate(invalid="ignore", divide="ignore"):
                s = cum + (x[r] - m) - np.log(np.exp(x[r] - m).sum())
            s = np.where(np.isnan(s), -np.inf, s)
            for t in np.argsort(-x[r], kind="stable")[:beams].tolist():
                cand.append((s[t], r, -x[r, t], t, t))
        cand.sort(key=lambda c: (-c[0], c[1], c[2], c[3]))
        for a, b in zip(cand[:beams], cand[1:]):
            if a[1] != b[1] and np.isfinite(a[0]) and np.isfinite(b[0]):
                gap = min(gap, a[0] - b[0])
        out += [(c[4], c[1], c[0], int(eos >= 0 and c[4] == eos)) for c in cand[:beams]]
    return [np.array(v) for v in zip(*out)] + [gap]


def ref(c):
    return C.byref(c.c)
