"""4-bit weights with group scales, logits' rules and token histories in plain numpy, written from the definitions in
include/gpt2_int4.h and include/gpt2_logits.h: the oracle of tests/test_gpu_int4.py and tests/test_gpu_logits.py."""
import ctypes as C

import numpy as np

U16 = 2.0 ** -11   # half a step of fp16, relative
TINY = 2.0 ** -25  # half a step of its smallest numbers
U32 = 2.0 ** -23   # a whole step of fp32: an addition on the matrix units may cut off


def cdiv(a, b):
    return -(-a // b)


def quantize(w, group):
    """fp16 [N][K] -> codes [N][K], scales fp16 [N][groups]."""
    x = np.clip(np.nan_to_num(w.astype(np.float32), nan=0.0, posinf=65504.0, neginf=-65504.0), -65504, 65504)
    codes, scales = np.zeros(w.shape, np.int8), np.zeros((w.shape[0], cdiv(w.shape[1], group)), np.float16)
    for g in range(scales.shape[1]):
        part = x[:, group * g:group * (g + 1)]
        s = (np.abs(part).max(axis=1) / np.float32(7)).astype(np.float16)
        s[s == 0] = 1
        scales[:, g] = s
        codes[:, group * g:group * (g + 1)] = np.clip(np.rint(part / s.astype(np.float32)[:, None]), -7, 7)
    return codes, scales


def pack(codes, scales, group, rest=8, rest_scale=1.0):
    """The two buffers.  `rest`: codes of rows past N (as held); `rest_scale`: their scales.  Codes past K are 0."""
    n, k = codes.shape
    nt, kb, per = cdiv(n, 16), cdiv(k, 128), 128 // group
    u = np.full((16 * nt, 128 * kb), 8, np.uint32)
    u[n:] = rest
    u[:n, :k] = codes.astype(np.int32) + 8
    out = np.zeros((nt, kb, 4, 16, 4), np.uint32)
    for e in range(8):
        # k = 128 kb + 32 i + 8 o + e
        part = u.reshape(nt, 16, kb, 4, 4, 8)[..., e]                      # [nt][n][kb][i][o]
        out |= part.transpose(0, 2, 4, 1, 3) << np.uint32(4 * (e // 2) + 16 * (e % 2))
    s = np.ones((16 * nt, per * kb), np.float16)
    s[n:] = rest_scale
    s[:n, :scales.shape[1]] = scales
    return out, np.ascontiguousarray(s.reshape(nt, 4, 4, kb, per).transpose(0, 3, 1, 4, 2))


def unpack(words, scales, N, K, group):
    """The codes and scales that the two buffers hold."""
    nt, kb = words.shape[:2]
    u = np.zeros((nt, 16, kb, 4, 4, 8), np.int32)
    for e in range(8):
        u[..., e] = (words >> np.uint32(4 * (e // 2) + 16 * (e % 2)) & np.uint32(15)).transpose(0, 3, 1, 4, 2)
    s = scales.transpose(0, 2, 4, 1, 3).reshape(16 * nt, -1)
    return (u.reshape(16 * nt, 128 * kb)[:N, :K] - 8).astype(np.int8), s[:N, :cdiv(K, group)]


def dequantized(codes, scales, group):
    """In 64 bits."""
    return codes * np.repeat(scales.astype(np.float64), group, axis=1)[:, :codes.shape[1]]


def gelu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))


def product(x, codes, scales, group, bias, epi, resid):
    """The product in 64 bits, and how far fp32 sums rounded to fp16 once may be from it.  Sums of K products and a row's groups in fp32, in
    any order: (K + groups) steps of the sum of the terms' sizes at most; the bias one more.  gelu's slope is at most 1.13; its exponent is
    off by a few steps of an argument of at most 2^7 where the result is not 0 or v (2^-23 * 2^7 * 4), and what it is applied to by the sums' error."""
    w, x = dequantized(codes, scales, group), x.astype(np.float64)
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    y, size = y + b, size + np.abs(b)
    tol = (w.shape[1] + scales.shape[1] + 2) * U32 * size
    if epi == 1:
        y = gelu(y)
        tol = 1.13 * tol + 2.0 ** -14 * np.abs(y) * (np.abs(y) < 8) + 16 * U32 * np.abs(y)
    elif epi == 2:
        y = resid.astype(np.float64) + y
        tol += U32 * (np.abs(y) + size)
    return y, tol + U16 * (np.abs(y) + tol) + TINY


class Weights:
    """Codes and scales on the device, and the struct."""

    def __init__(self, pkg, codes, scales, group, **kw):
        words, s = pack(codes, scales, group, **kw)
        self.words, self.s = pkg.Dev.from_numpy(words), pkg.Dev.from_numpy(s)
        self.w = pkg.GPT2Int4W(self.words.ptr, self.s.ptr, codes.shape[0], codes.shape[1], group, None)
        self.ref = C.byref(self.w)


def adjust(logits, seqs, starts, rep, pres, freq, ngram, biases, masks):
    """Logits after the rules in 64 bits, and how far fp32 rounded to fp16 once may be from them.  Per row: seqs a list of tokens or None, biases a
    list of (token, value), masks a list of booleans or None."""
    out = logits.astype(np.float64)
    size = np.abs(out)
    V = out.shape[1]
    for r in range(out.shape[0]):
        for t, v in dict(biases[r]).items():   # the last entry of a token
            if 0 <= t < V:
                out[r, t] += v
                size[r, t] += abs(v)
        if seqs is not None:
            s = list(seqs[r])
            for t in set(s):
                if not 0 <= t < V:
                    continue
                x = out[r, t]
                out[r, t] = x / rep[r] if x > 0 else x * rep[r]
                size[r, t] = size[r, t] * max(rep[r], 1 / rep[r])
                c = s[max(0, starts[r]):].count(t)
                if c:
                    out[r, t] -= freq[r] * c + pres[r]
                    size[r, t] += 2 * (abs(freq[r] * c) + abs(pres[r]))
            if ngram and len(s) >= ngram:
                tail = s[len(s) - (ngram - 1):]
                for i in range(len(s) - ngram + 1):
                    t = s[i + ngram - 1]
                    if s[i:i + ngram - 1] == tail and 0 <= t < V:
                        out[r, t] = -np.inf
        if masks[r] is not None:
            out[r, ~masks[r]] = -np.inf
    # three operations after one another, of 2^-24 each, the count's product one more: below 4 steps 2^-23 of the largest value on the way
    with np.errstate(invalid="ignore"):
        tol = 4 * U32 * np.where(np.isfinite(size), size, 0)
        return out, tol + U16 * (np.where(np.isfinite(out), np.abs(out), 0) + tol) + TINY


def mask_words(allowed):
    """Booleans [n][V] as the mask's words."""
    n, v = allowed.shape
    bits = np.zeros((n, cdiv(v, 32) * 32), np.uint8)
    bits[:, :v] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


class Histories:
    """Token histories in plain lists."""

    def __init__(self, n, room):
        self.n, self.room = n, room
        self.seq, self.start = [[] for _ in range(n)], [0] * n

    def step(self, parent, rows, ids, prompt):
        n_rows = len(ids)
        seq, start = [], []
        for s in range(self.n):
            p = s if parent is None else int(parent[s])
            old, st = (list(self.seq[p]), self.start[p]) if 0 <= p < self.n else ([], 0)
            a, b = (0, 0) if rows is None else (int(rows[s]), int(rows[s + 1]))
            if not 0 <= a <= b <= n_rows:
                a = b = 0
            new = (old + [int(t) for t in ids[a:b]])[:self.room]
            start.append(len(new) if prompt and len(new) > len(old) else st)
            seq.append(new)
        self.seq, self.start = seq, start
