"""Operators whose speed is measured, beside those of perf/operators.py: the two ends of a step of several sequences.

Weights of 4 bits with a scale for each group along k: their quantiser, and the product of one row (a sequence's next token), a
few rows (a batch's) or many (prompts) with them.  And what shapes logits before a token is chosen: penalties for tokens that a
sequence has already, n-gram bans, biases and grammar masks, with the token histories that they read, which follow the
beams' parents as the cache does.

A tile of codes is 16 outputs n by 128 inputs k, 1 KB: the 32-bit word at [k % 32 / 8][n % 16][k % 128 / 32] holds eight
k, the two of a pair 16 bits apart, pairs 4 bits apart, as q + 8.  Its scales: [n % 16 / 4][group in the tile][n % 4].
"""
import ctypes as C
import math
import random

import torch

own = False   # True: run() calls this library's kernels; False: the same in elementary torch operations

EMBD, VOCAB, CTX = 768, 50257, 1024
FFN, QKV = 4 * EMBD, 3 * EMBD
NONE, GELU, ADD = 0, 1, 2   # what follows a product


def listed():
    return [
        # One sequence's next token, its QKV product: the smallest call, latency.
        {"name": "row_qkv", "op": "matmul", "m": 1, "n": QKV, "k": EMBD, "group": 64, "epi": NONE, "bias": True},
        # The same with a layer of a large model: a stream of 33 MB.
        {"name": "row_8192", "op": "matmul", "m": 1, "n": 8192, "k": 8192, "group": 128, "epi": NONE, "bias": False},
        # The tied head for eight beams: an odd number of outputs.
        {"name": "head_8", "op": "matmul", "m": 8, "n": VOCAB, "k": EMBD, "group": 128, "epi": NONE, "bias": False},
        # A batch of 48 sequences, one token each: fc and its gelu, the finest scales.
        {"name": "batch_48_fc", "op": "matmul", "m": 48, "n": FFN, "k": EMBD, "group": 32, "epi": GELU, "bias": True},
        # A prompt of odd length: mlp-proj, added to the residual.
        {"name": "prompt_777_proj", "op": "matmul", "m": 777, "n": EMBD, "k": FFN, "group": 64, "epi": ADD, "bias": True},
        # A batch of prompts with a layer of a large model: matrix work.
        {"name": "prompts_2000_4096", "op": "matmul", "m": 2000, "n": 4096, "k": 4096, "group": 128, "epi": NONE, "bias": True},
        # One layer's matrix when a model is loaded, and the largest matrix of the model.
        {"name": "quantize_proj", "op": "quantize", "n": EMBD, "k": EMBD, "group": 64},
        {"name": "quantize_head", "op": "quantize", "n": VOCAB, "k": EMBD, "group": 128},
        # Two prompts with four beams each: repetition penalties and no repeated trigrams.
        {"name": "logits_8", "op": "logits", "rows": 8, "vocab": VOCAB, "past": 600, "ngram": 3, "biases": 0, "masks": 0},
        # A large batch under grammars, with biases, penalties by count and long histories.
        {"name": "logits_256_masked", "op": "logits", "rows": 256, "vocab": VOCAB, "past": 4096, "ngram": 0, "biases": 300, "masks": 256},
        # The histories of eight beams follow their parents and take a token each: latency.
        {"name": "history_8", "op": "history", "seqs": 8, "beams": 4, "past": 600, "room": CTX, "new": 1},
        # A thousand beams, long histories.
        {"name": "history_1024", "op": "history", "seqs": 1024, "beams": 8, "past": 4000, "room": 4096, "new": 1},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    op = rng.choice(("matmul", "matmul", "matmul", "quantize", "logits", "logits", "history"))
    if op == "matmul":
        m, n, k = size(1, 2000), size(64, VOCAB), size(64, 8192)
        if rng.random() < 0.6:
            k = max(64, k // 64 * 64)
        n = min(n, 8192 * 8192 // k)
        m = min(m, max(1, 2000 * 4096 * 4096 // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "group": rng.choice((32, 64, 128)), "epi": rng.choice((NONE, GELU, ADD)),
                "bias": rng.random() < 0.7}
    if op == "quantize":
        k = size(64, 8192)
        return {"op": op, "n": size(64, VOCAB * EMBD // k), "k": k, "group": rng.choice((32, 64, 128))}
    if op == "logits":
        return {"op": op, "rows": size(1, 256), "vocab": rng.choice((VOCAB, size(1000, 65536))), "past": size(8, 4096), "ngram": rng.choice((0, 2, 3, 4)),
                "biases": rng.choice((0, size(1, 300))), "masks": rng.choice((0, 1, 1, size(1, 256)))}
    past, seqs = size(16, 4000), size(1, 1024)
    return {"op": op, "seqs": seqs, "beams": rng.choice((1, 4, 8, 16)), "past": past, "room": past + size(16, 96), "new": rng.choice((1, 1, size(1, 16)))}


def _spread(n, hi, lo):
    """n lengths from hi down to lo, mixed."""
    v = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    random.Random(n * 31 + hi).shuffle(v)
    return v


def _ceil(a, b):
    return -(-a // b)


def _past(case):
    n = case["rows"] if case["op"] == "logits" else case["seqs"]
    return _spread(n, case["past"], case["past"] // 4)


def _parents(case):
    """As a beam search's selection picks them: a few beams of a group win, the order is mixed; the last group may be smaller."""
    rng, out = random.Random(case["seqs"] * 1000 + case["beams"]), []
    for g in range(0, case["seqs"], case["beams"]):
        b = min(case["beams"], case["seqs"] - g)
        out += [g + i for i in rng.choices(range(b), [rng.random() ** 2 + 1e-3 for _ in range(b)], k=b)]
    return out


def work(case):
    op = case["op"]
    if op in ("matmul", "quantize"):
        n, k = case["n"], case["k"]
        held = n * (_ceil(k, 2) + 2 * _ceil(k, case["group"]))
        if op == "quantize":   # with the values that the codes stand for, which are read back
            return {"bytes": 2 * n * k + 2 * held + 2 * n * k, "flops": 3 * n * k}
        m = case["m"]
        return {"bytes": held + 2 * m * k + 2 * m * n * (2 if case["epi"] == ADD else 1) + 2 * n * case["bias"], "flops": 2 * m * n * k}
    if op == "logits":
        rows, v = case["rows"], case["vocab"]
        masks = min(case["masks"], rows) * 4 * _ceil(v, 32)
        return {"bytes": 4 * rows * v + masks + 4 * sum(_past(case)) + 8 * rows * case["biases"], "flops": 2 * rows * v}
    past, parents = _past(case), _parents(case)
    moved = sum(past[p] for i, p in enumerate(parents) if p != i)
    return {"bytes": 8 * moved + 8 * case["seqs"] * case["new"] + 24 * case["seqs"], "flops": 0}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, std, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    rows = [0]
    for n in counts:
        rows.append(rows[-1] + n)
    return rows


def _weights(case, seed):
    """Codes [n][k] and scales [n][groups] as a quantiser leaves them: most codes small, scales of a spread of two."""
    g = _gen(seed)
    n, k, groups = case["n"], case["k"], _ceil(case["k"], case["group"])
    codes = _normal((n, k), 2.6, g).round_().clamp_(-8, 7).to(torch.int8)
    scales = ((0.5 + torch.rand((n, groups), generator=g, device="cuda")) * (0.4 / math.sqrt(k))).half()
    return codes, scales, g


def _matmul_inputs(case, seed):
    """Activations as after a LayerNorm, a few channels far wider; bias and residual as the model's."""
    codes, scales, g = _weights(case, seed)
    x = _normal((case["m"], case["k"]), 1.0, g)
    x[:, ::97] *= 8.0
    bias = _normal((case["n"],), 0.3, g).half() if case["bias"] else None
    resid = _normal((case["m"], case["n"]), 1.5, g).half() if case["epi"] == ADD else None
    return codes, scales, x.half(), bias, resid


def _pack(codes, scales, group):
    """Codes [n][k] and scales [n][groups] as tiles."""
    n, k = codes.shape
    nt, kb, per = _ceil(n, 16), _ceil(k, 128), 128 // group
    u = torch.full((16 * nt, 128 * kb), 8, dtype=torch.int32, device=codes.device)
    u[:n, :k] = codes.int() + 8
    u = u.view(nt, 16, kb, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)   # [nt][kb][octet][n][32s][pair][of the pair]
    shift = 4 * torch.arange(4, device=u.device)[:, None] + 16 * torch.arange(2, device=u.device)
    words = (u.long() << shift).sum(dim=(-2, -1))
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).int().contiguous()
    s = torch.ones((16 * nt, per * kb), dtype=torch.float16, device=codes.device)
    s[:n, :scales.shape[1]] = scales
    return words, s.view(nt, 4, 4, kb, per).permute(0, 3, 1, 4, 2).contiguous()


def _quantize_inputs(case, seed):
    """A trained matrix: rows of different sizes, a few values that stand out."""
    g = _gen(seed)
    w = _normal((case["n"], case["k"]), 1.0, g) * (0.05 + 0.1 * torch.rand((case["n"], 1), generator=g, device="cuda"))
    w *= 1.0 + 4.0 * (torch.rand(w.shape, generator=g, device="cuda") < 0.005)
    return w.half()


def _histories(case, seed):
    """Token histories of text: words come again, the more so the commoner they are, and phrases too."""
    g = _gen(seed + 77)
    past, vocab = _past(case), case.get("vocab", VOCAB)
    room = case.get("room", case["past"] + 16)
    u = torch.rand((len(past), room), generator=g, device="cuda")
    tokens = (torch.exp(u * math.log(vocab)) - 1.0).long() * 7919 % vocab
    tokens[:, 2::3] = tokens[:, :-2:3][:, :tokens[:, 2::3].shape[1]]
    prompt = (torch.rand(len(past), generator=g, device="cuda") * _ints(past)).int()
    return tokens.int().contiguous(), _ints(past), prompt


def _logits_inputs(case, seed):
    """Logits as a language model gives them, a row's penalties, bias lists of tokens of their own, grammar masks that allow
    anything from a few tokens to nearly all, some rows without one."""
    g, rows, v = _gen(seed), case["rows"], case["vocab"]
    i = {"logits": (_normal((rows, v), 2.5, g) - 2.0 + 8.0 * (torch.rand((rows, v), generator=g, device="cuda") < 20.0 / v)).half()}
    i["tokens"], i["len"], i["from"] = _histories(case, seed)
    i["repetition"] = 1.0 + 0.3 * torch.rand(rows, generator=g, device="cuda")
    i["presence"], i["frequency"] = (0.5 * torch.rand(rows, generator=g, device="cuda") for _ in range(2))
    i["bias_token"] = i["bias_value"] = i["bias_start"] = i["mask"] = i["mask_row"] = None
    if case["biases"]:
        n = min(case["biases"], v)
        counts = _spread(rows, n, n // 2)
        first = torch.randint(0, v, (rows, 1), generator=g, device="cuda")
        step = max(1, v // n)
        lists = (first + step * torch.arange(n, device="cuda")) % (step * n)
        i["bias_token"] = lists[torch.arange(n, device="cuda") < _ints(counts)[:, None]].int()
        i["bias_value"] = _normal(i["bias_token"].shape, 4.0, g)
        i["bias_start"] = _ints(_offsets(counts))
    if case["masks"]:
        n = case["masks"]
        allowed = torch.rand((n, 1), generator=g, device="cuda")
        bits = torch.rand((n, 32 * _ceil(v, 32)), generator=g, device="cuda") < allowed ** 2
        words = (bits.view(n, -1, 32).long() << torch.arange(32, device="cuda")).sum(-1)
        i["mask"] = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
        pick = torch.randperm(max(rows, n), generator=g, device="cuda")[:rows] % n
        i["mask_row"] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.1, -1, pick).int()
    return i


def prepare(case, seed):
    op = case["op"]
    s = {"op": op}
    if op == "matmul":
        codes, scales, s["x"], s["bias"], s["resid"] = _matmul_inputs(case, seed)
        s["codes"], s["scales"] = _pack(codes, scales, case["group"])
        s |= {"n": case["n"], "k": case["k"], "group": case["group"], "epi": case["epi"]}
        s["out"] = torch.empty((case["m"], case["n"]), dtype=torch.float16, device="cuda")
    elif op == "quantize":
        s["w"], s["group"] = _quantize_inputs(case, seed), case["group"]
        nt, kb = _ceil(case["n"], 16), _ceil(case["k"], 128)
        s["codes"] = torch.empty((nt, kb, 256), dtype=torch.int32, device="cuda")
        s["scales"] = torch.empty((nt, kb, 4, 128 // case["group"], 4), dtype=torch.float16, device="cuda")
        s["out"] = torch.empty_like(s["w"])
    elif op == "logits":
        s |= _logits_inputs(case, seed)
        s["ngram"] = case["ngram"]
        s["out"] = torch.empty_like(s["logits"])
    else:
        tokens, past, prompt = _histories(case, seed)
        n = case["seqs"]
        s["tokens"], s["book"] = tokens, torch.cat((past, prompt, _ints([0])))
        s["first"], s["len"], s["from"] = s["book"].clone(), s["book"][:n], s["book"][n:2 * n]
        s["parent"], s["rows"] = _ints(_parents(case)), _ints(_offsets([case["new"]] * n))
        s["ids"] = torch.randint(0, VOCAB, (n * case["new"],), generator=_gen(seed), device="cuda").int()
    if own:
        _bind(s)
    return s


def _bind(s):
    """The library's calls on a state's buffers."""
    import __graft_entry__
    pkg = __graft_entry__.load_package()
    lib, op = pkg.lib(), s["op"]
    p = lambda t: C.c_void_p(t.data_ptr() if t is not None else None)  # noqa: E731
    if op in ("matmul", "quantize"):
        w = pkg.GPT2Int4W()
        w.codes, w.scales, w.group = s["codes"].data_ptr(), s["scales"].data_ptr(), s["group"]
        w.N, w.K = (s["n"], s["k"]) if op == "matmul" else s["w"].shape
        s["held"], ref = w, C.byref(w)
        if op == "matmul":
            s["calls"] = [(lib.gpt2_matmul_int4, (p(s["out"]), p(s["x"]), ref, p(s["bias"]), s["x"].shape[0], s["epi"], p(s["resid"])))]
        else:
            s["calls"] = [(lib.gpt2_quantize_int4, (ref, p(s["w"]))), (lib.gpt2_dequantize_int4, (p(s["out"]), ref))]
        return
    h = pkg.GPT2History()
    h.tokens, h.len, h.start = s["tokens"].data_ptr(), s["len"].data_ptr(), s["from"].data_ptr()
    h.nSeq, h.room = s["tokens"].shape
    s["history"], ref = h, C.byref(h)
    if op == "history":
        h.arrived = s["book"].data_ptr() + 8 * h.nSeq
        s["calls"] = [(lib.gpt2_history_step, (ref, p(s["parent"]), p(s["rows"]), p(s["ids"]), s["ids"].numel(), 0))]
        return
    s["arrived"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    h.arrived = s["arrived"].data_ptr()
    r = pkg.GPT2LogitsRules()
    r.history = C.pointer(h)
    for name in ("repetition", "presence", "frequency", "bias_start", "bias_token", "bias_value", "mask", "mask_row"):
        setattr(r, name, s[name].data_ptr() if s[name] is not None else None)
    r.ngram = s["ngram"]
    r.n_bias = s["bias_token"].numel() if s["bias_token"] is not None else 0
    r.n_masks = s["mask"].shape[0] if s["mask"] is not None else 0
    s["rules"] = r
    rows, v = s["logits"].shape
    s["calls"] = [(lib.gpt2_logits_adjust, (p(s["out"]), p(s["logits"]), v, rows, v, C.byref(r)))]


def run(s):
    op = s["op"]
    if op == "history":
        s["book"].copy_(s["first"])   # the lengths are put back, so that every pass has the same to do
    if own:
        for call, args in s["calls"]:
            call(*args)
    else:
        {"matmul": _matmul, "quantize": _quantize, "logits": _logits, "history": _history}[op](s)
    if op == "history":
        return {"tokens": s["tokens"], "len": s["len"], "from": s["from"]}
    return s["out"]


# ----------------------------------------------------------------------------- the plain forms
def _unpack(s):
    """Tiles as codes times scales [n][k], in fp32 (a code has 4 bits and a scale 11: exact)."""
    shift = 4 * torch.arange(4, device="cuda")[:, None] + 16 * torch.arange(2, device="cuda")
    q = ((s["codes"][..., None, None] >> shift) & 15) - 8
    q = q.permute(0, 3, 1, 4, 2, 5, 6).flatten(2).flatten(0, 1)   # [16 nt][kb][128], still by tile
    q = q.reshape(-1, s["codes"].shape[1] * 128).float()
    scale = s["scales"].permute(0, 2, 4, 1, 3).reshape(q.shape[0], -1).float()
    return (q * scale.repeat_interleave(s["group"], dim=1))[:s["n"], :s["k"]]


def _matmul(s):
    y = torch.matmul(s["x"].float(), _unpack(s).t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["epi"] == GELU:
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif s["epi"] == ADD:
        y = s["resid"].float() + y
    s["out"].copy_(y)


def _quantize(s):
    n, k = s["w"].shape
    groups, seven = _ceil(k, s["group"]), torch.tensor(7.0, device="cuda")
    w = torch.zeros((n, groups * s["group"]), device="cuda")
    w[:, :k] = s["w"].float()
    w = w.view(n, groups, s["group"])
    scale = (w.abs().amax(dim=2, keepdim=True) / seven).half().float()
    scale = torch.where(scale == 0, 1.0, scale)
    s["out"].copy_((torch.round(w / scale).clamp(-7, 7) * scale).view(n, -1)[:, :k])


def _logits(s):
    rows, v = s["logits"].shape
    at = torch.arange(s["tokens"].shape[1], device="cuda")
    there = at < s["len"][:, None]
    tokens = s["tokens"].long()
    count = torch.zeros((2, rows, v), device="cuda")
    count[0].scatter_add_(1, tokens, there.float())
    count[1].scatter_add_(1, tokens, (there & (at >= s["from"][:, None])).float())
    x = s["logits"].float()
    if s["bias_token"] is not None:
        row = torch.bucketize(torch.arange(s["bias_token"].numel(), device="cuda"), s["bias_start"][1:].contiguous().long(), right=True)
        x = x.index_put((row, s["bias_token"].long()), s["bias_value"], accumulate=True)
    rep = s["repetition"][:, None]
    x = torch.where(count[0] > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (s["frequency"][:, None] * count[1] + s["presence"][:, None] * (count[1] > 0))
    n = s["ngram"]
    if n:
        window = tokens.unfold(1, n, 1)                                     # [row][i][token i .. i + n - 1]
        tail = (s["len"][:, None] - (n - 1) + torch.arange(n - 1, device="cuda")).clamp(min=0).long()
        same = (window[:, :, :n - 1] == tokens.gather(1, tail)[:, None]).all(dim=2)
        same &= at[:window.shape[1]] + n <= s["len"][:, None]
        banned = torch.zeros((rows, v), device="cuda").scatter_add_(1, window[:, :, n - 1], same.float())
        x = torch.where(banned > 0, -math.inf, x)
    if s["mask"] is not None:
        word = s["mask"][s["mask_row"].clamp(min=0).long()]
        t = torch.arange(v, device="cuda")
        allowed = (word[:, t // 32] >> (t % 32) & 1).bool() | (s["mask_row"] < 0)[:, None]
        x = torch.where(allowed, x, -math.inf)
    s["out"].copy_(x)


def _history(s):
    seqs, room = s["tokens"].shape
    parent, new = s["parent"].long(), s["rows"][1:] - s["rows"][:-1]
    past, start = s["len"][parent], s["from"][parent]
    after = (past + new).clamp(max=room)
    at = torch.arange(room, device="cuda")
    i = (s["rows"][:-1, None] + at - past[:, None]).clamp(0, s["ids"].numel() - 1).long()
    full = torch.where(at < past[:, None], s["tokens"][parent], s["ids"][i])
    s["tokens"].copy_(torch.where(at < after[:, None], full, s["tokens"]))
    s["len"].copy_(after)
    s["from"].copy_(start)


# ----------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """From the definitions: products group by group, logits row by row."""
    op = case["op"]
    if op == "matmul":
        codes, scales, x, bias, resid = _matmul_inputs(case, seed)
        group, x = case["group"], x.double()
        y = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for j in range(scales.shape[1]):
            k = slice(group * j, min(group * (j + 1), case["k"]))
            y += torch.matmul(x[:, k], codes[:, k].double().t()) * scales[:, j].double()
        if bias is not None:
            y += bias.double()
        if case["epi"] == GELU:
            z = math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)
            y = y / (1.0 + torch.exp(-2.0 * z))
        return y + resid.double() if case["epi"] == ADD else y
    if op == "quantize":
        w = _quantize_inputs(case, seed).double()
        out = torch.empty_like(w)
        for k in range(0, case["k"], case["group"]):
            part = w[:, k:k + case["group"]]
            scale = (part.abs().max(dim=1).values / 7.0).half().double()   # the scale is a number of 16 bits
            scale[scale == 0] = 1.0
            out[:, k:k + case["group"]] = torch.round(part / scale[:, None]).clamp(-7, 7) * scale[:, None]
        return out
    if op == "history":
        return None   # whole numbers
    i = _logits_inputs(case, seed)
    out, n, v = i["logits"].double(), case["ngram"], case["vocab"]
    start = i["bias_start"].tolist() if i["bias_start"] is not None else None
    for r in range(case["rows"]):
        seq = i["tokens"][r, :int(i["len"][r])].long()
        if start:
            own_tokens = i["bias_token"][start[r]:start[r + 1]].long()
            out[r, own_tokens] += i["bias_value"][start[r]:start[r + 1]].double()
        seen = torch.unique(seq)
        rep = float(i["repetition"][r])
        out[r, seen] = torch.where(out[r, seen] > 0, out[r, seen] / rep, out[r, seen] * rep)
        token, times = torch.unique(seq[int(i["from"][r]):], return_counts=True)
        out[r, token] -= float(i["frequency"][r]) * times.double() + float(i["presence"][r])
        if n:
            t = seq.tolist()
            tail = t[len(t) - n + 1:]
            ban = [t[j + n - 1] for j in range(len(t) - n + 1) if t[j:j + n - 1] == tail]
            out[r, torch.tensor(ban, dtype=torch.long, device="cuda")] = -math.inf
        m = int(i["mask_row"][r]) if i["mask"] is not None else -1
        if m >= 0:
            bits = i["mask"][m][:, None] >> torch.arange(32, device="cuda") & 1
            out[r, bits.flatten()[:v] == 0] = -math.inf
    return out
