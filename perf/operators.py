"""Operators whose speed is measured: what a program that serves several sequences has this library do beside
the model's matmuls (perf/cases.py has those).

Several sequences of GPT-2 (12 heads of 64) share one paged K/V cache: pages of 32 tokens, complete pages in INT8
with a scale for each page, head and K|V, the last, incomplete ("open") page of a sequence in fp16.  A program
appends the keys and values of new rows, attends over the cache, forks and reorders sequences as beam search
does, packs the pool's pages together, and chooses the beams' next tokens.

A tile is the 32 x 64 values of one page, head and K|V: K as [token][dim], V as [token / 8][dim][token % 8].
"""
import ctypes as C
import math
import random

import torch

own = False   # True: run() calls this library's kernels; False: the same in elementary torch operations

HEADS, HD, PAGE, LAYERS, VOCAB, CTX = 12, 64, 32, 12, 50257, 1024
E, TILE = HEADS * HD, PAGE * HD


def listed():
    return [
        # One prompt's four beams choose their next tokens: the smallest call, latency.
        {"name": "beam_1x4", "op": "beam", "groups": 1, "beams": 4, "vocab": VOCAB},
        # A batch of 64 prompts with 8 beams each: 51 MB of logits.
        {"name": "beam_64x8", "op": "beam", "groups": 64, "beams": 8, "vocab": VOCAB},
        # One sequence's next token over a nearly full context.
        {"name": "attn_decode_1_1000", "op": "attn", "seqs": 1, "cached": 999, "new": 1, "group": 1},
        # Eight prompts with eight beams each, which share all but their last pages.
        {"name": "attn_beams_8x8_900", "op": "attn", "seqs": 64, "cached": 900, "new": 1, "group": 8},
        # A batch of long, ragged contexts, one token each: streaming the cache.
        {"name": "attn_decode_16_16k", "op": "attn", "seqs": 16, "cached": 16384, "new": 1, "group": 1},
        # Prompts continued on top of cached contexts, a ragged batch: matrix work.
        {"name": "attn_rows_8_600", "op": "attn", "seqs": 8, "cached": 2000, "new": 600, "group": 1},
        # A decode step's rows of 48 sequences go into one layer's cache.
        {"name": "append_decode_48", "op": "append", "seqs": 48, "cached": 800, "new": 1},
        # Whole prompts go into one layer's cache.
        {"name": "append_prompts_48", "op": "append", "seqs": 48, "cached": 90, "new": 1000},
        # One prompt's four beams are reordered after a selection, all layers.
        {"name": "fork_4", "op": "fork", "seqs": 4, "beams": 4, "cached": 600},
        # 32 prompts with 8 beams each are reordered, all layers.
        {"name": "fork_256", "op": "fork", "seqs": 256, "beams": 8, "cached": 900},
        # A small pool, a quarter of it freed, is packed together.
        {"name": "compact_64", "op": "compact", "seqs": 3, "pages": 64, "live": 48},
        # A large pool, half of it freed, is packed together: hundreds of MB move.
        {"name": "compact_1500", "op": "compact", "seqs": 40, "pages": 1500, "live": 760},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["beam", "attn", "attn", "append", "fork", "compact"])
    if op == "beam":
        beams = _log_int(rng, 1, 16)
        return {"op": op, "groups": _log_int(rng, 1, 512 // beams), "beams": beams, "vocab": _log_int(rng, 100, VOCAB)}
    if op == "attn":
        kind = rng.choice(["decode", "decode", "beams", "rows"])
        if kind == "rows":
            seqs = _log_int(rng, 1, 8)
            return {"op": op, "seqs": seqs, "cached": _log_int(rng, 1, 2000), "new": _log_int(rng, 2, 600), "group": 1}
        seqs = _log_int(rng, 1, 64)
        group = rng.choice([2, 3, 4, 5, 8]) if kind == "beams" else 1
        seqs = max(1, seqs // group) * group
        return {"op": op, "seqs": seqs, "cached": _log_int(rng, 1, min(16384, 262144 // seqs)), "new": 1, "group": group}
    if op == "append":
        seqs = _log_int(rng, 1, 48)
        return {"op": op, "seqs": seqs, "cached": _log_int(rng, 1, CTX), "new": rng.choice([1, _log_int(rng, 2, 1000)])}
    if op == "fork":
        beams = rng.choice([2, 3, 4, 5, 8])
        return {"op": op, "seqs": beams * _log_int(rng, 1, 256 // beams), "beams": beams, "cached": _log_int(rng, 1, CTX)}
    pages = _log_int(rng, 16, 1500)
    live = max(2, int(pages * rng.uniform(0.3, 0.9)))
    return {"op": op, "seqs": rng.randint(1, min(40, live)), "pages": pages, "live": live}


# ----------------------------------------------------------------------------- sizes of a case
def _spread(n, hi, lo):
    """n lengths in [lo, hi], the first of them hi."""
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _lens(case):
    """Tokens cached before the call and new rows, by sequence."""
    n, hi, new = case["seqs"], case["cached"], case["new"]
    group = case.get("group", 1)
    cached = [c for c in _spread(n // group, hi, max(1, hi // 4)) for _ in range(group)]
    return cached, ([1] * n if new == 1 else _spread(n, new, max(1, new // 4))[::-1])


def _own_pages(cached):
    """Complete pages at its end that a beam has for itself."""
    return min(2, cached // PAGE)


def _parents(case):
    """Parents as a beam search's selection picks them, by sequence: a few beams win, the order is mixed."""
    rng, out = random.Random(case["seqs"] * 1000 + case["beams"]), []
    for g in range(case["seqs"] // case["beams"]):
        weights = [rng.random() ** 2 for _ in range(case["beams"])]
        out += [g * case["beams"] + b for b in rng.choices(range(case["beams"]), weights, k=case["beams"])]
    return out


def _fork_lens(case):
    return [c for c in _spread(case["seqs"] // case["beams"], case["cached"], max(1, case["cached"] // 2))
            for _ in range(case["beams"])]


def _moves(case):
    """The pool's live pages (a fixed choice), and how many of them lie past the place of the last one afterwards."""
    pages = sorted(random.Random(case["pages"] * 7 + case["live"]).sample(range(case["pages"]), case["live"]))
    return pages, sum(p >= case["live"] for p in pages)


def work(case):
    op = case["op"]
    if op == "beam":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (2 * case["vocab"] + 20), "flops": 4 * rows * case["vocab"]}
    tile = 2 * HEADS * (TILE + 4)   # a page's codes and scales, one layer
    if op == "attn":
        cached, new = _lens(case)
        pages = open_rows = pairs = 0
        for i, (c, n) in enumerate(zip(cached, new)):
            p = (c + n) // PAGE
            pages += p if i % case["group"] == 0 else min(p, _own_pages(c) + p - c // PAGE)
            open_rows += (c + n) % PAGE
            pairs += n * c + n * (n + 1) // 2
        return {"bytes": pages * tile + 4 * E * open_rows + 4 * E * sum(new), "flops": 4 * E * pairs}
    if op == "append":
        cached, new = _lens(case)
        made = sum((c + n) // PAGE - c // PAGE for c, n in zip(cached, new))
        opened = sum(min(n, (c + n) % PAGE) for c, n in zip(cached, new))
        kept = sum(c % PAGE for c, n in zip(cached, new) if (c + n) // PAGE > c // PAGE)
        back = sum(c + n - c // PAGE * PAGE for c, n in zip(cached, new))
        read = tile * made + 4 * E * sum((c + n) % PAGE for c, n in zip(cached, new))   # ... by the read back
        return {"bytes": 4 * E * (sum(new) + kept + opened + back) + tile * made + read, "flops": 4 * E * sum(new)}
    if op == "fork":
        lens, parents = _fork_lens(case), _parents(case)
        copied = sum(lens[p] % PAGE for i, p in enumerate(parents) if p in parents[:i])
        return {"bytes": 2 * LAYERS * 4 * E * copied + 8 * sum(n // PAGE for n in lens), "flops": 0}
    return {"bytes": 2 * LAYERS * tile * _moves(case)[1] + 8 * case["pages"], "flops": 0}


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


def _rows(n, g):
    """Rows of q | k | v: scores q.k / 8 of a spread of about 1.5, values of 0.6, some channels wider."""
    x = _normal((n, 3, E), 1.0, g)
    x[:, :2] *= 1.2
    x[:, 2] *= 0.6
    x[:, 1:, ::HD] *= 3.0
    return x.reshape(n, 3 * E).half()


def _cache(layers, pages, seqs, max_pages, g):
    """A cache whose pool holds what quantised normal keys and values look like; its bookkeeping is empty."""
    codes = (_normal((layers, pages, 2, HEADS, TILE), 35.0, g)).round_().clamp_(-127, 127).to(torch.int8)
    scales = 0.02 + 0.02 * torch.rand((layers, pages, 2, HEADS), generator=g, device="cuda")
    scales[:, :, 1] *= 0.5
    book = torch.zeros(seqs * max_pages + 3 * seqs + pages + 4, dtype=torch.int32, device="cuda")
    at, c = 0, {"codes": codes, "scales": scales, "book": book}
    c["open"] = _normal((layers, seqs, 2, HEADS, TILE), 1.0, g).half()
    for name, shape in (("table", (seqs, max_pages)), ("len", (seqs,)), ("start", (seqs,)), ("slot", (seqs,)),
                        ("refs", (pages,)), ("status", (4,))):
        n = math.prod(shape)
        c[name] = book[at:at + n].view(shape)
        at += n
    c["slot"].copy_(torch.randperm(seqs, generator=g, device="cuda"))
    return c


def _filled(case, seed):
    """The case's cache before the call, and its other inputs, from the seed; the sequences' pages lie anywhere
    in the pool."""
    op, g = case["op"], _gen(seed)
    spare = 3
    if op in ("attn", "append"):
        cached, new = _lens(case)
        after = [c + n for c, n in zip(cached, new)]
        have = cached if op == "append" else after
        max_pages = max(after) // PAGE + 1
        group = case.get("group", 1)
        tables, used = [], 0
        for i, n in enumerate(have):
            p = n // PAGE
            shared = 0 if i % group == 0 else max(0, cached[i] // PAGE - _own_pages(cached[i]))
            tables.append((tables[i - i % group][:shared] if shared else []) + list(range(used, used + p - shared)))
            used += p - shared
        pages = sum(a // PAGE for a in after) + spare if op == "append" else used + spare
        c = _cache(1, pages, case["seqs"], max_pages, g)
        c["len"].copy_(_ints(have))
        c["start"].copy_(_ints(cached))
        c["rows"] = _ints(_offsets(new))
        c["qkv"] = _rows(sum(new), g)
    elif op == "fork":
        have = _fork_lens(case)
        max_pages = CTX // PAGE
        tables, used = [], 0
        for i, n in enumerate(have):
            shared = 0 if i % case["beams"] == 0 else max(0, n // PAGE - _own_pages(n))
            tables.append((tables[i - i % case["beams"]][:shared] if shared else []) + list(range(used, used + n // PAGE - shared)))
            used += n // PAGE - shared
        pages = used + spare
        c = _cache(LAYERS, 1, case["seqs"], max_pages, g)   # only open pages move; one page's codes stand for the pool
        book = torch.zeros(c["book"].numel() + pages - 1, dtype=torch.int32, device="cuda")
        at = case["seqs"] * max_pages
        for name in ("len", "start", "slot"):
            v = book[at:at + case["seqs"]]
            v.copy_(c[name])
            c[name], at = v, at + case["seqs"]
        c["table"], c["refs"], c["status"] = book[:case["seqs"] * max_pages].view(case["seqs"], max_pages), book[at:at + pages], book[at + pages:]
        c["book"] = book
        c["len"].copy_(_ints(have))
        c["start"].copy_(_ints(have))
        c["parent"] = _ints(_parents(case))
    else:
        where, _ = _moves(case)
        rng = random.Random(case["live"])
        rng.shuffle(where)
        cuts = sorted(rng.sample(range(1, case["live"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
        tables = [where[a:b] for a, b in zip([0] + cuts, cuts + [case["live"]])]
        if case["seqs"] > 1 and len(tables[0]) > 1:
            tables[1] = tables[0][:1] + tables[1]   # a shared page
        max_pages = max(len(t) for t in tables) + 1
        c = _cache(LAYERS, case["pages"], case["seqs"], max_pages, g)
        c["open"] = c["open"][:, :, :, :, :0]
        c["len"].copy_(_ints([PAGE * len(t) for t in tables]))
        c["start"].copy_(c["len"])
    pages = c["refs"].numel()
    if op in ("attn", "append", "fork"):
        place = torch.randperm(pages, generator=g, device="cuda").tolist()
        tables = [[place[p] for p in t] for t in tables]
    c["table"].copy_(_ints([t + [0] * (c["table"].shape[1] - len(t)) for t in tables]))
    c["refs"].index_add_(0, _ints([p for t in tables for p in t]), _ints([1] * sum(map(len, tables))))
    c["first"] = c["book"].clone()   # the bookkeeping before the call
    return c


def _beam_inputs(case, seed):
    """Logits as a language model gives them (a few tokens stand out, the beams of a prompt are alike), some
    masked to -inf, cumulative scores, some beams done."""
    g = _gen(seed)
    n, b, v = case["groups"], case["beams"], case["vocab"]
    x = _normal((n, 1, v), 2.0, g) + _normal((n, b, v), 0.7, g) - 30.0
    x += 6.0 * (torch.rand((n, 1, v), generator=g, device="cuda") < 20.0 / v)
    x.masked_fill_(torch.rand((n, b, v), generator=g, device="cuda") < 0.02, -math.inf)
    score = -torch.rand((n, b), generator=g, device="cuda") * 6.0 - 10.0
    done = (torch.rand((n, b), generator=g, device="cuda") < 0.1).int()
    return x.half().view(n * b, v), score.view(-1), done.view(-1), v - 1


def prepare(case, seed):
    op = case["op"]
    if op == "beam":
        logits, score, done, eos = _beam_inputs(case, seed)
        s = {"op": op, "logits": logits, "score": score, "done": done, "eos": eos, "beams": case["beams"]}
        n = score.numel()
        s["out"] = {"token": torch.empty(n, dtype=torch.int32, device="cuda"), "parent": torch.empty(n, dtype=torch.int32, device="cuda"),
                    "score": torch.empty(n, device="cuda"), "done": torch.empty(n, dtype=torch.int32, device="cuda")}
    else:
        s = _filled(case, seed)
        s["op"] = op
        if op in ("attn", "append"):
            cached, new = _lens(case)
            after = [c + n for c, n in zip(cached, new)]
            s["total"], s["most"], s["group"] = sum(new), max(new), case.get("group", 1)
            s["att"] = torch.zeros((s["total"], E), dtype=torch.float16, device="cuda")
        if op == "append":
            # every token of the pages that the call touches is read back
            back = [c // PAGE * PAGE for c in cached]
            s["made"] = sum(a // PAGE - c // PAGE for a, c in zip(after, cached))
            s["touched"] = sum((a - 1) // PAGE - c // PAGE + 1 for a, c in zip(after, cached))
            s["back_pos"], s["back_rows"] = _ints(back), _ints(_offsets([a - b for a, b in zip(after, back)]))
            s["back"] = torch.empty((sum(after) - sum(back), 2 * E), dtype=torch.float16, device="cuda")
        if op == "fork":
            parents = _parents(case)
            s["extra"] = sum(p in parents[:i] for i, p in enumerate(parents))
        if op == "compact":
            s["moves"] = _moves(case)[1]
    if own:
        _bind(s)
    return s


def _bind(s):
    """The library's calls on a state's buffers."""
    import __graft_entry__
    pkg = __graft_entry__.load_package()
    lib, op = pkg.lib(), s["op"]
    p = lambda t: C.c_void_p(t.data_ptr() if t is not None else None)  # noqa: E731
    if op == "beam":
        groups, v = s["score"].numel() // s["beams"], s["logits"].shape[1]
        s["ws"] = torch.empty(lib.gpt2_beam_select_ws(groups, s["beams"], v), dtype=torch.uint8, device="cuda")
        o = s["out"]
        s["calls"] = [(lib.gpt2_beam_select, (p(o["token"]), p(o["parent"]), p(o["score"]), p(o["done"]), p(s["logits"]), v, p(s["score"]),
                                              p(s["done"]), groups, s["beams"], v, s["eos"], p(s["ws"]), s["ws"].numel()))]
        return
    c = pkg.GPT2PagedKV()
    c.nLayer, c.nHead, c.headDim, c.nPages = s["codes"].shape[0], HEADS, HD, s["refs"].numel()
    c.nSeq, c.maxPages = s["table"].shape
    s["plan"] = torch.zeros(pkg.pkv_plan_ints(c.nSeq, c.maxPages, c.nPages), dtype=torch.int32, device="cuda")
    for name in ("codes", "scales", "open", "table", "len", "start", "slot", "refs", "status", "plan"):
        setattr(c, name, s[name].data_ptr() or s["codes"].data_ptr())   # a compaction's state has no open pages, and touches none
    s["cache"], ref = c, C.byref(c)
    if op == "attn":
        s["ws"] = torch.empty(lib.gpt2_pkv_attn_ws(ref, s["total"]), dtype=torch.uint8, device="cuda")
        s["calls"] = [(lib.gpt2_pkv_attn, (p(s["att"]), p(s["qkv"]), ref, 0, p(s["rows"]), s["total"], s["group"], p(s["ws"]), s["ws"].numel()))]
    elif op == "append":
        s["calls"] = [(lib.gpt2_pkv_grow, (ref, p(s["rows"]), s["total"])),
                      (lib.gpt2_pkv_append, (ref, 0, p(s["qkv"]), p(s["rows"]), s["total"])),
                      (lib.gpt2_pkv_read, (p(s["back"]), ref, 0, p(s["back_rows"]), p(s["back_pos"]), s["back"].shape[0]))]
    elif op == "fork":
        s["calls"] = [(lib.gpt2_pkv_fork, (ref, p(s["parent"])))]
    else:
        s["calls"] = [(lib.gpt2_pkv_compact, (ref,))]


def run(s):
    op = s["op"]
    if op not in ("beam", "attn"):
        s["book"].copy_(s["first"])   # the bookkeeping is put back, so that every pass has the same to do
    if own:
        for call, args in s["calls"]:
            call(*args)
    else:
        {"beam": _beam, "attn": _attn, "append": _append, "fork": _fork, "compact": _compact}[op](s)
    if op == "beam":
        return s["out"]
    if op == "attn":
        return s["att"]
    out = {name: s[name] for name in ("table", "len", "start", "slot", "refs")}
    if op == "append":
        out |= {"open": s["open"], "scales": s["scales"], "back": s["back"]}
    elif op == "fork":
        out["open"] = s["open"]
    else:
        out |= {"codes": s["codes"], "scales": s["scales"]}   # whole pages, moved as they are
    return out


# ----------------------------------------------------------------------------- the plain forms
def _beam(s):
    b, v = s["beams"], s["logits"].shape[1]
    score_in, done = s["score"].view(-1, b), s["done"].view(-1, b) != 0
    x = torch.nan_to_num(s["logits"], nan=-math.inf, posinf=65504.0, neginf=-math.inf)
    # a row's best b logits, the lower token first among equal ones: keys without ties
    bits = (x + 0.0).view(torch.int16).int()
    order = torch.where(bits < 0, ~bits & 0x7FFF, bits | 0x8000)
    key = order * 65536 + (65535 - torch.arange(v, device=x.device))   # wraps into the sign for order >= 0x8000
    top = torch.topk(key ^ -0x80000000, min(b, v), dim=1).values ^ -0x80000000
    token = (65535 - (top & 65535)).view(-1, b, min(b, v))
    x = x.double()
    m = x.amax(dim=1, keepdim=True)
    total = torch.exp(x - m).sum(dim=1, keepdim=True)
    score = score_in.double()[..., None] + ((x.gather(1, token.view(x.shape[0], -1).long()) - m) - torch.log(total)).view_as(token)
    score = torch.nan_to_num(score, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    # a beam that is done goes on with the end token alone, its score as it was
    first = torch.arange(token.shape[2], device=x.device) == 0
    token = torch.where(done[..., None], s["eos"], token)
    score = torch.where(done[..., None], torch.where(first, score_in.double()[..., None], -math.inf), score)
    absent = (done[..., None] & ~first).flatten(1)
    at = torch.sort(absent, dim=1, stable=True).indices
    best, i = torch.sort(score.flatten(1).gather(1, at), dim=1, descending=True, stable=True)
    at = at.gather(1, i[:, :b])
    beam = at // token.shape[2]
    out = s["out"]
    token = token.flatten(1).gather(1, at)
    out["token"].copy_(token.flatten())
    out["parent"].copy_((beam + b * torch.arange(beam.shape[0], device=x.device)[:, None]).flatten())
    out["score"].copy_(best[:, :b].flatten())
    out["done"].copy_((done.gather(1, beam) | (token == s["eos"])).flatten())


def _unpack(tiles, values):
    """Tiles [..., K|V, head, 2048] as [..., K|V, head, token, dim]."""
    k, v = tiles.unbind(-3)
    v = v.unflatten(-1, (PAGE // 8, HD, 8)).transpose(-1, -2).flatten(-3, -2)
    return torch.stack((k.unflatten(-1, (PAGE, HD)), v), dim=-4).to(values)


def _pack(x):
    """[..., K|V, head, token, dim] as tiles."""
    k, v = x.unbind(-4)
    v = v.unflatten(-2, (PAGE // 8, 8)).transpose(-1, -2).flatten(-3)
    return torch.stack((k.flatten(-2), v), dim=-3)


def _attn(s):
    n = s["table"].shape[0]
    full = s["len"] // PAGE
    pages = s["table"].shape[1]
    is_open = torch.arange(pages, device="cuda") == full[:, None]
    tiles = _unpack(s["codes"][0][s["table"].long()], torch.float32)   # [seq, page, K|V, head, token, dim]
    tiles *= s["scales"][0][s["table"].long()][..., None, None]
    last = _unpack(s["open"][0][s["slot"].long()], torch.float32)
    tiles = torch.where(is_open[:, :, None, None, None, None], last[:, None], tiles)
    k, v = tiles.permute(2, 0, 3, 1, 4, 5).reshape(2, n, HEADS, pages * PAGE, HD)
    i = torch.arange(s["most"], device="cuda")
    row = torch.clamp(s["rows"][:-1, None] + i, max=s["total"] - 1).long()
    q = s["qkv"][:, :E].float()[row].view(n, s["most"], HEADS, HD).transpose(1, 2)
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(HD)
    at = torch.arange(pages * PAGE, device="cuda")
    scores.masked_fill_((at > (s["start"][:, None] + i)[..., None])[:, None], -math.inf)
    scores -= scores.amax(dim=-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores, v).transpose(1, 2).reshape(n, s["most"], E)
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), s["rows"].diff(), output_size=s["total"])
    s["att"].copy_(out[seq, torch.arange(s["total"], device="cuda") - s["rows"][seq]])


def _append(s):
    n = s["table"].shape[0]
    seqs = torch.arange(n, device="cuda")
    s["start"].copy_(s["len"])
    s["len"] += s["rows"].diff()
    # the lowest free pages, to the sequences in order
    had, need = s["start"] // PAGE, s["len"] // PAGE - s["start"] // PAGE
    seq = torch.repeat_interleave(seqs, need, output_size=s["made"])
    j = torch.arange(s["made"], device="cuda") - (need.cumsum(0) - need)[seq]
    page = torch.sort(s["refs"] != 0, stable=True).indices[:s["made"]]
    s["table"][seq, had[seq] + j] = page.int()
    s["refs"][page] = 1
    # the tiles of every touched page, from the open page and the new rows
    count = (s["len"] - 1) // PAGE - had + 1
    seq = torch.repeat_interleave(seqs, count, output_size=s["touched"])
    j = had[seq] + torch.arange(s["touched"], device="cuda") - (count.cumsum(0) - count)[seq]
    pos = j[:, None] * PAGE + torch.arange(PAGE, device="cuda")
    row = torch.clamp(s["rows"][:-1][seq, None] + pos - s["start"][seq, None], 0, s["total"] - 1)
    kv = torch.nan_to_num(s["qkv"][:, E:], nan=0.0, posinf=65504.0, neginf=-65504.0)
    fresh = kv[row.long()].view(-1, PAGE, 2, HEADS, HD).permute(0, 2, 3, 1, 4)
    kept = _unpack(s["open"][0][s["slot"][seq].long()], torch.float16)
    is_new = (pos >= s["start"][seq, None]) & (pos < s["len"][seq, None])
    x = torch.where(is_new[:, None, None, :, None], fresh, kept)
    whole = torch.sort((j + 1) * PAGE > s["len"][seq], stable=True).indices   # complete pages first
    done, left = whole[:s["made"]], whole[s["made"]:]
    full = x[done].float()
    peak = full.abs().amax(dim=(-1, -2))
    scale = torch.where(peak == 0, 1.0, peak / 127.0)
    page = s["table"][seq[done], j[done]].long()
    s["codes"][0][page] = _pack(torch.clamp(torch.round(full / scale[..., None, None]), -127, 127)).to(torch.int8)
    s["scales"][0][page] = scale
    stale = _unpack(s["open"][0][s["slot"][seq[left]].long()], torch.float16)
    s["open"][0][s["slot"][seq[left]].long()] = _pack(torch.where(is_new[left][:, None, None, :, None], x[left], stale))
    # the touched pages' tokens as the cache holds them
    total = s["back"].shape[0]
    seq = torch.repeat_interleave(seqs, s["back_rows"].diff(), output_size=total)
    pos = s["back_pos"][seq] + torch.arange(total, device="cuda") - s["back_rows"][seq]
    page, tok = s["table"][seq, pos // PAGE].long(), (pos % PAGE).long()
    k_at, v_at = tok[:, None] * HD + torch.arange(HD, device="cuda"), ((tok // 8)[:, None] * HD + torch.arange(HD, device="cuda")) * 8 + (tok % 8)[:, None]
    at = torch.stack((k_at, v_at), dim=1)[:, :, None].expand(-1, -1, HEADS, -1)
    held = s["codes"][0][page[:, None, None, None], torch.arange(2, device="cuda")[:, None, None], torch.arange(HEADS, device="cuda")[:, None], at]
    held = held.float() * s["scales"][0][page][..., None]
    opened = s["open"][0][s["slot"][seq].long()[:, None, None, None], torch.arange(2, device="cuda")[:, None, None], torch.arange(HEADS, device="cuda")[:, None], at]
    in_open = pos >= s["len"][seq] // PAGE * PAGE
    s["back"].copy_(torch.where(in_open[:, None, None, None], opened.float(), held).flatten(1))


def _fork(s):
    n, pages = s["table"].shape
    seqs, parent = torch.arange(n, device="cuda"), s["parent"].long()
    children = torch.zeros_like(s["len"]).index_add_(0, parent, torch.ones_like(s["len"]))
    heir = torch.full_like(seqs, n).scatter_reduce_(0, parent, seqs, "amin")[parent] == seqs   # the first child keeps the open page
    rank = (~heir).cumsum(0) - 1
    unheard = torch.sort(children != 0, stable=True).indices   # sequences that go, in order
    slot = torch.where(heir, s["slot"][parent], s["slot"][unheard[torch.clamp(rank, min=0)]])
    listed_ = torch.arange(pages, device="cuda") < (s["len"] // PAGE)[:, None]
    s["refs"].index_add_(0, torch.where(listed_, s["table"], 0).flatten(), ((children - 1)[:, None] * listed_).flatten().int())
    length = s["len"][parent]
    extra = torch.sort(heir, stable=True).indices[:s["extra"]]
    source, target = s["slot"][parent[extra]].long(), slot[extra].long()
    tok = torch.arange(PAGE, device="cuda")
    used = tok < (length[extra] % PAGE)[:, None]
    at = torch.arange(TILE, device="cuda")
    mask = torch.stack((used[:, at // HD], used[:, at // (8 * HD) * 8 + at % 8]), dim=1)[None, :, :, None]
    s["open"][:, target] = torch.where(mask, s["open"][:, source], s["open"][:, target])
    listed_ = torch.arange(pages, device="cuda") < (length // PAGE)[:, None]
    s["table"].copy_(torch.where(listed_, s["table"][parent], s["table"]))
    s["slot"].copy_(slot)
    s["len"].copy_(length)
    s["start"].copy_(length)


def _compact(s):
    pages = s["refs"].numel()
    ids = torch.arange(pages, device="cuda")
    live = s["refs"] != 0
    n = live.sum()
    hole = torch.sort(live | (ids >= n), stable=True).indices[:s["moves"]]
    mover = torch.sort(~(live & (ids >= n)), stable=True).indices[:s["moves"]]
    to = ids.clone()
    to[mover] = hole
    s["codes"][:, hole] = s["codes"][:, mover]
    s["scales"][:, hole] = s["scales"][:, mover]
    s["refs"][hole] = s["refs"][mover]
    s["refs"][mover] = 0
    listed_ = torch.arange(s["table"].shape[1], device="cuda") < (s["len"] // PAGE)[:, None]
    s["table"].copy_(torch.where(listed_, to[s["table"].long()].int(), s["table"]))


# ----------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """From the definitions, sequence by sequence."""
    op = case["op"]
    if op == "beam":
        logits, score, done, eos = _beam_inputs(case, seed)
        best = []
        for g in range(case["groups"]):
            cand = []
            for b in range(g * case["beams"], (g + 1) * case["beams"]):
                if done[b]:
                    cand.append(score[b:b + 1].double())
                else:
                    cand.append(score[b].double() + torch.log_softmax(logits[b].double(), dim=0))
            best.append(torch.sort(torch.cat(cand), descending=True).values[:case["beams"]])
        return {"token": None, "parent": None, "score": torch.cat(best), "done": None}
    if op not in ("attn", "append"):
        return None   # pages are copied as they are
    c = _filled(case, seed)
    cached, new = _lens(case)
    rows = _offsets(new)

    def history(i, upto):
        """Keys and values [2, HEADS, upto, HD] of sequence i as the cache holds them before the call."""
        parts = []
        for j in range(upto // PAGE):
            page = int(c["table"][i, j])
            parts.append(_tile64(c["codes"][0, page].double() * c["scales"][0, page].double()[..., None]))
        if upto % PAGE:
            parts.append(_tile64(c["open"][0, int(c["slot"][i])].double())[:, :, :upto % PAGE])
        return torch.cat(parts, dim=2)

    if op == "attn":
        out = torch.empty((rows[-1], E), dtype=torch.float64, device="cuda")
        for i, n in enumerate(new):
            k, v = history(i, cached[i] + n)
            q = c["qkv"][rows[i]:rows[i + 1], :E].double().view(n, HEADS, HD).transpose(0, 1)
            scores = torch.matmul(q, k.transpose(1, 2)) / 8.0
            later = torch.arange(cached[i] + n, device="cuda")[None] > (cached[i] + torch.arange(n, device="cuda"))[:, None]
            out[rows[i]:rows[i + 1]] = torch.matmul(torch.softmax(scores.masked_fill(later, -math.inf), dim=-1), v).transpose(0, 1).reshape(n, E)
        return out
    back = []
    for i, n in enumerate(new):
        start, end = cached[i], cached[i] + n
        x = c["qkv"][rows[i]:rows[i + 1], E:].double().view(n, 2, HEADS, HD).permute(1, 2, 0, 3)
        if start % PAGE:
            x = torch.cat((_tile64(c["open"][0, int(c["slot"][i])].double())[:, :, :start % PAGE], x), dim=2)
        whole = (end // PAGE - start // PAGE) * PAGE
        full = x[:, :, :whole].unflatten(2, (-1, PAGE))
        # the scale is a number of 32 bits, and the code is that of the quotient in 32 bits
        scale = (full.abs().amax(dim=(3, 4), keepdim=True).float() / 127.0)
        scale = torch.where(scale == 0, 1.0, scale)
        held = torch.round((full.float() / scale)).clamp(-127, 127).double() * scale.double()
        back.append(torch.cat((held.flatten(2, 3), x[:, :, whole:]), dim=2).permute(2, 0, 1, 3).reshape(-1, 2 * E))
    return {"table": None, "len": None, "start": None, "slot": None, "refs": None, "open": None, "scales": None, "back": torch.cat(back)}


def _tile64(t):
    """[K|V, HEADS, 2048] as [K|V, HEADS, token, dim]."""
    return torch.stack((t[0].view(HEADS, PAGE, HD), t[1].view(HEADS, PAGE // 8, HD, 8).transpose(2, 3).reshape(HEADS, PAGE, HD)))
