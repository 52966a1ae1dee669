"""What the paged cache's and the beam selection's calls refuse on the host: an error is recorded and nothing is launched
(these run without a GPU, where a launch would be an error of another kind)."""
import ctypes as C

import numpy as np
import pytest

ARG = 1000
ROWS = 0x1000   # an address that a refused call never reads


def cache(pkg, **kw):
    c = pkg.GPT2PagedKV()
    for i, n in enumerate(("codes", "scales", "open", "table", "len", "start", "slot", "refs", "status", "plan")):
        setattr(c, n, 0x10000 * (i + 1))
    c.nLayer, c.nHead, c.headDim, c.nPages, c.nSeq, c.maxPages = 2, 12, 64, 10, 4, 8
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(codes=None), dict(scales=0x10002), dict(codes=0x10004), dict(open=0x10008), dict(refs=0x10001), dict(table=None), dict(len=0x10002), dict(plan=None), dict(headDim=128),
              dict(nLayer=0), dict(nHead=0), dict(nHead=5000), dict(nPages=0), dict(nSeq=0), dict(nSeq=4097), dict(maxPages=0),
              dict(nSeq=4096, maxPages=1 << 25)]


@pytest.fixture(autouse=True)
def clean(L):
    L.gpt2_last_error()
    yield
    L.gpt2_last_error()


def calls(L, r):
    return [lambda: L.gpt2_pkv_reset(r), lambda: L.gpt2_pkv_status(r), lambda: L.gpt2_pkv_grow(r, ROWS, 4),
            lambda: L.gpt2_pkv_embed(ROWS, ROWS, ROWS, ROWS, r, ROWS, 4), lambda: L.gpt2_pkv_append(r, 0, ROWS, ROWS, 4),
            lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 1, ROWS, 1 << 40), lambda: L.gpt2_pkv_read(ROWS, r, 0, ROWS, ROWS, 4),
            lambda: L.gpt2_pkv_fork(r, ROWS), lambda: L.gpt2_pkv_compact(r)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches(pkg, L, bad):
    for call in calls(L, C.byref(cache(pkg, **bad))):
        call()
        assert L.gpt2_last_error() == ARG
    for call in calls(L, None):
        call()
        assert L.gpt2_last_error() == ARG


def test_bad_batches(pkg, L):
    r = C.byref(cache(pkg))
    for call in (lambda: L.gpt2_pkv_grow(r, None, 4), lambda: L.gpt2_pkv_grow(r, ROWS + 2, 4), lambda: L.gpt2_pkv_grow(r, ROWS, -1),
                 lambda: L.gpt2_pkv_grow(r, ROWS, (1 << 23) + 1),
                 lambda: L.gpt2_pkv_embed(ROWS + 2, ROWS, ROWS, ROWS, r, ROWS, 4), lambda: L.gpt2_pkv_embed(ROWS, ROWS, ROWS + 8, ROWS, r, ROWS, 4),
                 lambda: L.gpt2_pkv_embed(None, ROWS, ROWS, ROWS, r, ROWS, 4), lambda: L.gpt2_pkv_embed(ROWS, ROWS, ROWS, None, r, ROWS, 4),
                 lambda: L.gpt2_pkv_append(r, 2, ROWS, ROWS, 4), lambda: L.gpt2_pkv_append(r, -1, ROWS, ROWS, 4),
                 lambda: L.gpt2_pkv_append(r, 0, None, ROWS, 4), lambda: L.gpt2_pkv_append(r, 0, ROWS + 2, ROWS, 4),
                 lambda: L.gpt2_pkv_read(ROWS + 8, r, 0, ROWS, ROWS, 4), lambda: L.gpt2_pkv_read(ROWS, r, 0, ROWS, None, 4),
                 lambda: L.gpt2_pkv_read(ROWS, r, 5, ROWS, ROWS, 4), lambda: L.gpt2_pkv_fork(r, None), lambda: L.gpt2_pkv_fork(r, ROWS + 1),
                 lambda: L.gpt2_pkv_attn(None, ROWS, r, 0, ROWS, 4, 1, ROWS, 1 << 40), lambda: L.gpt2_pkv_attn(ROWS, ROWS + 2, r, 0, ROWS, 4, 1, ROWS, 1 << 40),
                 lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 0, ROWS, 1 << 40), lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 3, ROWS, 1 << 40),
                 lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 17, ROWS, 1 << 40), lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 1, None, 1 << 40),
                 lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 1, ROWS + 8, 1 << 40), lambda: L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 1, ROWS, 15)):
        call()
        assert L.gpt2_last_error() == ARG


def test_attention_workspace_is_checked(pkg, L):
    r = C.byref(cache(pkg, maxPages=4096))
    need = L.gpt2_pkv_attn_ws(r, 4)
    assert need > 16
    L.gpt2_pkv_attn(ROWS, ROWS, r, 0, ROWS, 4, 1, ROWS, need - 1)
    assert L.gpt2_last_error() == ARG
    assert L.gpt2_pkv_attn_ws(None, 4) == 16 and L.gpt2_pkv_attn_ws(r, 0) == 16


def test_empty_batches_do_nothing(pkg, L):
    r = C.byref(cache(pkg))
    L.gpt2_pkv_embed(None, None, None, None, r, ROWS, 0)
    L.gpt2_pkv_append(r, 0, None, ROWS, 0)
    L.gpt2_pkv_attn(None, None, r, 0, ROWS, 0, 1, None, 0)
    L.gpt2_pkv_read(None, r, 0, ROWS, None, 0)
    L.gpt2_beam_select(None, None, None, None, None, 0, None, None, 0, 0, 0, 0, None, 0)
    assert L.gpt2_last_error() in (0, 100)   # 100: no GPU here, as any call says


def test_alloc_sizes(pkg, L):
    c = pkg.GPT2PagedKV()
    for bad in ((0, 12, 10, 4, 100), (1, 0, 10, 4, 100), (1, 12, 0, 4, 100), (1, 12, 10, 0, 100), (1, 12, 10, 4097, 100), (1, 12, 10, 4, 0),
                (1, 12, 1 << 27, 4, 100), (16384, 4096, 1 << 26, 4, 100), (1 << 14, 1 << 11, 1 << 26, 1, 100), (1, 12, 10, 4096, 1 << 30)):
        assert L.gpt2_pkv_alloc(C.byref(c), *bad) != 0
        assert L.gpt2_last_error() == ARG
    assert L.gpt2_pkv_alloc(None, 1, 12, 10, 4, 100) != 0
    L.gpt2_pkv_free(None)
    L.gpt2_pkv_free(C.byref(c))


def test_beam_select_args(L):
    good = [ROWS, ROWS, ROWS, ROWS, ROWS, 100, ROWS, ROWS, 2, 4, 100, 99, ROWS, 1 << 40]
    need = L.gpt2_beam_select_ws(2, 4, 100)
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, None), (4, ROWS + 1), (5, 99), (6, None), (7, None), (8, -1), (8, 20000), (9, 0), (9, 17),
                 (10, 0), (10, 65537), (11, 100), (12, None), (12, ROWS + 4), (13, need - 1)):
        a = list(good)
        a[i] = v
        if (i, v) == (10, 65537):
            a[5] = 70000
        L.gpt2_beam_select(*a)
        assert L.gpt2_last_error() == ARG, (i, v)


def test_struct_layout(pkg, tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "l.c"
    names = [n for n, _ in pkg.GPT2PagedKV._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gpt2_pagedkv.h"\nint main(void) { printf("%zu", sizeof(GPT2PagedKV));'
                   + "".join(f'printf(" %zu", offsetof(GPT2PagedKV, {n}));' for n in names)
                   + 'printf(" %d %d %d %zu\\n", GPT2_PAGE_TOKENS, GPT2_PAGE_TILE, GPT2_BEAM_MAX, GPT2_PKV_PLAN_INTS(5, 7, 11)); return 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(pkg.GPT2PagedKV)] + [getattr(pkg.GPT2PagedKV, n).offset for n in names] + \
        [pkg.PAGE_TOKENS, pkg.PAGE_TILE, pkg.BEAM_MAX, pkg.pkv_plan_ints(5, 7, 11)]


def test_oracle_tiles_round_trip():
    from pagedkv_ref import quantize, tiles, untile
    x = np.arange(2 * 3 * 32 * 64, dtype=np.float32).reshape(2, 3, 32, 64)
    t = tiles(x)
    np.testing.assert_array_equal(untile(t), x)
    assert t[0, 1, 5 * 64 + 9] == x[0, 1, 5, 9] and t[1, 2, ((13 // 8) * 64 + 9) * 8 + 13 % 8] == x[1, 2, 13, 9]
    q, s = quantize(np.zeros((2, 1, 32, 64), np.float16))
    assert (q == 0).all() and (s == 1).all()
