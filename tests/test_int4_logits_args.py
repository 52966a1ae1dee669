"""What the calls on 4-bit weights, logits and histories refuse on the host: an error is recorded and nothing is launched (these run without a
GPU, where a launch would be an error of another kind); the structs' layouts; the oracle's own round trip."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from int4_ref import Histories, adjust, dequantized, mask_words, pack, quantize, unpack

ARG = 1000
AT = 0x10000   # an address that a refused call never reads


@pytest.fixture(autouse=True)
def clean(L):
    L.gpt2_last_error()
    yield
    L.gpt2_last_error()


def refused(L, call):
    call()
    assert L.gpt2_last_error() == ARG


def weights(pkg, **kw):
    w = pkg.GPT2Int4W(AT, AT, 32, 256, 64, None)
    for k, v in kw.items():
        setattr(w, k, v)
    return C.byref(w)


@pytest.mark.parametrize("bad", [dict(codes=None), dict(scales=None), dict(codes=AT + 8), dict(scales=AT + 2), dict(N=0), dict(K=0), dict(N=-1), dict(group=0), dict(group=16),
                                 dict(group=256), dict(group=96), dict(N=1 << 30, K=1 << 20)], ids=str)
def test_bad_weights(pkg, L, bad):
    w = weights(pkg, **bad)
    for call in (lambda: L.gpt2_quantize_int4(w, AT), lambda: L.gpt2_dequantize_int4(AT, w), lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, 0, None)):
        refused(L, call)


def test_bad_calls(pkg, L):
    w = weights(pkg)
    for call in (lambda: L.gpt2_quantize_int4(None, AT), lambda: L.gpt2_quantize_int4(w, None), lambda: L.gpt2_quantize_int4(w, AT + 1),
                 lambda: L.gpt2_dequantize_int4(None, w), lambda: L.gpt2_dequantize_int4(AT + 1, w), lambda: L.gpt2_dequantize_int4(AT, None),
                 lambda: L.gpt2_matmul_int4(AT, AT, None, None, 1, 0, None), lambda: L.gpt2_matmul_int4(None, AT, w, None, 1, 0, None),
                 lambda: L.gpt2_matmul_int4(AT, None, w, None, 1, 0, None), lambda: L.gpt2_matmul_int4(AT + 1, AT, w, None, 1, 0, None),
                 lambda: L.gpt2_matmul_int4(AT, AT + 1, w, None, 1, 0, None), lambda: L.gpt2_matmul_int4(AT, AT, w, AT + 1, 1, 0, None),
                 lambda: L.gpt2_matmul_int4(AT, AT, w, None, -1, 0, None), lambda: L.gpt2_matmul_int4(AT, AT, w, None, (1 << 21) + 1, 0, None),
                 lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, 3, None), lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, -1, None),
                 lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, 2, None), lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, 2, AT + 1),
                 lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, 0, AT), lambda: L.gpt2_matmul_int4(AT, AT, w, None, 1, 1, AT)):
        refused(L, call)
    L.gpt2_matmul_int4(None, None, w, None, 0, 0, None)   # no rows: nothing to do
    assert L.gpt2_last_error() in (0, 100)


def test_sizes(pkg, L):
    assert L.gpt2_int4_code_bytes(16, 128) == 1024 and L.gpt2_int4_code_bytes(17, 129) == 4096
    assert L.gpt2_int4_code_bytes(0, 5) == L.gpt2_int4_code_bytes(5, 0) == 0
    assert [L.gpt2_int4_scale_count(16, 128, g) for g in (32, 64, 128, 16)] == [64, 32, 16, 0]
    assert L.gpt2_int4_code_bytes(1 << 20, 1 << 20) == 1 << 39
    w = pkg.GPT2Int4W()
    for bad in ((0, 5, 32), (5, 0, 32), (5, 5, 48), (1 << 30, 1 << 20, 32)):
        assert L.gpt2_int4_alloc(C.byref(w), *bad) != 0
        assert L.gpt2_last_error() == ARG
    assert L.gpt2_int4_alloc(None, 16, 16, 32) != 0
    L.gpt2_int4_free(None)
    L.gpt2_int4_free(C.byref(w))


def history(pkg, **kw):
    h = pkg.GPT2History(AT, AT, AT, AT, 8, 100, None)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


BAD_HISTORIES = [dict(tokens=None), dict(len=None), dict(start=None), dict(arrived=None), dict(tokens=AT + 2), dict(arrived=AT + 1), dict(nSeq=0), dict(nSeq=4097), dict(room=0),
                 dict(room=(1 << 24) + 1)]


@pytest.mark.parametrize("bad", BAD_HISTORIES, ids=str)
def test_bad_histories(pkg, L, bad):
    h = history(pkg, **bad)
    r = pkg.GPT2LogitsRules(history=C.pointer(h))
    for call in (lambda: L.gpt2_history_reset(C.byref(h)), lambda: L.gpt2_history_step(C.byref(h), None, None, None, 0, 0),
                 lambda: L.gpt2_logits_adjust(AT, AT, 100, 4, 100, C.byref(r))):
        refused(L, call)


def test_bad_steps(pkg, L):
    h = C.byref(history(pkg))
    for call in (lambda: L.gpt2_history_step(None, None, None, None, 0, 0), lambda: L.gpt2_history_step(h, AT + 2, None, None, 0, 0),
                 lambda: L.gpt2_history_step(h, None, AT, None, 4, 0), lambda: L.gpt2_history_step(h, None, AT, AT, -1, 0),
                 lambda: L.gpt2_history_step(h, None, AT + 1, AT, 4, 0), lambda: L.gpt2_history_step(h, None, AT, AT + 2, 4, 0), lambda: L.gpt2_history_reset(None)):
        refused(L, call)
    x = pkg.GPT2History()
    for bad in ((0, 10), (4097, 10), (4, 0), (4, (1 << 24) + 1)):
        assert L.gpt2_history_alloc(C.byref(x), *bad) != 0
        assert L.gpt2_last_error() == ARG
    assert L.gpt2_history_alloc(None, 4, 10) != 0
    L.gpt2_history_free(None)
    L.gpt2_history_free(C.byref(x))


def test_bad_logits(pkg, L):
    h = history(pkg)

    def rules(**kw):
        r = pkg.GPT2LogitsRules(history=C.pointer(h))
        for k, v in kw.items():
            setattr(r, k, v)
        return C.byref(r)
    ok = rules()
    for a in ((None, AT, 100, 4, 100, ok), (AT, None, 100, 4, 100, ok), (AT + 1, AT, 100, 4, 100, ok), (AT, AT + 1, 100, 4, 100, ok), (AT, AT, 99, 4, 100, ok),
              (AT, AT, 100, -1, 100, ok), (AT, AT, 100, 65536, 100, ok), (AT, AT, 100, 4, 0, ok), (AT, AT, 1 << 25, 4, (1 << 24) + 1, ok), (AT, AT, 100, 4, 100, None),
              (AT, AT, 100, 9, 100, ok), (AT, AT, 100, 4, 100, rules(ngram=-1)), (AT, AT, 100, 4, 100, rules(n_bias=-1, bias_start=AT)),
              (AT, AT, 100, 4, 100, rules(n_bias=3, bias_start=AT)), (AT, AT, 100, 4, 100, rules(n_bias=3, bias_start=AT, bias_token=AT)),
              (AT, AT, 100, 4, 100, rules(mask=AT, n_masks=-1)), (AT, AT, 100, 4, 100, rules(mask=AT + 2, n_masks=1)), (AT, AT, 100, 4, 100, rules(repetition=AT + 1)),
              (AT, AT, 100, 4, 100, rules(mask=AT, n_masks=1, mask_row=AT + 3))):
        refused(L, lambda: L.gpt2_logits_adjust(*a))
    L.gpt2_logits_adjust(None, None, 0, 0, 0, None)   # no rows: nothing to do
    assert L.gpt2_last_error() in (0, 100)


def test_struct_layouts(pkg, tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "l.c"
    structs = ("GPT2Int4W", "GPT2History", "GPT2LogitsRules")
    body, want = "", []
    for s in structs:
        t = getattr(pkg, s)
        body += f'printf("%zu ", sizeof({s}));' + "".join(f'printf("%zu ", offsetof({s}, {n}));' for n, _ in t._fields_)
        want += [C.sizeof(t)] + [getattr(t, n).offset for n, _ in t._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gpt2_int4.h"\n#include "gpt2_logits.h"\nint main(void) { ' + body
                   + 'printf("%d %d %d", GPT2_EPI_NONE, GPT2_EPI_GELU, GPT2_EPI_ADD); return 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want + [pkg.EPI_NONE, pkg.EPI_GELU, pkg.EPI_ADD]


def test_oracle_weights():
    rng = np.random.default_rng(1)
    w = rng.standard_normal((37, 300)).astype(np.float16)
    for group in (32, 64, 128):
        codes, scales = quantize(w, group)
        words, s = pack(codes, scales, group)
        a, b = unpack(words, s, 37, 300, group)
        np.testing.assert_array_equal(a, codes)
        np.testing.assert_array_equal(b, scales)
        # n = 19, k = 170: tile (1, 1), octet 170 % 32 / 8 = 1, word 42 / 32 = 1, e = 2
        assert (words[1, 1, 1, 3, 1] >> 4 & 15) - 8 == codes[19, 170]
        off = np.abs(dequantized(codes, scales, group) - w)
        assert (off <= np.repeat(scales.astype(np.float64), group, axis=1)[:, :300] * 0.5 * (1 + 2.0 ** -6)).all()


def test_oracle_logits():
    x = np.array([[1, 2, -3, 4, 0]], np.float16)
    out, _ = adjust(x, [[1, 2, 1, 3, 1]], [2], [2.0], [0.5], [0.25], 2, [[(4, 1.0), (4, 7.0), (0, -1.0)]], [np.array([1, 1, 1, 1, 0], bool)])
    # token 1 ends no 2-gram after 1; 2 and 3 do
    assert out.tolist() == [[0.0, 1 - 0.5 - 2 * 0.25, -np.inf, -np.inf, -np.inf]]
    assert mask_words(np.arange(40)[None] % 2 == 0).tolist() == [[0x55555555, 0x55]]
    h = Histories(3, 4)
    h.step(None, [0, 2, 2, 7], [1, 2, 3, 4, 5, 6, 7], 1)
    assert h.seq == [[1, 2], [], [3, 4, 5, 6]] and h.start == [2, 0, 4]
    h.step([2, 0, 7], [0, 1, 2, 3], [9, 8, 7], 0)
    assert h.seq == [[3, 4, 5, 6], [1, 2, 8], [7]] and h.start == [4, 2, 0]
