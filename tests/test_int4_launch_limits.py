"""4-bit products of more results than one launch has threads for are refused on the host."""
import ctypes as C

import pytest

ARG = 1000
AT = 0x10000   # an address that a refused call never reads


@pytest.mark.parametrize("K", [30, 32])   # rows that are not at 16 bytes, and rows that are
def test_results_past_a_launch(pkg, L, K):
    L.gpt2_last_error()
    w = pkg.GPT2Int4W(AT, AT, 1 << 17, K, 32, None)
    L.gpt2_matmul_int4(AT, AT, C.byref(w), None, 1 << 21, 0, None)
    assert L.gpt2_last_error() == ARG
