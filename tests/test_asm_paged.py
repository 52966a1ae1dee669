"""Compiled-code checks of the paged cache's kernels: the attention's LDS ring, which global_load_lds fills, is waited for and
read in the right order; and no loop around a barrier has a lane-divergent latch."""
import re

import pytest

import asm_util
from asm_util import device_asm, functions
from test_asm_barriers import hazardous_loops
from test_asm_lds_dma import dma_alias_waits

asm_util.EXTRA.setdefault("attn_paged.hip", ["-mllvm", "-amdgpu-mfma-vgpr-form"])   # as in csrc/Makefile


def unordered_refills(lines):
    """Loads into LDS with a fragment read after the last wait for LDS reads before them, in the listing's order."""
    n, reading = 0, False
    for t in (x.strip() for x in lines):
        if re.match(r"ds_read_b128\b", t):
            reading = True
        elif re.match(r"s_waitcnt .*lgkmcnt\(0\)", t):
            reading = False
        elif t.startswith("global_load_lds") and reading:
            n += 1
    return n


def test_scanner_flags_the_pattern():
    read, fill, wait = "\tds_read_b128 v[0:3], v4", "\tglobal_load_lds_dwordx4 v[0:1], off", "\ts_waitcnt lgkmcnt(0)"
    assert unordered_refills([read, wait, fill]) == 0
    assert unordered_refills([read, wait, read, "\ts_waitcnt lgkmcnt(1)", fill]) == 1
    assert unordered_refills([fill, read]) == 0


def test_attention_ring():
    fns = {k: v for k, v in functions(device_asm("attn_paged.hip")).items() if any("global_load_lds" in x for x in v)}
    assert len(fns) == 6, sorted(fns)   # one row or a group of beams on four and eight waves, 16 and 32 rows
    for name, lines in fns.items():
        assert dma_alias_waits(lines) == 0, name
        assert unordered_refills(lines) == 0, name


@pytest.mark.parametrize("src", ["attn_paged.hip", "pagedkv.hip", "beam.hip"])
def test_uniform_loops_around_barriers(src):
    assert hazardous_loops(device_asm(src)) == []
