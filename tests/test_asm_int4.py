"""Compiled-code checks of the 4-bit products and the logits' kernels: the tiles' LDS ring, which global_load_lds fills, is waited for by count
and not emptied ahead of the fragment reads; no loop around a barrier has a lane-divergent latch; nothing spills."""
import re

import pytest

import asm_util
from asm_util import device_asm, functions
from test_asm_barriers import hazardous_loops
from test_asm_lds_dma import dma_alias_waits

asm_util.EXTRA.setdefault("int4.hip", ["-mllvm", "-amdgpu-mfma-vgpr-form"])   # as in csrc/Makefile


@pytest.mark.parametrize("src", ["int4.hip", "logits.hip"])
def test_uniform_loops_around_barriers(src):
    asm = device_asm(src)
    assert "s_barrier" in asm and "Loop Header" in asm
    assert hazardous_loops(asm) == []


def test_tiles_ring():
    fns = {k: v for k, v in functions(device_asm("int4.hip")).items() if any("global_load_lds" in x for x in v)}
    assert len(fns) == 27   # nine forms, three groups
    for name, lines in fns.items():
        assert "k_int4_tile" in name
        assert dma_alias_waits(lines) == 0, name
        assert any(re.match(r"\s*v_mfma_f32_16x16x32_f16", x) for x in lines), name


@pytest.mark.parametrize("src", ["int4.hip", "logits.hip"])
def test_no_spills_and_no_packed_fp32(src):
    asm = device_asm(src)
    spills = re.findall(r"\.vgpr_spill_count:\s*(\d+)", asm)
    assert spills and all(int(s) == 0 for s in spills)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", asm)
