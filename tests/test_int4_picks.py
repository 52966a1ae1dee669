"""The table that picks a form for 4-bit products of more than 16 rows (csrc/int4.hip: tile_form), read from the source: how many work-groups of a form
a CU has room for is what the compiled kernels' registers and LDS allow, and the sizes of the exact products' tests reach every form, in every group size."""
import math
import os
import re

import pytest

import asm_util
from asm_util import device_asm
from int4_ref import cdiv
from test_int4_exact import SIZES

asm_util.EXTRA.setdefault("int4.hip", ["-mllvm", "-amdgpu-mfma-vgpr-form"])   # as in csrc/Makefile
GROUPS = (32, 64, 128)
LDS, SIMDS, REGISTERS, WAVES = 160 * 1024, 4, 512, 8   # a CU's; a SIMD's


def forms(group):
    """{table: [(the template's arguments, room, start, step, start2, step2)]} as tile_form<group> has them."""
    src = open(os.path.join(asm_util.CSRC, "int4.hip")).read()
    src = src[src.index("static const Q4Form &tile_form"):]
    out = {}
    for table in ("by_loads", "by_registers"):
        body = re.search(r"Q4Form " + table + r"\[\] = \{(.*?)\};", src, re.S).group(1)
        out[table] = []
        for args, room, *times in re.findall(r"q4_form<G, ([^>]*)>\(([^,]+), ([\d.]+)f, ([\d.]+)f, ([\d.]+)f, ([\d.]+)f\)", body):
            m = re.match(r"G == (\d+) \? (\d) : (\d)$", room)
            room = int(room) if not m else int(m[2] if group == int(m[1]) else m[3])
            out[table].append((tuple(v.strip() for v in args.split(",")), room, *map(float, times)))
        assert len(out[table]) == body.count("q4_form<") > 0
    return out


def compiled():
    """{(group, the template's arguments): (threads, registers, bytes of LDS)}."""
    out = {}
    for lds, name, vgprs in re.findall(r"\.group_segment_fixed_size: (\d+).*?\.name:\s+(\S+).*?\.vgpr_count:\s+(\d+)", device_asm("int4.hip"), re.S):
        m = re.search(r"k_int4_tileI((?:L[ib]\d+E)+)E", name)
        if m:
            v = re.findall(r"L([ib])(\d+)E", m.group(1))
            args = tuple(("false", "true")[int(x)] if t == "b" else x for t, x in v[1:])
            out[int(v[0][1]), args] = (64 * int(args[2]) * int(args[3]) * int(args[4]), int(vgprs), int(lds))
    return out


@pytest.mark.parametrize("group", GROUPS)
def test_room(group):
    kernels = compiled()
    for table in forms(group).values():
        for args, room, *_ in table:
            threads, vgprs, lds = kernels[group, args]
            waves = SIMDS * min(WAVES, REGISTERS // (cdiv(vgprs, 8) * 8))
            assert room == min(waves * 64 // threads, LDS // lds), (group, args, vgprs, lds)


@pytest.mark.parametrize("group", GROUPS)
def test_every_form_is_reached(group):
    for table, direct in (("by_loads", True), ("by_registers", False)):
        reached = set()
        for m, n, k in SIZES:
            if m <= 16 or (k % 8 == 0) != direct:
                continue
            best, least = None, math.inf
            for i, (args, room, start, step, start2, step2) in enumerate(forms(group)[table]):
                bm, bn, _, _, ks = map(int, args[:5])
                a_cu, steps = math.ceil(cdiv(m, bm) * cdiv(n, bn) / 256), cdiv(cdiv(k, 128), ks)
                rounds = math.ceil(a_cu / room)
                us = rounds * (start + steps * step) + (a_cu - rounds) * (start2 + steps * step2)
                if us < least:
                    best, least = i, us
            reached.add(best)
        assert reached == set(range(len(forms(group)[table]))), table
