"""Compiled-code check of the history step, which changes its sequences in place: at the barriers between what is read and what is written over it
(a piece's tokens, twice, by blocks and by columns; the lengths at the end) a wave waits for all of its loads, by an instruction that the source
writes, not one that the compiler happens to place for a use."""
import re

from asm_util import device_asm, functions


def waits_at_barriers(lines):
    """For each barrier whether a written wait for every load is ahead of it, no load in between."""
    out, waited, written = [], False, False
    for x in lines:
        if "ASMSTART" in x:
            written = True
        elif "ASMEND" in x:
            written = False
        elif written and re.match(r"\s*s_waitcnt vmcnt\(0\)", x):
            waited = True
        elif re.match(r"\s*(global|flat|buffer|scratch)_load|\s*(global|flat)_atomic", x) or re.match(r"^\.LBB", x):
            waited = False
        elif re.match(r"\s*s_barrier", x):
            out.append(waited)
            waited = False
    return out


def test_scanner():
    wait = ["\t;;#ASMSTART", "\ts_waitcnt vmcnt(0)", "\t;;#ASMEND"]
    load, barrier = ["\tglobal_load_dword v1, v2, s[0:1]"], ["\ts_barrier"]
    assert waits_at_barriers(load + wait + barrier) == [True]
    assert waits_at_barriers(wait + load + barrier) == [False]
    assert waits_at_barriers(load + ["\ts_waitcnt vmcnt(0)"] + barrier) == [False]
    assert waits_at_barriers(wait + barrier + barrier) == [True, False]


def test_loads_are_in_before_they_are_written_over():
    fns = {k: v for k, v in functions(device_asm("logits.hip")).items() if "k_history_step" in k}
    assert len(fns) == 2
    for name, lines in fns.items():
        assert sum(waits_at_barriers(lines)) == 3, (name, waits_at_barriers(lines))
