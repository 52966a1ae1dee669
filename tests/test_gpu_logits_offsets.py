"""Offsets of bias lists that cannot be, at both ends of a row's list: they are cut to the list, so none reaches past it."""
import numpy as np
import pytest

from test_gpu_logits import Rules, check, some_logits

pytestmark = pytest.mark.gpu

LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("n_bias", [40, 700])   # 700: more entries than a work-group has threads
@pytest.mark.parametrize("rows,masks", [(17, 0), (17, 3), (272, 0), (272, 3)])   # both forms of the kernel
def test_offsets_past_both_ends(pkg, L, rows, masks, n_bias):
    rng = np.random.default_rng([rows, masks, n_bias])
    V = 300
    rules = Rules(pkg, rng, rows, V, [20] * rows, 2, 0, masks)
    dev = lambda a, t: rules.keep.append(pkg.Dev.from_numpy(np.asarray(a, t))) or rules.keep[-1].ptr  # noqa: E731
    # every one is the end of a row and the start of the next
    ends = [0, -1, 5, LOW, LOW, 7, LOW + 1, 3, LOW + 511, n_bias, LOW + 512, HIGH, -513, n_bias + 1, n_bias - 2, HIGH, 0, n_bias]
    offsets = np.resize(np.array(ends, np.int64), rows + 1)
    flat = list(zip(rng.integers(-3, V + 3, n_bias).tolist(), (rng.standard_normal(n_bias).astype(np.float32) * 5).tolist()))
    rules.r.n_bias, rules.r.bias_start = n_bias, dev(offsets, np.int32)
    rules.r.bias_token, rules.r.bias_value = dev([t for t, _ in flat], np.int32), dev([v for _, v in flat], np.float32)
    cut = np.clip(offsets, 0, n_bias)
    rules.biases = [flat[a:b] for a, b in zip(cut[:-1], cut[1:])]
    x = some_logits(rng, rows, V)
    for kw in ({}, {"out_shift": 0}):
        check(pkg, L, x, rules, **kw)
