"""What pages of INT8 cost: one sequence's attention over them, its prompt in one call, in pieces and token by token, against 64 bits over
the keys and values as they came and against the fp16 prefill attention."""
import numpy as np
import pytest

from pagedkv_ref import D, P, Ws, ref
from test_gpu_pagedkv import qkv_of, rows_of

pytestmark = pytest.mark.gpu
H, E = 12, 12 * D


def paged(pkg, L, x, cuts):
    """att of a prompt whose rows go into the cache in those pieces."""
    c = pkg.PagedKV(20, 1, 512, 1, H)
    d_x, att = pkg.Dev.from_numpy(x), pkg.Dev(len(x) * E * 2)
    ws = Ws(pkg, max(L.gpt2_pkv_attn_ws(ref(c), n) for n in set(cuts)))
    at, keep = 0, []
    for n in cuts:
        rows = pkg.Dev.from_numpy(rows_of([n]))
        keep.append(rows)
        L.gpt2_pkv_grow(ref(c), rows.ptr, n)
        L.gpt2_pkv_append(ref(c), 0, d_x.at(at * 3 * E * 2), rows.ptr, n)
        L.gpt2_pkv_attn(att.at(at * E * 2), d_x.at(at * 3 * E * 2), ref(c), 0, rows.ptr, n, 1, *ws.args)
        at += n
    assert at == len(x) and L.gpt2_pkv_status(ref(c)) == 0
    pkg.check("paged")
    out = att.numpy(np.float16, (len(x), E)).astype(np.float64)
    c.free()
    return out


@pytest.mark.parametrize("n", [20, 70, 300])
def test_prompt_in_one_call_and_in_pieces(pkg, L, n):
    """A page's key is off by half a code s_k / 2 in each dim, so a score by d = sum |q| s_k / 16 at most and a share of the softmax by
    a factor of exp(2 d); a value by s_v / 2.  A row's pages are those that are complete when its call attends: with the prompt in one call
    the page that the row itself is in may be, and its scale then has later tokens in it."""
    x = qkv_of(np.random.default_rng(70 + n), n, H)
    q, k, v = x.astype(np.float64).reshape(n, 3, H, D).transpose(1, 2, 0, 3)
    ends = {1: np.arange(n) + 1, 37: np.minimum((np.arange(n) // 37 + 1) * 37, n), n: np.full(n, n)}
    exact, bound = np.empty((n, H, D)), {c: np.empty((n, H, D)) for c in ends}
    for h in range(H):
        page = [slice(j * P, (j + 1) * P) for j in range(n // P)]
        sk, sv = (np.array([np.abs(t[h, s]).max() / 127 for s in page]) for t in (k, v))
        for i in range(n):
            sc = k[h, :i + 1] @ q[h, i] / 8
            w = np.exp(sc - sc.max())
            w /= w.sum()
            exact[i, h] = w @ v[h, :i + 1]
            away, vmax = w @ np.abs(v[h, :i + 1] - exact[i, h]), np.abs(v[h, :i + 1]).max()
            for c, end in ends.items():   # with no page yet the kernel's own roundings are all
                m = min(end[i] // P, -(-(i + 1) // P))   # complete pages that the row sees
                d = np.abs(q[h, i]).sum() * sk[:m].max(initial=0) / 16
                # those: fp16 weights and output, 3 half steps 2^-11 of the largest value, scores' sums 2^-10
                bound[c][i, h] = (np.exp(2 * d) - 1) * away + sv[:m].max(initial=0) / 2 + vmax * (3 * 2.0 ** -11 + 2.0 ** -10)
    exact = exact.reshape(n, E)
    got = {c: paged(pkg, L, x, [c] * (n // c) + ([n % c] if n % c else [])) for c in ends}
    for c, a in got.items():
        assert (np.abs(a - exact) <= bound[c].reshape(n, E)).all(), c
    d_x, att = pkg.Dev.from_numpy(x), pkg.Dev(n * E * 2)
    L.gpt2_attention_flash(att.ptr, d_x.ptr, n, E, H, D)
    L.gpt2_sync()
    flash = att.numpy(np.float16, (n, E)).astype(np.float64)
    for c, a in got.items():
        assert (np.abs(a - flash) <= bound[c].reshape(n, E) + np.abs(v).max() * (3 * 2.0 ** -11 + 2.0 ** -10)).all(), c
