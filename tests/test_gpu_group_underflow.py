"""Values of V that are not finite under weights that underflow.

A query that sees such a value has something non-finite in its dim, however small
the weight is (0 x Inf is NaN): also where the value lies in a part of the row's
work (a stream's tiles, a CTA's stretch, an earlier piece, the prefix) whose
maximum is so far below the other parts' that the part as a whole weighs 0.  The
other dims are held against the 64-bit form.
"""
import numpy as np
import pytest

import tgkv
from group_model import bf16
from test_gpu_group import BF16, F32, JUNK, Setup, put

pytestmark = pytest.mark.gpu

C = tgkv.C

CASES = {  # old lengths, new tokens, prefix, heads, kv heads, head_dim; where the low scores are, their positions
    "full rows, first stream": ([200], [10], None, 4, 1, 64, "own", 0, 128),
    "full rows, second stream": ([370], [10], None, 4, 1, 128, "own", 128, 256),
    "full rows, first CTAs": ([5000], [10], None, 8, 2, 64, "own", 0, 2560),
    "full rows, CTAs between": ([5000], [200], 300, 6, 2, 128, "own", 1024, 3584),
    "full rows, shared prefix": ([5] * 6, [70] * 6, 9000, 16, 4, 128, "prefix", 0, 9000),
    "full rows, own parts": ([5] * 6, [70] * 6, 9000, 16, 4, 128, "own", 0, 75),
    "full rows, earlier piece": ([4200], [1152], None, 16, 4, 64, "own", 0, 4096),
    "few rows, first stream": ([200], [1], None, 4, 1, 64, "own", 0, 128),
    "few rows, second stream": ([370, 3], [1, 2], None, 8, 4, 128, "own", 128, 256),
    "few rows, first CTAs": ([9000, 20], [1, 1], None, 8, 2, 64, "own", 0, 4096),
    "few rows, shared prefix": ([5, 0, 300, 9], [1] * 4, 20000, 32, 8, 128, "prefix", 0, 20000),
    "few rows, own parts": ([300] * 4, [1] * 4, 20000, 32, 8, 128, "own", 0, 301),
    "few rows, earlier piece": ([4300] * 36, [1] * 36, None, 16, 4, 64, "own", 0, 4096),
}


def shaped(s, rows, low):
    """Rows whose K gives scores of about +160 (head_dim 64) or +226 to queries near 1, and as far below 0 in `low`."""
    sign = np.ones(rows.shape[1])
    sign[low] = -1
    rows = np.stack([20 * sign[:, None] + rows[0], rows[1]])
    return bf16(rows)[1]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("case", CASES)
def test_an_underflowing_part_keeps_what_is_not_finite(cuda, devbuf, case, act):
    old, new, P, nh, nkv, hd, where, a, b = CASES[case]
    low, n, total = slice(a, b), len(old), sum(new)
    s = Setup(cuda, old, [t + 3 for t in new], P, nh, nkv, hd, act, seed=len(case))
    cols = [3, hd - 1, s.kvd - 1]                             # of V, at one position of the low ones
    at = (a + min([b] + [o for o in old if o > a])) // 2 if where == "own" else (a + b) // 2

    def fill(c, cap, rows, mine):
        clean = shaped(s, rows, low if mine else slice(0, 0))
        dirty = clean.copy()
        if mine and at < clean.shape[1]:
            clean[1, at, cols] = 0
            dirty[1, at, cols] = np.inf, np.nan, -np.inf
        put(cuda, c, BF16, cap, s.kvd, dirty, JUNK)
        return clean
    for i in range(n):
        s.rows[i] = fill(s.caches[i], s.cap[i], s.rows[i], where == "own")
    if P:
        s.prefix_rows = fill(s.prefix, P + 5, s.prefix_rows, where == "prefix")
    sees = [where == "prefix" or at < o for o in old]
    assert any(sees)
    # queries near 1; the new rows' K like the others' (low if the low positions reach them)
    (_, q), (_, k), (_, v) = s.new(total)
    sign = -1.0 if where == "own" and b > max(old) else 1.0
    put_in = []
    for x in (1 + 0.1 * q, 20 * sign + k, v):
        bits, value = bf16(x)
        put_in.append((bits, value) if act == BF16 else (x.astype(np.float32), x.astype(np.float32).astype(np.float64)))
    (qb, q), (kb, k), (vb, v) = put_in
    s.grow(new, k, v)
    bufs = [devbuf(x) for x in (qb, kb, vb)] + [devbuf(nbytes=qb.nbytes)]
    tgkv.check(cuda.tg_kv_group_prompt(s.g, (C.c_uint32 * n)(*new), *[x.ptr for x in bufs], None), cuda)
    assert cuda.tg_cuda_kv_sync(None)
    got, (want, tol) = s.read(bufs[3], total), s.expect(q, new)
    bad = np.zeros((n, nkv, hd), bool)
    bad[np.ix_(np.flatnonzero(sees), [0], [3, hd - 1])] = True
    bad[np.ix_(np.flatnonzero(sees), [nkv - 1], [hd - 1])] = True
    bad = np.repeat(bad.repeat(nh // nkv, 1), new, 0)
    assert not np.isfinite(got[bad]).any(), (np.isfinite(got[bad]).mean(), got[bad][:4])
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all()
    assert cuda.tg_cuda_kv_device_error() == 0
    s.close()
