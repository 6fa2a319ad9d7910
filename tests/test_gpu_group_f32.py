"""fp32 activations: long histories, and what a head's row may be off by.

A full row tile that sees more than 32 K/V tiles of 128 positions is worked in
pieces of 32 tiles whose sums meet in the group's scratch.  The cases hold such
items whole in one CTA, by the plan for 148 SMs that a test without a device
looks at; on the GPU every element is held against a plain 64-bit form within
the roundings of group_model.py, and every head's row within the bound that
tgai_kv_group.h states.

group_model.py adds the roundings up as if all had one sign.  The bounds on a
head's row (error over the row's largest value) let them average out, so that a
lost term shows:
  5e-5  full row tiles, q and weights as two bf16 terms.  A term is off by at most
        half a step of 8 bits, so two by 2^-16, about 2^-19 on average (rms);
        over the positions both roundings move an output by 1.4 * 2^-19 = 2.7e-6
        of its rms, at worst of 10^5 outputs by 4.5 times that, and the truncated
        fp32 sums (at most 128 steps of 16 positions, each for two terms, half a
        step of 2^-23 of a sum that on average is half its end) by 7.7e-6.  One
        term alone moves it by 2^-10.
  2e-6  few rows, three terms (2^-24 at most), up to 400 positions: the scores'
        sums and the exponential, 2^-21 of a weight, move an output by 4.8e-7 of
        its rms, at worst by 4.5 times that, against a row maximum of at least
        twice the rms; 16 steps of truncated sums by 6.4e-7: 1.8e-6 in all.  Two
        terms alone move it by 2.7e-6 rms.
"""
import numpy as np
import pytest

import tgkv
from conftest import rel_head_err
from group_model import bf16, reference
from test_gpu_group import F32, Setup
from test_group_host import plan

C = tgkv.C
FULL, FEW = 5e-5, 2e-6

LONG = [  # old lengths, new tokens, prefix, heads, kv heads, head_dim; tiles that an item in one CTA passes
    ([4200], [1152], None, 16, 4, 128, 32),
    ([50], [1152], 4200, 16, 4, 64, 32),
    ([0] * 3, [500] * 3, 4200, 12, 4, 64, 32),               # row tiles of 42 tokens: two rows unused
    ([4500], [700], None, 32, 8, 128, 32),                   # beside items over several CTAs
    ([1000 + 37 * i for i in range(24)], [40] * 24, 6000, 32, 8, 128, 32),
    ([8200] * 9, [128] * 9, None, 16, 4, 64, 64),
    ([12300] * 9, [125] * 9, None, 16, 4, 128, 96),
]


def whole_items(lib, old, new, P, nh, nkv):
    """(share, [(K/V tiles, query rows)] of the items that one CTA of line 0 does whole)."""
    P = P or 0
    share, (starts, light) = plan(lib, old, new, P, nh, nkv, F32, 148)
    assert not light
    g = nh // nkv
    per, pre = 128 // g, 0 if share else -(-P // 128)
    cut = {s[:3] for s in starts if s[3]}
    return share, [(pre + -(-(o + min((r + 1) * per, t)) // 128), g * min(per, t - r * per))
                   for i, (o, t) in enumerate(zip(old, new)) for h in range(nkv) for r in range(-(-t // per))
                   if (i + 1, h, r) not in cut]


@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_items_lie_whole_in_a_cta(lib, case):
    old, new, P, nh, nkv, _, passed = LONG[case]
    share, items = whole_items(lib, old, new, P, nh, nkv)
    assert not share
    # rows of all four warps of a row tile, in pieces of 32 tiles
    assert sum(tiles > passed and rows > 96 for tiles, rows in items) >= 16


def attend(s, devbuf, n_new):
    """One call that appends, on fresh tokens: (result, 64-bit form, tolerance)."""
    total = sum(n_new)
    (qb, q), (kb, k), (vb, v) = s.new(total)
    s.grow(n_new, k, v)
    bufs = [devbuf(x) for x in (qb, kb, vb)] + [devbuf(nbytes=qb.nbytes)]
    tgkv.check(s.lib.tg_kv_group_prompt(s.g, (C.c_uint32 * len(n_new))(*n_new), *[b.ptr for b in bufs], None), s.lib)
    assert s.lib.tg_cuda_kv_sync(None)
    got = s.read(bufs[3], total)
    s.check_caches()
    assert s.lib.tg_cuda_kv_device_error() == 0
    return got, *s.expect(q, n_new)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_items(cuda, devbuf, case):
    old, new, P, nh, nkv, hd, _ = LONG[case]
    s = Setup(cuda, old, [n + 3 for n in new], P, nh, nkv, hd, F32, seed=150 + case)
    got, want, tol = attend(s, devbuf, new)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])
    assert rel_head_err(got, want) < FULL
    s.close()


@pytest.mark.parametrize("terms,bound,holds", [(1, FULL, False), (2, FULL, True), (2, FEW, False), (3, FEW, True)])
def test_bounds_tell_the_terms(terms, bound, holds):
    """q and the weights as that many bf16 terms, all else in 64 bits."""
    def rounded(x):
        out, rest = np.zeros_like(x), x
        for _ in range(terms):
            t = bf16(rest)[1]
            out, rest = out + t, rest - t
        return out
    rng = np.random.default_rng(terms)
    got, want = [], []
    for _ in range(24):                                      # heads
        q, k, v = (rng.standard_normal((n, 128)).astype(np.float32).astype(np.float64) for n in (8, 400, 400))
        want.append(reference(q, [(k, v)], 128 ** -0.5, False)[0])
        w = rounded(np.exp(np.where(np.arange(400) <= 392 + np.arange(8)[:, None], rounded(q) @ k.T * 128 ** -0.5, -np.inf)))
        got.append(w @ v / w.sum(1, keepdims=True))
    assert (rel_head_err(np.array(got), np.array(want)) < bound) == holds


BOUNDS = [  # old lengths, new tokens, prefix, heads, kv heads, head_dim; what of a head's row
    ([390, 0, 127, 128], [1] * 4, None, 16, 4, 128, FEW),
    ([100] * 40, [1] * 40, 250, 32, 8, 64, FEW),
    ([7, 200, 380], [2, 2, 1], 0, 8, 2, 128, FEW),           # two tokens of four heads
    ([380, 40, 3], [10, 0, 9], None, 4, 4, 64, FEW),
    ([300, 0, 77], [200, 129, 11], None, 12, 4, 128, FULL),
    ([10] * 12, [22, 9, 11, 4, 31, 8, 1, 1, 3, 5, 6, 7], 700, 16, 2, 64, FULL),
    ([2000], [300], 500, 32, 8, 128, FULL),
    ([17] * 40, [1] * 40, 4000, 6, 3, 64, FULL),             # the prefix on full row tiles, own rows on few
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(BOUNDS)))
def test_a_head_row_within_its_bound(cuda, devbuf, case):
    old, new, P, nh, nkv, hd, bound = BOUNDS[case]
    starts = plan(cuda, old, new, P or 0, nh, nkv, F32, 148)[1]
    assert (bound == FEW) == (not starts[0])                 # all of it on the kernel of few rows
    s = Setup(cuda, old, [2 * n + 3 for n in new], P, nh, nkv, hd, F32, seed=170 + case)
    for _ in range(2):
        got, want, tol = attend(s, devbuf, new)
        assert (np.abs(got - want) <= tol).all()
        assert rel_head_err(got, want) < bound
    s.close()
