"""fp32 activations over long histories.

A full row tile that sees more than 32 K/V tiles of 128 positions is worked in
pieces of 32 tiles whose sums meet in the group's scratch.  The cases hold such
items whole in one CTA, by the plan for 148 SMs that a test without a device
looks at; on the GPU every element is held against a plain 64-bit form within
the roundings of group_model.py, and every head's row within the bound that
tgai_kv_group.h states.
"""
import numpy as np
import pytest

import tgkv
from conftest import rel_head_err
from test_gpu_group import F32, Setup
from test_group_host import plan

C = tgkv.C

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
    assert rel_head_err(got, want) < 5e-5
    s.close()
