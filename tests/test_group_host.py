"""Refusals of the group operators that need no device: bad arguments end with
a reason before any device call.  Addresses are only looked at, never followed."""
import ctypes as C

import pytest

u32 = C.c_uint32


class Call(C.Structure):
    """TGCudaGroupCall of include/tgai_cuda_bridge.h."""
    _fields_ = [("act", C.c_int), ("n_seq", u32), ("n_heads", u32), ("n_kv_heads", u32),
                ("head_dim", u32), ("prefix_len", u32), ("table_dev", C.c_void_p),
                ("old_len", C.POINTER(u32)), ("n_new", C.POINTER(u32)), ("q", C.c_void_p),
                ("k_new", C.c_void_p), ("v_new", C.c_void_p), ("out", C.c_void_p),
                ("scale", C.c_float), ("scratch", C.c_void_p)]


def caches(*rows):
    return (C.c_uint64 * (2 * len(rows)))(*[x for r in rows for x in r])


def test_null_objects(lib):
    null = (C.c_void_p * 2)(None, None)
    n1 = (u32 * 1)(1)
    assert not lib.tg_kv_group_create(None, None, 1, 8, 0)
    assert not lib.tg_kv_group_create(None, null, 0, 8, 0)
    assert not lib.tg_kv_group_create(None, null, 1025, 8, 0)
    assert b"1..1024" in lib.tg_kv_last_error()
    assert not lib.tg_kv_group_create(None, null, 2, 8, 0)
    assert b"null cache 0" in lib.tg_kv_last_error()
    lib.tg_kv_group_destroy(None)
    assert lib.tg_kv_group_truncate(None, n1) == 0
    assert lib.tg_kv_group_decode(None, 16, None, None, 16, None) == 0
    assert lib.tg_kv_group_prompt(None, n1, 16, None, None, 16, None) == 0
    assert b"null argument" in lib.tg_kv_last_error()
    assert lib.tg_kv_fork(None, 1, null, 1, 1, None) == 0
    assert lib.tg_kv_fork(null, 1, null, 0, 1, None) == 0
    assert lib.tg_kv_fork(null, 512, null, 3, 1, None) == 0
    assert b"1..1024 copies" in lib.tg_kv_last_error()
    assert lib.tg_kv_fork(null, 1, null, 1, 1, None) == 0
    assert b"null cache" in lib.tg_kv_last_error()
    assert lib.tg_kv_compact(None, 1, n1, n1, 1, None) == 0
    assert lib.tg_kv_compact(null, 1, None, n1, 1, None) == 0
    assert lib.tg_kv_compact(null, 1, n1, n1, 1025, None) == 0
    assert b"1024 ranges" in lib.tg_kv_last_error()
    assert lib.tg_kv_compact(null, 2, n1, n1, 1, None) == 0
    assert b"null cache" in lib.tg_kv_last_error()


@pytest.mark.parametrize("src,dst,n_src,fan,row,n,why", [
    ([(16, 8)], [(32, 8)], 1, 1, 24, 4, b"rows of 24 bytes"),
    ([(16, 8)], [(32, 8)], 1, 1, 0, 4, b"rows of 0 bytes"),
    ([(24, 8)], [(32, 8)], 1, 1, 32, 4, b"source 0"),
    ([(16, 8)], [(32, 3)], 1, 1, 32, 4, b"copy 0"),
    ([(16, 3)], [(32, 8)], 1, 1, 32, 4, b"source 0"),
    ([(16, 8)], [(32, 8), (0, 8)], 1, 2, 32, 4, b"copy 1"),
    ([(16, 8)], [(32, 8)], 0, 1, 32, 4, b"0 sources"),
    ([(16, 8)], [(32, 8)], 1025, 1, 32, 4, b"1025 sources"),
])
def test_fork_rows_refuses(lib, src, dst, n_src, fan, row, n, why):
    assert lib.tg_cuda_kv_fork_rows(caches(*src), n_src, caches(*dst), fan, row, n, None) == 0
    assert why in lib.tg_cuda_kv_last_error()


@pytest.mark.parametrize("cache,start,count,row,why", [
    ((16, 8), [0], [0], 32, b"range 0"),
    ((16, 8), [0, 2], [3, 1], 32, b"range 1"),
    ((16, 8), [4, 2], [1, 1], 32, b"range 1"),
    ((16, 8), [4], [5], 32, b"fewer than 9 rows"),
    ((16, 8), [0xffffffff], [0xffffffff], 32, b"fewer than 8589934590 rows"),
    ((8, 8), [4], [1], 32, b"16-byte aligned"),
    ((16, 8), [4], [1], 20, b"rows of 20 bytes"),
])
def test_compact_rows_refuses(lib, cache, start, count, row, why):
    n = len(start)
    assert lib.tg_cuda_kv_compact_rows(caches(cache), 1, row, (u32 * n)(*start), (u32 * n)(*count), n, None) == 0
    assert why in lib.tg_cuda_kv_last_error()


@pytest.mark.parametrize("change,why", [
    ({"q": None}, b"NULL pointer"), ({"out": None}, b"NULL pointer"), ({"table_dev": None}, b"NULL pointer"),
    ({"scratch": None}, b"NULL pointer"), ({"old_len": None}, b"NULL pointer"), ({"n_new": None}, b"NULL pointer"),
    ({"k_new": None}, b"go together"), ({"v_new": None}, b"go together"),
    ({"q": 0x1008}, b"16-byte aligned"), ({"out": 0x1004}, b"16-byte aligned"),
    ({"k_new": 0x1002}, b"16-byte aligned"), ({"v_new": 0x1008}, b"16-byte aligned"),
    ({"n_seq": 0}, b"no kernel"), ({"n_seq": 1025}, b"no kernel"), ({"head_dim": 96}, b"no kernel"),
    ({"n_heads": 6}, b"no kernel"), ({"n_kv_heads": 0}, b"no kernel"),
    ({"n_heads": 516, "n_kv_heads": 4}, b"no kernel"), ({"act": 2}, b"no kernel"),
    ({"new": 0x7fffffff}, b"too many query rows"), ({"prefix_len": 0x80000000}, b"too long"),
])
def test_group_attention_refuses(lib, change, why):
    change = dict(change)
    old, new = (u32 * 1)(0), (u32 * 1)(change.pop("new", 1))
    a = dict(act=0, n_seq=1, n_heads=8, n_kv_heads=4, head_dim=64, prefix_len=0, table_dev=0x1000, old_len=old,
             n_new=new, q=0x1000, k_new=0x2000, v_new=0x3000, out=0x4000, scale=1.0, scratch=0x5000)
    a.update(change)
    c = Call(**a)
    assert lib.tg_cuda_kv_group_attention(C.byref(c), None) == 0
    assert why in lib.tg_cuda_kv_last_error()


def test_group_table_refuses(lib):
    for n, nkv, hd in ((0, 4, 64), (1025, 4, 64), (1, 0, 64), (1, 4, 96)):
        assert not lib.tg_cuda_kv_group_table(caches((16, 8), (0, 0)), n, nkv, hd)
        assert b"bad argument" in lib.tg_cuda_kv_last_error()


def plan(lib, old, new, prefix, nh, nkv, act, sms):
    """(share, CTA starts of the two kernels) of a call; the last start is what follows the line."""
    n = len(old)
    c = Call(act=act, n_seq=n, n_heads=nh, n_kv_heads=nkv, head_dim=64, prefix_len=prefix, old_len=(u32 * n)(*old),
             n_new=(u32 * n)(*new))
    share, n_cta, starts = u32(), (u32 * 2)(), (u32 * (2 * 161 * 4))()
    assert lib.tg_cuda_kv_group_plan(C.byref(c), sms, C.byref(share), n_cta, starts), lib.tg_cuda_kv_last_error()
    return share.value, [[tuple(starts[644 * ln + 4 * b:644 * ln + 4 * b + 4]) for b in range(n_cta[ln] + 1)]
                         if n_cta[ln] else [] for ln in range(2)]


def lines(old, new, prefix, nh, nkv, share, act):
    """Every (item, tile) of the two lines in order, from the description of the cut alone."""
    g = nh // nkv
    heavy, light = 128 // g * (1 + act), (16 if act else 10) // g
    own_light = max(new) <= light
    pre_light = own_light and (not share or sum(new) <= light)
    got = [[], []]

    def add(line, seq, tokens, tiles_of):
        per = light if line else heavy
        got[line] += [(seq, h, r, j) for h in range(nkv) for r in range(-(-tokens // per)) for j in range(tiles_of(r, per))]
    pre = -(-prefix // 128)
    if share:
        add(int(pre_light), 0, sum(new), lambda r, per: pre)
    for i, (o, t) in enumerate(zip(old, new)):
        add(int(own_light), i + 1, t, lambda r, per: (0 if share else pre) + -(-(o + min((r + 1) * per, t)) // 128))
    return got


@pytest.mark.parametrize("old,new,prefix,nh,nkv,share", [
    ([0], [1], 0, 1, 1, 0), ([0], [1], 1, 1, 1, 0), ([5] * 64, [1] * 64, 32768, 32, 8, 1),
    ([100] * 1024, [1] * 1024, 300, 8, 8, 1), ([5, 9], [1, 1], 64, 8, 8, 0), ([0, 3, 900], [0, 7, 0], 500, 12, 4, 0),
    ([0] * 5, [0] * 5, 100, 4, 4, 0), ([0, 0], [5000, 1], 0, 16, 4, 0),
    ([10] * 12, [2, 9, 0, 4, 0, 8, 1, 1, 3, 5, 6, 7], 70000, 16, 2, 1), ([0, 9], [1, 1], 30000, 8, 8, 1),
    ([77] * 9, [40] * 9, 40000, 16, 4, 1), ([77] * 9, [40] * 9, 1000, 16, 4, 0), ([77] * 9, [60] * 9, 4000, 16, 4, 0), ([1], [3], 129, 128, 1, 0),
    ([200000], [1], 0, 7, 1, 0), ([0] * 30, [600] * 30, 100, 32, 8, 0), ([3, 0, 5], [2, 0, 1], 0, 8, 4, 0),
])
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("sms", [148, 1, 7, 0])
def test_plan_covers_the_lines(lib, old, new, prefix, nh, nkv, share, sms, act):
    """The CTAs' stretches are the lines of tiles, cut in order into parts of about one size."""
    got_share, starts = plan(lib, old, new, prefix, nh, nkv, act, sms)
    if sms == 148:                                               # what it saves is weighed against the SMs
        assert got_share == share
    share = got_share
    both = [len(st) - 1 if st else 0 for st in starts]
    want = lines(old, new, prefix, nh, nkv, share, act)
    assert sum(both) <= max(2 if all(want) else 1, sms or 160)
    for tiles, st in zip(want, starts):
        if not tiles:
            assert not st
            continue
        index = {t: k for k, t in enumerate(tiles)}
        cuts = [index[s] for s in st[:-1]] + [len(tiles)]
        after = min([i + 1 for i, t in enumerate(new) if t and i + 1 > tiles[-1][0]], default=len(new) + 1)
        assert st[-1] == (after, 0, 0, 0)
        assert cuts[0] == 0 and all(a <= b for a, b in zip(cuts, cuts[1:]))
        n_cta = len(st) - 1
        items = len({t[:3] for t in tiles})
        if n_cta == items and all(s[3] == 0 for s in st):
            continue                                             # a CTA per item
        cost = 4 if st is starts[1] else 1 if act else 5         # of an item beside its tiles
        most = max(b - a + cost * len({t[:3] for t in tiles[a:b]}) for a, b in zip(cuts, cuts[1:]))
        assert most <= (len(tiles) + cost * items) / n_cta + 2 * cost + 1
