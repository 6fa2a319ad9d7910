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
                ("scale", C.c_float)]


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
    ({"k_new": None}, b"go together"), ({"v_new": None}, b"go together"),
    ({"q": 0x1008}, b"16-byte aligned"), ({"out": 0x1004}, b"16-byte aligned"),
    ({"k_new": 0x1002}, b"16-byte aligned"), ({"v_new": 0x1008}, b"16-byte aligned"),
    ({"n_seq": 0}, b"no kernel"), ({"n_seq": 1025}, b"no kernel"), ({"head_dim": 96}, b"no kernel"),
    ({"n_heads": 6}, b"no kernel"), ({"n_kv_heads": 0}, b"no kernel"),
    ({"n_heads": 516, "n_kv_heads": 4}, b"no kernel"), ({"act": 2}, b"no kernel"),
    ({"new": 0x7fffffff}, b"too many query rows"),
])
def test_group_attention_refuses(lib, change, why):
    change = dict(change)
    old, new = (u32 * 1)(0), (u32 * 1)(change.pop("new", 1))
    a = dict(act=0, n_seq=1, n_heads=8, n_kv_heads=4, head_dim=64, prefix_len=0, table_dev=0x1000, old_len=old,
             n_new=new, q=0x1000, k_new=0x2000, v_new=0x3000, out=0x4000, scale=1.0)
    a.update(change)
    c = Call(**a)
    assert lib.tg_cuda_kv_group_attention(C.byref(c), None) == 0
    assert why in lib.tg_cuda_kv_last_error()


def test_group_table_refuses(lib):
    for n, nkv, hd in ((0, 4, 64), (1025, 4, 64), (1, 0, 64), (1, 4, 96)):
        assert not lib.tg_cuda_kv_group_table(caches((16, 8), (0, 0)), n, nkv, hd)
        assert b"bad argument" in lib.tg_cuda_kv_last_error()
