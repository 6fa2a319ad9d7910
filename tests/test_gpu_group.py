"""Groups of caches on the GPU: decode over a shared prefix, packed prompts,
fork and compaction, against plain 64-bit forms.

Rows behind a cache's length hold NaN, Inf or huge values (what a truncated
turn may leave), so every result also shows that they take no part.  The
tolerances are the roundings the kernels make (group_model.py), element by
element.
"""
import numpy as np
import pytest

import tgkv
from conftest import rel_head_err
from group_model import bf16, group_reference

pytestmark = pytest.mark.gpu

F32, BF16 = tgkv.TG_KV_F32, tgkv.TG_KV_BF16
C = tgkv.C


def put(lib, c, dtype, cap, kvd, rows, junk):
    """The whole buffer of cache c: `rows` [2][n][kvd], then junk rows."""
    n = rows.shape[1]
    full = np.empty((2, cap, kvd), np.float32)
    full[:, :n] = rows
    full[:, n:] = np.resize(np.array(junk, np.float32), (2, cap - n, kvd))
    raw = bf16(full)[0] if dtype == BF16 else full
    assert lib.tg_cuda_kv_h2d(lib.tg_kv_device_handle(c), raw.ctypes.data, raw.nbytes, None)
    lib.tg_kv_reset(c)
    lib.tg_kv_advance(c, n)
    return raw


def get(lib, c, dtype, cap, kvd):
    raw = np.empty(lib.tg_kv_bytes(c), np.uint8)
    tgkv.check(lib.tg_kv_download(c, raw.ctypes.data), lib)
    return raw.view(np.uint16 if dtype == BF16 else np.float32).reshape(2, cap, kvd)


JUNK = [np.nan, np.inf, -np.inf, 3e38, -1.0]


class Setup:
    """n caches with old[i] rows each (and a prefix of P), a group over them."""

    def __init__(self, lib, old, room, P, nh, nkv, hd, act, seed=0, mscale=None):
        self.lib, self.nh, self.nkv, self.hd, self.act, self.P = lib, nh, nkv, hd, act, P
        self.rng = np.random.default_rng(seed)
        self.kvd, self.q_scale = nkv * hd, 1
        self.old, self.cap = list(old), [o + r for o, r in zip(old, room)]
        self.rows, self.caches = [], []
        for o, cap in zip(self.old, self.cap):
            self._cache(cap, o)
        self.prefix = None
        if P is not None:
            self._cache(P + 5, P)
            self.prefix, self.prefix_rows = self.caches.pop(), self.rows.pop()
        scale = hd ** -0.5
        if mscale is not None:
            scale *= mscale
            for c in self.caches + [self.prefix] * (P is not None):
                lib.tg_kv_set_attn_mscale(c, mscale)
        self.scale = float(np.float32(scale))
        self.arr = (C.c_void_p * len(old))(*self.caches)
        self.g = lib.tg_kv_group_create(self.prefix, self.arr, len(old), nh, act)
        tgkv.check(self.g, lib, "group")

    def _cache(self, cap, n):
        c = self.lib.tg_kv_create_ex(cap, self.nkv, self.hd, BF16)
        tgkv.check(c, self.lib)
        x = self.rng.standard_normal((2, n, self.kvd))
        put(self.lib, c, BF16, cap, self.kvd, x, JUNK)
        self.caches.append(c)
        self.rows.append(bf16(x)[1])

    def new(self, total):
        """q, k, v of `total` tokens: (device-ready array, float64 value) each."""
        got = []
        for cols, mul in ((self.nh * self.hd, self.q_scale), (self.kvd, 1), (self.kvd, 1)):
            x = (mul * self.rng.standard_normal((total, cols))).astype(np.float32)
            b, v = bf16(x)
            got.append((b, v) if self.act == BF16 else (x, x.astype(np.float64)))
        return got

    def expect(self, q, n_new):
        """The reference for the rows as they are in self.rows now."""
        def heads(r):
            return r[0].reshape(-1, self.nkv, self.hd), r[1].reshape(-1, self.nkv, self.hd)
        pre = heads(self.prefix_rows) if self.P else None
        return group_reference(q.reshape(-1, self.nh, self.hd), pre, [heads(r) for r in self.rows], n_new, self.nkv,
                               self.scale, self.act == BF16)

    def grow(self, n_new, k, v):
        at = 0
        for i, t in enumerate(n_new):
            add = np.stack([bf16(k[at:at + t])[1], bf16(v[at:at + t])[1]])
            self.rows[i] = np.concatenate([self.rows[i], add], 1)
            at += t

    def read(self, buf, total):
        if self.act == BF16:
            import oracle as O
            return O.bf16_to_f32(buf.get(np.uint16, (total, self.nh, self.hd))).astype(np.float64)
        return buf.get(np.float32, (total, self.nh, self.hd)).astype(np.float64)

    def check_caches(self):
        """Every cache holds its rows, and what lay behind them as it was."""
        for c, cap, r in zip(self.caches, self.cap, self.rows):
            n = r.shape[1]
            assert self.lib.tg_kv_len(c) == n
            raw = get(self.lib, c, BF16, cap, self.kvd)
            assert np.array_equal(raw[:, :n], bf16(r)[0])

    def close(self):
        self.lib.tg_kv_group_destroy(self.g)
        for c in self.caches + [self.prefix] * (self.prefix is not None):
            self.lib.tg_kv_destroy(c)


def call(s, devbuf, n_new, append=True, decode=False, stream=None):
    """One call on fresh tokens; checks outputs, caches and what lies behind out."""
    lib, total = s.lib, sum(n_new)
    (qb, q), (kb, k), (vb, v) = s.new(total)
    if append:
        s.grow(n_new, k, v)
    qd, kd, vd = devbuf(qb), devbuf(kb), devbuf(vb)
    guard = np.full(qb.size + 4096, 0x55, qb.dtype)
    od = devbuf(guard)
    ptrs = (qd.ptr, kd.ptr if append else None, vd.ptr if append else None, od.ptr, stream)
    if decode:
        tgkv.check(lib.tg_kv_group_decode(s.g, *ptrs), lib, "decode")
    else:
        tgkv.check(lib.tg_kv_group_prompt(s.g, (C.c_uint32 * len(n_new))(*n_new), *ptrs), lib, "prompt")
    assert lib.tg_cuda_kv_sync(stream)
    got = s.read(od, total)
    assert np.all(od.get(qb.dtype, guard.shape)[qb.size:] == 0x55)
    want, tol = s.expect(q, n_new)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    s.check_caches()
    assert lib.tg_cuda_kv_device_error() == 0
    return got


DECODE = [  # old lengths, prefix (None: no cache), heads, kv heads, head_dim
    ([0], None, 1, 1, 64),
    ([0], 0, 4, 2, 128),
    ([0, 1, 5], 1, 8, 8, 64),
    ([127, 128, 129, 0, 63], 127, 16, 4, 128),
    ([300, 31, 2], 128, 12, 4, 128),
    ([500] * 9, 129, 32, 8, 128),
    ([1, 700, 40], 1000, 7, 1, 64),
    (list(range(0, 140, 2)), 640, 16, 2, 128),
    ([2000], 3001, 128, 1, 64),
    ([17] * 40, 4000, 6, 3, 64),
    ([33] * 64, 1030, 32, 8, 128),                           # a long enough prefix for many: shared
    ([5, 0, 300, 9], 20000, 32, 8, 128),                     # shared by four
    ([9000, 20], None, 8, 2, 64),                            # several CTAs per sequence
    ([70000], None, 2, 1, 64),                               # more than 32 CTAs for one row
    ([255, 256, 383], 130, 32, 2, 128),                      # 16 query heads per KV head
    ([90, 4], 200, 36, 2, 128),                              # 18
]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(cuda, devbuf, case, act):
    old, P, nh, nkv, hd = DECODE[case]
    s = Setup(cuda, old, [4] * len(old), P, nh, nkv, hd, act, seed=case)
    ones = [1] * len(old)
    call(s, devbuf, ones, decode=True)
    call(s, devbuf, ones, decode=True)                       # the second step reads the first one's row
    call(s, devbuf, ones, decode=True, append=False)         # other queries of the same last rows
    tgkv.check(cuda.tg_kv_group_truncate(s.g, (C.c_uint32 * len(old))(*old)), cuda)
    s.rows = [r[:, :o] for r, o in zip(s.rows, old)]
    s.check_caches()
    call(s, devbuf, ones, decode=True)
    s.close()


PROMPT = [  # old lengths, new tokens, prefix, heads, kv heads, head_dim
    ([0], [1], None, 1, 1, 64),
    ([0], [130], None, 2, 2, 128),
    ([0, 0, 0], [1, 5, 17], 0, 8, 8, 64),
    ([40, 129, 0, 7], [0, 3, 64, 0], 100, 16, 4, 128),
    ([300, 0, 77], [200, 129, 1], None, 12, 4, 128),
    ([0, 500], [257, 128], 383, 32, 8, 128),
    ([10] * 12, [2, 9, 1, 4, 31, 8, 1, 1, 3, 5, 6, 7], 700, 16, 2, 128),
    ([0, 20], [70, 33], 65, 7, 1, 64),
    ([1500], [600], 900, 4, 1, 64),
    ([0, 0], [3, 2], 50, 128, 1, 128),
    ([10] * 12, [2, 9, 1, 4, 31, 8, 1, 1, 3, 5, 6, 7], 9000, 16, 2, 128),
    ([7] * 20, [6] * 20, 3000, 16, 4, 128),
    ([126, 300, 5], [2, 1, 2], 77, 8, 2, 64),                # few tokens, over a tile's end
    ([125, 0], [5, 3], None, 2, 2, 128),
]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("case", range(len(PROMPT)))
def test_prompt(cuda, devbuf, case, act):
    old, new, P, nh, nkv, hd = PROMPT[case]
    s = Setup(cuda, old, [n + 3 for n in new], P, nh, nkv, hd, act, seed=50 + case)
    call(s, devbuf, new)
    call(s, devbuf, new, append=False)                       # other queries of the rows just appended
    call(s, devbuf, [1] * len(old), decode=True)
    s.close()


def test_scale_with_mscale(cuda, devbuf):
    s = Setup(cuda, [200, 3], [8, 8], 150, 8, 2, 128, F32, seed=7, mscale=1.37)
    call(s, devbuf, [5, 2])
    call(s, devbuf, [1, 1], decode=True)
    s.close()


@pytest.mark.parametrize("act", [F32, BF16])
def test_large_scores(cuda, devbuf, act):
    """Scores in the hundreds: one key takes nearly all the weight."""
    s = Setup(cuda, [260, 140], [8, 8], 300, 8, 2, 128, act, seed=9)
    s.q_scale = 40
    call(s, devbuf, [2, 1])
    s.close()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("new", [None, 40])                 # a decode step, or packed prompts of 40 tokens
def test_repeats_are_identical(cuda, devbuf, act, new):
    """Long stretches per CTA: the same call gives the same bits every time."""
    n = 24
    s = Setup(cuda, [1000 + 37 * i for i in range(n)], [41] * n, 6000, 32, 8, 128, act, seed=3)
    n_new = [new or 1] * n
    (qb, q), (kb, k), (vb, v) = s.new(sum(n_new))
    qd, kd, vd, od = devbuf(qb), devbuf(kb), devbuf(vb), devbuf(nbytes=qb.nbytes)
    arr, first = (C.c_uint32 * n)(*n_new), None
    tgkv.check(cuda.tg_kv_group_prompt(s.g, arr, qd.ptr, kd.ptr, vd.ptr, od.ptr, None), cuda)
    for _ in range(8):
        tgkv.check(cuda.tg_kv_group_prompt(s.g, arr, qd.ptr, None, None, od.ptr, None), cuda)
        assert cuda.tg_cuda_kv_sync(None)
        got = od.get(qb.dtype, qb.shape)
        first = got if first is None else first
        assert np.array_equal(got.view(np.uint8), first.view(np.uint8))
    s.close()


def test_matches_the_single_cache_operators(cuda, devbuf):
    """The same history in one plain cache: tg_kv_append_attention and tg_kv_attention agree."""
    lib, nh, nkv, hd, P = cuda, 16, 4, 128, 200
    s = Setup(lib, [90, 0], [300, 300], P, nh, nkv, hd, F32, seed=21)
    for n_new in ([150, 70], [1, 1]):
        (qb, q), (kb, k), (vb, v) = s.new(sum(n_new))
        before = [r.copy() for r in s.rows]
        s.grow(n_new, k, v)
        qd, kd, vd, od = devbuf(qb), devbuf(kb), devbuf(vb), devbuf(nbytes=qb.nbytes)
        tgkv.check(lib.tg_kv_group_prompt(s.g, (C.c_uint32 * 2)(*n_new), qd.ptr, kd.ptr, vd.ptr, od.ptr, None), lib)
        got, at = s.read(od, sum(n_new)), 0
        for i, t in enumerate(n_new):
            one = lib.tg_kv_create_ex(1000, nkv, hd, BF16)
            put(lib, one, BF16, 1000, s.kvd, np.concatenate([s.prefix_rows, before[i]], 1), JUNK)
            part = [devbuf(np.ascontiguousarray(x[at:at + t])) for x in (kb, vb, qb)]
            o1 = devbuf(nbytes=t * nh * hd * 4)
            tgkv.check(lib.tg_kv_append_attention(one, part[0].ptr, part[1].ptr, part[2].ptr, o1.ptr, nh, t, None), lib)
            assert lib.tg_cuda_kv_sync(None)
            # both sit within 5e-5 of the head's output scale of the 64-bit value
            assert rel_head_err(got[at:at + t], o1.get(np.float32, (t, nh, hd))) < 1e-4
            lib.tg_kv_destroy(one)
            at += t
    s.close()


# ------------------------------------------------------------- row moves
FORK = [(1, 1, 1, 1, 64, F32), (1, 3, 37, 2, 64, F32), (3, 2, 1000, 4, 128, BF16), (2, 5, 513, 1, 128, F32),
        (24, 8, 65, 3, 32, BF16), (2, 1, 0, 4, 64, BF16), (600, 1, 4, 1, 32, BF16)]


@pytest.mark.parametrize("n_src,fan,rows,nkv,hd,dtype", FORK)
def test_fork(cuda, n_src, fan, rows, nkv, hd, dtype):
    lib, kvd = cuda, nkv * hd
    rng = np.random.default_rng(rows)
    src, dst, want, before = [], [], [], []
    for i in range(n_src):
        cap = rows + 1 + i % 3
        src.append(lib.tg_kv_create_ex(cap, nkv, hd, dtype))
        want.append(put(lib, src[-1], dtype, cap, kvd, rng.standard_normal((2, rows + 1, kvd)), JUNK))
    for j in range(n_src * fan):
        cap = rows + 1 + j % 2
        dst.append(lib.tg_kv_create_ex(cap, nkv, hd, dtype))
        before.append(put(lib, dst[-1], dtype, cap, kvd, rng.standard_normal((2, min(j % 3, cap), kvd)), JUNK))
    tgkv.check(lib.tg_kv_fork((C.c_void_p * n_src)(*src), n_src, (C.c_void_p * len(dst))(*dst), fan, rows, None), lib)
    assert lib.tg_cuda_kv_sync(None)
    bits = np.uint16 if dtype == BF16 else np.uint32
    for j, c in enumerate(dst):
        assert lib.tg_kv_len(c) == rows
        raw = get(lib, c, dtype, lib.tg_kv_capacity(c), kvd).view(bits)
        assert np.array_equal(raw[:, :rows], want[j // fan].view(bits)[:, :rows])
        assert np.array_equal(raw[:, rows:], before[j].view(bits)[:, rows:])
    for i, c in enumerate(src):
        assert lib.tg_kv_len(c) == rows + 1
        assert np.array_equal(get(lib, c, dtype, lib.tg_kv_capacity(c), kvd).view(bits), want[i].view(bits))
    for c in src + dst:
        lib.tg_kv_destroy(c)


COMPACT = [  # caches, rows, kv heads, head_dim, dtype, ranges
    (1, 1, 1, 64, F32, "all"), (1, 50, 1, 64, BF16, "none"), (1, 50, 2, 64, F32, "last"),
    (3, 700, 4, 128, BF16, "window"), (1, 20000, 8, 128, BF16, "window"), (2, 5000, 8, 64, F32, 300),
    (24, 900, 4, 128, BF16, 40), (1, 9001, 1, 128, BF16, 1024), (1, 30000, 3, 32, F32, 7),
    (2, 333, 5, 64, BF16, "shift"), (1, 4096, 4, 128, BF16, "halves"), (1, 300, 1, 8, BF16, 9),
]


@pytest.mark.parametrize("n,rows,nkv,hd,dtype,kind", COMPACT)
def test_compact(cuda, n, rows, nkv, hd, dtype, kind):
    lib, kvd, cap = cuda, nkv * hd, rows + 3
    rng = np.random.default_rng(rows + n)
    if kind == "all":
        start, count = [0], [rows]
    elif kind == "none":
        start, count = [], []
    elif kind == "last":
        start, count = [rows - 1], [1]
    elif kind == "window":                                   # 4 sinks and the last third
        start, count = [0, rows - rows // 3], [4, rows // 3]
    elif kind == "shift":                                    # everything moves by one row
        start, count = [1], [rows - 1]
    elif kind == "halves":                                   # adjoining ranges, nothing dropped between
        start, count = [1, 101, 2000], [100, 1899, rows - 2000]
    else:
        cuts = np.sort(rng.choice(rows + 1, 2 * kind, replace=False))
        start, count = list(cuts[0::2]), list(cuts[1::2] - cuts[0::2])
    index = np.concatenate([np.arange(a, a + c) for a, c in zip(start, count)] + [np.arange(0)]).astype(int)
    caches, before = [], []
    for i in range(n):
        caches.append(lib.tg_kv_create_ex(cap, nkv, hd, dtype))
        before.append(put(lib, caches[-1], dtype, cap, kvd, rng.standard_normal((2, rows, kvd)), JUNK))
    tgkv.check(lib.tg_kv_compact((C.c_void_p * n)(*caches), n, (C.c_uint32 * len(start))(*start),
                                 (C.c_uint32 * len(start))(*count), len(start), None), lib)
    assert lib.tg_cuda_kv_sync(None)
    bits = np.uint16 if dtype == BF16 else np.uint32
    for c, b in zip(caches, before):
        assert lib.tg_kv_len(c) == len(index)
        raw = get(lib, c, dtype, cap, kvd).view(bits)
        assert np.array_equal(raw[:, :len(index)], b.view(bits)[:, index])
        assert np.array_equal(raw[:, len(index):], b.view(bits)[:, len(index):])   # the rest as it was
        lib.tg_kv_destroy(c)


# ------------------------------------------------------- used together, and refused
def test_a_thousand_sequences(cuda, devbuf):
    n = 1024
    s = Setup(cuda, [i % 7 for i in range(n)], [2] * n, 300, 2, 1, 64, BF16, seed=31)
    call(s, devbuf, [1] * n, decode=True)
    call(s, devbuf, [(i % 3 == 0) * 1 for i in range(n)])
    s.close()


def test_on_a_stream_and_replayed_from_a_graph(cuda, devbuf):
    """A step on its own stream, then captured once and replayed over new inputs in the same buffers."""
    import torch
    lib, n = cuda, 6
    s = Setup(lib, [50 * i for i in range(n)], [40] * n, 700, 16, 4, 128, BF16, seed=41)
    stream = torch.cuda.Stream()
    handle = C.c_void_p(stream.cuda_stream)
    call(s, devbuf, [1] * n, decode=True, stream=handle)
    call(s, devbuf, [3, 0, 31, 1, 2, 5], stream=handle)
    old = [r.shape[1] for r in s.rows]
    (qb, _), (kb, _), (vb, _) = s.new(n)
    qd, kd, vd, od = devbuf(qb), devbuf(kb), devbuf(vb), devbuf(nbytes=qb.nbytes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        tgkv.check(lib.tg_kv_group_decode(s.g, qd.ptr, kd.ptr, vd.ptr, od.ptr, handle), lib)
    before = s.rows
    for _ in range(3):                           # each replay stores the row at the captured length
        (qb, q), (kb, k), (vb, v) = s.new(n)
        for d, b in ((qd, qb), (kd, kb), (vd, vb)):
            assert lib.tg_cuda_kv_h2d(d.ptr, b.ctypes.data, b.nbytes, None)
        graph.replay()
        torch.cuda.synchronize()
        s.rows = [r[:, :o] for r, o in zip(before, old)]
        s.grow([1] * n, k, v)
        want, tol = s.expect(q, [1] * n)
        assert (np.abs(s.read(od, n) - want) <= tol).all()
        s.check_caches()
    del graph
    s.close()


def test_two_groups_over_one_prefix(cuda, devbuf):
    """Groups with their own caches and scratch, on two streams at once."""
    import torch
    lib = cuda
    a = Setup(lib, [100, 40, 7], [9] * 3, 2000, 8, 2, 128, F32, seed=51)
    b = Setup(lib, [300, 2], [9] * 2, None, 8, 2, 128, F32, seed=52)
    lib.tg_kv_group_destroy(b.g)
    b.g = lib.tg_kv_group_create(a.prefix, b.arr, 2, 8, F32)
    tgkv.check(b.g, lib)
    b.P, b.prefix_rows = a.P, a.prefix_rows
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s, st in zip((a, b), streams):
        n = len(s.old)
        (qb, q), (kb, k), (vb, v) = s.new(n)
        bufs = devbuf(qb), devbuf(kb), devbuf(vb), devbuf(nbytes=qb.nbytes)
        s.grow([1] * n, k, v)
        outs.append((s, q, n, bufs))
    for _ in range(4):
        for (s, q, n, bufs), st in zip(outs, streams):
            ptrs = [x.ptr for x in bufs]
            lens = (C.c_uint32 * n)(*s.old)
            tgkv.check(lib.tg_kv_group_truncate(s.g, lens), lib)
            tgkv.check(lib.tg_kv_group_decode(s.g, *ptrs, C.c_void_p(st.cuda_stream)), lib)
    torch.cuda.synchronize()
    for s, q, n, bufs in outs:
        want, tol = s.expect(q, [1] * n)
        assert (np.abs(s.read(bufs[3], n) - want) <= tol).all()
        s.check_caches()
    b.close()
    a.close()


def test_a_serving_loop(cuda, devbuf):
    """A system prompt through tg_kv_append_attention, chats behind it, a fork, an eviction, and on."""
    lib, nh, nkv, hd, P = cuda, 16, 4, 128, 150
    s = Setup(lib, [0, 0, 0], [400] * 3, 0, nh, nkv, hd, F32, seed=61)
    lib.tg_kv_group_destroy(s.g)                             # a prefix cache with room, filled through the API
    lib.tg_kv_destroy(s.prefix)
    s.prefix = lib.tg_kv_create_ex(P + 50, nkv, hd, BF16)
    s.g = lib.tg_kv_group_create(s.prefix, s.arr, 3, nh, F32)
    tgkv.check(s.g, lib)
    (qb, q), (kb, k), (vb, v) = s.new(P)
    bufs = [devbuf(x) for x in (kb, vb, qb)] + [devbuf(nbytes=qb.nbytes)]
    tgkv.check(lib.tg_kv_append_attention(s.prefix, *[x.ptr for x in bufs], nh, P, None), lib)
    s.P, s.prefix_rows = P, np.stack([bf16(k)[1], bf16(v)[1]])
    call(s, devbuf, [90, 0, 33])
    call(s, devbuf, [1, 1, 1], decode=True)
    # chat 1 becomes a branch of chat 0 (its own rows), then both go on
    tgkv.check(lib.tg_kv_fork((C.c_void_p * 1)(s.caches[0]), 1, (C.c_void_p * 1)(s.caches[1]), 1, 60, None), lib)
    s.rows[1] = s.rows[0][:, :60]
    s.check_caches()
    call(s, devbuf, [2, 40, 1])
    # chat 0 keeps its first 4 and last 50 positions
    n0 = s.rows[0].shape[1]
    tgkv.check(lib.tg_kv_compact((C.c_void_p * 1)(s.caches[0]), 1, (C.c_uint32 * 2)(0, n0 - 50), (C.c_uint32 * 2)(4, 50),
                                 2, None), lib)
    s.rows[0] = np.concatenate([s.rows[0][:, :4], s.rows[0][:, n0 - 50:]], 1)
    s.check_caches()
    call(s, devbuf, [1, 1, 1], decode=True)
    # the prefix grows: all sequences see it from the next call on
    extra = s.rng.standard_normal((2, 20, s.kvd)).astype(np.float32)
    tgkv.check(lib.tg_kv_append(s.prefix, extra[0].ctypes.data, extra[1].ctypes.data, 20), lib)
    s.prefix_rows = np.concatenate([s.prefix_rows, bf16(extra)[1]], 1)
    call(s, devbuf, [5, 1, 0])
    s.close()


@pytest.mark.parametrize("act", [F32, BF16])
def test_a_nan_query_stays_in_its_row(cuda, devbuf, act):
    s = Setup(cuda, [200, 10, 40], [8, 8, 8], 300, 8, 2, 128, act, seed=71)
    n_new = [40, 1, 3]
    s.cap = [c + 40 for c in s.cap]
    normal = s.new

    def new(total):
        (qb, q), k, v = normal(total)
        qb, q = qb.copy().reshape(total, 8, 128), q.copy().reshape(total, 8, 128)
        qb[5, 3] = 0x7fc0 if act == BF16 else np.nan
        q[5, 3] = np.nan
        return [(qb.reshape(total, -1), q.reshape(total, -1)), k, v]
    s.new = new
    (qb, q), _, _ = s.new(44)
    qd, od = devbuf(qb), devbuf(nbytes=qb.nbytes)
    tgkv.check(cuda.tg_kv_group_prompt(s.g, (C.c_uint32 * 3)(*n_new), qd.ptr, None, None, od.ptr, None), cuda)
    assert cuda.tg_cuda_kv_sync(None)
    got, (want, tol) = s.read(od, 44), s.expect(q, n_new)
    assert np.isnan(got[5, 3]).all()
    rest = ~np.isnan(want)
    assert rest.sum() == want.size - 128 and (np.abs(got - want)[rest] <= tol[rest]).all()
    s.close()


NON_FINITE = [  # old lengths, new tokens, prefix, heads, kv heads, head_dim
    ([0, 100], [300, 40], 70, 8, 2, 128),                    # pairs of row tiles, sequences joined with the prefix
    ([60], [700], None, 2, 2, 64),                           # 256 tokens an item
    ([5, 5, 5, 5, 5, 5], [70] * 6, 9000, 16, 4, 128),        # the prefix shared
    ([5000], [200], 300, 6, 2, 128),                         # an item over several CTAs, or in pieces
    ([3, 126, 255, 0], [2, 2, 1, 2], 40, 8, 2, 128),         # few rows
    ([125, 9000], [3, 3], None, 6, 2, 64),
]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("case", range(len(NON_FINITE)))
def test_non_finite_values_reach_only_who_sees_them(cuda, devbuf, case, act):
    """NaN and infinities among a call's own V: queries before them are as if they
    were not there, those that see them have something non-finite in their dims and
    in no others: exactly the sum with bf16 activations."""
    old, new, P, nh, nkv, hd = NON_FINITE[case]
    s = Setup(cuda, old, [n + 3 for n in new], P, nh, nkv, hd, act, seed=90 + case)
    total = sum(new)
    (qb, q), (kb, k), (vb, v) = s.new(total)
    bad = np.zeros_like(v)
    at = 0
    for i, t in enumerate(new):
        bad[at + t - 1, (3 * i + 1) % s.kvd] = np.nan
        bad[at + t // 2, [5, 9, s.kvd - 1]] = np.inf, -np.inf, np.inf
        bad[at + (3 * t) // 4, [9, 7]] = np.inf, -np.inf      # dim 9 gets both infinities
        if t > 64:
            bad[at + 33, s.kvd // 2:] = np.inf                # half a row
        at += t
    raw = np.where(bad != 0, bad, v).astype(np.float32)
    clean = np.where(bad != 0, 0, v)
    s.grow(new, k, clean)
    qd, kd, vd = devbuf(qb), devbuf(kb), devbuf(bf16(raw)[0] if act == BF16 else raw)
    od = devbuf(nbytes=qb.nbytes)
    for again in (False, True):                               # with the rows appended, then as they lie there
        tgkv.check(cuda.tg_kv_group_prompt(s.g, (C.c_uint32 * len(new))(*new), qd.ptr, None if again else kd.ptr,
                                           None if again else vd.ptr, od.ptr, None), cuda)
        assert cuda.tg_cuda_kv_sync(None)
        got, (want, tol) = s.read(od, total), s.expect(q, new)
        at = 0
        for t in new:
            with np.errstate(invalid="ignore"):
                add = np.cumsum(bad[at:at + t], 0).reshape(t, nkv, hd).repeat(nh // nkv, 1)
                want[at:at + t] += add
            at += t
        fin = np.isfinite(want)
        assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all()
        if act == BF16:
            assert np.array_equal(got[~fin], want[~fin], equal_nan=True)
        else:
            # a weight enters as hi + lo parts, and lo is often 0 or below it: 0 x Inf and Inf - Inf
            # are NaN, so an infinity that a whole item sees may come out as NaN
            assert not np.isfinite(got[~fin]).any()
        assert cuda.tg_cuda_kv_device_error() == 0
    s.close()


@pytest.mark.parametrize("as_prefix", [False, True])
def test_offsets_past_32_bits(cuda, devbuf, as_prefix):
    """Halves of 4.5 GB.  K is zero, so every weight is 1 and a result is the sum of the
    few V rows that are not zero over the length: one rounding of the output, and the
    division's."""
    lib, nkv, hd, n = cuda, 8, 128, 2_200_000
    kvd, cap, rng = nkv * hd, 2_200_001, np.random.default_rng(123)
    mk = lambda cap: lib.tg_kv_create_ex(cap, nkv, hd, BF16)  # noqa: E731
    big, copy, small = mk(cap), mk(cap), mk(8)
    tgkv.check(big and copy and small, lib)
    at = [0, 1, n // 2, n - 2, n - 1]
    bits, v = bf16(rng.standard_normal((len(at), kvd)) * 2.0 ** 20)
    row = lambda c, r, half=1: lib.tg_kv_device_handle(c) + (half * cap + r) * kvd * 2  # noqa: E731
    for r, b in zip(at, bits):
        assert lib.tg_cuda_kv_h2d(row(big, r), b.ctypes.data, b.nbytes, None)
    lib.tg_kv_advance(big, n)
    caches = (C.c_void_p * 1)(small if as_prefix else big)
    g = lib.tg_kv_group_create(big if as_prefix else None, caches, 1, 16, BF16)
    tgkv.check(g, lib)
    new_bits, new = bf16(rng.standard_normal((1, kvd)) * 2.0 ** 20)
    q, k = devbuf(bf16(rng.standard_normal((1, 16 * hd)))[0]), devbuf(np.zeros((1, kvd), np.uint16))
    vd, od = devbuf(new_bits), devbuf(nbytes=16 * hd * 2)
    tgkv.check(lib.tg_kv_group_decode(g, q.ptr, k.ptr, vd.ptr, od.ptr, None), lib)
    assert lib.tg_cuda_kv_sync(None)
    import oracle as O
    got = O.bf16_to_f32(od.get(np.uint16, (nkv, 2, hd))).astype(np.float64)
    want = ((v.sum(0) + new[0]) / (n + 1)).reshape(nkv, 1, hd)
    mag = ((np.abs(v).sum(0) + np.abs(new[0])) / (n + 1)).reshape(nkv, 1, hd)
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * mag).all()
    assert lib.tg_cuda_kv_device_error() == 0
    if not as_prefix:
        def read(c, r):
            out = np.empty(kvd, np.uint16)
            assert lib.tg_cuda_kv_d2h(out.ctypes.data, row(c, r), out.nbytes, None) and lib.tg_cuda_kv_sync(None)
            return out
        assert np.array_equal(read(big, n), new_bits[0])
        tgkv.check(lib.tg_kv_fork((C.c_void_p * 1)(big), 1, (C.c_void_p * 1)(copy), 1, n + 1, None), lib)
        every = list(zip(at + [n], np.concatenate([bits, new_bits])))
        assert all(np.array_equal(read(copy, r), b) for r, b in every)
        start, count = (C.c_uint32 * 3)(1, n // 2, n - 2), (C.c_uint32 * 3)(1, 1, 3)
        tgkv.check(lib.tg_kv_compact((C.c_void_p * 1)(copy), 1, start, count, 3, None), lib)
        assert lib.tg_kv_len(copy) == 5
        assert all(np.array_equal(read(copy, i), b) for i, (_, b) in enumerate(every[1:]))
    lib.tg_kv_group_destroy(g)
    for c in (big, copy, small):
        lib.tg_kv_destroy(c)


def test_refusals_change_nothing(cuda, devbuf):
    lib = cuda
    mk = lambda cap=64, nkv=2, hd=64, dt=BF16: lib.tg_kv_create_ex(cap, nkv, hd, dt)  # noqa: E731
    a, b, p = mk(), mk(), mk()
    f32, other, wide, hd32 = mk(dt=F32), mk(nkv=4), mk(hd=128), mk(hd=32)
    arr = lambda *c: (C.c_void_p * len(c))(*c)  # noqa: E731
    u = lambda *x: (C.c_uint32 * len(x))(*x)  # noqa: E731
    err = lambda: lib.tg_kv_last_error()  # noqa: E731
    for caches, pre, nh, act, why in [
            (arr(a, a), None, 4, F32, b"twice"), (arr(a, b), a, 4, F32, b"twice"), (arr(a, other), None, 4, F32, b"differs"),
            (arr(a, wide), None, 4, F32, b"differs"), (arr(a, f32), None, 4, F32, b"differs"), (arr(a), f32, 4, F32, b"differs"),
            (arr(f32), None, 4, F32, b"no attention kernel"), (arr(hd32), None, 4, F32, b"no attention kernel"),
            (arr(a), None, 3, F32, b"multiple"), (arr(a), None, 0, F32, b"multiple"), (arr(a), None, 258, F32, b"128 times"),
            (arr(a), None, 4, 7, b"invalid dtype")]:
        assert not lib.tg_kv_group_create(pre, caches, len(caches), nh, act)
        assert why in err(), (why, err())
    for c in (a, b, p):
        lib.tg_kv_advance(c, 60)
    g = lib.tg_kv_group_create(p, arr(a, b), 2, 4, F32)
    d = devbuf(nbytes=1 << 20)
    args = (d.ptr, d.ptr, d.ptr, d.ptr, None)
    assert lib.tg_kv_group_prompt(g, u(4, 5), *args) == 0 and b"capacity exceeded at cache 1" in err()
    assert lib.tg_kv_group_prompt(g, u(1, 61), d.ptr, None, None, d.ptr, None) == 0 and b"61 queries" in err()
    assert lib.tg_kv_group_decode(g, d.ptr, d.ptr, None, d.ptr, None) == 0 and b"together" in err()
    assert lib.tg_kv_group_decode(g, d.ptr + 4, d.ptr, d.ptr, d.ptr, None) == 0 and b"16-byte" in err()
    assert lib.tg_kv_group_truncate(g, u(10, 61)) == 0 and b"beyond" in err()
    lib.tg_kv_set_attn_mscale(b, 1.5)
    assert lib.tg_kv_group_decode(g, *args) == 0 and b"mscale" in err()
    for c in (a, b, p):
        lib.tg_kv_set_attn_mscale(c, -1.0)
    assert lib.tg_kv_group_decode(g, *args) == 0 and b"positive" in err()
    assert lib.tg_kv_group_prompt(g, u(0, 0), d.ptr, None, None, d.ptr, None) == 0
    for c in (a, b, p):
        lib.tg_kv_set_attn_mscale(c, 1.0)
    assert lib.tg_kv_group_prompt(g, u(0, 0), *args) == 1                   # nothing to do
    assert lib.tg_kv_fork(arr(a), 1, arr(a), 1, 3, None) == 0 and b"source" in err()
    assert lib.tg_kv_fork(arr(a), 1, arr(b, b), 2, 3, None) == 0 and b"twice" in err()
    assert lib.tg_kv_fork(arr(a), 1, arr(b), 1, 61, None) == 0 and b"61 rows" in err()
    assert lib.tg_kv_fork(arr(a), 1, arr(other), 1, 3, None) == 0 and b"differs" in err()
    tiny = mk(cap=2)
    assert lib.tg_kv_fork(arr(a), 1, arr(tiny), 1, 3, None) == 0 and b"capacity" in err()
    assert lib.tg_kv_compact(arr(a, a), 2, u(0), u(1), 1, None) == 0 and b"twice" in err()
    assert lib.tg_kv_compact(arr(a, tiny), 2, u(0), u(1), 1, None) == 0 and b"rows" in err()
    assert lib.tg_kv_compact(arr(a), 1, u(59), u(2), 1, None) == 0 and b"beyond length 60" in err()
    assert lib.tg_kv_compact(arr(a), 1, u(5, 6), u(2, 2), 2, None) == 0 and b"out of order" in err()
    assert [lib.tg_kv_len(c) for c in (a, b, p, tiny)] == [60, 60, 60, 0]
    # a cache of another device (by what its record says; nothing runs): the record's seventh word
    device = C.c_int32.from_address(b + 24)
    assert device.value == lib.tg_cuda_kv_device()
    device.value += 1
    assert not lib.tg_kv_group_create(None, arr(a, b), 2, 4, F32) and b"cache 1 lies on device" in err()
    assert not lib.tg_kv_group_create(b, arr(a), 1, 4, F32) and b"prefix: cache 0 lies on device" in err()
    assert lib.tg_kv_fork(arr(a), 1, arr(b), 1, 3, None) == 0 and b"copies: cache 0 lies on device" in err()
    assert lib.tg_kv_fork(arr(b), 1, arr(a), 1, 3, None) == 0 and b"lies on device" in err()
    assert lib.tg_kv_compact(arr(a, b), 2, u(0), u(1), 1, None) == 0 and b"cache 1 lies on device" in err()
    device.value -= 1
    assert [lib.tg_kv_len(c) for c in (a, b, p, tiny)] == [60, 60, 60, 0]
    lib.tg_kv_group_destroy(g)
    for c in (a, b, p, f32, other, wide, hd32, tiny):
        lib.tg_kv_destroy(c)
