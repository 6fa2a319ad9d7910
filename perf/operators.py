"""The operators over groups of KV caches, as cases to measure.

Four operators of one serving loop: sequences that share a prefix (a system
prompt) take packed prompts of different lengths, decode one token each per
step, and have rows of their caches forked and compacted.

  decode   one token of each of n sequences attends a prefix that all share and
           its own cache, where its K/V row is appended first (`append`), or
           was appended before the call
  prompt   n_new[i] tokens of each sequence, packed, causal over the prefix (if
           any) and the sequence's own cache, where they are appended first
  fork     the first rows of each source cache copied into `fan` others
  compact  ranges of a cache's positions moved to its front, in place

A cache is [2][capacity][kv_heads * head_dim], K then V.  With `own` false,
run() computes the plain form with elementary torch operations; with `own`
true it calls libtgkv.so as a user's program does.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # two chats just opened on a short system prompt: the latency of one call
        {"name": "decode 2 short", "op": "decode", "n": 2, "prefix": 64, "own_min": 0, "own_max": 32,
         "heads": 8, "kv_heads": 8, "head_dim": 64, "act": "f32", "append": True, "pick": 1},
        # a small server: 16 chats on a 1k system prompt
        {"name": "decode 16 x 1k prefix", "op": "decode", "n": 16, "prefix": 1024, "own_min": 64,
         "own_max": 512, "heads": 16, "kv_heads": 4, "head_dim": 128, "act": "bf16",
         "append": True, "pick": 2},
        # many short questions about one document, odd sizes, a group of 3 query heads, fp32 activations;
        # the rows were appended with the rotation
        {"name": "decode 200 x 4099 prefix", "op": "decode", "n": 200, "prefix": 4099, "own_min": 0,
         "own_max": 299, "heads": 12, "kv_heads": 4, "head_dim": 128, "act": "f32",
         "append": False, "pick": 3},
        # 64 long chats about one 32k document: the largest batch
        {"name": "decode 64 x 32k prefix", "op": "decode", "n": 64, "prefix": 32768, "own_min": 1000,
         "own_max": 4000, "heads": 32, "kv_heads": 8, "head_dim": 128, "act": "bf16",
         "append": False, "pick": 4},
        # three tiny turns in one call
        {"name": "prompt 3 tiny", "op": "prompt", "n": 3, "prefix": 0, "own_min": 0, "own_max": 130,
         "new_min": 1, "new_max": 17, "heads": 8, "kv_heads": 8, "head_dim": 64, "act": "f32", "pick": 5},
        # eight chat turns of 64-512 tokens behind their kept history, fp32 activations
        {"name": "prompt 8 turns", "op": "prompt", "n": 8, "prefix": 0, "own_min": 300, "own_max": 2000,
         "new_min": 64, "new_max": 512, "heads": 16, "kv_heads": 4, "head_dim": 128, "act": "f32", "pick": 6},
        # 32 whole prompts of 1 to 2048 tokens into empty caches
        {"name": "prompt 32 ragged", "op": "prompt", "n": 32, "prefix": 0, "own_min": 0, "own_max": 0,
         "new_min": 1, "new_max": 2048, "heads": 32, "kv_heads": 8, "head_dim": 128, "act": "bf16", "pick": 7},
        # 6 long prompts behind an 8k system prompt: the largest dense work
        {"name": "prompt 6 long, 8k prefix", "op": "prompt", "n": 6, "prefix": 8192, "own_min": 0,
         "own_max": 100, "new_min": 1000, "new_max": 8000, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "act": "bf16", "pick": 8},
        # three branches of one short fp32 cache
        {"name": "fork 1 into 3", "op": "fork", "layers": 1, "fan": 3, "rows": 37, "kv_heads": 2,
         "head_dim": 64, "cache": "f32"},
        # five samples of one 2000-token chat, twelve layers
        {"name": "fork 12 layers into 5", "op": "fork", "layers": 12, "fan": 5, "rows": 2000,
         "kv_heads": 4, "head_dim": 128, "cache": "bf16"},
        # odd ranges kept in four small fp32 caches (eviction by score)
        {"name": "compact 4 x 300 ranges", "op": "compact", "layers": 4, "len": 5000, "ranges": 300,
         "kv_heads": 8, "head_dim": 64, "cache": "f32", "pick": 9},
        # 24 layers of a 32k chat shrink to 4 sinks and the last 16k positions
        {"name": "compact 24 x 32k window", "op": "compact", "layers": 24, "len": 32768, "ranges": 2,
         "kv_heads": 4, "head_dim": 128, "cache": "bf16", "pick": 0},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    heads, kv = rng.choice([(8, 8), (16, 4), (32, 8), (12, 4), (16, 2), (7, 1)])
    hd = rng.choice([64, 128, 128])
    act = rng.choice(["f32", "bf16"])
    pick = rng.randrange(1 << 20)
    op = rng.choice(["decode", "decode", "prompt", "prompt", "fork", "compact"])
    if op == "decode":
        n, append = _log(rng, 1, 200), rng.random() < 0.5
        n = min(n, 60) if append else n                        # each sequence's new rows are an output
        hi = _log(rng, 1, 4000)
        return {"op": op, "n": n, "prefix": rng.choice([0, _log(rng, 1, 16000), _log(rng, 64, 16000)]),
                "own_min": rng.randrange(hi), "own_max": hi, "heads": heads, "kv_heads": kv,
                "head_dim": hd, "act": act, "append": append, "pick": pick}
    if op == "prompt":
        n = _log(rng, 1, 32)
        hi = _log(rng, 1, 2048)
        old = _log(rng, 1, 3000)
        return {"op": op, "n": n, "prefix": rng.choice([0, _log(rng, 1, 4000)]),
                "own_min": rng.randrange(old), "own_max": old, "new_min": rng.randrange(hi) + 1,
                "new_max": hi, "heads": heads, "kv_heads": kv, "head_dim": hd, "act": act, "pick": pick}
    if op == "fork":
        fan = rng.randrange(8) + 1
        return {"op": op, "layers": _log(rng, 1, 60 // fan), "fan": fan, "rows": _log(rng, 1, 2000),
                "kv_heads": kv, "head_dim": hd, "cache": act}
    length = _log(rng, 64, 8000)
    return {"op": op, "layers": _log(rng, 1, 24), "len": length, "ranges": rng.randrange(min(400, length // 16)) + 1,
            "kv_heads": kv, "head_dim": hd, "cache": act, "pick": pick}


def _lengths(case):
    """(rows each sequence's cache holds before the call, rows it gets), from the case alone."""
    r = random.Random(case["pick"])
    old = [r.randint(case["own_min"], case["own_max"]) for _ in range(case["n"])]
    if case["op"] == "decode":
        return old, [1] * case["n"]
    return old, [r.randint(case["new_min"], case["new_max"]) for _ in range(case["n"])]


def _kept(case):
    """The kept ranges (first positions, counts) of a compaction, from the case alone."""
    n, k = case["len"], case["ranges"]
    if case["pick"] == 0:
        return [0, n // 2], [4, n - n // 2]
    r = random.Random(case["pick"])
    cuts = sorted(r.sample(range(n), 2 * k))
    return cuts[0::2], [b - a for a, b in zip(cuts[0::2], cuts[1::2])]


def work(case):
    kv_dim = case["kv_heads"] * case["head_dim"]
    if case["op"] in ("decode", "prompt"):
        old, new = _lengths(case)
        es = 4 if case["act"] == "f32" else 2
        row = 2 * 2 * kv_dim                                   # K and V of a position, bf16
        pairs = sum(n * (case["prefix"] + o) + n * (n + 1) // 2 for o, n in zip(old, new))
        moved = (case["prefix"] + sum(old) + sum(new)) * row   # cached rows read; new rows written, or read
        acts = sum(new) * (2 * case["heads"] * case["head_dim"] + (2 * kv_dim if case.get("append", True) else 0)) * es
        return {"bytes": moved + acts, "flops": 4 * case["head_dim"] * case["heads"] * pairs}
    row = 2 * kv_dim * (4 if case["cache"] == "f32" else 2)
    if case["op"] == "fork":
        return {"bytes": case["layers"] * case["rows"] * (1 + case["fan"]) * row, "flops": 0}
    at, n = 0, 0
    for s, c in zip(*_kept(case)):
        n += c if s != at else 0                               # rows that stay need no copy
        at += c
    return {"bytes": case["layers"] * n * 2 * row, "flops": 0}


# ------------------------------------------------------------------ state
class _Handle:
    """The caches of a state (and the group over them), freed with it."""

    def __init__(self, lib):
        self.lib, self.caches, self.group, self.extra = lib, [], None, []

    def cache(self, capacity, kv_heads, head_dim, dtype, rows):
        """A cache whose first rows are `rows` ([2][n][kv_dim]), and its buffer as a tensor."""
        c = self.lib.tg_kv_create_ex(capacity, kv_heads, head_dim, 1 if dtype == torch.bfloat16 else 0)
        assert c, self.lib.tg_kv_last_error()
        self.caches.append(c)
        view = _tensor(self, self.lib.tg_kv_device_handle(c), (2, capacity, kv_heads * head_dim), dtype)
        if rows is not None:
            view[:, :rows.shape[1]] = rows
            self.lib.tg_kv_advance(c, rows.shape[1])
        return c, view

    def __del__(self):
        torch.cuda.synchronize()
        if self.group:
            self.lib.tg_kv_group_destroy(self.group)
        for c in self.caches:
            self.lib.tg_kv_destroy(c)


class _Memory:
    """Part of a cache as torch sees it; keeps the owner, so that a tensor outlives its state."""

    def __init__(self, owner, address, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (address, False), "shape": shape, "typestr": kind, "version": 3}


def _tensor(owner, address, shape, dtype):
    """Device memory of `owner` as a tensor, without a copy."""
    if dtype == torch.bfloat16:
        return torch.as_tensor(_Memory(owner, address, shape, "<i2"), device=DEV).view(torch.bfloat16)
    return torch.as_tensor(_Memory(owner, address, shape, "<f4"), device=DEV)


def _library():
    at = os.path.join(os.getcwd(), "tgai-go_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tgkv
    lib = tgkv.load()
    tgkv.check(lib.tg_be_select(b"cuda"), lib, "tg_be_select")
    return tgkv, lib


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kv_dim = case["kv_heads"] * case["head_dim"]
    if case["op"] in ("decode", "prompt"):
        return _prepare_attention(case, g, kv_dim)
    dtype = DT[case["cache"]]
    s = {"case": case}
    if case["op"] == "fork":
        rows, L, fan = case["rows"], case["layers"], case["fan"]
        s["src"] = [_normal(g, 2, rows, kv_dim).to(dtype) for _ in range(L)]
        if own:
            tgkv, lib = _library()
            h = s["h"] = _Handle(lib)
            src = [h.cache(rows, case["kv_heads"], case["head_dim"], dtype, x)[0] for x in s["src"]]
            dst = [h.cache(rows + 64, case["kv_heads"], case["head_dim"], dtype, None) for _ in range(L * fan)]
            s["src_c"], s["dst_c"] = (tgkv.C.c_void_p * L)(*src), (tgkv.C.c_void_p * (L * fan))(*[c for c, _ in dst])
            s["dst"] = [v[:, :rows] for _, v in dst]
        else:
            s["dst"] = [torch.zeros(2, rows + 64, kv_dim, device=DEV, dtype=dtype)[:, :rows] for _ in range(L * fan)]
        return s
    start, count = _kept(case)
    s["start"], s["count"], s["kept"] = start, count, sum(count)
    s["index"] = torch.cat([torch.arange(a, a + c) for a, c in zip(start, count)]).to(DEV)
    bufs = [_normal(g, 2, case["len"], kv_dim).to(dtype) for _ in range(case["layers"])]
    if own:
        tgkv, lib = _library()
        h = s["h"] = _Handle(lib)
        made = [h.cache(case["len"], case["kv_heads"], case["head_dim"], dtype, b) for b in bufs]
        bufs = [v for _, v in made]
        s["caches"] = [c for c, _ in made]
        s["caches_c"] = (tgkv.C.c_void_p * len(made))(*s["caches"])
        s["start_c"], s["count_c"] = (tgkv.u32 * len(start))(*start), (tgkv.u32 * len(start))(*count)
    s["bufs"] = bufs
    s["out"] = [b[:, :s["kept"]] for b in bufs]
    return s


def _prepare_attention(case, g, kv_dim):
    old, new = _lengths(case)
    n, act, cap = case["n"], DT[case["act"]], max(o + t for o, t in zip(old, new))
    total = sum(new)
    s = {"case": case, "old": old, "new": new}
    s["prefix"] = _normal(g, 2, case["prefix"], kv_dim).bfloat16()
    s["q"] = _normal(g, total, case["heads"], case["head_dim"]).to(act)
    s["k"], s["v"] = _normal(g, total, kv_dim).to(act), _normal(g, total, kv_dim).to(act)
    # the sequences' caches in one block, rows behind a sequence's length unused
    s["block"] = _normal(g, n, 2, cap, kv_dim).bfloat16()
    s["old_t"] = torch.tensor(old, device=DEV)
    s["append"] = case.get("append", True)
    held = old
    if not s["append"]:                                        # decode over rows that are there already
        at, held = torch.arange(n, device=DEV), [o + 1 for o in old]
        s["block"][at, 0, s["old_t"]] = s["k"].bfloat16()
        s["block"][at, 1, s["old_t"]] = s["v"].bfloat16()
    if own:
        tgkv, lib = _library()
        h = s["h"] = _Handle(lib)
        geo = (case["kv_heads"], case["head_dim"], torch.bfloat16)
        made = [h.cache(cap, *geo, s["block"][i, :, :held[i]]) for i in range(n)]
        prefix = h.cache(case["prefix"], *geo, s["prefix"])[0] if case["prefix"] else None
        h.group = lib.tg_kv_group_create(prefix, (tgkv.C.c_void_p * n)(*[c for c, _ in made]), n, case["heads"],
                                         tgkv.TG_KV_BF16 if case["act"] == "bf16" else tgkv.TG_KV_F32)
        tgkv.check(h.group, lib, "tg_kv_group_create")
        s["old_c"], s["new_c"] = (tgkv.u32 * n)(*old), (tgkv.u32 * n)(*new)
        s["out"] = torch.empty_like(s["q"])
        s["rows"] = [v[:, o:o + t] for (_, v), o, t in zip(made, old, new)]
        s["block"] = None
        s["ptr"] = [tgkv.ptr(s[x]) if x in ("q", "out") or s["append"] else None for x in ("q", "k", "v", "out")]
    else:
        s["rows"] = [s["block"][i, :, o:o + t] for i, (o, t) in enumerate(zip(old, new))]
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"decode": _plain_decode, "prompt": _plain_prompt, "fork": _plain_fork,
            "compact": _plain_compact}[s["case"]["op"]](s)


def _run_own(s):
    tgkv, lib = _library_loaded()
    case, h = s["case"], s["h"]
    stream = tgkv.stream_handle()
    op = case["op"]
    if op == "fork":
        ok = lib.tg_kv_fork(s["src_c"], case["layers"], s["dst_c"], case["fan"], case["rows"], stream)
        result = s["dst"]
    elif op == "compact":
        ok = lib.tg_kv_compact(s["caches_c"], case["layers"], s["start_c"], s["count_c"], case["ranges"], stream)
        for c in s["caches"]:                      # the next pass compacts caches of the same length
            lib.tg_kv_advance(c, case["len"] - s["kept"])
        result = s["out"]
    else:
        # back to the lengths before the call, then the step
        ok = not s["append"] or lib.tg_kv_group_truncate(h.group, s["old_c"])
        q, k, v, out = s["ptr"]
        if op == "decode":
            ok = ok and lib.tg_kv_group_decode(h.group, q, k, v, out, stream)
        else:
            ok = ok and lib.tg_kv_group_prompt(h.group, s["new_c"], q, k, v, out, stream)
        result = [s["out"], s["rows"]] if s["append"] else [s["out"]]
    tgkv.check(ok, lib, op)
    return result


def _library_loaded():
    import tgkv
    return tgkv, tgkv.load()


def _softmax(x):
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return x / x.sum(-1, keepdim=True)


def _plain_decode(s):
    case = s["case"]
    n, kvh, hd, P = case["n"], case["kv_heads"], case["head_dim"], case["prefix"]
    G, block, old = case["heads"] // kvh, s["block"], s["old_t"]
    at = torch.arange(n, device=DEV)
    if s["append"]:
        block[at, 0, old] = s["k"].bfloat16()
        block[at, 1, old] = s["v"].bfloat16()
    q = s["q"].float().view(n, kvh, G, hd) * hd ** -0.5
    kp, vp = s["prefix"].float().view(2, P, kvh, hd).permute(0, 2, 1, 3)                   # [kvh][P][hd]
    ki, vi = block.float().view(n, 2, -1, kvh, hd).permute(1, 0, 3, 2, 4)                  # [n][kvh][cap][hd]
    cap = ki.shape[2]
    # stale rows behind a sequence's end take no part
    seen = torch.arange(cap, device=DEV) <= old[:, None]
    sp = q.permute(1, 0, 2, 3).reshape(kvh, n * G, hd) @ kp.transpose(1, 2)
    si = (q @ ki.transpose(2, 3)).masked_fill(~seen[:, None, None], float("-inf"))
    p = _softmax(torch.cat([sp.view(kvh, n, G, P).transpose(0, 1), si], -1))
    out = (p[..., :P].transpose(0, 1).reshape(kvh, n * G, P) @ vp).view(kvh, n, G, hd).transpose(0, 1)
    out = out + p[..., P:] @ vi.masked_fill(~seen[:, None, :, None], 0.0)
    out = out.reshape(n, case["heads"], hd).to(s["q"].dtype)
    return [out, s["rows"]] if s["append"] else [out]


def _plain_prompt(s):
    case = s["case"]
    kvh, hd, P = case["kv_heads"], case["head_dim"], case["prefix"]
    G, at, outs = case["heads"] // kvh, 0, []
    for i, (o, t) in enumerate(zip(s["old"], s["new"])):       # ragged: one sequence after another
        part = slice(at, at + t)
        at += t
        s["rows"][i][0] = s["k"][part].bfloat16()
        s["rows"][i][1] = s["v"][part].bfloat16()
        kv = torch.cat([s["prefix"], s["block"][i, :, :o + t]], 1).float().view(2, P + o + t, kvh, 1, hd)
        k, v = kv.permute(0, 2, 3, 1, 4)                                                   # [kvh][1][L][hd]
        q = s["q"][part].float().view(t, kvh, G, hd).permute(1, 2, 0, 3) * hd ** -0.5
        later = torch.arange(P + o + t, device=DEV) > torch.arange(P + o, P + o + t, device=DEV)[:, None]
        p = _softmax((q @ k.transpose(2, 3)).masked_fill_(later, float("-inf")))
        outs.append((p @ v).permute(2, 0, 1, 3).reshape(t, case["heads"], hd).to(s["q"].dtype))
    return [torch.cat(outs), s["rows"]]


def _plain_fork(s):
    fan = s["case"]["fan"]
    for i, d in enumerate(s["dst"]):
        d.copy_(s["src"][i // fan])
    return s["dst"]


def _plain_compact(s):
    for b, o in zip(s["bufs"], s["out"]):
        o.copy_(b[:, s["index"]])
    return s["out"]


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """What run() returns, from the definition, in 64 bits and sequence by sequence."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "fork":
        return [x.double() for x in s["src"] for _ in range(case["fan"])]
    if case["op"] == "compact":
        place = [a + j for a, c in zip(s["start"], s["count"]) for j in range(c)]
        place = torch.tensor(place, device=DEV)
        return [torch.index_select(b, 1, place).double() for b in s["bufs"]]
    H, kvh, hd, P = case["heads"], case["kv_heads"], case["head_dim"], case["prefix"]
    outs, rows, at = [], [], 0
    for i, (o, t) in enumerate(zip(s["old"], s["new"])):
        k_new, v_new = s["k"][at:at + t].double(), s["v"][at:at + t].double()
        rows.append(torch.stack([k_new, v_new]))
        # what the cache holds of the new rows is their bf16 rounding
        keys = torch.cat([s["prefix"][0].double(), s["block"][i, 0, :o].double(), k_new.bfloat16().double()])
        values = torch.cat([s["prefix"][1].double(), s["block"][i, 1, :o].double(), v_new.bfloat16().double()])
        out = torch.empty(t, H, hd, dtype=torch.float64, device=DEV)
        first = P + o
        for h in range(H):
            c = h * kvh // H * hd
            score = s["q"][at:at + t, h].double() @ keys[:, c:c + hd].T / hd ** 0.5
            past = torch.ones_like(score, dtype=torch.bool).tril(first)
            score = torch.where(past, score, float("-inf"))
            weight = (score - score.max(1, keepdim=True).values).exp()
            out[:, h] = weight @ values[:, c:c + hd] / weight.sum(1, keepdim=True)
        outs.append(out)
        at += t
    return [torch.cat(outs), rows] if s["append"] else [torch.cat(outs)]
