"""The serving operators around the MoE layer, as cases to be timed and compared: block tables and
slot maps (``extend``), rotary positions (``rope``), writing keys and values into the 8-bit paged
cache (``append``, read back with ``read``) and attention over that cache (``attend``).

``own`` chooses between the operators' plain form (elementary torch operations in 32 bits) and
this package's entry points (``rusty_engine_b200.kv``).  Cache layout, in both: codes
[blocks, kv heads, block size, head dim], one f32 scale per block and head for K and for V.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest code
TINY = 1.1754943508222875e-38  # the smallest normal f32: a smaller scale is 0


# ---- cases --------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a handful of requests: the smallest table update
        dict(name="extend-decode-8", op="extend", reqs=8, new=1, ctx=500, block=16),
        # admission of a large batch: ragged prompts beside requests that add one token
        dict(name="extend-prompts-512", op="extend", reqs=512, new=1024, ctx=4000, block=64),
        # q and k of a decode batch, in the f32 that the stack's projections give
        dict(name="rope-decode-f32", op="rope", tokens=16, nq=32, nkv=4, dim=128, rot=128, layout="half", scaling="none",
             dtype="f32", fused=False, max_pos=8192),
        # a long-context prompt: interleaved pairs on half of the head, YaRN, views of one fused qkv buffer
        dict(name="rope-prompt-bf16", op="rope", tokens=8192, nq=32, nkv=4, dim=128, rot=64, layout="interleaved",
             scaling="yarn", dtype="bf16", fused=True, max_pos=131072),
        # the cache write of one decode step (a token per request, blocks partly filled), rope of q and k with it
        dict(name="append-decode-f32", op="append", reqs=32, new=1, ctx=3000, nq=32, nkv=4, dim=128, rot=128,
             layout="half", block=16, code="int8", dtype="f32", rope=True),
        # the cache write of a prompt batch, rope of q and k with it
        dict(name="append-prompt-bf16", op="append", reqs=4, new=2048, ctx=0, nq=32, nkv=4, dim=128, rot=128,
             layout="half", block=64, code="int8", dtype="bf16", rope=True),
        # chunks of odd length behind earlier context, e4m3 codes, no rope (positions learned elsewhere)
        dict(name="append-chunk-e4m3", op="append", reqs=5, new=247, ctx=777, nq=16, nkv=8, dim=64, rot=0, layout="half",
             block=32, code="e4m3", dtype="f16", rope=False),
        # one request, one token, a short context: latency
        dict(name="attend-decode-1-f32", op="attend", reqs=1, new=1, long=1, ctx=97, nq=32, nkv=4, dim=128, block=16,
             code="int8", dtype="f32", window=0),
        # a decode batch of ragged contexts
        dict(name="attend-decode-32", op="attend", reqs=32, new=1, long=1, ctx=8192, nq=32, nkv=4, dim=128, block=64,
             code="int8", dtype="bf16", window=0),
        # long contexts of few requests: the cache is split over the whole chip
        dict(name="attend-decode-long", op="attend", reqs=2, new=1, long=1, ctx=131071, nq=32, nkv=4, dim=128, block=128,
             code="e4m3", dtype="f16", window=0),
        # the 2048-token prompt of the stack benchmark, in the stack's f32
        dict(name="attend-prompt-f32", op="attend", reqs=1, new=2048, long=2048, ctx=2048, nq=32, nkv=4, dim=128, block=64,
             code="int8", dtype="f32", window=0),
        # continuous batching: a prompt chunk of one request beside decoding ones
        dict(name="attend-mixed-bf16", op="attend", reqs=4, new=1, long=4096, ctx=8192, nq=32, nkv=4, dim=128, block=64,
             code="int8", dtype="bf16", window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["extend", "rope", "append", "append", "attend", "attend", "attend"])
    block = rng.choice([16, 32, 64, 128])
    if op == "extend":
        reqs = _log(rng, 1, 512)
        return dict(op=op, reqs=reqs, new=rng.choice([1, _log(rng, 1, min(4096, 262144 // reqs))]), ctx=_log(rng, 1, 8000),
                    block=block)
    dim = rng.choice([64, 128, 128, 256])
    nkv = rng.choice([1, 2, 4, 8])
    nq = nkv * rng.choice([1, 4, 5, 8]) if dim < 256 else nkv * rng.choice([1, 2, 4])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    layout = rng.choice(["half", "interleaved"])
    rot = rng.choice([dim, dim, dim // 2])
    if op == "rope":
        tokens = min(32768, _log(rng, 1, 8192 * 30 * 128 * 2 // ((nq + nkv) * dim * SIZE[dtype])))
        return dict(op=op, tokens=tokens, nq=nq, nkv=nkv, dim=dim, rot=rot, layout=layout,
                    scaling=rng.choice(["none", "linear", "yarn"]), dtype=dtype, fused=rng.random() < 0.5,
                    max_pos=_log(rng, max(2048, tokens), 131072))
    code = rng.choice(["int8", "int8", "e4m3"])
    if op == "append":
        if rng.random() < 0.5:
            reqs, new = _log(rng, 1, 64), rng.choice([1, 1, 2])
        else:
            reqs = rng.choice([1, 2, 5])
            new = _log(rng, 3, 1 + 2048 * 4 * 128 * 2 // (reqs * dim * nkv * SIZE[dtype]) // max(1, nq // nkv // 4))
            new = min(new, 8192 // reqs)
        return dict(op=op, reqs=reqs, new=new, ctx=rng.choice([0, _log(rng, 1, 4000)]), nq=nq, nkv=nkv, dim=dim, rot=rot,
                    layout=layout, block=block, code=code, dtype=dtype, rope=rng.random() < 0.7)
    kind = rng.choice(["decode", "decode", "prompt", "mixed"])
    per = nkv * dim  # cache bytes of a token, and a measure of a head's work
    if kind == "decode":
        reqs, new = _log(rng, 1, 48), rng.choice([1, 1, 1, 2, 3])
        ctx = max(new, _log(rng, 1, min(131071, 131071 * 2 * 512 // (reqs * per))))
        return dict(op=op, reqs=reqs, new=new, long=new, ctx=ctx, nq=nq, nkv=nkv, dim=dim, block=block, code=code,
                    dtype=dtype, window=rng.choice([0, 0, 0, 1024]))
    reqs = rng.choice([1, 2, 3, 4]) if kind == "mixed" else 1
    ctx = _log(rng, 17, min(8192, int(4096 * math.sqrt(4096 / (nq * dim)))))
    long = ctx if kind == "prompt" else max(1, ctx // rng.choice([2, 3, 5]))
    return dict(op=op, reqs=reqs, new=1, long=long, ctx=ctx, nq=nq, nkv=nkv, dim=dim, block=block, code=code, dtype=dtype,
                window=rng.choice([0, 0, 0, 1024]))


def _spread(r, top):
    """A length between a quarter of `top` and `top`, the same for every seed (request 0: `top`)."""
    return max(1, int(top * (1.0 - 0.75 * ((r * 0.6180339887) % 1.0))))


def _lengths(c):
    """(tokens in the cache after the call, new tokens of the call) of every request."""
    if c["op"] == "attend":
        new = [c["long"] if r == 0 else c["new"] for r in range(c["reqs"])]
        return [max(new[r], _spread(r, c["ctx"])) for r in range(c["reqs"])], new
    if c["op"] == "append":
        new = [c["new"]] * c["reqs"]
        return [(_spread(r, c["ctx"]) if c["ctx"] else 0) + new[r] for r in range(c["reqs"])], new
    new = [_spread(r, c["new"]) if r % 2 == 0 else 1 for r in range(c["reqs"])]
    return [_spread(r, c["ctx"]) + new[r] for r in range(c["reqs"])], new


def _pairs(n, new, window):
    """Visible (query, key) pairs of a request with n cached tokens, its last `new` being queries."""
    total = 0
    for lo, hi in ((n - new + 1, n),):  # query i sees min(position + 1, window) keys
        if window and lo <= window < hi:
            total += (lo + window) * (window - lo + 1) // 2 + (hi - window) * window
        elif window and lo > window:
            total += (hi - lo + 1) * window
        else:
            total += (lo + hi) * (hi - lo + 1) // 2
    return total


def work(case):
    c = case
    if c["op"] == "extend":
        lens, new = _lengths(c)
        blocks = sum(-(-n // c["block"]) - -(-(n - m) // c["block"]) for n, m in zip(lens, new))
        return {"bytes": 16 * c["reqs"] + 8 * sum(new) + 8 * blocks, "flops": 2 * sum(new)}
    es = SIZE[c["dtype"]]
    if c["op"] == "rope":
        rows = c["tokens"] * (c["nq"] + c["nkv"])
        return {"bytes": 2 * rows * c["dim"] * es + c["tokens"] * (4 + c["rot"] * 4), "flops": rows * c["rot"] * 3}
    lens, new = _lengths(c)
    t = sum(new)
    if c["op"] == "append":
        kv = t * c["nkv"] * c["dim"] * 2
        touched = sum(-(-n // c["block"]) - (n - m) // c["block"] for n, m in zip(lens, new))
        moved = kv * es + kv + kv * es + touched * c["nkv"] * 8  # in, codes, read back, scales
        if c["rope"]:
            moved += 2 * t * c["nq"] * c["dim"] * es + t * (4 + c["rot"] * 4)
        return {"bytes": moved + 8 * t, "flops": kv * 4 + (t * (c["nq"] + c["nkv"]) * c["rot"] * 3 if c["rope"] else 0)}
    seen = [min(n, m + c["window"] - 1) if c["window"] else n for n, m in zip(lens, new)]
    cache = sum(seen) * c["nkv"] * c["dim"] * 2 + sum(-(-n // c["block"]) for n in seen) * (c["nkv"] * 8 + 4)
    flops = 4 * c["nq"] * c["dim"] * sum(_pairs(n, m, c["window"]) for n, m in zip(lens, new))
    return {"bytes": cache + t * c["nq"] * (2 * c["dim"] * es + 4), "flops": flops}


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _frequencies(c):
    """Angle per position of each pair, in 64 bits, and the factor of cos and sin."""
    rot, base = c["rot"], 1e6
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    scaling = c.get("scaling", "none")
    if scaling == "linear":
        return [x / 4.0 for x in f], 1.0
    if scaling == "yarn":
        factor, orig = 4.0, 32768
        at = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        keep = [1.0 - min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        return [x * k + x / factor * (1.0 - k) for x, k in zip(f, keep)], 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rope_plan(c, max_pos):
    if own:
        from rusty_engine_b200 import kv

        scaling = {"none": kv.RopeScaling.NoScaling, "linear": kv.RopeScaling.Linear, "yarn": kv.RopeScaling.Yarn}
        layout = {"half": kv.RopeLayout.Half, "interleaved": kv.RopeLayout.Interleaved}
        s = scaling[c.get("scaling", "none")]
        cfg = kv.RopeConfig(rot_dim=c["rot"], base=1e6, layout=layout[c["layout"]], scaling=s,
                            factor=1.0 if s == kv.RopeScaling.NoScaling else 4.0, orig_ctx=32768)
        return kv.Rope(cfg, max_pos)
    f, m = _frequencies(c)
    angle = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * torch.tensor(f, device="cuda", dtype=torch.float64)
    return ((angle.cos() * m).float(), (angle.sin() * m).float())


def _qkv(c, g, t):
    """q, k, v [t, heads, dim]: keys with a few strong channels, as trained models have."""
    nq, nkv, d, dt = c["nq"], c["nkv"], c["dim"], DTYPES[c["dtype"]]
    loud = 1.0 + 4.0 * (torch.rand((1, nkv, d), generator=g, device="cuda") < 0.05)
    return (2.0 * _randn(g, t, nq, d)).to(dt), (_randn(g, t, nkv, d) * loud).to(dt), _randn(g, t, nkv, d).to(dt)


def _codes(c, g, n):
    x = _randn(g, n, c["nkv"], c["block"], c["dim"])
    if c["code"] == "int8":
        return (x * 32.0).round().clamp(-127, 127).to(torch.int8)
    return (x * 100.0).clamp(-448, 448).to(torch.float8_e4m3fn)


def _cache(c, g, n):
    """Codes and scales of n blocks, as a running server's cache holds them (stale blocks too)."""
    one = 1.0 / (32.0 if c["code"] == "int8" else 100.0)
    scale = lambda: one * (0.7 + 0.6 * torch.rand((n, c["nkv"]), generator=g, device="cuda"))  # noqa: E731
    s = {"k": _codes(c, g, n), "v": _codes(c, g, n), "ks": scale(), "vs": scale()}
    if own:
        from rusty_engine_b200 import kv

        s["cache"] = kv.KVCache.from_buffers(s["k"], s["v"], s["ks"], s["vs"])
    return s


def _table(c, g, lens):
    """A block table for these lengths, blocks in random order; entries past a request's end are -1."""
    need = [-(-n // c["block"]) for n in lens]
    n = sum(need)
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    inside = torch.arange(width, device="cuda")[None] < _ints(need)[:, None]
    table[inside] = order
    return table, max(1, n)


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = {"case": c}
    if c["op"] == "rope":
        s["rope"] = _rope_plan(c, c["max_pos"])
        q, k, v = _qkv(c, g, c["tokens"])
        if c["fused"]:  # views of the one buffer that a fused projection writes
            both = torch.cat((q, k, v), dim=1)
            q, k = both[:, :c["nq"]], both[:, c["nq"]:c["nq"] + c["nkv"]]
        last = torch.randint(c["tokens"] - 1, c["max_pos"], (1,), generator=g, device="cuda")
        s |= {"q": q, "k": k, "positions": (last - c["tokens"] + 1 + torch.arange(c["tokens"], device="cuda")).to(torch.int32)}
        return s
    lens, new = _lengths(c)
    if c["op"] == "extend":
        off = torch.randint(0, c["block"], (c["reqs"],), generator=g, device="cuda").to(torch.int32)
        before = _ints([n - m for n, m in zip(lens, new)]) + off
        have = (before + c["block"] - 1) // c["block"]
        width = max(-(-(n + c["block"]) // c["block"]) for n in lens) + 3
        table = torch.full((c["reqs"], width), -1, dtype=torch.int32, device="cuda")
        blocks = sum(-(-(n + c["block"]) // c["block"]) for n in lens) + 17
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        inside = torch.arange(width, device="cuda")[None] < have[:, None]
        used = int(have.sum())
        table[inside] = order[:used]
        s |= {"table": table, "lens": before, "new": _ints(new), "free": order[used:].contiguous(),
              "n_free": _ints([blocks - used]), "total": sum(new), "block": c["block"]}
        return s
    table, blocks = _table(c, g, lens)
    s |= _cache(c, g, blocks)
    q, k, v = _qkv(c, g, sum(new))
    s["q"] = q
    if c["op"] == "append":
        # where extend puts these tokens, request after request
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).cuda()
        req = torch.cat([torch.full((m,), r) for r, m in enumerate(new)]).cuda()
        s |= {"k_new": k, "v_new": v, "positions": pos.to(torch.int32),
              "slots": (table[req, pos // c["block"]] * c["block"] + pos % c["block"]).to(torch.int32)}
        if c["rope"]:
            s["rope"] = _rope_plan(c, max(lens))
        return s
    s |= {"table": table, "lens": _ints(lens), "cu": _ints([sum(new[:r]) for r in range(c["reqs"] + 1)]),
          "max_new": max(new), "scale": 1.0 / math.sqrt(c["dim"])}
    return s


# ---- the operators, plain -----------------------------------------------------------------------
def _extend(s):
    lens, table, free, bs, total = s["lens"], s["table"], s["free"], s["block"], s["total"]
    new = s["new"].clamp(min=0)
    cu = torch.cat((new.new_zeros(1), new.cumsum(0))).to(torch.int32)
    have = (lens + bs - 1) // bs
    fits = (lens + new <= table.shape[1] * bs) & (cu[1:] <= total)
    need = torch.where(fits, (lens + new + bs - 1) // bs - have, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= s["n_free"]))
    # the j-th new block of request r is the (upto - need + j)-th from the top of the free stack
    col = torch.arange(table.shape[1], device="cuda")[None]
    j = col - have[:, None]
    at = s["n_free"] - 1 - (upto - need)[:, None] - j
    fresh = granted[:, None] & (j >= 0) & (j < need[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    t = torch.arange(total, device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True)
    inside = r < lens.numel()
    r = r.clamp(max=lens.numel() - 1)
    pos = torch.where(inside, lens[r] + (t - cu[r]), 0)
    slot = table[r, (pos // bs).clamp(max=table.shape[1] - 1)] * bs + pos % bs
    slot = torch.where(inside & granted[r], slot, -1)
    left = s["n_free"] - torch.where(granted, upto, 0).amax()
    return {"table": table, "cu": cu, "positions": pos.to(torch.int32), "slots": slot.to(torch.int32),
            "lens": torch.where(granted, lens + new, lens).to(torch.int32), "n_free": left.to(torch.int32)}


def _rotate(x, cos, sin, rot, layout):
    """x [t, heads, dim] in f32, cos and sin [t, rot / 2]."""
    c, n = cos[:, None], sin[:, None]
    y = x.clone()
    if layout == "half":
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = x0 * c - x1 * n, x1 * c + x0 * n
    else:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = x0 * c - x1 * n, x1 * c + x0 * n
    return y


def _rope(s):
    c, (cos, sin) = s["case"], s["rope"]
    cos, sin = cos[s["positions"]], sin[s["positions"]]
    return {n: _rotate(s[n].float(), cos, sin, c["rot"], c["layout"]).to(s[n].dtype) for n in ("q", "k")}


def _round(x, code):
    x = torch.where(x.isnan(), 0.0, x).clamp(-TOP[code], TOP[code])
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _write(x, codes, scales, slots, code):
    """x [t, heads, dim] f32 into the cache: one scale per block and head, grown where the new tokens need it."""
    bs = codes.shape[2]
    page, off = slots // bs, slots % bs
    before = torch.cat((slots.new_full((1,), -2), slots[:-1]))
    lead = (off == 0) | (before != slots - 1)  # the first token of each run in one block
    run = lead.cumsum(0) - 1
    at, first = page[lead].long(), off[lead]
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(dim=-1)
    amax = torch.zeros((at.numel(), x.shape[1]), device="cuda").index_reduce_(0, run, top, "amax")
    want = amax / TOP[code]
    want = torch.where(want < TINY, 0.0, want)
    old = torch.where(first[:, None] > 0, scales[at], 0.0)
    scale = torch.maximum(old, want)
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    held = codes[at]
    again = _round(held.float() * (old * inv)[:, :, None, None], code)
    keep = torch.arange(bs, device="cuda")[None] < first[:, None]
    raw = lambda v: v.view(torch.uint8)  # noqa: E731
    raw(codes)[at] = torch.where(keep[:, None, :, None], raw(again), raw(held))
    scales[at] = scale
    raw(codes)[page.long(), :, off.long()] = raw(_round(x * inv[run][:, :, None], code))


def _append(s):
    c = s["case"]
    k, v, slots = s["k_new"].float(), s["v_new"].float(), s["slots"]
    out = {}
    if c["rope"]:
        cos, sin = (x[s["positions"]] for x in s["rope"])
        k = _rotate(k, cos, sin, c["rot"], c["layout"])
        out["q"] = _rotate(s["q"].float(), cos, sin, c["rot"], c["layout"]).to(s["q"].dtype)
    page, off = (slots // c["block"]).long(), (slots % c["block"]).long()
    for name, x, codes, scales in (("k", k, s["k"], s["ks"]), ("v", v, s["v"], s["vs"])):
        _write(x, codes, scales, slots, c["code"])
        out[name] = (codes[page, :, off].float() * scales[page][:, :, None]).to(s["q"].dtype)
    return out | {"ks": s["ks"], "vs": s["vs"]}


def _attend(s):
    q, table, lens, cu, bs = s["q"], s["table"], s["lens"], s["cu"], s["case"]["block"]
    reqs, wide, heads, dim, rows = table.shape[0], table.shape[1] * bs, s["case"]["nkv"], q.shape[2], s["max_new"]
    group, at = q.shape[1] // heads, table.clamp(min=0).long()
    key = torch.arange(wide, device="cuda")
    held = (key[None] < lens[:, None])[:, None, :, None]
    gather = lambda x, n: (x[at].float() * n[at][..., None, None]).transpose(1, 2).reshape(reqs, heads, wide, dim)  # noqa: E731
    k, v = gather(s["k"], s["ks"]), gather(s["v"], s["vs"])
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    new = cu[1:] - cu[:-1]
    i = torch.arange(rows, device="cuda")
    real = i[None] < new[:, None]
    x = q[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)].float()  # [reqs, rows, q heads, dim]
    x = x.view(reqs, rows, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(reqs, heads, rows * group, dim)
    p = torch.matmul(x, k.transpose(2, 3)).mul_(s["scale"])
    pos = (lens - new)[:, None] + i
    seen = key <= pos[..., None]
    if s["case"]["window"]:
        seen &= key > pos[..., None] - s["case"]["window"]
    p = p.view(reqs, heads, rows, group, wide).masked_fill_(~seen[:, None, :, None], -math.inf)
    m = p.amax(dim=-1, keepdim=True)
    p = p.sub_(torch.where(m.isinf(), 0.0, m)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(reqs, heads, rows * group, wide), v).view(reqs, heads, rows, group, dim)
    o = (o / torch.where(total > 0, total, 1.0)).permute(0, 2, 1, 3, 4).reshape(reqs, rows, heads * group, dim)
    lse = (m + total.log()).squeeze(-1).permute(0, 2, 1, 3).reshape(reqs, rows, heads * group)
    return {"out": o[real].to(q.dtype), "lse": lse[real]}


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"extend": _extend, "rope": _rope, "append": _append, "attend": _attend}[op](s)
    if op == "extend":
        from rusty_engine_b200 import kv

        step = kv.extend_tables(s["table"], s["lens"], s["new"], s["free"], s["n_free"], s["total"], s["block"])
        return {"table": s["table"], "cu": step.cu, "positions": step.positions, "slots": step.slots, "lens": step.lens,
                "n_free": step.n_free}
    if op == "rope":
        q, k = s["rope"].apply(s["q"], s["positions"], s["k"])
        return {"q": q, "k": k}
    if op == "append":
        q = s["cache"].append(s["k_new"], s["v_new"], s["slots"], rope=s.get("rope"), positions=s["positions"],
                              q=s["q"] if "rope" in s else None)
        k, v = s["cache"].read(s["slots"], s["q"].dtype)
        return ({"q": q} if q is not None else {}) | {"k": k, "v": v, "ks": s["ks"], "vs": s["vs"]}
    out, lse = s["cache"].attend(s["q"], s["table"], s["lens"], s["cu"], scale=s["scale"], window=s["case"]["window"],
                                 max_new=s["max_new"], return_lse=True)
    return {"out": out, "lse": lse}


# ---- 64 bits, from the definitions --------------------------------------------------------------
def _exact_angles(c, positions):
    f, m = _frequencies(c)
    a = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    return a, m


def _exact_rope(c, x, positions):
    """Each pair as a complex number times m * exp(i * angle)."""
    a, m = _exact_angles(c, positions)
    turn = torch.polar(torch.full_like(a, m), a)[:, None]
    x, rot = x.double().clone(), c["rot"]
    if c["layout"] == "half":
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        x[..., :rot // 2], x[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * turn
        x[..., :rot] = torch.view_as_real(z).flatten(-2)
    return x


def _exact_round(x, code):
    if code == "int8":
        return x.round().clamp(-127, 127)
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e): steps of 2^(e-4), of 2^-9 below 2^-6
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(c, s):
    lens, new = _lengths(c)
    bs, out = c["block"], {}
    k, v = s["k_new"].double(), s["v_new"].double()
    if c["rope"]:
        out["q"], k = _exact_rope(c, s["q"], s["positions"]), _exact_rope(c, s["k_new"], s["positions"])
    slots = s["slots"].tolist()
    for name, x, scales in (("k", k, s["ks"].double().clone()), ("v", v, s["vs"].double().clone())):
        y, t, ends = torch.empty_like(x), 0, []
        for n, m in zip(lens, new):  # a request's tokens, block by block
            p = n - m
            while p < n:
                q = min(n, (p // bs + 1) * bs)
                ends.append((t, t + q - p, slots[t] // bs, p % bs))
                t, p = t + q - p, q
        for t0, t1, b, first in ends:
            scale = x[t0:t1].abs().amax(dim=2).amax(dim=0) / TOP[c["code"]]
            if first:
                scale = torch.maximum(scale, scales[b])
            scales[b] = scale
            y[t0:t1] = _exact_round(x[t0:t1] / scale[None, :, None], c["code"]) * scale[None, :, None]
        out[name], out[name + "s"] = y, scales
    return out


def _exact_attend(c, s):
    lens, new = _lengths(c)
    group, d, bs, at = c["nq"] // c["nkv"], c["dim"], c["block"], 0
    outs, lses = [], []
    for r, (n, m) in enumerate(zip(lens, new)):
        blocks = s["table"][r, :-(-n // bs)].long()
        o = torch.empty((m, c["nq"], d), dtype=torch.float64, device="cuda")
        lse = torch.empty((m, c["nq"]), dtype=torch.float64, device="cuda")
        key, pos = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda")[:, None]
        hidden = (key > pos) | (key <= pos - c["window"]) if c["window"] else key > pos
        for h in range(c["nq"]):
            g = h // group
            k = (s["k"][blocks, g].double() * s["ks"][blocks, g].double()[:, None, None]).reshape(-1, d)[:n]
            v = (s["v"][blocks, g].double() * s["vs"][blocks, g].double()[:, None, None]).reshape(-1, d)[:n]
            z = (s["q"][at:at + m, h].double() @ k.T) * s["scale"]
            z[hidden] = -math.inf
            lse[:, h] = torch.logsumexp(z, dim=1)
            o[:, h] = torch.exp(z - lse[:, h:h + 1]) @ v
        outs.append(o)
        lses.append(lse)
        at += m
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def exact(case, seed):
    c = case
    if c["op"] == "extend":
        return None  # whole numbers: equal or not
    s = prepare(c, seed)
    if c["op"] == "rope":
        return {n: _exact_rope(c, s[n], s["positions"]) for n in ("q", "k")}
    return _exact_append(c, s) if c["op"] == "append" else _exact_attend(c, s)
