"""TEST INFRASTRUCTURE ONLY: the paged 8-bit KV cache operators restated plainly on the CPU, the
checkers of tests/test_kv*.py: block tables as Python loops, rotary positions and attention in
float64, the cache's codes in the float32 steps that define them."""
from __future__ import annotations

import math

import numpy as np
import torch

TINY = np.float32(1.1754943508222875e-38)
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def extend(table, lens, new, free, n_free, total, bs):
    """Python loops over requests and tokens; tables and lists of ints."""
    R, mb = len(lens), len(table[0]) if table else 0
    table = [list(r) for r in table]
    cu, pos, slots, out = [0], [0] * total, [-1] * total, []
    taken, ran_out = 0, False
    for r in range(R):
        n, ln = max(new[r], 0), max(lens[r], 0)
        first = cu[-1]
        cu.append(first + n)
        have, want = -(-ln // bs), -(-(ln + n) // bs)
        fits = ln + n <= mb * bs and first + n <= total
        need = want - have if fits else 0
        ok = fits and (need == 0 or (not ran_out and taken + need <= n_free))
        if fits and not ok:
            ran_out = True
        if ok:
            for j in range(need):
                table[r][have + j] = free[n_free - 1 - taken - j]
            taken += need
        out.append(ln + n if ok else lens[r])
        for i in range(n):
            t, p = first + i, ln + i
            if t < total:
                pos[t] = p
                if ok and table[r][p // bs] >= 0:
                    slots[t] = table[r][p // bs] * bs + p % bs
    return table, cu, pos, slots, out, n_free - taken


def frequencies(rot, base, scaling="none", factor=1.0, orig=0, fast=32.0, slow=1.0, ff=None):
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    m = 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        at = lambda n: rot * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
        g = [1 - min(max((i - lo) / max(hi - lo, 0.001), 0), 1) for i in range(rot // 2)]
        f = [x * k + x / factor * (1 - k) for x, k in zip(f, g)]
        m = 0.1 * math.log(factor) + 1
    if ff is not None:
        f = [x / float(np.float32(y)) for x, y in zip(f, ff)]
    return np.array(f), m


def rope(x, positions, freq, m, half, inverse=False):
    """x [T, heads, d] -> float64, every pair turned by position * freq and scaled by m."""
    x = x.double().cpu().numpy().copy()
    rot = 2 * len(freq)
    a = np.asarray(positions, dtype=np.float64)[:, None] * freq[None] * (-1 if inverse else 1)
    c, s = (m * np.cos(a))[:, None], (m * np.sin(a))[:, None]
    i0 = np.arange(rot // 2) if half else np.arange(0, rot, 2)
    i1 = i0 + rot // 2 if half else i0 + 1
    x0, x1 = x[..., i0].copy(), x[..., i1].copy()
    x[..., i0], x[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    return torch.from_numpy(x)


def e4m3_round(x):
    """float32 -> the nearest e4m3 value (ties to even), saturating: the format's definition."""
    x = np.clip(np.asarray(x, dtype=np.float64), -448, 448)
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 4, -9).astype(np.float64))
    return np.clip(np.round(x / step) * step, -448, 448).astype(np.float32)


def code_round(x, code):
    x = np.where(np.isnan(x), np.float32(0), x)
    return np.clip(np.round(np.clip(x, -127, 127)), -127, 127).astype(np.float32) if code == "int8" else e4m3_round(x)


def append(values, scales, x, slots, bs, code):
    """One of K / V: values [blocks, heads, bs, d] (the codes as float32 numbers) and scales
    [blocks, heads], both changed in place; x [T, heads, d] float32."""
    per = np.float32(1.0) / np.float32(127.0 if code == "int8" else 448.0)
    t, T = 0, len(slots)
    while t < T:
        if slots[t] < 0:
            t += 1
            continue
        b, first, n = slots[t] // bs, slots[t] % bs, 1
        while t + n < T and first + n < bs and slots[t + n] == slots[t] + n:
            n += 1
        for h in range(x.shape[1]):
            new = x[t:t + n, h]
            mag = np.abs(new[np.isfinite(new)])
            want = np.float32(mag.max() if mag.size else 0) * per
            want = np.float32(0) if want < TINY else want
            old = scales[b, h] if first else np.float32(0)
            s = max(old, want)
            inv = np.float32(1) / s if s > 0 else np.float32(0)
            values[b, h, :first] = code_round(values[b, h, :first] * (old * inv), code)
            with np.errstate(invalid="ignore", over="ignore"):
                values[b, h, first:first + n] = code_round(new * inv, code)
            scales[b, h] = s
        t += n


def attend(q, k, v, ks, vs, table, lens, cu, scale, window=0):
    """q [T, heads, d]; k, v values [blocks, kv heads, bs, d] with scales; float64 (out, lse)."""
    q, k, v, ks, vs = (np.asarray(torch.as_tensor(a).double().cpu()) for a in (q, k, v, ks, vs))
    T, nq, d = q.shape
    nkv, bs = k.shape[1], k.shape[2]
    out, lse = np.zeros((T, nq, d)), np.full((T, nq), -np.inf)
    for r in range(len(lens)):
        n, m = lens[r], cu[r + 1] - cu[r]
        blocks = [b for b in table[r][: -(-max(n, 0) // bs)]]
        for h in range(nq):
            g = h // (nq // nkv)
            if not blocks or m <= 0:
                continue
            kk = (k[blocks, g] * ks[blocks, g][:, None, None]).reshape(-1, d)[:n]
            vv = (v[blocks, g] * vs[blocks, g][:, None, None]).reshape(-1, d)[:n]
            for i in range(m):
                p = n - m + i
                lo, hi = (max(0, p - window + 1) if window else 0), p + 1
                if hi <= 0:
                    continue
                z = kk[lo:hi] @ q[cu[r] + i, h] * scale
                top = z.max()
                e = np.exp(z - top)
                out[cu[r] + i, h] = e @ vv[lo:hi] / e.sum()
                lse[cu[r] + i, h] = top + np.log(e.sum())
    return torch.from_numpy(out), torch.from_numpy(lse)
