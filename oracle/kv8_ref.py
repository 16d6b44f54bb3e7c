"""Paged 8-bit KV cache from its definitions, in numpy: the oracle of the
kv8 operators. Pools are dicts of int8 codes `k`, `v` [pages, KV, P, D] and
E8M0 bytes `k_exp`, `v_exp` [pages, KV]."""
import math

import numpy as np


def pow2(e):
    """2^(e - 127), NaN for 255, in 64 bits."""
    return np.where(e == 255, np.nan, np.ldexp(1.0, np.asarray(e, np.int64) - 127))


def scale_byte(amax: float) -> int:
    """The smallest e >= 0 with amax <= 127 * 2^(e - 127); 255 when amax is not finite."""
    if not np.isfinite(amax):
        return 255
    e = 0
    while amax > 127.0 * math.ldexp(1.0, e - 127):
        e += 1
    return e


def sequences(pos, n, starts=None):
    """(sequence, its first row, number of rows, first position)."""
    b = len(pos)
    starts = np.arange(b + 1) * (n // b) if starts is None else starts
    return [(i, int(starts[i]), int(starts[i + 1] - starts[i]), int(pos[i])) for i in range(b)]


def rotate(x, cos, sin, p):
    """Rotate-half at position p, fp32 with every product and sum rounded; x [heads, D]."""
    h = x.shape[-1] // 2
    c, s = cos[p], sin[p]
    x1, x2 = x[:, :h], x[:, h:]
    return np.concatenate([x1 * c - x2 * s, x2 * c + x1 * s], -1).astype(np.float32)


def append(pool, qkv, table, pos, cos, sin, heads, bias=None, starts=None):
    """Updates `pool` in place; returns q [N, heads, D] in fp32."""
    kv, page, d = pool["k"].shape[1:]
    n = len(qkv)
    x = np.asarray(qkv, np.float32)
    if bias is not None:
        x = x + bias
    x = x.reshape(n, heads + 2 * kv, d)
    q = np.zeros((n, heads, d), np.float32)
    for b, r0, rows, p0 in sequences(pos, n, starts):
        turned = {}
        for t in range(rows):
            p = p0 + t
            if p < 0 or p >= len(cos):
                continue
            q[r0 + t] = rotate(x[r0 + t, :heads], cos, sin, p)
            if p < table.shape[1] * page and 0 <= table[b, p // page] < len(pool["k"]):
                turned[p] = (rotate(x[r0 + t, heads:heads + kv], cos, sin, p), x[r0 + t, heads + kv:])
        for o in sorted({p // page for p in turned}):
            new = sorted(p for p in turned if p // page == o)
            i, s0 = table[b, o], new[0] % page
            for which, name in enumerate("kv"):
                codes, exps = pool[name], pool[name + "_exp"]
                for h in range(kv):
                    part = np.stack([turned[p][which][h] for p in new])
                    old = 0 if s0 == 0 else int(exps[i, h])
                    e = max(old, scale_byte(float(np.abs(part).max()) if np.isfinite(part).all() else np.inf))
                    top = 63 if e == 249 else 127  # 64 * 2^122 is past the largest float
                    codes[i, h, :s0] = np.clip(np.rint(codes[i, h, :s0] * math.ldexp(1.0, max(old - e, -126))), -top, top)
                    codes[i, h, s0:s0 + len(new)] = 0 if e == 255 else np.clip(
                        np.rint(part.astype(np.float64) * math.ldexp(1.0, 127 - e)), -top, top)
                    exps[i, h] = e
    return q


def attention(pool, q, table, pos, starts=None, window=0, scale=None):
    """out [N, H, D] in 64 bits, with sum_j p_j |v_j| [N, H, D] and
    max_j scale * sum_d |q_d k_jd| [N, H], the magnitudes its rounding errors
    scale with."""
    kv, page, d = pool["k"].shape[1:]
    q = np.asarray(q, np.float64)
    n, heads, _ = q.shape
    g = heads // kv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out, mag, size = np.zeros((n, heads, d)), np.zeros((n, heads, d)), np.zeros((n, heads))
    for b, r0, rows, p0 in sequences(pos, n, starts):
        last = p0 + rows
        if last <= 0 or rows == 0:
            continue
        ids = table[b, :-(-last // page)]
        k = (pool["k"][ids] * pow2(pool["k_exp"][ids])[..., None, None]).transpose(1, 0, 2, 3).reshape(kv, -1, d)
        v = (pool["v"][ids] * pow2(pool["v_exp"][ids])[..., None, None]).transpose(1, 0, 2, 3).reshape(kv, -1, d)
        for t in range(rows):
            p = p0 + t
            if p < 0:
                continue
            lo = max(0, p - window + 1) if window else 0
            for h in range(heads):
                kk, vv, qq = k[h // g, lo:p + 1], v[h // g, lo:p + 1], q[r0 + t, h]
                s = scale * (kk @ qq)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r0 + t, h] = w @ vv
                mag[r0 + t, h] = w @ np.abs(vv)
                size[r0 + t, h] = scale * (np.abs(kk) @ np.abs(qq)).max()
    return out, mag, size
