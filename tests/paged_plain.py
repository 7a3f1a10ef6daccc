"""Plain 64-bit forms of the 8-bit paged cache's operators, written from their
definitions with numpy, one request, page and head at a time."""

from __future__ import annotations

import numpy as np
import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def scale_of(amax: float, store: str) -> float:
    """Least power of two s >= 2^-100 with amax <= TOP s."""
    s = 2.0**-100
    while amax > TOP[store] * s:
        s *= 2.0
    return s


def round_code(y: np.ndarray, store: str) -> np.ndarray:
    """Nearest representable code value, ties to even, saturating."""
    if store == "int8":
        return np.clip(np.rint(y), -127, 127)
    _, e = np.frexp(np.maximum(np.abs(y), 2.0**-6))
    step = np.ldexp(1.0, e - 4)
    return np.clip(np.rint(y / step) * step, -448.0, 448.0)


def tables(cached, new, table, free, page, capacity):
    """(ok, table, lens, cu, slots, positions, free left) of one step."""
    table, free = [list(r) for r in table], list(free)
    slots, pos, cu = [-1] * capacity, [0] * capacity, [0]
    need = sum(-(-(c + t) // page) + (-c // page) for c, t in zip(cached, new))
    width = len(table[0])
    bad = any(c < 0 or t < 0 or c + t > width * page for c, t in zip(cached, new))
    if bad or need > len(free) or sum(new) > capacity:
        return False, table, list(cached), [0] * (len(cached) + 1), slots, pos, len(free)
    i = 0
    for b, (c, t) in enumerate(zip(cached, new)):
        for j in range(-(-c // page), -(-(c + t) // page)):
            table[b][j] = free.pop()
        for p in range(c, c + t):
            slots[i], pos[i] = table[b][p // page] * page + p % page, p
            i += 1
        cu.append(i)
    return True, table, [c + t for c, t in zip(cached, new)], cu, slots, pos, len(free)


def append(codes, scales, slots, rows, store):
    """codes (pages, H, page, D) and scales (pages, H) after rows (n, H, D) are
    stored at slots, run by run; arrays of float64, codes as their values."""
    codes, scales = codes.copy(), scales.copy()
    page = codes.shape[2]
    i = 0
    while i < len(slots):
        if slots[i] < 0 or slots[i] >= codes.shape[0] * page:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % page:
            n += 1
        p, o = divmod(int(slots[i]), page)
        for h in range(codes.shape[1]):
            x = rows[i : i + n, h]
            fin = np.abs(x[np.isfinite(x)])
            s = scale_of(fin.max() if fin.size else 0.0, store)
            if o:
                s = max(s, scales[p, h])
                if s > scales[p, h]:
                    codes[p, h, :o] = round_code(codes[p, h, :o] * (scales[p, h] / s), store)
            y = np.where(np.isnan(x), 0.0, x) / s
            codes[p, h, o : o + n] = round_code(y, store)
            scales[p, h] = s
        i += n
    return codes, scales


def dense(codes, scales, table, n):
    """(H, n, D) of the first n tokens of one request (its row of the table)."""
    page = codes.shape[2]
    out = np.zeros((codes.shape[1], n, codes.shape[3]))
    for t in range(n):
        p = table[t // page]
        out[:, t] = codes[p, :, t % page] * scales[p][:, None]
    return out


def attention(q, k, v, scaling, window=0, start=0, vs=None):
    """q (n, Hq, D), k and v (H, len, D), all float64, vs (H, len) the values'
    scale of each token.  Returns out (n, Hq, D), lse (n, Hq), and what the error
    bounds are made of: weight (n, Hq, D) = sum w |v|, size (n, Hq) = the largest
    scaling * sum |q_d k_d| a row sees, flush (n, Hq, D) = max(w vs) sum |v| / vs
    (0 without vs)."""
    n, hq, dim = q.shape
    heads, length = k.shape[:2]
    out, lse = np.zeros(q.shape), np.full((n, hq), -np.inf)
    weight, size, flush = np.zeros(q.shape), np.zeros((n, hq)), np.zeros(q.shape)
    for i in range(n):
        hi = min(length, length - n + i + 1)
        lo = max(start, hi - window) if window else start
        if hi <= lo:
            continue
        for h in range(hq):
            g = h // (hq // heads)
            x = k[g, lo:hi] @ q[i, h] * scaling
            m = x.max()
            w = np.exp(x - m)
            lse[i, h] = m + np.log(w.sum())
            w /= w.sum()
            out[i, h] = w @ v[g, lo:hi]
            weight[i, h] = w @ np.abs(v[g, lo:hi])
            size[i, h] = (np.abs(k[g, lo:hi]) @ np.abs(q[i, h])).max() * abs(scaling)
            if vs is not None:
                s = vs[g, lo:hi]
                flush[i, h] = (w * s).max() * (np.abs(v[g, lo:hi]) / s[:, None]).sum(0)
    return out, lse, weight, size, flush


def bounds(ref, lse, weight, size, flush, dim, length, dtype):
    """How far (out, lse) may be off, elementwise.

    Scores: products are exact in fp32 and summed there, dim terms, each sum off
    by at most 2^-23 of the running magnitude; q's split or rounding and the
    scales' products add 2^-22.  A weight is off by that times size, by 2^-21
    from the exponential, and by 2^-11 (16-bit types: one rounding to f16) or
    2^-21 (fp32: two f16 parts); sums over the tokens add length 2^-23.  What is
    rounded to f16 is w vs; under 2^-14 of its largest value f16 is spaced 2^-24 of
    that, an absolute error of 2^-25 max(w vs) in w vs, so of 2^-25 flush in the
    sum over w vs (v / vs).  The result's own rounding is half a step."""
    score = ((dim + 8) * 2.0**-23 + 2.0**-21) * size
    rel = score + 2.0**-21 + length * 2.0**-22 + (2.0**-21 if dtype == torch.float32 else 2.0**-11)
    half = torch.finfo(dtype).eps / 2
    out = half * np.abs(ref) * 1.001 + rel[..., None] * weight * 2 + 2.0**-25 * flush + 1e-30
    le = np.where(np.isfinite(lse), score + 2.0**-20 + length * 2.0**-22 + 2.0**-22 * np.abs(lse), 0.0)
    return out, le
