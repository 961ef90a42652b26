"""The operators of a step over an 8-bit cache in 64 bits, written from their formulas with numpy: what the kernels of store8.hip, attention8.hip
and verify.hip are checked against.  Arrays are float64 (ints where they are numbers of things); a cache is held as the numbers its entries are."""
from __future__ import annotations

import math

import numpy as np

LOWEST = -64


def e4m3_numbers() -> np.ndarray:
    """The 127 values from 0 to 448, in order: 2^-9 apart up to 2^-6, then eight to a power of two."""
    return np.array([i * 2.0 ** -9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 3) for e in range(-6, 9) for i in range(8)])[:127]


def e4m3(x: np.ndarray) -> np.ndarray:
    """The nearest of them, of two equally near ones the one with the even last digit; NaN stays."""
    numbers = e4m3_numbers()
    a = np.abs(x)
    hi = np.searchsorted(numbers, a).clip(1, 126)
    lo = hi - 1
    up = numbers[hi] - a
    down = a - numbers[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isnan(x), np.nan, np.copysign(numbers[pick], x))


def exponent_for(top: float) -> int:
    """The least e >= LOWEST with top <= 448 * 2^e."""
    e = LOWEST
    while top > 448.0 * 2.0 ** e:
        e += 1
    return e


def heads(x, w, eps, cos, sin, places):
    """Norm and rotation of [n, heads, d]."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos is not None:
        c, s, h = cos[places][:, None], sin[places][:, None], cos.shape[1]
        x = np.concatenate([x[..., :h] * c - x[..., h:2 * h] * s, x[..., h:2 * h] * c + x[..., :h] * s, x[..., 2 * h:]], -1)
    return x


def store(qkv, nq, nkv, d, k, v, scales, q_w, k_w, eps, cos, sin, table, cu, k_len):
    """q [T, nq, d] (NaN for rows of no sequence); k [pages, nkv, P, d], v [pages, nkv, d, P] and scales [pages, nkv, 2] are written in place."""
    x = qkv.reshape(len(qkv), nq + 2 * nkv, d)
    q = np.full((len(qkv), nq, d), np.nan)
    P = k.shape[2]
    for s in range(len(k_len)):
        a, b = int(cu[s]), int(cu[s + 1])
        n, first = b - a, int(k_len[s]) - (b - a)
        if n <= 0:
            continue
        places = np.arange(first, first + n)
        q[a:b] = heads(x[a:b, :nq], q_w, eps, cos, sin, places)
        new = (heads(x[a:b, nq:nq + nkv], k_w, eps, cos, sin, places), x[a:b, nq + nkv:])
        for j in range(first // P, (first + n - 1) // P + 1) if nkv else ():
            page = int(table[s, j])
            if not 0 <= page < len(k):
                continue
            mine = (places // P) == j
            off = int(places[mine][0]) - j * P
            for which, cache in ((0, k), (1, v.swapaxes(2, 3))):
                for h in range(nkv):
                    rows = new[which][mine][:, h]
                    fine = rows[np.isfinite(rows)]
                    e = exponent_for(np.abs(fine).max() if fine.size else 0.0)
                    stood = math.frexp(scales[page, h, which])[1] - 1 if scales[page, h, which] > 0 else -127
                    if off > 0:
                        e = max(e, stood)
                    if e > stood:
                        cache[page, h] = e4m3(cache[page, h] * 2.0 ** (stood - e))
                    with np.errstate(invalid="ignore"):
                        cache[page, h, off:off + len(rows)] = e4m3(np.where(np.isfinite(rows), rows, np.nan) * 2.0 ** -e)
                    scales[page, h, which] = 2.0 ** e
    return q


def attention(q, k, v, scales, table, cu, k_len, scale, window=0):
    """(out, weighted |v|, largest sum of |q k| scale, sum of |v - out| over the keys seen) of every row [T, nq, d] ([T, nq, 1] the third): rows of no sequence are NaN."""
    T, nq, d = q.shape
    nkv, P = k.shape[1], k.shape[2]
    group = nq // nkv
    out, weighted, most, flushed = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((T, nq, 1)), np.zeros(q.shape)
    for s in range(len(k_len)):
        a, b = int(cu[s]), int(cu[s + 1])
        n, keys = b - a, int(k_len[s])
        if n <= 0:
            continue
        pages = [int(p) for p in table[s, :-(-keys // P)]]
        there = np.repeat([0 <= p < len(k) for p in pages], P)[:keys] if pages else np.zeros(0, bool)
        kept = [p if 0 <= p < len(k) else 0 for p in pages]
        for h in range(nkv):
            kk = np.concatenate([k[p, h] * scales[p, h, 0] for p in kept])[:keys] if kept else np.zeros((0, d))
            vv = np.concatenate([v[p, h].T * scales[p, h, 1] for p in kept])[:keys] if kept else np.zeros((0, d))
            for r in range(n):
                pos = keys - n + r
                j = np.arange(keys)
                see = there & (j <= pos) & ((j > pos - window) if window else True)
                for m in range(h * group, (h + 1) * group):
                    if not see.any():
                        out[a + r, m] = 0
                        continue
                    x = kk[see] @ q[a + r, m] * scale
                    w = np.exp(x - np.max(x))
                    w = w / w.sum()
                    out[a + r, m] = w @ vv[see]
                    weighted[a + r, m] = w @ np.abs(vv[see])
                    most[a + r, m] = (np.abs(kk[see]) @ np.abs(q[a + r, m])).max() * scale
                    flushed[a + r, m] = np.abs(vv[see] - out[a + r, m]).sum(0)
    return out, weighted, most, flushed


def chances(x, t):
    """softmax(x / t), or 1 at the maximum (a NaN, else the first of the largest) where t is not positive or the maximum not finite."""
    nan = np.isnan(x)
    at = int(np.argmax(nan)) if nan.any() else int(np.argmax(x))
    if not t > 0 or not np.isfinite(x[at]):
        return np.eye(1, len(x), at)[0]
    z = np.zeros(len(x)) if math.isinf(t) else (x - x[at]) / t
    p = np.where(np.isneginf(x), 0.0, np.exp(z))
    return p / p.sum()


def verify(logits, ids, cu, draft_logits, temps, accept_u, draw_u):
    """(tokens [R], counts [S], accept [D]); places that nothing is written to are -7."""
    R, V = logits.shape
    S = len(cu) - 1
    tokens, counts, accept = np.full(R, -7), np.zeros(S, int), np.full(len(ids), np.nan)
    m = 0
    for s in range(S):
        n = int(cu[s + 1]) - int(cu[s]) - 1
        if n < 0:
            continue
        t = temps[s] if temps is not None else 0.0
        stand, left = n, None
        for i in range(n):
            p, d = chances(logits[cu[s] + i], t), int(ids[m + i])
            known = 0 <= d < V
            q = chances(draft_logits[m + i], t) if draft_logits is not None else np.eye(1, V, d)[0] if known else np.zeros(V)
            pd, qd = (p[d], q[d]) if known else (0.0, 0.0)
            accept[m + i] = min(1.0, pd / qd) if qd > 0 else float(pd > 0)
            if stand == n and left is None and not (accept_u[m + i] if accept_u is not None else 0.0) * qd < pd:
                stand, left = i, np.maximum(p - q, 0)
        p = chances(logits[cu[s] + stand], t)
        if left is None or left.sum() == 0:
            left = p
        line = np.cumsum(left)
        j = int(np.searchsorted(line, (draw_u[s] if draw_u is not None else 0.0) * line[-1], side="right"))
        tokens[cu[s]:cu[s + 1]] = -1
        tokens[cu[s]:cu[s] + stand] = ids[m:m + stand]
        tokens[cu[s] + stand] = min(j, int(np.nonzero(left)[0][-1]))
        counts[s] = stand + 1
        m += n
    return tokens, counts, accept
