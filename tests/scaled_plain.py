"""The block-scaled cache in plain numpy and 64 bits: what the GPU tests compare with.

Written from the format's definition alone (a value is ``code * 2 ** e``, one ``e`` for the K
and one for the V rows of a (block, head); the least ``e`` under which the rows' largest finite
value fits 448), on caches in the order block, token, head, value.
"""

from __future__ import annotations

import numpy as np

LOW, HIGH = -100, 100


def _code_values() -> np.ndarray:
    c = np.arange(256)
    exp, man = (c >> 3) & 15, c & 7
    v = np.where(exp > 0, np.ldexp(1 + man / 8.0, exp - 7), np.ldexp(man / 8.0, -6))
    v[(c & 127) == 127] = np.nan
    return np.where(c > 127, -v, v)


VALUES = _code_values()
_POS = VALUES[:127]  # codes 0 to 126, ascending


def decode(codes: np.ndarray) -> np.ndarray:
    return VALUES[codes]


def exponents(scales: np.ndarray) -> np.ndarray:
    return np.clip(scales.astype(np.int64) - 127, LOW, HIGH)


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest code, ties to the even one; what is larger than 448 saturates; NaN: 0x7F."""
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    hi = np.clip(np.searchsorted(_POS, a), 1, 126)
    lo = hi - 1
    up, down = _POS[hi] - a, a - _POS[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = code | np.where(np.signbit(x), 128, 0)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def exponent_for(rows: np.ndarray) -> int:
    a = np.abs(rows[np.isfinite(rows)])
    top = float(a.max()) if a.size else 0.0
    if top == 0.0:
        return LOW
    e = -400
    while top > 448.0 * 2.0 ** e:
        e += 1
    return min(max(e, LOW), HIGH)


def step_slots(held, new, tables, free, free_at, bs):
    """(tables, starts, slots, positions, free_at) of a step that fits."""
    tables, starts, slots, pos = tables.copy(), [0], [], []
    for r, (h, n) in enumerate(zip(held, new)):
        for b in range(-(-h // bs), -(-(h + n) // bs)):
            tables[r, b] = free[free_at]
            free_at += 1
        for p in range(h, h + n):
            slots.append(int(tables[r, p // bs]) * bs + p % bs)
            pos.append(p)
        starts.append(starts[-1] + n)
    return tables, starts, slots, pos, free_at


def store(codes, scales, k, v, tables, starts, lens, bs):
    """In place.  ``codes`` uint8 [blocks, bs, heads, 2, D], ``scales`` uint8 [blocks, heads, 2],
    ``k`` and ``v`` float64 [tokens, heads, D]."""
    new = np.stack((k, v), 2)
    for r, last in enumerate(lens):
        s0, s1 = starts[r], starts[r + 1]
        pos = last - (s1 - s0)
        t = s0
        while t < s1:
            p = pos + t - s0
            off, n = p % bs, min(bs - p % bs, s1 - t)
            b = tables[r][p // bs]
            for h in range(new.shape[1]):
                for w in range(2):
                    e = exponent_for(new[t:t + n, h, w])
                    if off:
                        was = int(exponents(scales[b, h, w]))
                        if e > was:
                            old = decode(codes[b, :off, h, w])
                            codes[b, :off, h, w] = encode(old * 2.0 ** (was - e))
                        e = max(e, was)
                    codes[b, off:off + n, h, w] = encode(new[t:t + n, h, w] * 2.0 ** -e)
                    scales[b, h, w] = e + 127
            t += n


def rows(codes, scales, table, n, bs):
    """float64 [n, heads, 2, D]: positions 0 to n through a block table."""
    p = np.arange(n)
    b = np.asarray(table)[p // bs]
    return decode(codes[b, p % bs]) * 2.0 ** exponents(scales[b])[..., None].astype(np.float64)


def attend(codes, scales, q, tables, starts, lens, bs, scale):
    """float64 [tokens, query heads, D]; rows that see nothing are zeros, rows of nobody NaN."""
    out = np.full(q.shape, np.nan)
    group = q.shape[1] // codes.shape[2]
    for r, last in enumerate(lens):
        s0, s1 = starts[r], starts[r + 1]
        x = rows(codes, scales, tables[r], max(last, 0), bs)
        for t in range(s0, s1):
            sees = last - (s1 - s0) + (t - s0) + 1
            for h in range(q.shape[1]):
                if sees <= 0:
                    out[t, h] = 0.0
                    continue
                kk, vv = x[:sees, h // group, 0], x[:sees, h // group, 1]
                s = kk @ q[t, h] * scale
                p = np.exp(s - s.max())
                out[t, h] = (p / p.sum()) @ vv
    return out


def shift(src, src_scales, dst, dst_scales, spans, src_table, dst_table, sbs, dbs, inv_freq):
    """In place on ``dst`` and ``dst_scales``: one layer.  K turns in fp32, product by product."""
    half = len(inv_freq)
    for src_pos, dst_pos, si, di, n, delta, _, _ in spans:
        p = src_pos + np.arange(n)
        b = np.asarray(src_table)[si + p // sbs]
        x = (decode(src[b, p % sbs])
             * 2.0 ** exponents(src_scales[b])[..., None].astype(np.float64)).astype(np.float32)
        if delta and half:
            a = (np.float32(delta) * inv_freq).astype(np.float64)
            c, s = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
            lo, hi = x[..., 0, :half].copy(), x[..., 0, half:2 * half].copy()
            x[..., 0, :half] = lo * c + hi * -s
            x[..., 0, half:2 * half] = hi * c + lo * s
        for first in range(0, n, dbs):
            m = min(dbs, n - first)
            d = np.asarray(dst_table)[di + (dst_pos + first) // dbs]
            for h in range(x.shape[1]):
                for w in range(2):
                    e = exponent_for(x[first:first + m, h, w])
                    dst[d, :m, h, w] = encode(x[first:first + m, h, w].astype(np.float64) * 2.0 ** -e)
                    dst_scales[d, h, w] = e + 127
