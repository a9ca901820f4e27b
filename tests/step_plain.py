"""A step's operators around the block-scaled cache in plain numpy and 64 bits: what the GPU
tests compare with, and how far fp32 arithmetic may be from it."""

from __future__ import annotations

import numpy as np
import torch

from tests import scaled_plain as plain

#: Half an fp32 step, relative.
U = 2.0 ** -24

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
#: Half the smallest step of a type.
LEAST = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in HALF_STEP}


def turned(x, weight, positions, inv_freq, eps):
    """(heads normalised and turned, and the size that fp32's roundings are relative to).

    ``x`` float64 [tokens, heads, D]; weight [D] or None; positions [tokens]; inv_freq [half] or
    None; eps None: no norm.

    How far fp32 may be off, in U relative to the second value (|a| + |b| of a value's pair): the
    squares' sum 20 roundings (16 fused, at most 4 exchanges), halved by the root, the mean and
    eps 1, the root 2, two scalings 2: 15; cos and sin 4 absolutely (the reduced angle's rounding
    0.4, the series' last steps); two products' 2.  32 covers it."""
    y = np.asarray(x, np.float64)
    if eps is not None:
        y = y / np.sqrt(np.mean(y * y, -1, keepdims=True) + eps)
        if weight is not None:
            y = y * weight
    out, size = y.copy(), np.abs(y)
    half = 0 if inv_freq is None else len(inv_freq)
    if half:
        # the angle's product in 80 bits, brought into one turn before it is rounded
        whole = np.asarray(positions).astype(np.longdouble)[:, None] * np.asarray(inv_freq).astype(np.longdouble)
        turn = 2 * np.longdouble("3.14159265358979323846264338327950288")
        angle = (whole - np.rint(whole / turn) * turn).astype(np.float64)[:, None]
        c, s = np.cos(angle), np.sin(angle)
        a, b = y[..., :half], y[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
        size[..., :half] = size[..., half:2 * half] = np.abs(a) + np.abs(b)
    return out, size


def check_turned(got: torch.Tensor, want, size):
    """A type's rounding (half a step, or half the smallest one) behind fp32's roundings."""
    tolerance = HALF_STEP[got.dtype] * np.abs(want) * (1 + 2 * U) + LEAST[got.dtype] + 33 * U * size
    off = np.abs(got.double().cpu().numpy() - want) - tolerance
    assert (off <= 0).all(), f"past the tolerance by {off.max()} at {np.unravel_index(off.argmax(), off.shape)}"


def check_store(cache, codes, scales, k, size, v, tables, starts, lens, bs):
    """The cache (``codes``, ``scales`` as read back) after rows ``k`` (float64, with the ``size``
    of their roundings) and ``v`` went in; ``cache`` is the state from before."""
    before, was = cache
    new = np.stack((k, v), 2)
    slack = np.stack((33 * U * size, np.zeros_like(v)), 2)
    touched = np.zeros(codes.shape[0], bool)
    for r, last in enumerate(lens):
        t = starts[r]
        while t < starts[r + 1]:
            p = last - starts[r + 1] + t
            off, n = p % bs, min(bs - p % bs, starts[r + 1] - t)
            b = tables[r][p // bs]
            touched[b] = True
            for h in range(new.shape[1]):
                for w in range(2):
                    x, d = new[t:t + n, h, w], slack[t:t + n, h, w]
                    e = int(plain.exponents(scales[b, h, w]))
                    lo = plain.exponent_for(np.maximum(np.abs(x) - d, 0))
                    hi = plain.exponent_for(np.abs(x) + d)
                    if off:
                        old = int(plain.exponents(was[b, h, w]))
                        lo, hi = max(lo, old), max(hi, old)
                        kept = plain.decode(before[b, :off, h, w])
                        if e > old:
                            kept = plain.decode(plain.encode(kept * 2.0 ** (old - e)))
                        assert np.array_equal(plain.decode(codes[b, :off, h, w]), kept, equal_nan=True)
                    assert lo <= e <= hi, (b, h, w, e, lo, hi)
                    got = plain.decode(codes[b, off:off + n, h, w]) * 2.0 ** e
                    # half a step of a normal code, or of the smallest ones; 448 is not passed
                    # by more than x's own roundings
                    tolerance = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** (e - 10)) + 2 * d
                    assert (np.abs(got - x) <= tolerance).all(), (b, h, w)
            assert np.array_equal(codes[b, off + n:], before[b, off + n:])
            t += n
    assert np.array_equal(codes[~touched], before[~touched])
    assert np.array_equal(scales[~touched], was[~touched])
