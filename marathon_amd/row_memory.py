"""Where a tensor's rows lie in memory, and whether two tensors' rows share any of it.

Rows of ``width`` bytes stand at ``base + sum(i_k * stride_k)``, ``0 <= i_k < count_k``: a paged
cache's blocks, heads and tokens.  Caches of several layers may interleave in one allocation
(a block's layers side by side, K's row before V's), so that address ranges alone do not say
whether they share memory."""

from __future__ import annotations

from dataclasses import dataclass


@dataclass(frozen=True)
class Rows:
    """``dims``: (stride in bytes, count), in the tensors' common order."""

    base: int
    width: int
    dims: tuple

    @property
    def end(self) -> int:
        """Behind the last byte; ``base`` where there is none."""
        if not all(n for _, n in self.dims):
            return self.base
        return self.base + self.width + sum(s * (n - 1) for s, n in self.dims)

    def apart(self) -> bool:
        """Whether no row lies in another: each stride is at least as long as all that the
        smaller ones reach."""
        reach = self.width
        for s, n in sorted(d for d in self.dims if d[1] > 1):
            if s < reach:
                return False
            reach += s * (n - 1)
        return True


def share(a: Rows, b: Rows) -> bool:
    """Whether a row of ``a`` and one of ``b`` have a byte in common: exactly where their strides
    agree (a dimension of one element has any); where ranges interleave in strides that differ,
    it is taken that they do."""
    if a.end <= b.base or b.end <= a.base or a.end == a.base or b.end == b.base:
        return False
    dims = []
    for (s, n), (t, m) in zip(a.dims, b.dims):
        if n > 1 and m > 1 and s != t:
            return True
        s = s if n > 1 else t
        if s and (n > 1 or m > 1):  # (a stride of 0 leads nowhere else)
            dims.append((s, n, m))
    return _meet(b.base - a.base, sorted(dims, reverse=True), a.width, b.width)


def _meet(delta: int, dims: list, wa: int, wb: int) -> bool:
    """Whether ``-wb < delta + sum(q_k * s_k) < wa`` for some ``-n_k < q_k < m_k``."""
    if not dims:
        return -wb < delta < wa
    (s, n, m), rest = dims[0], dims[1:]
    # what the smaller strides can still add or take away bounds q
    up = wa + sum(t * (k - 1) for t, k, _ in rest)
    down = wb + sum(t * (k - 1) for t, _, k in rest)
    lo = max(1 - n, (-down - delta) // s + 1)
    hi = min(m - 1, -((delta - up) // s) - 1)
    return any(_meet(delta + q * s, rest, wa, wb) for q in range(lo, hi + 1))
