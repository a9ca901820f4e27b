"""An engine step around the block-scaled 8-bit cache: from its projections to its attention.

* :func:`norm_rotate`   -- every query and key head normalised (root mean square, a weight for
  each value) and turned to its token's position, in one pass; for a cache of any type;
* :func:`store_rotated` -- the same for a step's projections with the keys and values written
  straight into a :class:`~marathon_amd.scaled_cache.ScaledCache`: what :func:`norm_rotate` and
  :func:`~marathon_amd.scaled_cache.store_scaled` do, in one launch, the keys rounded once;
* :func:`attend_shared` -- :func:`~marathon_amd.scaled_cache.attend_scaled` for a batch whose
  requests begin, in groups, with the same cached tokens (a system prompt, a document, one
  history that several drafts continue): those are read once for all of a group's rows.

A step's requests are described as in :mod:`marathon_amd.scaled_cache` (``block_tables``,
``starts``, ``lens``), all on the GPU; every call is asynchronous on the current stream and can
be captured into a graph.  The turn is the rotate-half one of the rest of this package, over the
first ``2 * len(inv_freq)`` values of each head: its keys are what :class:`ScaledShifts` and
:func:`~marathon_amd.scatter_shifted` move (kvshift.py:44-61).

The calls on tensors that need no conversion go through the CPython binding, as the cache's do.

There is no CPU path and no gradient: tensors that are not on a HIP device raise, and so do
rows that require a gradient or carry a tangent.  C ABI: ``include/marathon_kvstep.h``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .row_memory import share
from .scaled_cache import (
    HEAD_SIZES,
    ScaledCache,
    _attend_desc,
    _current,
    _flags,
    _int32,
    _no_gradient,
    _rows_of,
    _steps,
    _table,
    _usual,
)
from .shift_kernels import current_stream, dtype_code
from .spans import _on

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _vector(name: str, t: torch.Tensor, device, n: int) -> int:
    """The address of a contiguous vector of ``n`` values."""
    if t.device != device or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous [{n}] on {device}, got {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _turn(who: str, device, head_size: int, inv_freq, q_weight, k_weight, eps) -> _lib.Turn:
    turn = _lib.Turn()
    _no_gradient(who, inv_freq=inv_freq, q_weight=q_weight, k_weight=k_weight)
    if inv_freq is not None:
        if inv_freq.dtype != torch.float32:
            raise TypeError(f"inv_freq {inv_freq.dtype}: float32")
        rotary = 2 * inv_freq.numel()
        if rotary % 32 or rotary > head_size:
            raise ValueError(f"rotary {rotary}: a multiple of 32, at most {head_size}")
        if rotary:
            turn.inv_freq = _vector("inv_freq", inv_freq, device, rotary // 2)
        turn.rotary = rotary
    weights = [w for w in (q_weight, k_weight) if w is not None]
    if eps is None:
        if weights:
            raise ValueError(f"{who}: weights without a norm (eps is None)")
        return turn
    turn.norm, turn.eps = 1, float(eps)
    if not 0.0 <= turn.eps < float("inf"):
        raise ValueError(f"eps {eps}")
    for w in weights:
        if w.dtype not in _DTYPES or w.dtype != weights[0].dtype:
            raise TypeError(f"weights {[w.dtype for w in weights]}: of one type, one of {_DTYPES}")
        turn.weight_dtype = dtype_code(w.dtype)
    if q_weight is not None:
        turn.q_weight = _vector("q_weight", q_weight, device, head_size)
    if k_weight is not None:
        turn.k_weight = _vector("k_weight", k_weight, device, head_size)
    return turn


def _check_rows(who: str, dtype, device, **rows: torch.Tensor) -> None:
    for name, t in rows.items():
        if t.dtype not in _DTYPES or t.dtype != dtype:
            raise TypeError(f"{name} {t.dtype}: rows of one type, one of {_DTYPES}")
        if t.device != device:
            raise ValueError(f"{name} on {t.device}, not {device}")
        if t.stride(2) != 1:
            raise ValueError(f"{name}'s rows must be contiguous in the last dimension")
    _no_gradient(who, **rows)


def _output(who: str, name: str, x: torch.Tensor, out, others: dict, inputs: tuple,
            caches: tuple = ()) -> torch.Tensor:
    """``out``, or a fresh one, for rows of ``x``'s shape: in ``x``'s place or apart from it, from
    the rows of ``others``, from the ``inputs`` and from the ``caches``."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(2) != 1:
        raise ValueError(f"out_{name} {out.dtype} {tuple(out.shape)} on {out.device} does not fit {name}")
    _no_gradient(who, **{f"out_{name}": out})
    rows = _rows_of(out)
    if not (out.data_ptr() == x.data_ptr() and _steps(out) == _steps(x)) and share(rows, _rows_of(x)):
        raise ValueError(f"out_{name} shares memory with {name} and is not {name} itself")
    for what, other in others.items():
        if share(rows, _rows_of(other)):
            raise ValueError(f"out_{name} shares memory with {what}")
    for r in caches:
        if rows.base < r.end and r.base < rows.end:
            raise ValueError(f"out_{name} lies among the cache's rows")
    for t in inputs:
        if t is not None and t.numel():
            last = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
            if rows.base < t.data_ptr() + last * t.element_size() and t.data_ptr() < rows.end:
                raise ValueError(f"out_{name} shares memory with an input")
    return out


def _head_rows(x: torch.Tensor, out: torch.Tensor) -> _lib.HeadRows:
    rows = _lib.HeadRows()
    rows.x, (rows.token_stride, rows.head_stride) = x.data_ptr(), _steps(x)
    rows.out, (rows.out_token_stride, rows.out_head_stride) = out.data_ptr(), _steps(out)
    rows.heads = x.shape[1]
    return rows


def norm_rotate(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor | None,
                inv_freq: torch.Tensor | None, *, q_weight: torch.Tensor | None = None,
                k_weight: torch.Tensor | None = None, eps: float | None = 1e-6,
                out_q: torch.Tensor | None = None,
                out_k: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Query and key heads (``[tokens, heads, D]``, bf16, fp16 or fp32; views of one projection
    are taken as they are) normalised and turned: ``x / sqrt(mean(x ** 2) + eps) * weight``, then
    each pair ``(i, i + rotary / 2)`` by ``positions * inv_freq[i]``.

    ``positions``: int32 or int64 ``[tokens]`` (:func:`~marathon_amd.step_slots` makes them);
    ``inv_freq``: fp32 ``[rotary / 2]`` on the GPU, ``rotary`` a multiple of 32, at most D; with
    None nothing is turned and ``positions`` is not read.  Weights: ``[D]`` of one type, ones where
    None.  ``eps`` None: no norm, the heads are only turned.  ``out_q`` and ``out_k`` may be ``q``
    and ``k`` themselves; otherwise they share no memory with them or each other.

    fp32 throughout and rounded once; angles are taken in 64 bits.  A head of zeros with eps 0 is
    NaN.  An infinity under the norm is NaN itself and, where it is turned, in its pair; the rest of
    its head is zeros."""
    made = _usual.rotate(q, k, positions, inv_freq, q_weight, k_weight, eps, out_q, out_k)
    if made is not None:
        if type(made) is int:
            _lib.check(made)
        return made
    for name, t in (("q", q), ("k", k)):
        if not t.is_cuda:
            raise RuntimeError(f"norm_rotate: {name} is not on a HIP device; there is no CPU path")
        if t.dim() != 3:
            raise ValueError(f"{name} {tuple(t.shape)}: [tokens, heads, D]")
    device, d = q.device, q.shape[2]
    if d not in HEAD_SIZES or k.shape[2] != d or k.shape[0] != q.shape[0]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)}: [tokens, heads, D], D one of "
                         f"{HEAD_SIZES}")
    _check_rows("norm_rotate", q.dtype, device, q=q, k=k)
    desc = _lib.NormRotateDesc()
    desc.turn = _turn("norm_rotate", device, d, inv_freq, q_weight, k_weight, eps)
    if desc.turn.rotary:
        if positions is None or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions: int32 or int64 "
                            f"[tokens], got {None if positions is None else positions.dtype}")
        desc.positions = _vector("positions", positions, device, q.shape[0])
        desc.position_bytes = positions.element_size()
    inputs = (positions, inv_freq, q_weight, k_weight)
    given = {} if out_k is None else {"out_k": out_k}
    out_q = _output("norm_rotate", "q", q, out_q, {"k": k, **given}, inputs)
    out_k = _output("norm_rotate", "k", k, out_k, {"q": q, "out_q": out_q}, inputs)
    desc.q, desc.k = _head_rows(q, out_q), _head_rows(k, out_k)
    desc.tokens, desc.head_size, desc.dtype = q.shape[0], d, dtype_code(q.dtype)
    with _on(device, _current(device)):
        _lib.check(_lib.lib().mkv_norm_rotate(ctypes.byref(desc), current_stream(device)))
    return out_q, out_k


def store_rotated(cache: ScaledCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  block_tables: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor,
                  inv_freq: torch.Tensor | None, *, q_weight: torch.Tensor | None = None,
                  k_weight: torch.Tensor | None = None, eps: float | None = 1e-6,
                  out_q: torch.Tensor | None = None,
                  error_flags: torch.Tensor | None = None) -> torch.Tensor:
    """A step's projections: the query heads normalised and turned (returned, or written to
    ``out_q``, which may be ``q`` itself), the key heads too and, with the values, into their
    blocks.

    Row i of request r stands at position ``lens[r] - new[r] + i``, by which it is turned.
    ``q`` ``[tokens, query heads, D]``, ``k`` and ``v`` ``[tokens, heads, D]`` of one type; weights,
    ``eps`` and ``inv_freq`` as :func:`norm_rotate` takes them, blocks, scales and flags as
    :func:`~marathon_amd.scaled_cache.store_scaled` does.  Keys are rounded once, to their codes.
    Rows of no request are not read, and of ``out_q`` left as they were (in a fresh one,
    undefined)."""
    made = _usual.put(*cache.handle, q, k, v, block_tables, starts, lens, inv_freq, q_weight, k_weight,
                      eps, out_q, error_flags)
    if made is not None:
        if type(made) is int:
            _lib.check(made)
        return made
    device, d = cache.device, cache.head_size
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3 or t.shape[2] != d or t.shape[0] != q.shape[0]:
            raise ValueError(f"{name} {tuple(t.shape)}: [{q.shape[0]}, heads, {d}]")
    if k.shape[1] != cache.heads or v.shape[1] != cache.heads:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)}: {cache.heads} heads")
    _check_rows("store_rotated", q.dtype, device, q=q, k=k, v=v)
    desc = _lib.StoreRotatedDesc()
    desc.turn = _turn("store_rotated", device, d, inv_freq, q_weight, k_weight, eps)
    out_q = _output("store_rotated", "q", q, out_q, {"k": k, "v": v},
                    (inv_freq, q_weight, k_weight, block_tables, starts, lens),
                    (*cache.rows, cache.scale_rows))
    desc.cache, desc.q = cache.desc, _head_rows(q, out_q)
    desc.k, (desc.k_token_stride, desc.k_head_stride) = k.data_ptr(), _steps(k)
    desc.v, (desc.v_token_stride, desc.v_head_stride) = v.data_ptr(), _steps(v)
    (desc.block_tables, desc.table_stride, desc.requests,
     desc.table_width) = _table(block_tables, device)
    desc.starts = _int32("starts", starts, device, desc.requests + 1)
    desc.lens = _int32("lens", lens, device, desc.requests)
    desc.error_flags = _flags(error_flags, device)
    desc.tokens, desc.dtype = q.shape[0], dtype_code(q.dtype)
    with _on(device, _current(device)):
        _lib.check(_lib.lib().mkv_store_rotated(ctypes.byref(desc), current_stream(device)))
    return out_q


def attend_shared(cache: ScaledCache, q: torch.Tensor, block_tables: torch.Tensor,
                  starts: torch.Tensor, lens: torch.Tensor, groups: torch.Tensor,
                  shared: torch.Tensor, *, softmax_scale: float | None = None,
                  max_new: int | None = None, max_shared: int | None = None,
                  max_own: int | None = None, out: torch.Tensor | None = None,
                  error_flags: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`~marathon_amd.scaled_cache.attend_scaled` where requests ``groups[g]`` to
    ``groups[g + 1]`` (int32 ``[groups + 1]``) begin with the same ``shared[g]`` tokens (int32
    ``[groups]``), both on the GPU.

    Of the shared tokens whole blocks are read once for the group, through the block table of its
    first request; the others' entries for them are not read.  Where a group's tables agree, as
    those of requests that share blocks do, the result is ``attend_scaled``'s but for the order of
    sums and the roundings of p named there, by the rows of a request, however many share: 2^-17 of
    itself for fp16 queries and for bf16 ones of at most 32 rows (``max_new``, or without it the tokens,
    times the query heads of a KV head), 2^-8 of more.  Requests in no group share nothing.  Groups that
    leave the requests or descend, and negative ``shared``, are flagged (``MKV_FLAG_SPAN``) and share
    nothing.

    ``max_new``, ``max_shared`` and ``max_own``: the largest number of new tokens of a request, of
    tokens that a group shares and of tokens that a request has behind them, where the host knows
    them.  They choose launch shapes, and a result only by the order of its sums and the roundings
    above."""
    made = _usual.attend_shared(*cache.handle, q, block_tables, starts, lens, groups, shared,
                                softmax_scale, max_new, max_shared, max_own, out, error_flags)
    if made is not None:
        if type(made) is int:
            _lib.check(made)
        return made
    desc = _lib.AttendSharedDesc()
    desc.attend, out = _attend_desc("attend_shared", cache, q, block_tables, starts, lens,
                                    softmax_scale, max_new, max_own, out, error_flags)
    device = cache.device
    desc.n_groups = shared.shape[0] if shared.dim() == 1 else 0
    desc.shared = _int32("shared", shared, device, None)
    desc.groups = _int32("groups", groups, device, desc.n_groups + 1)
    desc.max_shared = max(-1, min(int(max_shared or 0), 2**31 - 1))
    L = _lib.lib()
    need = L.mkv_attend_shared_workspace_size(ctypes.byref(desc))
    with _on(device, _current(device)):
        if need > 0:  # the allocator hands it on in stream order
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            desc.attend.workspace, desc.attend.workspace_bytes = workspace.data_ptr(), need
        _lib.check(L.mkv_attend_shared(ctypes.byref(desc), current_stream(device)))
    return out
