"""A paged KV cache held in 8 bits, with a scale for each block of tokens and KV head.

The cache's rows are e4m3fn codes in the layouts of the other caches here (HND ``[blocks,
heads, bs, 2D]``, NHD ``[blocks, bs, heads, 2D]``, or K and V planes apart); a value is ``code
* 2 ** e`` with one ``e`` for the K rows and one for the V rows of each (block, head), held as
``float8_e8m0fnu`` in ``scales`` ``[blocks, heads, 2]`` (``include/marathon_kvscaled.h`` has
the format).  Four operators work on it, each one launch (attention over long histories two),
asynchronous on the current stream:

* :func:`step_slots`    -- an engine step's block tables, slot map and positions, built on
  the GPU from the requests' lengths: :func:`marathon_amd.slots` for a whole batch, without
  its host loop (shift_store.py:56-60);
* :func:`store_scaled`  -- the step's new K and V rows into their blocks;
* :func:`attend_scaled` -- the step's queries over the cache, causal, grouped heads;
* :class:`ScaledShifts` -- reused spans into other blocks, K re-rotated by each span's delta,
  every layer at once: :class:`marathon_amd.spans.SmallShifts` for this cache.

A step's requests are described by ``block_tables`` (int32 ``[requests, width]``), ``starts``
(int32 ``[requests + 1]``: request r's new tokens are rows ``starts[r]`` to ``starts[r + 1]``
of the step's token arrays) and ``lens`` (int32 ``[requests]``: tokens held with the new ones),
all on the GPU, so that a captured step replays with the lengths of its day.  Rows behind
``starts[-1]`` (a padded batch) are neither read nor written.

The calls on tensors that need no conversion go through the CPython binding, which makes these
functions' checks on the tensors themselves; it answers None, with nothing launched, for any
other call, which the code here takes (and refuses, where it must).

There is no CPU path and no gradient: tensors that are not on a HIP device raise, and so do
rows, queries and outputs that require a gradient or carry a tangent.
"""

from __future__ import annotations

import ctypes
import warnings
from dataclasses import dataclass, field
from itertools import chain

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from .row_memory import Rows, share
from .shift_kernels import current_stream, dtype_code
from .spans import _on, _span_struct

HEAD_SIZES = (64, 128, 256)
BLOCK_SIZES = (16, 32, 64, 128)

_ROW_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_QUERY_DTYPES = (torch.bfloat16, torch.float16)


class _Usual:
    """The binding's calls, loaded at the first use; where the module cannot be loaded, calls
    that always answer None (the general path launches the same kernels)."""

    def __getattr__(self, name):
        try:
            call = getattr(_lib.binding(), name)
        except (RuntimeError, ImportError, OSError) as e:
            warnings.warn(f"{name}: the general path is taken, slower on the host: {e}",
                          RuntimeWarning, stacklevel=3)

            def call(*args):
                return None
        setattr(self, name, call)
        return call


_usual = _Usual()


def _current(device: torch.device) -> bool:
    return device.index == torch.cuda.current_device()


@dataclass
class ScaledCache:
    """One layer's cache: ``kv`` (``float8_e4m3fn``, fused rows ``[..., 2D]`` of K then V) and
    ``scales`` (``float8_e8m0fnu`` ``[blocks, heads, 2]``, contiguous), of ``layout`` ``"hnd"``
    or ``"nhd"``.  With ``v_cache``, ``kv`` holds K and ``v_cache`` V, rows ``[..., D]`` of the
    same shape and strides.  No row lies in another.  The tensors are checked once, here, and
    kept."""

    kv: torch.Tensor
    scales: torch.Tensor
    layout: str
    block_size: int = 16
    v_cache: torch.Tensor | None = None
    desc: _lib.ScaledCacheDesc = field(init=False, repr=False)

    def __post_init__(self):
        kv, scales, v = self.kv, self.scales, self.v_cache
        if self.layout not in ("hnd", "nhd"):
            raise ValueError(f"layout {self.layout!r}: 'hnd' or 'nhd'")
        if not kv.is_cuda:
            raise RuntimeError("ScaledCache: kv is not on a HIP device; there is no CPU path")
        if kv.dim() != 4:
            raise ValueError(f"a {self.layout} cache is 4-D, got {tuple(kv.shape)}")
        if kv.dtype != torch.float8_e4m3fn:
            raise TypeError(f"cache dtype {kv.dtype}: float8_e4m3fn")
        if kv.shape[2 if self.layout == "hnd" else 1] != self.block_size:
            raise ValueError(f"{self.layout} cache {tuple(kv.shape)} has no blocks of "
                             f"{self.block_size} tokens")
        if v is not None and (v.shape != kv.shape or v.dtype != kv.dtype or v.device != kv.device
                              or v.stride() != kv.stride()):
            raise ValueError("v_cache differs from kv in shape, strides, dtype or device")
        width = kv.shape[3]
        if v is None and width % 2:
            raise ValueError(f"fused rows of {width} values")
        self.head_size = width if v is not None else width // 2
        if self.head_size not in HEAD_SIZES:
            raise ValueError(f"head_size {self.head_size}: one of {HEAD_SIZES}")
        if self.block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size {self.block_size}: one of {BLOCK_SIZES}")
        if kv.stride(3) != 1:
            raise ValueError("rows must be contiguous in the last dimension")
        self.heads = kv.shape[1 if self.layout == "hnd" else 2]
        if self.heads == 0:
            raise ValueError(f"a cache of no heads: {tuple(kv.shape)}")
        self.device = kv.device
        if (scales.dtype != torch.float8_e8m0fnu or scales.device != kv.device
                or tuple(scales.shape) != (kv.shape[0], self.heads, 2)
                or not scales.is_contiguous()):
            raise ValueError(f"scales: contiguous float8_e8m0fnu {(kv.shape[0], self.heads, 2)} "
                             f"on {kv.device}, got {scales.dtype} {tuple(scales.shape)}")
        # a dimension of one element never advances an address, and torch gives it any stride
        strides = [s if n > 1 else 0 for s, n in zip(kv.stride(), kv.shape)]
        block, head, token = (strides[:3] if self.layout == "hnd" else
                              (strides[0], strides[2], strides[1]))
        steps = ((block, kv.shape[0]), (head, self.heads), (token, self.block_size))
        self.rows = [Rows(kv.data_ptr(), width, steps)]
        if v is not None:
            self.rows.append(Rows(v.data_ptr(), width, steps))
        self.scale_rows = Rows(scales.data_ptr(), 2 * self.heads, ((2 * self.heads, kv.shape[0]),))
        # (an expanded cache, of stride 0, is one whose rows lie in one another)
        if not self.rows[0].apart():
            raise ValueError(f"a cache of shape {tuple(kv.shape)} and strides {kv.stride()} has "
                             "rows that overlap")
        if v is not None and share(*self.rows):
            raise ValueError("kv and v_cache share memory")
        if any(s % 16 for s in strides[:3]) or kv.data_ptr() % 16 or (
                v is not None and v.data_ptr() % 16) or scales.data_ptr() % 2:
            raise ValueError("the cache's base and strides must be multiples of 16 bytes")
        d = self.desc = _lib.ScaledCacheDesc()
        if kv.numel():
            d.k_base = kv.data_ptr()
            d.v_base = kv.data_ptr() + self.head_size if v is None else v.data_ptr()
            d.scales = scales.data_ptr()
        d.num_blocks, d.block_stride, d.head_stride, d.token_stride = kv.shape[0], block, head, token
        d.block_size, d.heads, d.head_size = self.block_size, self.heads, self.head_size
        self.handle = (ctypes.addressof(d), kv.get_device())  # for the binding; `desc` is kept


def _no_gradient(who: str, **tensors: torch.Tensor | None) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{who} has no backward pass; detach {name} or use torch.no_grad()")
        if forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{who} has no derivative for the tangent of {name}")


def _flags(error_flags: torch.Tensor | None, device) -> int | None:
    if error_flags is None:
        return None
    if error_flags.dtype != torch.int32 or error_flags.device != device or error_flags.numel() < 1:
        raise ValueError(f"error_flags: int32 [1] on {device}")
    return error_flags.data_ptr()


def _int32(name: str, t: torch.Tensor, device, n: int | None) -> int:
    """The address of a contiguous int32 vector (of ``n`` entries)."""
    if t.dtype != torch.int32 or t.device != device or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 vector on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} has {t.shape[0]} entries, not {n}")
    return t.data_ptr()


def _table(t: torch.Tensor, device) -> tuple[int, int, int, int]:
    """(address, row stride, requests, width) of a block table."""
    if t.dtype != torch.int32 or t.device != device or t.dim() != 2:
        raise ValueError(f"block_tables: int32 [requests, width] on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    n, width = t.shape
    if width > 1 and t.stride(1) != 1:
        raise ValueError("block_tables' rows must be contiguous")
    return t.data_ptr(), t.stride(0) if n > 1 else width, n, width


@dataclass
class StepSlots:
    """What :func:`step_slots` makes, all on the GPU: ``starts`` int32 ``[requests + 1]``,
    ``lens`` int32 ``[requests]``, ``slots`` int64 ``[max_tokens]`` (-1 behind the last token),
    ``positions`` int32 ``[max_tokens]`` (0 there) and ``free_at`` int32 ``[1]``."""

    starts: torch.Tensor
    lens: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    free_at: torch.Tensor


def step_slots(held: torch.Tensor, new: torch.Tensor, block_tables: torch.Tensor,
               free_blocks: torch.Tensor, free_at: torch.Tensor, block_size: int,
               max_tokens: int, *, error_flags: torch.Tensor | None = None) -> StepSlots:
    """Block tables and slot map of a step, from the requests' lengths on the GPU.

    Request r holds ``held[r]`` tokens and gets ``new[r]`` more (int32).  The blocks that it
    needs beyond ``ceil(held / block_size)`` are taken from ``free_blocks[free_at[0]:]``,
    requests in order, and entered into ``block_tables`` in place; ``max_tokens`` bounds the
    step's tokens (the length of the slot map).  ``slots`` is what :func:`scatter_shifted` and
    a slot-addressed shift take, ``starts`` and ``lens`` what :func:`store_scaled` and
    :func:`attend_scaled` take; the next step's ``held`` is ``lens`` and its ``free_at``
    the one returned.  Ids are taken as they are; a token whose block's id is negative gets slot -1.

    All or nothing: where the free list runs out, a request exceeds its table, the tokens
    exceed ``max_tokens`` or a length is negative, bit ``MKV_FLAG_DST_RANGE`` is set in
    ``error_flags``, the tables are left alone and the step is empty (``lens`` is ``held``,
    every slot -1)."""
    made = _usual.slots(held, new, block_tables, free_blocks, free_at, block_size, max_tokens,
                        error_flags)
    if made is not None:
        if type(made) is int:
            _lib.check(made)
        return StepSlots(*made)
    device = block_tables.device
    if not block_tables.is_cuda:
        raise RuntimeError("step_slots: block_tables is not on a HIP device; there is no CPU path")
    at, stride, n, width = _table(block_tables, device)
    if n > _lib.MKV_MAX_REQUESTS:
        raise ValueError(f"{n} requests: at most {_lib.MKV_MAX_REQUESTS}")
    if n > 1 and stride < width:
        raise ValueError("block_tables' rows overlap")
    block_size, max_tokens = int(block_size), int(max_tokens)
    if block_size <= 0 or max_tokens < 0 or max_tokens >= 2**31:
        raise ValueError(f"block_size {block_size}, max_tokens {max_tokens}")
    held_at, new_at = _int32("held", held, device, n), _int32("new", new, device, n)
    free_list = _int32("free_blocks", free_blocks, device, None)
    free_from = _int32("free_at", free_at, device, 1)
    flags = _flags(error_flags, device)

    def out(size, dtype=torch.int32):
        return torch.empty(size, dtype=dtype, device=device)

    step = StepSlots(out(n + 1), out(n), out(max_tokens, torch.int64), out(max_tokens), out(1))
    with _on(device, _current(device)):
        _lib.check(_lib.lib().mkv_step_slots(
            held_at, new_at, n, at, stride, width, free_list, free_blocks.shape[0], free_from,
            block_size, step.starts.data_ptr(), step.lens.data_ptr(), step.slots.data_ptr(),
            step.positions.data_ptr(), max_tokens, step.free_at.data_ptr(), flags,
            current_stream(device)))
    return step


def store_scaled(cache: ScaledCache, k: torch.Tensor, v: torch.Tensor,
                 block_tables: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, *,
                 error_flags: torch.Tensor | None = None) -> None:
    """Write the step's new rows ``k`` and ``v`` (``[tokens, heads, D]``, bf16, fp16 or fp32)
    into their blocks.

    A block that its request begins here gets the smallest scale that fits its new rows.  A
    block begun in an earlier step keeps its rows and at least its scale; where the new rows
    need a larger one, the old rows are encoded again under it, which keeps their values but
    for codes that become subnormal.  Infinities saturate, NaNs stay NaN."""
    done = _usual.store(*cache.handle, k, v, block_tables, starts, lens, error_flags)
    if done is not None:
        if done is not True:
            _lib.check(done)
        return
    device = cache.device
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (cache.heads, cache.head_size):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)}: [tokens, {cache.heads}, "
                         f"{cache.head_size}]")
    if k.dtype not in _ROW_DTYPES or v.dtype != k.dtype:
        raise TypeError(f"k {k.dtype} and v {v.dtype}: one of {_ROW_DTYPES}")
    if k.device != device or v.device != device:
        raise ValueError(f"k on {k.device}, v on {v.device}, the cache on {device}")
    _no_gradient("store_scaled", k=k, v=v)
    if k.stride(2) != 1 or v.stride(2) != 1:
        raise ValueError("rows must be contiguous in the last dimension")
    at, stride, n, width = _table(block_tables, device)
    args = (
        ctypes.byref(cache.desc), k.data_ptr(), *_steps(k), v.data_ptr(), *_steps(v), k.shape[0],
        dtype_code(k.dtype), at, stride, width, _int32("starts", starts, device, n + 1),
        _int32("lens", lens, device, n), n, _flags(error_flags, device))
    with _on(device, _current(device)):
        _lib.check(_lib.lib().mkv_store_scaled(*args, current_stream(device)))


def _steps(t: torch.Tensor) -> tuple[int, int]:
    """Token and head strides; of a dimension of one element, 0 (torch gives it any)."""
    return (t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0)


def _rows_of(t: torch.Tensor) -> Rows:
    size = t.element_size()
    steps = ((size * s, n) for s, n in zip(_steps(t), t.shape))
    return Rows(t.data_ptr(), size * t.shape[2], tuple(steps))


def attend_scaled(cache: ScaledCache, q: torch.Tensor, block_tables: torch.Tensor,
                  starts: torch.Tensor, lens: torch.Tensor, *, softmax_scale: float | None = None,
                  max_new: int | None = None, max_len: int | None = None,
                  out: torch.Tensor | None = None,
                  error_flags: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the step's queries ``q`` (``[tokens, query heads, D]``, bf16 or
    fp16) over the cache; query head h reads KV head ``h // (query heads / heads)``.

    Row i of request r stands at position ``lens[r] - new[r] + i`` and sees the positions up
    to its own: store the step's rows first.  ``softmax_scale``: ``D ** -0.5`` unless given.
    A row that sees nothing is zeros; rows of ``out`` behind ``starts[-1]`` are left as they
    were (in a fresh ``out``, undefined).  ``out``'s rows share no memory with each other, ``q`` or
    the cache (ranges that interleave in strides that differ are taken to); it is refused.
    Sums and softmax statistics are fp32.  Where a probability meets V it is off by at most 2^-17
    of itself, or by 2^-8, as a bf16 output itself is, for bf16 queries in the kernel of more than
    32 rows (``max_new``, or without it the tokens, times the query heads of a KV head).

    ``max_new`` and ``max_len``: the largest number of new tokens and of tokens of a request,
    where the host knows them (a captured step: the largest that will be replayed).  They choose
    launch shapes, and a result only by the order of its sums and the roundings above.  Without
    ``max_new`` a batch's decode step is taken for one request's chunk."""
    got = _usual.attend(*cache.handle, q, block_tables, starts, lens, softmax_scale, max_new,
                        max_len, out, error_flags)
    if got is not None:
        if type(got) is int:
            _lib.check(got)
        return got
    desc, out = _attend_desc("attend_scaled", cache, q, block_tables, starts, lens, softmax_scale,
                             max_new, max_len, out, error_flags)
    device = cache.device
    L = _lib.lib()
    need = L.mkv_attend_workspace_size(ctypes.byref(desc))
    with _on(device, _current(device)):
        if need > 0:  # the allocator hands it on in stream order
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            desc.workspace, desc.workspace_bytes = workspace.data_ptr(), need
        _lib.check(L.mkv_attend_scaled(ctypes.byref(desc), current_stream(device)))
    return out


def _attend_desc(who: str, cache: ScaledCache, q, block_tables, starts, lens, softmax_scale, max_new,
                 max_len, out, error_flags) -> tuple[_lib.AttendDesc, torch.Tensor]:
    """An attention call's descriptor, but for its workspace, and its output."""
    device, d = cache.device, cache.head_size
    if q.dim() != 3 or q.shape[2] != d or q.shape[1] == 0 or q.shape[1] % cache.heads:
        raise ValueError(f"q {tuple(q.shape)}: [tokens, a multiple of {cache.heads}, {d}]")
    if q.dtype not in _QUERY_DTYPES:
        raise TypeError(f"q {q.dtype}: one of {_QUERY_DTYPES}")
    if q.device != device:
        raise ValueError(f"q on {q.device}, the cache on {device}")
    _no_gradient(who, q=q, out=out)
    if q.stride(2) != 1:
        raise ValueError("q's rows must be contiguous in the last dimension")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or out.stride(2) != 1:
        raise ValueError(f"out {out.dtype} {tuple(out.shape)} on {out.device} does not fit q")
    else:
        written = _rows_of(out)
        if share(written, _rows_of(q)):
            raise ValueError("out shares memory with q")
        if any(share(written, r) for r in (*cache.rows, cache.scale_rows)):
            raise ValueError("out shares memory with the cache")
    at, stride, n, width = _table(block_tables, device)
    desc = _lib.AttendDesc()
    ctypes.memmove(ctypes.byref(desc), ctypes.byref(cache.desc), ctypes.sizeof(cache.desc))
    desc.q, (desc.q_token_stride, desc.q_head_stride) = q.data_ptr(), _steps(q)
    desc.out, (desc.out_token_stride, desc.out_head_stride) = out.data_ptr(), _steps(out)
    desc.block_tables, desc.table_stride, desc.table_width, desc.requests = at, stride, width, n
    desc.starts = _int32("starts", starts, device, n + 1)
    desc.lens = _int32("lens", lens, device, n)
    desc.error_flags = _flags(error_flags, device)
    desc.tokens, desc.q_heads, desc.dtype = q.shape[0], q.shape[1], dtype_code(q.dtype)
    # (no request has more than 2^31 - 1 tokens, whatever the hints say)
    desc.max_new, desc.max_len = (max(-1, min(int(m or 0), 2**31 - 1)) for m in (max_new, max_len))
    desc.softmax_scale = d ** -0.5 if softmax_scale is None else float(softmax_scale)
    return desc, out


class ScaledShifts:
    """Shifts between block-scaled caches: ``src`` and ``dst`` are lists of one
    :class:`ScaledCache` a layer, of one geometry each (block sizes and layouts may differ
    between the two).  ``inv_freq``: fp32 ``[rotary / 2]``, ``rotary`` a multiple of 32; None
    moves keys without turning them.

    Layers may share memory, of one list or of both, where they are one cache or views of whole
    blocks of one: :meth:`run` then refuses to read a block that it writes, in any layer.  A layer
    that stands in both lists twice is moved once.  No two of ``dst`` share memory otherwise.

    One runner serves every step over the same caches (:meth:`run`).  A graph that captured a
    step reads the runner's buffers: the runner outlives it."""

    def __init__(self, src: list, dst: list, inv_freq: torch.Tensor | None):
        if len(src) != len(dst) or not src:
            raise ValueError(f"src has {len(src)} layers, dst {len(dst)}")
        for caches in (src, dst):
            first = caches[0]
            for c in caches[1:]:
                if _geometry(c) != _geometry(first) or c.device != first.device:
                    raise ValueError("the layers of one side differ in geometry or device")
        a, b = src[0], dst[0]
        if (a.heads, a.head_size) != (b.heads, b.head_size) or a.device != b.device:
            raise ValueError("src and dst differ in heads, head_size or device")
        # a pair of caches that is there before writes the same bytes to the same place
        pairs = list({(bytes(s.desc), bytes(d.desc)): (s, d) for s, d in zip(src, dst)}.values())
        src, dst = [s for s, _ in pairs], [d for _, d in pairs]
        self.src, self.dst, self.device, self.layers = src, dst, b.device, len(dst)
        # where a source block n is the destination's block n + offset of some layer
        offsets = set()
        for i, j in _near(src + dst):
            if i >= len(src) and _offset(dst[i - len(src)], dst[j - len(src)]) is not None:
                raise ValueError("two layers of dst share memory")
            if i < len(src) <= j:
                offsets.add(_offset(src[i], dst[j - len(src)]))
        offsets.discard(None)
        self.rotary = 0 if inv_freq is None else 2 * int(inv_freq.numel())
        if self.rotary % 32 or self.rotary > b.head_size:
            raise ValueError(f"rotary {self.rotary}: a multiple of 32, at most {b.head_size}")
        self.inv_freq = None if inv_freq is None else inv_freq.detach().to(
            "cpu", torch.float32).contiguous()
        d = self.desc = _lib.ScaledShiftDesc()
        d.src, d.dst = a.desc, b.desc
        d.layers, d.rotary = self.layers, self.rotary
        self._one_cache = 0 in offsets and _geometry(a) == _geometry(b)
        self._offsets = sorted(offsets - {0} if self._one_cache else offsets)
        self._unit_bytes = 4 * _lib.unit_words(a.block_size, b.block_size)
        with _on(self.device, _current(self.device)):
            # (a copy from pageable memory: it is there when the call returns)
            self._bases = torch.tensor(
                [[[c.desc.k_base or 0, c.desc.v_base or 0, c.desc.scales or 0] for c in caches]
                 for caches in (src, dst)], dtype=torch.int64).to(self.device)
            self._streams = {current_stream(self.device)}
        d.src_layers = self._bases[0].data_ptr()
        d.dst_layers = self._bases[1].data_ptr()

    def run(self, rows: list, src_table, dst_table, *,
            error_flags: torch.Tensor | None = None) -> None:
        """Shift ``rows`` on the current stream: ``mkv_span_t`` field tuples (src_pos, dst_pos,
        src_index, dst_index, n_tokens, delta, 0, 0), positions through the block tables
        ``src_table`` and ``dst_table`` (int32, on the host; a span's tables begin at its
        src_index and dst_index).  ``dst_pos`` is a multiple of the destination's block size:
        a span writes whole blocks, each anew under the scale of its rows; behind a span's
        last row the codes stay, but not the values, whose scale was another.  A block one of
        whose rows has no source (a table too short, an id out of range) is left as it was,
        with ``MKV_FLAG_SRC_RANGE`` in ``error_flags``.  The destination blocks of one call are
        distinct, and none is one of its source blocks (in one cache; both are refused)."""
        n, bs = len(rows), self.dst[0].block_size
        if n > _lib.MKV_MAX_SPANS:
            raise ValueError(f"{n} spans: at most {_lib.MKV_MAX_SPANS}")
        src, src_at, src_len = _host_table(src_table)
        dst, dst_at, dst_len = _host_table(dst_table)
        most = deltas = tokens = 0
        for r in rows:
            if r[0] < 0 or r[1] < 0 or r[4] < 0:
                raise ValueError("a span's position or length is negative")
            if r[1] % bs:
                raise ValueError(f"a destination position is not a multiple of {bs}")
            tokens |= int(r[4])
            most += min(-(-int(r[4]) // bs), dst_len)  # units: blocks beyond the table get none
            deltas |= int(r[5])
        if tokens == 0:
            return
        spans = _span_struct(n).pack(*chain.from_iterable(rows))
        # Units, then the spans' rotation tables, in one buffer.  What fits into one launch's
        # arguments goes along in them, more through pinned memory and a copy (377 units: 41 us
        # against 49 for the launches it would take, 1,388 units: 634 against 786).  A capture
        # takes all of it in arguments: it may not allocate pinned memory, and its replays
        # then read nothing on the host.
        turns = n * 8 * self.rotary if deltas else 0
        room = most * self._unit_bytes
        small = room + turns <= _lib.SHIFT_HOST_BYTES or self._capturing()
        host = torch.empty(room + turns, dtype=torch.uint8, pin_memory=not small)
        at, d, L = host.data_ptr(), self.desc, _lib.lib()
        made, flag = ctypes.c_int64(), ctypes.c_int32()
        _lib.check(L.mkv_scaled_units(
            spans, n, src_at, src_len, dst_at, dst_len,
            ctypes.byref(d.dst if self._one_cache else d.src), ctypes.byref(d.dst), at, most,
            ctypes.byref(made), ctypes.byref(flag)))
        if self._offsets:
            self._refuse_shared(host.numpy()[:made.value * self._unit_bytes].view(np.int32))
        if turns:
            steps = np.ascontiguousarray(np.frombuffer(spans, _lib.SPAN_DTYPE)["delta"])
            _lib.check(L.mkv_rope_tables(steps.ctypes.data, n, self.inv_freq.data_ptr(),
                                         self.rotary, at + room))
        flags = _flags(error_flags, self.device)
        desc = _lib.ScaledShiftDesc.from_buffer_copy(d)
        desc.n_spans, desc.n_units = n, made.value
        if not turns:
            desc.rotary = 0
        with _on(self.device, _current(self.device)):
            stream = current_stream(self.device)
            if stream not in self._streams:
                self._bases.record_stream(torch.cuda.current_stream(self.device))
                self._streams.add(stream)
            if flag.value and flags:
                error_flags[(0,) * error_flags.dim()].bitwise_or_(flag.value)
            if not desc.n_units:
                return
            blob = host
            if small:
                desc.on_host = 1
            else:
                # the caching host allocator keeps ``host`` until this copy has completed
                blob = host.to(self.device, non_blocking=True)
            at = blob.data_ptr()
            desc.units, desc.tables = at, at + room if turns else None
            _lib.check(L.mkv_shift_scaled(ctypes.byref(desc), stream))

    def _refuse_shared(self, units: np.ndarray) -> None:
        """Raise where a unit's source block is another's destination, in views of one cache."""
        u = units.reshape(-1, self._unit_bytes // 4)
        bs = self.src[0].block_size
        used = (u[:, 3] + u[:, 1] + bs - 1) // bs
        ids = u[:, 4:]
        ids = ids[(np.arange(ids.shape[1]) < used[:, None]) & (ids >= 0)]
        for offset in self._offsets:
            both = np.intersect1d(ids.astype(np.int64) + offset, u[:, 0])
            if both.size:
                raise _lib.KVShiftError(
                    _lib.MKV_ERR_ARG, f"block {both[0]} is a destination and, {offset} blocks "
                    "behind, a source")

    def _capturing(self) -> bool:
        with _on(self.device, _current(self.device)):
            return torch.cuda.is_current_stream_capturing()


def _near(caches: list) -> set:
    """The pairs of places, the lower first, of caches whose address ranges meet."""
    ranges = sorted((r.base, r.end, i) for i, c in enumerate(caches)
                    for r in (*c.rows, c.scale_rows))
    pairs, open_ranges = set(), []
    for base, end, i in ranges:
        open_ranges = [r for r in open_ranges if r[0] > base]
        pairs.update((min(i, j), max(i, j)) for _, j in open_ranges if i != j)
        open_ranges.append((end, i))
    return pairs


def _offset(a: ScaledCache, b: ScaledCache) -> int | None:
    """The n by which block i of ``a`` is block i + n of ``b``; None where they share nothing."""
    if not (share(a.scale_rows, b.scale_rows)
            or any(share(x, y) for x in a.rows for y in b.rows)):
        return None
    x, y = a.desc, b.desc
    step = max(x.block_stride, y.block_stride)  # (0 in a cache of one block)
    n, rest = divmod((x.k_base or 0) - (y.k_base or 0), step) if step else (0, x.k_base != y.k_base)
    if (rest or x.v_base - y.v_base != n * step or x.scales - y.scales != 2 * a.heads * n
            or _geometry(a)[2:] != _geometry(b)[2:] or len(a.rows) != len(b.rows)
            or (x.block_stride != y.block_stride and min(x.num_blocks, y.num_blocks) > 1)):
        raise ValueError("two caches share memory, but not as views of one cache's blocks")
    return n


def _geometry(c: ScaledCache) -> tuple:
    d = c.desc
    return (d.num_blocks, d.block_stride, d.head_stride, d.token_stride, d.block_size, d.heads,
            d.head_size)


def _host_table(t) -> tuple:
    """A block table on the host: what keeps it alive, its address and its length."""
    if isinstance(t, torch.Tensor):
        if t.is_cuda:
            raise ValueError("a shift's block tables are on the host")
        if t.dtype == torch.int32 and t.is_contiguous():
            return t, t.data_ptr(), t.numel()
        t = t.detach().numpy()
    t = np.asarray(t).reshape(-1)
    if t.dtype != np.int32:
        if t.dtype.kind not in "iu" or (t.size and (t.min() < -2**31 or t.max() >= 2**31)):
            raise ValueError("a shift's block tables hold int32 block ids")
    t = np.ascontiguousarray(t, dtype=np.int32)
    return t, t.ctypes.data, t.size
