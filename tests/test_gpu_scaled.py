"""The block-scaled cache's operators on the GPU against their definitions in 64 bits
(:mod:`tests.scaled_plain`): slots, store and shift exactly, attention within its roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import (
    ScaledCache,
    ScaledShifts,
    attend_scaled,
    scatter_shifted,
    step_slots,
    store_scaled,
)
from marathon_amd import _lib
from marathon_amd.shift_kernels import inv_freq_for
from tests import scaled_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def i32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def requests_of(new, held, bs, rng, spare=3, gap=1):
    """Shuffled tables for requests that hold ``held`` tokens before ``new``; the numpy tables
    and the block count.  Entries behind a request's last block hold ids out of range."""
    need = [-(-(h + n) // bs) for h, n in zip(held, new)]
    count = sum(need) + spare
    ids = rng.permutation(count).astype(np.int32)
    tables = np.full((len(new), max(need, default=0) + gap), 2**31 - 1, np.int32)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = ids[at:at + n]
        at += n
    return tables, count


class Cache:
    """A cache on the GPU and its twin on the host."""

    def __init__(self, gpu, rng, blocks, heads, d, bs, layout="hnd", split=False, fill="values"):
        self.bs, self.layout = bs, layout
        if fill == "values":
            x = rng.standard_normal((blocks, bs, heads, 2, d)) * np.exp2(
                rng.integers(-6, 7, (blocks, 1, heads, 2, 1)))
            self.codes = np.zeros(x.shape, np.uint8)
            self.scales = np.zeros((blocks, heads, 2), np.uint8)
            for b in range(blocks):
                for h in range(heads):
                    for w in range(2):
                        e = plain.exponent_for(x[b, :, h, w])
                        self.codes[b, :, h, w] = plain.encode(x[b, :, h, w] * 2.0 ** -e)
                        self.scales[b, h, w] = e + 127
        else:  # anything: NaN codes and NaN scales among it
            self.codes = rng.integers(0, 256, (blocks, bs, heads, 2, d)).astype(np.uint8)
            self.scales = rng.integers(0, 256, (blocks, heads, 2)).astype(np.uint8)
        x = self.codes if layout == "nhd" else self.codes.transpose(0, 2, 1, 3, 4)
        if split:
            planes = [torch.from_numpy(np.ascontiguousarray(x[..., w, :])).to(gpu) for w in (0, 1)]
            self.planes = [p.view(torch.float8_e4m3fn) for p in planes]
            kv, v = self.planes
        else:
            kv = torch.from_numpy(x.reshape(*x.shape[:3], 2 * d).copy()).to(gpu)
            kv, v = kv.view(torch.float8_e4m3fn), None
            self.planes = [kv]
        self.dev_scales = torch.from_numpy(self.scales.copy()).to(gpu).view(torch.float8_e8m0fnu)
        self.dev = ScaledCache(kv, self.dev_scales, layout, bs, v)

    def read(self):
        """(codes, scales) of the GPU's cache in the host's order."""
        got = [p.view(torch.uint8).cpu().numpy() for p in self.planes]
        x = np.stack(got, -2) if len(got) == 2 else got[0].reshape(*got[0].shape[:3], 2, -1)
        x = x if self.layout == "nhd" else x.transpose(0, 2, 1, 3, 4)
        return x, self.dev_scales.view(torch.uint8).cpu().numpy()

    def check(self):
        codes, scales = self.read()
        nan = (self.codes & 127) == 127
        assert np.array_equal((codes & 127) == 127, nan)
        assert np.array_equal(codes[~nan], self.codes[~nan])
        assert np.array_equal(scales, self.scales)


# ------------------------------------------------------------------------------- slots


@pytest.mark.parametrize("requests,bs,most,long", [
    (1, 16, 1, 0), (1, 16, 700, 90), (5, 16, 1, 40), (64, 32, 9, 100), (65, 16, 30, 100),
    (700, 16, 3, 300), (1300, 7, 40, 50), (4096, 1, 2, 9), (3, 128, 5000, 4000)])
def test_slots_equal_the_plain_ones(gpu, requests, bs, most, long):
    rng = np.random.default_rng(requests * 131 + bs)
    held = rng.integers(0, long + 1, requests)
    new = rng.integers(0, most + 1, requests)
    if most == 1:
        new[:] = 1
    width = int(max(-(-(held + new) // bs))) + 2
    tables = rng.integers(0, 1 << 20, (requests, width)).astype(np.int32)
    total = int(new.sum())
    need = int((-(-(held + new) // bs) - -(-held // bs)).sum())
    free = rng.permutation(need + 5).astype(np.int32) + 7
    wt, ws, wslots, wpos, wat = plain.step_slots(held.tolist(), new.tolist(), tables, free, 3, bs)
    dev = torch.from_numpy(tables).to(gpu)
    flags = i32([0], gpu)
    pad = 13
    step = step_slots(i32(held, gpu), i32(new, gpu), dev, i32(free, gpu), i32([3], gpu), bs,
                      total + pad, error_flags=flags)
    assert flags.item() == 0
    assert np.array_equal(dev.cpu().numpy(), wt)
    assert step.starts.tolist() == ws and step.lens.tolist() == (held + new).tolist()
    assert step.slots.tolist() == wslots + [-1] * pad
    assert step.positions.tolist() == wpos + [0] * pad
    assert step.free_at.item() == wat


@pytest.mark.parametrize("why", ["free", "width", "tokens", "negative", "held", "cursor"])
def test_slots_are_all_or_nothing(gpu, why):
    held, new = [20, 5, 0], [30, 2, 40]
    width, free, cap, at = 4, 6, 72, 1
    if why == "free":
        free = 5  # blocks needed: 2 + 0 + 3 from free_at 1
    elif why == "width":
        width = 3
    elif why == "tokens":
        cap = 71
    elif why == "negative":
        new[1] = -1
    elif why == "held":
        held[0] = -3
    else:
        at = -1
    tables = torch.full((3, width), 9, dtype=torch.int32, device=gpu)
    flags = i32([0], gpu)
    step = step_slots(i32(held, gpu), i32(new, gpu), tables, i32(list(range(free)), gpu),
                      i32([at], gpu), 16, cap, error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_DST_RANGE
    assert (tables == 9).all()
    assert step.starts.tolist() == [0] * 4 and step.lens.tolist() == held
    assert (step.slots == -1).all() and (step.positions == 0).all()
    assert step.free_at.item() == at


def test_slots_of_nobody_and_of_no_tokens(gpu):
    none = torch.zeros((0, 4), dtype=torch.int32, device=gpu)
    step = step_slots(i32([], gpu), i32([], gpu), none, i32([1], gpu), i32([0], gpu), 16, 5)
    assert step.starts.tolist() == [0] and step.slots.tolist() == [-1] * 5
    tables = torch.zeros((2, 3), dtype=torch.int32, device=gpu)
    step = step_slots(i32([4, 0], gpu), i32([0, 0], gpu), tables, i32([1], gpu), i32([1], gpu), 16, 0)
    assert step.starts.tolist() == [0, 0, 0] and step.lens.tolist() == [4, 0]
    assert step.slots.numel() == 0 and step.free_at.tolist() == [1]


def test_slots_feed_the_shift_path(gpu):
    """A step's slots address the plain paged cache: scatter_shifted writes the same rows that
    the host's slots name, and padding slots write nothing."""
    heads, d, bs = 2, 64, 16
    held, new = [10, 0, 33], [7, 20, 1]
    tables = torch.zeros((3, 4), dtype=torch.int32, device=gpu)
    tables[0, 0], tables[2, :3] = 5, i32([1, 2, 3], gpu)
    step = step_slots(i32(held, gpu), i32(new, gpu), tables, i32([9, 8, 7, 6], gpu), i32([0], gpu),
                      bs, 30)
    kv = torch.zeros((10, heads, bs, 2 * d), dtype=torch.bfloat16, device=gpu)
    src = torch.randn(30, heads, 2 * d, dtype=torch.bfloat16, device=gpu)
    scatter_shifted(src, kv, step.slots, bs, True, None)
    want = torch.zeros_like(kv)
    for t, slot in enumerate(step.slots.tolist()):
        if slot >= 0:
            want[slot // bs, :, slot % bs] = src[t]
    assert step.slots.tolist()[28:] == [-1, -1]
    assert torch.equal(kv, want)


# ------------------------------------------------------------------------------- store


def loud(rng, shape, spread=6):
    """Normal values whose rows differ in size by powers of two."""
    return rng.standard_normal(shape) * np.exp2(rng.integers(-spread, spread + 1, (*shape[:2], 1)))


STORES = [  # new tokens, held tokens, heads, D, bs, layout, dtype, split planes
    ([1], [0], 1, 128, 16, "hnd", "bf16", False),
    ([1, 1, 1], [15, 16, 33], 8, 128, 16, "hnd", "bf16", False),
    ([5, 0, 40, 1], [3, 9, 0, 31], 3, 64, 16, "nhd", "fp16", False),
    ([33, 2, 100], [31, 62, 7], 2, 256, 32, "hnd", "fp32", True),
    ([70, 1], [63, 64], 5, 128, 64, "nhd", "bf16", True),
    ([300, 129], [1, 127], 2, 64, 128, "hnd", "fp32", False),
    ([4200, 37, 1, 900], [5, 0, 77, 15], 1, 64, 16, "nhd", "bf16", False),
    ([17, 16, 15], [16, 0, 1], 4, 256, 16, "hnd", "fp16", False),
]


@pytest.mark.parametrize("new,held,heads,d,bs,layout,dtype,split", STORES)
def test_store_equals_the_plain_one(gpu, new, held, heads, d, bs, layout, dtype, split):
    rng = np.random.default_rng(sum(new) + bs + d)
    tables, blocks = requests_of(new, held, bs, rng)
    cache = Cache(gpu, rng, blocks, heads, d, bs, layout, split)
    first, pad = 2, 3  # rows before the first request and behind the last belong to nobody
    starts = np.cumsum([first] + new)
    lens = [h + n for h, n in zip(held, new)]
    rows = []
    for _ in range(2):
        x = torch.from_numpy(loud(rng, (int(starts[-1]) + pad, heads, d))).to(gpu, DTYPES[dtype])
        rows.append(x)
    flags = i32([0], gpu)
    store_scaled(cache.dev, *rows, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu),
                 error_flags=flags)
    plain.store(cache.codes, cache.scales, *(x.double().cpu().numpy() for x in rows), tables,
                starts.tolist(), lens, bs)
    assert flags.item() == 0
    cache.check()


def test_store_takes_strided_rows_and_tables(gpu):
    rng = np.random.default_rng(3)
    new, held = [9, 20], [4, 0]
    tables, blocks = requests_of(new, held, 16, rng)
    cache = Cache(gpu, rng, blocks, 2, 128, 16)
    qkv = torch.from_numpy(loud(rng, (29, 2, 5 * 128))).to(gpu, torch.bfloat16)
    k, v = qkv[:, :, 128:256], qkv[:, :, 384:512]
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    wide[:, :tables.shape[1]] = i32(tables, gpu)
    store_scaled(cache.dev, k, v, wide[:, :tables.shape[1]], i32([0, 9, 29], gpu), i32([13, 20], gpu))
    plain.store(cache.codes, cache.scales, k.double().cpu().numpy(), v.double().cpu().numpy(),
                tables, [0, 9, 29], [13, 20], 16)
    cache.check()


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_store_of_infinities_nans_zeros_and_extremes(gpu, bs):
    rng = np.random.default_rng(bs)
    new, held = [bs + 5], [bs - 3]
    tables, blocks = requests_of(new, held, bs, rng)
    cache = Cache(gpu, rng, blocks, 3, 64, bs, fill="anything")
    cache.scales[...] = rng.integers(100, 140, cache.scales.shape)
    cache.dev_scales.view(torch.uint8).copy_(torch.from_numpy(cache.scales).to(gpu))
    k, v = (loud(rng, (new[0], 3, 64)).astype(np.float32) for _ in range(2))
    k[0, 0, :3] = np.inf, -np.inf, np.nan
    k[4, 1] = 0.0
    v[3:, 1] = 0.0
    k[3:, 2] = 3e38          # beyond 448 * 2^100
    k[5, 2, 7] = -1e-38
    v[6, 2] = 1e-40          # below the smallest scale's smallest code
    v[7, 0, 5] = np.nan
    v[:, 0, 9] = -0.0
    dev = [torch.from_numpy(x).to(gpu) for x in (k, v)]
    store_scaled(cache.dev, *dev, i32(tables, gpu), i32([0, new[0]], gpu), i32([2 * bs + 2], gpu))
    plain.store(cache.codes, cache.scales, k.astype(np.float64), v.astype(np.float64), tables,
                [0, new[0]], [2 * bs + 2], bs)
    cache.check()


def test_store_token_by_token_grows_the_scale(gpu):
    """One block filled a token at a time, each larger than the last: every earlier row is
    encoded again, and its value kept."""
    rng = np.random.default_rng(8)
    tables, blocks = requests_of([16], [0], 16, rng)
    cache = Cache(gpu, rng, blocks, 2, 128, 16)
    k, v = (rng.standard_normal((16, 2, 128)) * np.exp2(np.arange(16) / 2)[:, None, None]
            for _ in range(2))
    k, v = (torch.from_numpy(x).to(gpu, torch.bfloat16) for x in (k, v))
    for t in range(16):
        store_scaled(cache.dev, k[t:t + 1], v[t:t + 1], i32(tables, gpu), i32([0, 1], gpu),
                     i32([t + 1], gpu))
        plain.store(cache.codes, cache.scales, k[t:t + 1].double().cpu().numpy(),
                    v[t:t + 1].double().cpu().numpy(), tables, [0, 1], [t + 1], 16)
    cache.check()


def test_store_refuses_what_leaves_the_cache(gpu):
    """Ids out of range, a table too short, starts that leave the rows or descend, a request
    with more new tokens than tokens: flagged, nothing written for them, the others are."""
    rng = np.random.default_rng(5)
    new, held = [20, 18, 4, 3], [0, 16, 0, 0]
    tables, blocks = requests_of(new, held, 16, rng, gap=0)
    cache = Cache(gpu, rng, blocks, 1, 64, 16)
    k, v = (torch.from_numpy(loud(rng, (45, 1, 64))).to(gpu, torch.bfloat16) for _ in range(2))
    bad = tables.copy()
    bad[0, 1] = blocks          # the first request's second block
    flags = i32([0], gpu)
    store_scaled(cache.dev, k, v, i32(bad, gpu), i32([0, 20, 38, 42, 45], gpu),
                 i32([20, 60, 4, 2], gpu), error_flags=flags)  # lens: past the table; below new
    assert flags.item() == _lib.MKV_FLAG_DST_RANGE | _lib.MKV_FLAG_SPAN
    host = [x.double().cpu().numpy() for x in (k, v)]
    plain.store(cache.codes, cache.scales, *host, tables, [0, 16], [16], 16)
    # of the second request, positions 42 to 47 lie in its table
    plain.store(cache.codes, cache.scales, *(x[20:26] for x in host), tables[1:2], [0, 6], [48], 16)
    plain.store(cache.codes, cache.scales, *(x[38:42] for x in host), tables[2:3], [0, 4], [4], 16)
    cache.check()
    flags.zero_()
    store_scaled(cache.dev, k[:10], v[:10], i32(tables[:2], gpu), i32([0, 8, 30], gpu),
                 i32([8, 38], gpu), error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SPAN
    plain.store(cache.codes, cache.scales, *host, tables, [0, 8], [8], 16)
    cache.check()


# ------------------------------------------------------------------------------ attend


def bound_of(cache, q, tables, starts, lens, bs, scale, want, dtype):
    """How far an output may be from the exact one, entry by entry, from the roundings.

    Of the output: half a step, eps / 2 of it.  Of p: 2^-9 of each term for bf16 queries, 2^-17
    for fp16; of a score s: fp32 sums of D products and the scaling, (D + 4) * 2^-24 of the sum
    of the products' sizes, which multiplies p; of the exponential, the sums and the quotient:
    2^-20 in all at these lengths.  Each moves the output by at most that share of sum(p |v|)
    (and of |out| for the denominator): bounded by twice it."""
    eps = torch.finfo(dtype).eps / 2
    out = np.zeros(want.shape)
    group = q.shape[1] // cache.codes.shape[2]
    d = q.shape[2]
    for r, last in enumerate(lens):
        s0, s1 = starts[r], starts[r + 1]
        x = plain.rows(cache.codes, cache.scales, tables[r], max(last, 0), bs)
        for t in range(s0, s1):
            sees = last - (s1 - s0) + (t - s0) + 1
            if sees <= 0:
                continue
            for h in range(q.shape[1]):
                kk, vv = x[:sees, h // group, 0], x[:sees, h // group, 1]
                s = kk @ q[t, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                size = (np.abs(kk) @ np.abs(q[t, h]) * scale).max()
                share = (2.0 ** -9 if dtype == torch.bfloat16 else 2.0 ** -17) + 2.0 ** -20
                share += (d + 4) * 2.0 ** -24 * size
                out[t, h] = 2 * share * (p @ np.abs(vv))
    return out + eps * (np.abs(want) + out) + 1e-30


def attend_case(gpu, rng, new, held, heads, group, d, bs, layout, dtype, split=False, dirty=True,
                scale=None, loud_keys=False, **kw):
    tables, blocks = requests_of(new, held, bs, rng)
    cache = Cache(gpu, rng, blocks, heads, d, bs, layout, split)
    lens = [h + n for h, n in zip(held, new)]
    if dirty:  # rows behind a request's last one hold NaNs, on the GPU alone
        raw = [p.view(torch.uint8) for p in cache.planes]
        for r, n in enumerate(lens):
            if n % bs:
                b = int(tables[r, n // bs])
                for p in raw:
                    (p[b, n % bs:] if layout == "nhd" else p[b, :, n % bs:]).fill_(0x7F)
    starts = np.cumsum([0] + new)
    pad = 2
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]) + pad, heads * group, d))
                         * (4.0 if loud_keys else 1.0)).to(gpu, DTYPES[dtype])
    out = torch.full_like(q, 77.0)
    flags = i32([0], gpu)
    got = attend_scaled(cache.dev, q, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), out=out,
                        softmax_scale=scale, error_flags=flags, **kw)
    assert got is out and flags.item() == 0
    assert (out[int(starts[-1]):] == 77.0).all()
    qh = q.double().cpu().numpy()
    s = scale or d ** -0.5
    want = plain.attend(cache.codes, cache.scales, qh, tables, starts, lens, bs, s)[:starts[-1]]
    tol = bound_of(cache, qh, tables, starts, lens, bs, s, want, q.dtype)
    off = np.abs(out.double().cpu().numpy()[:starts[-1]] - want)
    assert (off <= tol).all(), float((off / tol).max())


ATTENDS = [  # new, held, heads, group, D, bs, layout, dtype
    ([1], [0], 1, 1, 64, 16, "hnd", "bf16"),
    ([1], [700], 2, 5, 128, 16, "hnd", "bf16"),
    ([1, 1, 1, 1], [0, 15, 16, 300], 2, 4, 128, 16, "nhd", "bf16"),
    ([1, 1], [31, 1000], 1, 16, 128, 32, "hnd", "fp16"),
    ([3, 0, 1, 17], [5, 40, 0, 100], 3, 3, 64, 16, "nhd", "fp16"),
    ([2, 5], [600, 63], 2, 8, 256, 64, "hnd", "bf16"),
    ([1, 40], [127, 200], 1, 7, 128, 128, "nhd", "bf16"),
    ([129, 1, 64], [0, 517, 3], 1, 2, 128, 16, "hnd", "bf16"),
    ([70], [530], 2, 1, 256, 16, "nhd", "fp16"),
    ([33, 150], [0, 90], 2, 5, 64, 32, "hnd", "bf16"),
    ([1], [3], 1, 40, 128, 16, "hnd", "bf16"),
    # a chunk beside decoding requests, which get a launch of their own
    ([1, 1, 260, 3, 1, 0, 2], [700, 3, 40, 75, 15, 8, 90], 2, 8, 128, 16, "hnd", "bf16"),
    ([300, 1, 1], [600, 1400, 0], 1, 8, 64, 16, "nhd", "fp16"),
]


@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("new,held,heads,group,d,bs,layout,dtype", ATTENDS)
def test_attend_matches_the_plain_one(gpu, new, held, heads, group, d, bs, layout, dtype, known):
    rng = np.random.default_rng(sum(new) * 7 + d + bs)
    kw = dict(max_new=max(new), max_len=max(h + n for h, n in zip(held, new))) if known else {}
    attend_case(gpu, rng, new, held, heads, group, d, bs, layout, dtype, split=d == 256, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_with_sharp_scores(gpu, dtype):
    """Scores that spread over hundreds: the running largest moves often."""
    rng = np.random.default_rng(4)
    attend_case(gpu, rng, [1, 30], [900, 200], 2, 4, 128, 16, "hnd", dtype, loud_keys=True)


def test_attend_hints_change_nothing_but_the_order(gpu):
    """Wrong hints: fewer tokens and shorter requests than there are."""
    rng = np.random.default_rng(6)
    attend_case(gpu, rng, [1, 50, 3], [2000, 10, 40], 1, 4, 128, 16, "hnd", "bf16", max_new=1,
                max_len=16)


def test_rows_that_see_nothing_are_zeros(gpu):
    rng = np.random.default_rng(9)
    cache = Cache(gpu, rng, 4, 2, 128, 16, fill="anything")
    q = torch.randn(9, 4, 128, device=gpu, dtype=torch.bfloat16)
    tables = i32([[0, 1], [2, 3], [1, 2]], gpu)
    # no tokens at all; fewer tokens than new ones: the first rows stand before position 0
    out = attend_scaled(cache.dev, q, tables, i32([0, 3, 6, 9], gpu), i32([0, -5, 1], gpu))
    assert (out[:8] == 0).all() and out[8].isfinite().sum() >= 0
    empty = attend_scaled(cache.dev, q[:0], tables, i32([0, 0, 0, 0], gpu), i32([5, 5, 5], gpu))
    assert empty.shape == (0, 4, 128)


@pytest.mark.parametrize("new,group,d", [([6], 2, 128), ([40], 3, 64), ([300], 2, 128),
                                         ([20], 2, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_nan_reaches_only_the_rows_that_see_it(gpu, new, group, d, dtype):
    """NaN and large values among a chunk's own tokens: rows before them are as without."""
    rng = np.random.default_rng(d + new[0])
    held = [75]
    tables, blocks = requests_of(new, held, 16, rng)
    cache = Cache(gpu, rng, blocks, 1, d, 16)
    n = held[0] + new[0]
    q = torch.randn(new[0], group, d, device=gpu).to(DTYPES[dtype])
    args = (i32(tables, gpu), i32([0, new[0]], gpu), i32([n], gpu))
    clean = attend_scaled(cache.dev, q, *args)
    at = held[0] + new[0] // 2
    block, row = int(tables[0, at // 16]), at % 16
    raw = cache.planes[0].view(torch.uint8)
    raw[block, 0, row, 2 * d - 3] = 0x7F  # one dimension of V
    got = attend_scaled(cache.dev, q, *args)
    before = new[0] // 2
    assert torch.equal(got[:before], clean[:before])
    assert got[before:, :, d - 3].isnan().all()
    keep = [i for i in range(d) if i != d - 3]
    assert torch.equal(got[before:][..., keep], clean[before:][..., keep])
    raw[block, 0, row, 5] = 0xFF  # and K: the whole row's scores
    got = attend_scaled(cache.dev, q, *args)
    assert torch.equal(got[:before], clean[:before]) and got[before:].isnan().all()


def test_a_nan_query_row_stays_alone(gpu):
    rng = np.random.default_rng(2)
    tables, blocks = requests_of([5], [60], 16, rng)
    cache = Cache(gpu, rng, blocks, 1, 128, 16)
    q = torch.randn(5, 4, 128, device=gpu, dtype=torch.bfloat16)
    args = (i32(tables, gpu), i32([0, 5], gpu), i32([65], gpu))
    clean = attend_scaled(cache.dev, q, *args)
    q[2, 1, 7], q[3, 0, 1] = float("nan"), float("inf")
    got = attend_scaled(cache.dev, q, *args)
    hurt = torch.zeros(5, 4, dtype=torch.bool, device=gpu)
    hurt[2, 1] = hurt[3, 0] = True
    assert got[hurt].isnan().all() and torch.equal(got[~hurt], clean[~hurt])


def test_pages_out_of_range_are_not_seen(gpu):
    """A bad block id in the middle of a history, and a history past its table."""
    rng = np.random.default_rng(12)
    cache = Cache(gpu, rng, 6, 2, 128, 16)
    q = torch.randn(2, 4, 128, device=gpu, dtype=torch.bfloat16)
    flags = i32([0], gpu)
    for bad in (-1, 6, 2**31 - 1):
        flags.zero_()
        got = attend_scaled(cache.dev, q, i32([[0, 1, bad, 3], [4, 5, 0, 1]], gpu),
                            i32([0, 1, 2], gpu), i32([64, 64], gpu), error_flags=flags)
        assert flags.item() == _lib.MKV_FLAG_SRC_RANGE
        want = attend_scaled(cache.dev, q, i32([[0, 1, 3], [4, 5, 0]], gpu), i32([0, 1, 1], gpu),
                             i32([48, 48], gpu))
        assert torch.allclose(got[0].float(), want[0].float(), atol=0.02, rtol=0.02)
    flags.zero_()
    got = attend_scaled(cache.dev, q[:1], i32([[0, 1]], gpu), i32([0, 1], gpu), i32([50], gpu),
                        error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SRC_RANGE
    assert torch.equal(got, attend_scaled(cache.dev, q[:1], i32([[0, 1]], gpu), i32([0, 1], gpu),
                                          i32([32], gpu)))
    flags.zero_()  # starts that leave q: skipped
    out = torch.full_like(q, 5.0)
    attend_scaled(cache.dev, q, i32([[0, 1], [2, 3]], gpu), i32([0, 1, 9], gpu), i32([20, 30], gpu),
                  out=out, error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SPAN and (out[1] == 5.0).all() and (out[0] != 5.0).any()


def test_attend_strides_and_scale(gpu):
    rng = np.random.default_rng(21)
    new, held = [4, 1], [100, 37]
    tables, blocks = requests_of(new, held, 16, rng)
    cache = Cache(gpu, rng, blocks, 2, 64, 16)
    wide = torch.randn(5, 4, 3 * 64, device=gpu, dtype=torch.bfloat16)
    q = wide[:, :, 64:128]
    out = torch.zeros(5, 4, 128, device=gpu, dtype=torch.bfloat16)
    args = (i32(tables, gpu), i32([0, 4, 5], gpu), i32([104, 38], gpu))
    attend_scaled(cache.dev, q, *args, out=out[..., 64:], softmax_scale=0.3)
    want = attend_scaled(cache.dev, q.contiguous(), *args, softmax_scale=0.3)
    assert torch.equal(out[..., 64:], want) and (out[..., :64] == 0).all()


def test_attend_long_history_in_parts(gpu):
    """A history cut into parts and joined, against the plain softmax in fp64 on the GPU."""
    rng = np.random.default_rng(31)
    d, heads, group, n = 128, 2, 4, 20011
    blocks = -(-n // 16) + 1
    codes = torch.randint(0, 0x60, (blocks, heads, 16, 2 * d), device=gpu, dtype=torch.uint8)
    codes |= torch.randint(0, 2, codes.shape, device=gpu, dtype=torch.uint8) << 7
    scales = torch.randint(121, 125, (blocks, heads, 2), device=gpu, dtype=torch.uint8)
    cache = ScaledCache(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), "hnd")
    table = torch.from_numpy(rng.permutation(blocks)[:blocks - 1].astype(np.int32)).to(gpu)[None]
    q = torch.randn(3, heads * group, d, device=gpu, dtype=torch.bfloat16)
    got = attend_scaled(cache, q, table, i32([0, 3], gpu), i32([n], gpu))
    x = codes[table[0].long()].view(torch.float8_e4m3fn).double()
    x = x.transpose(1, 2).reshape(-1, heads, 2, d)
    s = torch.exp2(scales[table[0].long()].double() - 127).repeat_interleave(16, 0)
    x = (x * s[..., None])[:n]
    for t in range(3):
        sees = n - 2 + t
        for h in range(heads * group):
            score = x[:sees, h // group, 0] @ q[t, h].double() * d ** -0.5
            p = torch.softmax(score, 0)
            want = p @ x[:sees, h // group, 1]
            tol = 2 * (2.0 ** -9 + 2.0 ** -16) * (p @ x[:sees, h // group, 1].abs())
            tol = tol + 2.0 ** -8 * (want.abs() + tol)
            assert ((got[t, h].double() - want).abs() <= tol).all()


# ------------------------------------------------------------------------------- shift


SHIFTS = [  # spans (src_pos, dst_pos, n, delta), heads, D, rotary, sbs, dbs, layouts
    ([(0, 0, 16, 0)], 1, 128, 128, 16, 16, "hnd", "hnd"),
    ([(5, 16, 33, 11), (100, 64, 1, -36)], 8, 128, 128, 16, 16, "nhd", "hnd"),
    ([(3, 32, 100, 700)], 3, 64, 32, 16, 32, "hnd", "nhd"),
    ([(17, 0, 40, -17), (70, 64, 64, 0), (150, 128, 3, 9)], 2, 256, 128, 32, 64, "nhd", "nhd"),
    ([(1, 128, 200, 127)], 2, 64, 64, 64, 128, "hnd", "hnd"),
    ([(9, 16, 50, -100000)], 5, 128, 0, 128, 16, "nhd", "hnd"),
    # more units than a launch's arguments hold
    ([(7, 0, 1500, 21), (2100, 1504, 501, -9)], 1, 64, 64, 16, 16, "hnd", "nhd"),
]


@pytest.mark.parametrize("spans,heads,d,rotary,sbs,dbs,lay_s,lay_d", SHIFTS)
def test_shift_equals_the_plain_one(gpu, spans, heads, d, rotary, sbs, dbs, lay_s, lay_d):
    rng = np.random.default_rng(len(spans) * 100 + d + dbs)
    layers = 2
    sn = max(a + n for a, _, n, _ in spans)
    dn = max(b + n for _, b, n, _ in spans)
    sb, db = -(-sn // sbs) + 1, -(-dn // dbs) + 2
    src = [Cache(gpu, rng, sb, heads, d, sbs, lay_s) for _ in range(layers)]
    dst = [Cache(gpu, rng, db, heads, d, dbs, lay_d, split=True) for _ in range(layers)]
    st = rng.permutation(sb).astype(np.int32)
    dt = rng.permutation(db).astype(np.int32)
    inv = inv_freq_for(d, 1e6, rotary / d) if rotary else None
    # the source table begins one entry in, the destination's two
    rows = [(a, b, 1, 2, n, delta, 0, 0) for a, b, n, delta in spans]
    flags = i32([0], gpu)
    runner = ScaledShifts([c.dev for c in src], [c.dev for c in dst], inv)
    runner.run(rows, np.concatenate(([99], st)), np.concatenate(([7, 8], dt)), error_flags=flags)
    assert flags.item() == 0
    for a, b in zip(src, dst):
        plain.shift(a.codes, a.scales, b.codes, b.scales, rows, np.concatenate(([99], st)),
                    np.concatenate(([7, 8], dt)), sbs, dbs,
                    inv.numpy() if rotary else np.zeros(0, np.float32))
        a.check()
        b.check()


def test_shift_of_anything_and_of_bad_ids(gpu):
    """NaN codes and scales out of their range in the source; ids out of range on both sides."""
    rng = np.random.default_rng(17)
    src = Cache(gpu, rng, 8, 2, 128, 16, fill="anything")
    dst = Cache(gpu, rng, 8, 2, 128, 16)
    inv = inv_freq_for(128, 1e6)
    st, dt = rng.permutation(8).astype(np.int32), rng.permutation(8).astype(np.int32)
    rows = [(3, 16, 0, 0, 50, 13, 0, 0)]
    runner = ScaledShifts([src.dev], [dst.dev], inv)
    flags = i32([0], gpu)
    runner.run(rows, st, dt, error_flags=flags)
    assert flags.item() == 0
    plain.shift(src.codes, src.scales, dst.codes, dst.scales, rows, st, dt, 16, 16, inv.numpy())
    dst.check()
    bad = dt.copy()
    bad[2] = 8
    runner.run(rows, st, bad, error_flags=flags)  # the block is not written
    assert flags.item() == _lib.MKV_FLAG_DST_RANGE
    dst.check()
    flags.zero_()
    runner.run(rows, st[:3], dt, error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SRC_RANGE


# ------------------------------------------------------------------- as they are used


def test_a_session_through_all_four(gpu):
    """Prompts stored, decoded token by token, one's history moved by an edit and decoded on:
    each step's attention against the plain softmax over what the cache should hold."""
    rng = np.random.default_rng(77)
    heads, group, d, bs, blocks = 2, 2, 64, 16, 40
    cache = Cache(gpu, rng, blocks, heads, d, bs)
    inv = inv_freq_for(d, 1e4)
    free = torch.from_numpy(rng.permutation(blocks).astype(np.int32)).to(gpu)
    tables = torch.full((3, 9), -1, dtype=torch.int32, device=gpu)
    held, at = i32([0, 0, 0], gpu), i32([0], gpu)

    def step(new):
        nonlocal held, at
        total = sum(new)
        s = step_slots(held, i32(new, gpu), tables, free, at, bs, total)
        k, v = (torch.from_numpy(loud(rng, (total, heads, d), 2)).to(gpu, torch.bfloat16)
                for _ in range(2))
        q = torch.randn(total, heads * group, d, device=gpu, dtype=torch.bfloat16)
        store_scaled(cache.dev, k, v, tables, s.starts, s.lens)
        out = attend_scaled(cache.dev, q, tables, s.starts, s.lens, max_new=max(new))
        held, at = s.lens, s.free_at
        host, starts, lens = tables.cpu().numpy(), s.starts.tolist(), s.lens.tolist()
        plain.store(cache.codes, cache.scales, k.double().cpu().numpy(), v.double().cpu().numpy(),
                    host, starts, lens, bs)
        cache.check()
        qh = q.double().cpu().numpy()
        want = plain.attend(cache.codes, cache.scales, qh, host, starts, lens, bs, d ** -0.5)
        tol = bound_of(cache, qh, host, starts, lens, bs, d ** -0.5, want, torch.bfloat16)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()

    step([37, 20, 1])
    for _ in range(3):
        step([1, 1, 1])
    step([5, 0, 30])
    # request 0's positions 9 to 40 become request 1's positions 32 on: its 23 tokens end in a
    # block of their own, and 9 blank ones would be recomputed
    host = tables.cpu().numpy()
    fresh = free[int(at):int(at) + 2].cpu().numpy()
    at = at + 2
    tables[1, 2:4] = torch.from_numpy(fresh).to(gpu)
    row = [(9, 0, 0, 0, 31, 23, 0, 0)]
    ScaledShifts([cache.dev], [cache.dev], inv).run(row, host[0], fresh)
    plain.shift(cache.codes, cache.scales, cache.codes, cache.scales, row, host[0], fresh, bs, bs,
                inv.numpy())
    cache.check()
    held[1] = 63
    step([1, 2, 0])
    step([1, 1, 1])


def test_a_captured_step_replays_with_other_lengths(gpu):
    """slots, store and attention in one graph, replayed while the lengths on the GPU change;
    eager work and a second graph's replays between."""
    rng = np.random.default_rng(41)
    heads, group, d, bs, blocks, n = 2, 4, 128, 16, 64, 3
    caches = [Cache(gpu, rng, blocks, heads, d, bs) for _ in range(2)]
    free = torch.from_numpy(rng.permutation(blocks).astype(np.int32)).to(gpu)
    start = [30, 5, 300]
    need = [-(-x // bs) for x in start]
    tables = torch.zeros((n, 24), dtype=torch.int32, device=gpu)
    order = free.tolist()
    for r in range(n):
        tables[r, :need[r]] = i32(order[sum(need[:r]):sum(need[:r + 1])], gpu)
    states = []
    for c in caches:
        states.append(dict(cache=c.dev, tables=tables.clone(), held=i32(start, gpu),
                           new=i32([1, 1, 1], gpu), at=i32([sum(need)], gpu),
                           k=torch.zeros(n, heads, d, device=gpu, dtype=torch.bfloat16),
                           v=torch.zeros(n, heads, d, device=gpu, dtype=torch.bfloat16),
                           q=torch.zeros(n, heads * group, d, device=gpu, dtype=torch.bfloat16)))

    def step(s):
        p = step_slots(s["held"], s["new"], s["tables"], free, s["at"], bs, n)
        store_scaled(s["cache"], s["k"], s["v"], s["tables"], p.starts, p.lens)
        o = attend_scaled(s["cache"], s["q"], s["tables"], p.starts, p.lens, max_new=1)
        s["held"].copy_(p.lens)
        s["at"].copy_(p.free_at)
        return o

    captured, eager = states
    keep = {k: t.clone() for k, t in captured.items() if isinstance(t, torch.Tensor)}
    kv0, sc0 = captured["cache"].kv.clone(), captured["cache"].scales.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(captured)
    side.synchronize()
    for k, t in keep.items():
        captured[k].copy_(t)
    captured["cache"].kv.view(torch.uint8).copy_(kv0.view(torch.uint8))
    captured["cache"].scales.view(torch.uint8).copy_(sc0.view(torch.uint8))
    eager["cache"].kv.view(torch.uint8).copy_(kv0.view(torch.uint8))
    eager["cache"].scales.view(torch.uint8).copy_(sc0.view(torch.uint8))
    with torch.cuda.graph(graph):
        result = step(captured)
    for i in range(20):
        for name in ("k", "v", "q"):
            x = torch.randn_like(captured[name])
            captured[name].copy_(x)
            eager[name].copy_(x)
        if i == 7:  # one request pauses, its row belongs to the next
            captured["new"].copy_(i32([1, 0, 1], gpu))
            eager["new"].copy_(i32([1, 0, 1], gpu))
        if i == 9:
            captured["new"].fill_(1)
            eager["new"].fill_(1)
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        rows = int(eager["new"].sum())
        assert torch.equal(result[:rows], want[:rows])
        assert captured["held"].tolist() == eager["held"].tolist()
    assert torch.equal(captured["cache"].kv.view(torch.uint8), eager["cache"].kv.view(torch.uint8))


def test_a_captured_shift_keeps_its_spans(gpu):
    rng = np.random.default_rng(51)
    src, dst = Cache(gpu, rng, 6, 2, 64, 16), Cache(gpu, rng, 6, 2, 64, 16)
    inv = inv_freq_for(64, 1e4)
    runner = ScaledShifts([src.dev], [dst.dev], inv)
    table = np.arange(6, dtype=np.int32)
    rows = [(4, 16, 0, 0, 40, 12, 0, 0)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        runner.run(rows, table, table)
    plain.shift(src.codes, src.scales, dst.codes, dst.scales, rows, table, table, 16, 16, inv.numpy())
    for _ in range(3):
        runner.run([(0, 0, 0, 0, 16, 0, 0, 0)], table, table)  # eager work between
        dst.planes[0].view(torch.uint8)[2].zero_()  # a block that the graph writes whole
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
    plain.shift(src.codes, src.scales, dst.codes, dst.scales, [(0, 0, 0, 0, 16, 0, 0, 0)], table,
                table, 16, 16, inv.numpy())
    dst.check()


@pytest.mark.parametrize("spans", [1, 60])  # one launch's arguments, and more
def test_a_captured_shift_next_to_eager_ones(gpu, spans):
    rng = np.random.default_rng(52)
    src, dst = Cache(gpu, rng, 61, 2, 64, 16), Cache(gpu, rng, 130, 2, 64, 16)
    inv = inv_freq_for(64, 1e4)
    runner = ScaledShifts([src.dev], [dst.dev], inv)
    table = np.arange(130, dtype=np.int32)
    rows = [(3 + i, 32 * i, 0, 0, 17, i - 7, 0, 0) for i in range(spans)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        runner.run(rows, table, table)
    for i in range(4):
        other = [(5 * i + j, 32 * j, 0, 0, 32, i + j, 0, 0) for j in range(spans)]
        runner.run(other, table, table)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for r in (other, rows):
            plain.shift(src.codes, src.scales, dst.codes, dst.scales, r, table, table, 16, 16,
                        inv.numpy())
        dst.check()


def test_on_another_stream(gpu):
    """Each operator on a side stream, with the default stream busy."""
    rng = np.random.default_rng(61)
    new, held = [20, 1], [0, 50]
    tables, blocks = requests_of(new, held, 16, rng, gap=0)
    src, dst = (Cache(gpu, rng, blocks, 2, 128, 16) for _ in range(2))
    runner = ScaledShifts([src.dev], [dst.dev], inv_freq_for(128, 1e6))
    k, v = (torch.from_numpy(loud(rng, (21, 2, 128))).to(gpu, torch.bfloat16) for _ in range(2))
    q = torch.randn(21, 4, 128, device=gpu, dtype=torch.bfloat16)
    args = i32(tables, gpu), i32([0, 20, 21], gpu), i32([20, 51], gpu)
    perm = np.arange(blocks, dtype=np.int32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        store_scaled(src.dev, k, v, *args)
        runner.run([(0, 0, 0, 0, 16 * blocks, 5, 0, 0)], perm, perm)
        out = attend_scaled(dst.dev, q, *args)
    side.synchronize()
    plain.store(src.codes, src.scales, k.double().cpu().numpy(), v.double().cpu().numpy(), tables,
                [0, 20, 21], [20, 51], 16)
    src.check()
    plain.shift(src.codes, src.scales, dst.codes, dst.scales,
                [(0, 0, 0, 0, 16 * blocks, 5, 0, 0)], perm, perm, 16, 16,
                inv_freq_for(128, 1e6).numpy())
    dst.check()
    assert torch.equal(out, attend_scaled(dst.dev, q, *args))


def test_offsets_past_32_bits(gpu):
    """A cache of over 4 GiB: its last blocks are stored, read and moved like its first."""
    heads, d, bs = 8, 256, 128
    blocks = 4 * 2**30 // (heads * bs * 2 * d) + 40
    kv = torch.zeros((blocks, heads, bs, 2 * d), dtype=torch.uint8, device=gpu)
    scales = torch.full((blocks, heads, 2), 127, dtype=torch.uint8, device=gpu)
    big = ScaledCache(kv.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), "hnd", bs)
    small_kv, small_scales = torch.zeros_like(kv[:3]), torch.full_like(scales[:3], 127)
    small = ScaledCache(small_kv.view(torch.float8_e4m3fn),
                        small_scales.view(torch.float8_e8m0fnu), "hnd", bs)
    k, v = (torch.randn(200, heads, d, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn(200, heads, d, device=gpu, dtype=torch.bfloat16)
    last = [blocks - 1, blocks - 3]
    rest = i32([0, 200], gpu), i32([200], gpu)
    store_scaled(big, k, v, i32([last], gpu), *rest)
    store_scaled(small, k, v, i32([[0, 2]], gpu), *rest)
    assert torch.equal(kv[last], small_kv[[0, 2]]) and torch.equal(scales[last], small_scales[[0, 2]])
    assert torch.equal(attend_scaled(big, q, i32([last], gpu), *rest),
                       attend_scaled(small, q, i32([[0, 2]], gpu), *rest))
    inv = inv_freq_for(d, 1e6)
    row = [(5, 0, 0, 0, 128, 40, 0, 0)]
    ScaledShifts([big], [big], inv).run(row, last, [blocks - 5])
    ScaledShifts([small], [small], inv).run(row, [0, 2], [1])
    assert torch.equal(kv[blocks - 5], small_kv[1]) and int(kv[1:blocks - 6].any()) == 0


# ---------------------------------------------------------------------------- refusals


def test_python_refusals(gpu):
    rng = np.random.default_rng(1)
    cache = Cache(gpu, rng, 4, 2, 64, 16)
    kv, scales = cache.planes[0], cache.dev_scales
    for bad, error in [
        (lambda: ScaledCache(kv, scales, "flat"), ValueError),
        (lambda: ScaledCache(kv.view(torch.uint8), scales, "hnd"), TypeError),
        (lambda: ScaledCache(kv, scales, "nhd"), ValueError),
        (lambda: ScaledCache(kv, scales, "hnd", 32), ValueError),
        (lambda: ScaledCache(kv, scales.view(torch.uint8), "hnd"), ValueError),
        (lambda: ScaledCache(kv, scales[:3], "hnd"), ValueError),
        (lambda: ScaledCache(kv[..., :96], scales, "hnd"), ValueError),
        (lambda: ScaledCache(kv, scales, "hnd", 16, kv[:2]), ValueError),
        (lambda: ScaledCache(kv[:1].expand(4, -1, -1, -1), scales, "hnd"), ValueError),
        (lambda: ScaledCache(kv[0], scales, "hnd"), ValueError),
    ]:
        with pytest.raises(error):
            bad()
    tables, starts, lens = i32([[0, 1]], gpu), i32([0, 3], gpu), i32([3], gpu)
    q = torch.zeros(3, 4, 64, device=gpu, dtype=torch.bfloat16)
    k = torch.zeros(3, 2, 64, device=gpu, dtype=torch.bfloat16)
    for args, kw, error in [
        ((q.float(), tables, starts, lens), {}, TypeError),
        ((q[:, :3], tables, starts, lens), {}, ValueError),
        ((q.cpu(), tables, starts, lens), {}, ValueError),
        ((q.transpose(1, 2).contiguous().transpose(1, 2), tables, starts, lens), {}, ValueError),
        ((q.clone().requires_grad_(), tables, starts, lens), {}, RuntimeError),
        ((q, tables.long(), starts, lens), {}, ValueError),
        ((q, tables, starts[:1], lens), {}, ValueError),
        ((q, tables, starts, lens.long()), {}, ValueError),
        ((q, tables, starts, lens.cpu()), {}, ValueError),
        ((q, tables, starts, lens), dict(out=q), ValueError),
        ((q, tables, starts, lens), dict(out=q.float()), ValueError),
        ((q, tables, starts, lens), dict(softmax_scale=-1.0), _lib.KVShiftError),
        ((q, tables, starts, lens), dict(error_flags=lens.long()), ValueError),
    ]:
        with pytest.raises(error):
            attend_scaled(cache.dev, *args, **kw)
    for args, error in [
        ((k, k[:2], tables, starts, lens), ValueError),
        ((k.double(), k.double(), tables, starts, lens), TypeError),
        ((k, k.float(), tables, starts, lens), TypeError),
        ((k[:, :1], k[:, :1], tables, starts, lens), ValueError),
        ((k.cpu(), k, tables, starts, lens), ValueError),
        ((k, k, tables[0], starts, lens), ValueError),
    ]:
        with pytest.raises(error):
            store_scaled(cache.dev, *args)
    one = i32([1], gpu)
    for args in [(lens, lens, tables, one, one, 0, 4), (lens, lens, tables, one, one, 16, -1),
                 (starts, lens, tables, one, one, 16, 4), (lens, lens.long(), tables, one, one, 16, 4),
                 (lens, lens, tables, one[None], one, 16, 4), (lens, lens, tables, one, starts, 16, 4)]:
        with pytest.raises(ValueError):
            step_slots(*args)
    other = Cache(gpu, rng, 4, 1, 64, 16).dev
    with pytest.raises(ValueError):
        ScaledShifts([cache.dev], [other], None)
    with pytest.raises(ValueError):
        ScaledShifts([cache.dev], [cache.dev], torch.ones(8))
    with pytest.raises(ValueError):
        ScaledShifts([], [], None)
    runner = ScaledShifts([cache.dev], [cache.dev], None)
    for rows, tab in [([(0, 8, 0, 0, 16, 0, 0, 0)], [0, 1]), ([(0, 0, 0, 0, -1, 0, 0, 0)], [0]),
                      ([(-1, 0, 0, 0, 4, 0, 0, 0)], [0]), ([(0, 0, 0, 0, 4, 0, 0, 0)], [2**40]),
                      ([(0, 0, 0, 0, 4, 0, 0, 0)], tables[0])]:
        with pytest.raises(ValueError):
            runner.run(rows, tab, [2, 3])
    runner.run([], [0], [1])
    runner.run([(0, 0, 0, 0, 0, 5, 0, 0)], [0], [1])
    for tab, to in ([[0, 1], [2, 2]], [[0, 1], [3, 1]]):  # a block written twice, or read too
        with pytest.raises(_lib.KVShiftError):
            runner.run([(0, 0, 0, 0, 32, 0, 0, 0)], tab, to)
    flags = i32([0, 0, 0], gpu)  # a span far longer than its tables
    runner.run([(0, 0, 0, 0, 2**31 - 1, 0, 0, 0)], [0], [-1], error_flags=flags)
    assert flags.tolist() == [_lib.MKV_FLAG_DST_RANGE, 0, 0]
    cache.check()
    q = torch.zeros(3, 2, cache.dev.head_size, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(_lib.KVShiftError, match="overlap"):
        attend_scaled(cache.dev, q, tables, starts, lens, out=q[:1].clone().expand(3, -1, -1))
