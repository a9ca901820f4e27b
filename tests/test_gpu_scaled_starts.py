"""Requests whose starts leave the token arrays, or descend: skipped by the block-scaled store
and attention, and flagged, wherever they stand."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import _lib, attend_scaled, store_scaled
from tests import scaled_plain as plain
from tests.test_gpu_scaled import Cache, i32, loud

pytestmark = pytest.mark.gpu

T = 40  # rows of the token arrays
CASES = {  # starts; requests that are whole
    "behind": ([0, 40, 45], [0]),
    "all behind": ([41, 50, 90], []),
    "straddles": ([0, 8, 44], [0]),
    "negative": ([-3, 5, 40], [1]),
    "all negative": ([-30, -20, -10], []),
    "long": ([2, 30, 2**31 - 1], [0]),
    "far": ([-2**31, 3, 2**31 - 1], []),
}
GOOD = {"padded": [0, 8, 8, 8], "empty": [0, 0, 0], "full": [0, 20, 40], "late": [30, 40, 40]}


def tables_of(rng, starts, bs, lens):
    width = max(1, -(-max(max(lens), 1) // bs))
    n = len(starts) - 1
    return rng.permutation(n * width).reshape(n, width).astype(np.int32)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("bs,heads", [(16, 3), (64, 1)])
def test_store_flags_requests_that_leave_the_rows(gpu, case, bs, heads):
    starts, whole = CASES[case]
    rng = np.random.default_rng(len(case))
    lens = [60] * (len(starts) - 1)
    tables = tables_of(rng, starts, bs, lens)
    cache = Cache(gpu, rng, tables.size, heads, 64, bs)
    k, v = (torch.from_numpy(loud(rng, (T, heads, 64))).to(gpu, torch.bfloat16) for _ in range(2))
    flags = i32([0], gpu)
    store_scaled(cache.dev, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu),
                 error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SPAN
    for r in whole:
        s0, s1 = starts[r], starts[r + 1]
        plain.store(cache.codes, cache.scales, *(x[s0:s1].double().cpu().numpy() for x in (k, v)),
                    tables[r:r + 1], [0, s1 - s0], lens[r:r + 1], bs)
    cache.check()


@pytest.mark.parametrize("case", GOOD)
def test_store_flags_no_other(gpu, case):
    starts = GOOD[case]
    rng = np.random.default_rng(3)
    lens = [b - a + 5 for a, b in zip(starts, starts[1:])]
    tables = tables_of(rng, starts, 16, lens)
    cache = Cache(gpu, rng, tables.size, 2, 64, 16)
    k, v = (torch.from_numpy(loud(rng, (T, 2, 64))).to(gpu, torch.bfloat16) for _ in range(2))
    flags = i32([0], gpu)
    store_scaled(cache.dev, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu),
                 error_flags=flags)
    plain.store(cache.codes, cache.scales, *(x.double().cpu().numpy() for x in (k, v)), tables,
                starts, lens, 16)
    assert flags.item() == 0
    cache.check()


# query heads a KV head, hint: 16 and 32 rows a tile, 128, and the two launches of a chunk
# beside decoding requests
SHAPES = [(1, 1), (8, 4), (4, None), (64, None)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("group,most", SHAPES)
def test_attend_flags_requests_that_leave_the_rows(gpu, case, group, most):
    starts, whole = CASES[case]
    rng = np.random.default_rng(7)
    lens = [60] * (len(starts) - 1)
    tables = tables_of(rng, starts, 16, lens)
    cache = Cache(gpu, rng, tables.size, 2, 64, 16)
    q = torch.randn(T, 2 * group, 64, device=gpu, dtype=torch.bfloat16)
    out, flags = torch.full_like(q, 5.0), i32([0], gpu)
    attend_scaled(cache.dev, q, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), out=out,
                  max_new=most, error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SPAN
    seen = torch.zeros(T, dtype=torch.bool, device=gpu)
    for r in whole:
        s0, s1 = starts[r], starts[r + 1]
        seen[s0:s1] = True
        alone = attend_scaled(cache.dev, q[s0:s1], i32(tables[r:r + 1], gpu), i32([0, s1 - s0], gpu),
                              i32(lens[r:r + 1], gpu))
        # The same rows under another launch shape.  Each is off by half a step of the output
        # (2^-8) and twice p's rounding (2 * 2^-9) of V's largest: 2^-7, and both 2^-6.
        size = cache_size(cache, tables[r], lens[r])
        assert (out[s0:s1].double() - alone.double()).abs().max() <= 2 ** -6 * size
    assert (out[~seen] == 5.0).all()


def cache_size(cache, table, n):
    return float(np.abs(plain.rows(cache.codes, cache.scales, table, n, cache.bs)[:, :, 1]).max())


@pytest.mark.parametrize("case", GOOD)
@pytest.mark.parametrize("group,most", SHAPES)
def test_attend_flags_no_other(gpu, case, group, most):
    starts = GOOD[case]
    rng = np.random.default_rng(3)
    lens = [b - a + 5 for a, b in zip(starts, starts[1:])]
    tables = tables_of(rng, starts, 16, lens)
    cache = Cache(gpu, rng, tables.size, 2, 64, 16)
    q = torch.randn(T, 2 * group, 64, device=gpu, dtype=torch.bfloat16)
    out, flags = torch.full_like(q, 5.0), i32([0], gpu)
    attend_scaled(cache.dev, q, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), out=out,
                  max_new=most, error_flags=flags)
    assert flags.item() == 0
    assert (out[:starts[0]] == 5.0).all() and (out[starts[-1]:] == 5.0).all()


@pytest.mark.parametrize("starts", [[0, 30, 10, 40], [40, 20, 0], [5, 4, 40, 40]])
def test_starts_that_descend_are_flagged(gpu, starts):
    """Their rows stay or go to a neighbour; the flag says so either way."""
    rng = np.random.default_rng(1)
    lens = [60] * (len(starts) - 1)
    tables = tables_of(rng, starts, 16, lens)
    cache = Cache(gpu, rng, tables.size, 1, 64, 16)
    x = torch.randn(T, 1, 64, device=gpu, dtype=torch.bfloat16)
    args = i32(tables, gpu), i32(starts, gpu), i32(lens, gpu)
    for most in (1, None):
        flags = i32([0], gpu)
        attend_scaled(cache.dev, x, *args, max_new=most, error_flags=flags)
        assert flags.item() == _lib.MKV_FLAG_SPAN
    flags = i32([0], gpu)
    store_scaled(cache.dev, x, x, *args, error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SPAN


def test_a_request_of_no_new_tokens_holds_anything(gpu):
    """Rows of a batch that no request has taken: empty, their length whatever it was."""
    rng = np.random.default_rng(2)
    cache = Cache(gpu, rng, 4, 1, 64, 16)
    x = torch.from_numpy(loud(rng, (T, 1, 64))).to(gpu, torch.bfloat16)
    tables = np.array([[0, 1], [2, 3], [-1, -1]], np.int32)
    args = i32(tables, gpu), i32([0, 20, 20, 20], gpu), i32([20, -1, -2**31], gpu)
    flags = i32([0], gpu)
    store_scaled(cache.dev, x, x, *args, error_flags=flags)
    attend_scaled(cache.dev, x, *args, error_flags=flags)
    assert flags.item() == 0
    x = x.double().cpu().numpy()
    plain.store(cache.codes, cache.scales, x, x, tables[:1], [0, 20], [20], 16)
    cache.check()
