"""Groups that do not fit, among few and many: the others share what they share."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import _lib
from tests.test_gpu_attend_shared import Batch, run
from tests.test_gpu_scaled import Cache

pytestmark = pytest.mark.gpu


def two_each(gpu, groups, seed):
    """Groups of two requests, a token each, over a block of their own."""
    rng = np.random.default_rng(seed)
    batch = Batch(rng, [(16, [(int(a), 1), (int(b), 1)]) for a, b in rng.integers(0, 40, (groups, 2))],
                  [(20, 1)], 16)
    cache = Cache(gpu, rng, batch.blocks, 1, 64, 16)
    q = torch.from_numpy(rng.standard_normal((2 * groups + 1, 2, 64))).to(gpu, torch.bfloat16)
    return batch, cache, q


# groups, the entry that does not fit, what stands there
BAD = [(3, 0, -1), (3, 2, -1), (3, 2, 9), (5, 3, -2**31), (64, 40, -7), (64, 63, 1000),
       (65, 64, -1), (65, 64, 2**31 - 1), (130, 64, -1), (130, 64, 4095), (130, 128, -1), (130, 128, 600),
       (130, 64, 20), (700, 64, -1), (700, 512, -1), (700, 512, 2000), (700, 640, 5), (700, 1, -1)]


@pytest.mark.parametrize("groups,entry,value", BAD)
def test_a_group_that_does_not_fit_leaves_the_others_theirs(gpu, groups, entry, value):
    batch, cache, q = two_each(gpu, groups, groups + entry)
    clean = run(gpu, batch, cache, q, max_new=1)
    # who shares nothing reads its own table from its first token on; the others' entries are not read
    lost = np.zeros(2 * groups + 1, bool)
    lost[2 * max(entry - 1, 0):2 * entry + 2] = True
    if 0 <= value < 2 * groups:  # back among requests in front: theirs until the next entry
        lost[value:2 * entry] = True
    batch.given[lost] = batch.tables[lost]
    batch.groups[entry] = value
    flags = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = run(gpu, batch, cache, q, torch.full_like(q, 7.0), flags, max_new=1)
    assert flags.item() == _lib.MKV_FLAG_SPAN
    keep = torch.from_numpy(~lost).to(gpu)
    assert torch.equal(got[keep], clean[keep])
    if not 0 <= value < 2 * groups:
        # one rounding of p (2^-8) and of the output (2^-8) on either side, as with few groups
        assert (got.float() - clean.float()).abs().max() <= 2.0 ** -6 * clean.float().abs().max()


@pytest.mark.parametrize("groups", [64, 65, 200, 1100])
def test_many_groups_are_found(gpu, groups):
    """Against the same requests in no group."""
    batch, cache, q = two_each(gpu, groups, groups)
    flags = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = run(gpu, batch, cache, q, flags=flags, max_new=1)
    batch.given, batch.groups, batch.shared = batch.tables, np.array([0]), []
    want = run(gpu, batch, cache, q, flags=flags, max_new=1)
    assert flags.item() == 0
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()


def test_starts_that_descend_leave_other_requests_right(gpu):
    """Request 0 ends before it begins, and leads the group by which 64 are found: the requests whose
    group is not found read their own tables.  (15 rows a token: the first group's tiles would begin
    behind those of tokens up to 93.)"""
    groups, begins = 100, 190
    batch, cache, _ = two_each(gpu, groups, 1)
    q = torch.from_numpy(np.random.default_rng(2).standard_normal((201, 15, 64))).to(gpu, torch.bfloat16)
    batch.given = batch.tables
    clean = run(gpu, batch, cache, q, max_new=1)
    batch.starts[0] = begins
    flags = torch.zeros(1, dtype=torch.int32, device=gpu)
    torch.cuda.empty_cache()  # a workspace is then cut out of what held these
    spoilt = torch.empty((64, 1 << 20), device=gpu).fill_(float("nan"))
    del spoilt
    got = run(gpu, batch, cache, q, torch.full_like(q, 7.0), flags, max_new=1)
    assert flags.item() == _lib.MKV_FLAG_SPAN
    # (rows of the first 64 requests may stay untouched: they too are found by request 0's start)
    # one rounding of p (2^-8) and of the output (2^-8) on either side, as with few groups
    off = (got[64:].float() - clean[64:].float()).abs().max().item()
    assert off == off and off <= 2.0 ** -6 * clean.float().abs().max().item()
