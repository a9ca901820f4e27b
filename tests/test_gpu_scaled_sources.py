"""A block-scaled shift whose source blocks are missing: a destination block is written with all
of its rows or left as it was, its scale among it."""

from __future__ import annotations

import numpy as np
import pytest

from marathon_amd import ScaledShifts, _lib
from marathon_amd.shift_kernels import inv_freq_for
from tests import scaled_plain as plain
from tests.test_gpu_scaled import Cache, i32

pytestmark = pytest.mark.gpu


def shift_and_compare(gpu, rows, src_table, dst_table, sbs, dbs, layout, heads=2, d=64):
    """Runs ``rows`` over caches of values, and over the twins each destination block whose
    sources are all there; returns how many were left."""
    rng = np.random.default_rng(len(rows) * 10 + sbs + dbs)
    sb, db = 40, max(int(max(dst_table)) + 1, 8)
    src = Cache(gpu, rng, sb, heads, d, sbs, layout)
    dst = Cache(gpu, rng, db, heads, d, dbs, layout)
    inv = inv_freq_for(d, 1e4)
    flags = i32([0], gpu)
    ScaledShifts([src.dev], [dst.dev], inv).run(rows, src_table, dst_table, error_flags=flags)
    left = 0
    for sp, dp, si, di, n, delta, _, _ in rows:
        for at in range(0, n, dbs):
            m = min(dbs, n - at)
            index = si + np.arange((sp + at) // sbs, (sp + at + m - 1) // sbs + 1)
            if any(i >= len(src_table) or not 0 <= src_table[i] < sb for i in index):
                left += 1
                continue
            plain.shift(src.codes, src.scales, dst.codes, dst.scales,
                        [(sp + at, dp + at, si, di, m, delta, 0, 0)], src_table, dst_table, sbs, dbs,
                        inv.numpy())
    assert flags.item() == (_lib.MKV_FLAG_SRC_RANGE if left else 0)
    dst.check()
    src.check()
    return left


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("sbs,dbs", [(16, 16), (16, 64), (32, 128), (64, 16), (128, 128)])
@pytest.mark.parametrize("bad", [-1, 40, 2**31 - 1])
def test_a_block_without_a_source_is_left(gpu, bad, sbs, dbs, layout):
    """Sources missing at the front, in the middle and behind the table's end: units that lack
    all of their rows, and units that lack some."""
    n = 6 * max(sbs, dbs) + 5
    need = (n + 3) // sbs + 1
    table = (np.arange(need) * 3 % 40).astype(np.int32)
    table[[0, need // 2]] = bad
    dst = np.arange(8, dtype=np.int32)[::-1].copy()
    dst = np.concatenate((dst, np.arange(8, 8 + n // dbs, dtype=np.int32)))
    left = shift_and_compare(gpu, [(3, 0, 0, 0, n, 17, 0, 0)], table[:need - 1], dst, sbs, dbs, layout)
    assert left >= 2


def test_a_span_with_one_source_writes_that_block_alone(gpu):
    left = shift_and_compare(gpu, [(0, 0, 0, 0, 40, 9, 0, 0), (0, 64, 1, 0, 16, 0, 0, 0)],
                             np.array([-1, 3, -7, -1], np.int32), np.arange(8, dtype=np.int32), 16,
                             16, "hnd")
    assert left == 2  # the first span's first and third block


def test_a_span_without_any_source_changes_nothing(gpu):
    left = shift_and_compare(gpu, [(5, 0, 0, 0, 40, 9, 0, 0)], np.full(4, -1, np.int32),
                             np.arange(8, dtype=np.int32), 16, 16, "nhd")
    assert left == 3


def test_blocks_without_a_source_among_many_units(gpu):
    """More units than a launch's arguments hold: they come from device memory."""
    rows = [(1 + 16 * i, 32 * i, 0, 0, 31, i - 40, 0, 0) for i in range(90)]
    table = (np.arange(100) * 7 % 40).astype(np.int32)
    table[11::9] = -1
    left = shift_and_compare(gpu, rows, table, np.arange(180, dtype=np.int32), 16, 16, "nhd")
    assert left > 20
