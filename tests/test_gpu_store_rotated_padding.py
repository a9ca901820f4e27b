"""Rows of no request: a step's arrays may end before them, or begin behind them."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from marathon_amd import _lib, store_rotated
from marathon_amd.shift_kernels import current_stream, dtype_code
from tests.test_gpu_norm_rotate import DTYPES, freq
from tests.test_gpu_scaled import Cache, i32

pytestmark = pytest.mark.gpu

APART = 1 << 29  # bytes between tokens: rows of nobody would lie in no allocation


def head_rows(d, x, out, steps, out_steps, heads):
    d.x, d.out, d.heads = x, out, heads
    d.token_stride, d.head_stride = steps
    d.out_token_stride, d.out_head_stride = out_steps


@pytest.mark.parametrize("tokens,first,count", [(300, 150, 3), (300, 0, 2), (300, 298, 2), (9, 4, 1), (2000, 777, 3)])
@pytest.mark.parametrize("heads,d,bs,dtype", [(1, 64, 16, "bf16"), (1, 64, 64, "fp16"), (3, 128, 16, "bf16"),
                                              (40, 128, 16, "bf16"), (2, 256, 32, "fp32")])
def test_rows_of_nobody_are_not_read(gpu, tokens, first, count, heads, d, bs, dtype):
    """Only the request's rows lie in memory, the others' addresses in none."""
    rng = np.random.default_rng(tokens + heads)
    element = DTYPES[dtype].itemsize
    step = APART // element
    room = torch.zeros((count - 1) * step + (heads + 2) * d, dtype=DTYPES[dtype], device=gpu)
    both = room.as_strided((count, heads + 2, d), (step, d, 1))
    both.copy_(torch.from_numpy(rng.standard_normal(both.shape)))
    starts, lens, inv = i32([first, first + count], gpu), i32([count + 5], gpu), freq(d).to(gpu)
    table = i32([[2, 0, 1]], gpu)
    caches = [Cache(gpu, np.random.default_rng(1), 3, 1, d, bs) for _ in range(2)]

    # the same step with rows everywhere
    dense = torch.full((tokens, heads + 2, d), float("nan"), dtype=DTYPES[dtype], device=gpu)
    dense[first:first + count] = both
    want = torch.full((tokens, heads, d), 77.0, dtype=DTYPES[dtype], device=gpu)
    store_rotated(caches[0].dev, *dense.split((heads, 1, 1), 1), table, starts, lens, inv, out_q=want)

    got = torch.full_like(want, 77.0)
    at = room.data_ptr() - first * APART
    desc = _lib.StoreRotatedDesc()
    desc.cache = caches[1].dev.desc
    head_rows(desc.q, at, got.data_ptr(), (step, d), (heads * d, d), heads)
    desc.turn.inv_freq, desc.turn.rotary, desc.turn.norm, desc.turn.eps = inv.data_ptr(), d, 1, 1e-6
    desc.k, desc.v = at + heads * d * element, at + (heads + 1) * d * element
    desc.k_token_stride = desc.v_token_stride = step
    desc.block_tables, desc.table_stride, desc.table_width = table.data_ptr(), 3, 3
    desc.starts, desc.lens, desc.requests = starts.data_ptr(), lens.data_ptr(), 1
    desc.tokens, desc.dtype = tokens, dtype_code(DTYPES[dtype])
    print(f"rows {first} to {first + count} of {tokens}, {heads} heads of {d}", flush=True)
    _lib.check(_lib.lib().mkv_store_rotated(ctypes.byref(desc), current_stream(gpu)))
    assert torch.equal(got, want)
    for a, b in zip(*([*c.planes, c.dev_scales] for c in caches)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
