"""The block-scaled store at each number of tokens that its workgroups look through."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import store_scaled
from tests import scaled_plain as plain
from tests.test_gpu_scaled import DTYPES, Cache, i32, loud, requests_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,held,heads,d,bs,layout,dtype", [
    ([1] * 900, [3] * 900, 2, 64, 16, "hnd", "bf16"),       # 1
    ([1] * 1100, [15] * 1100, 8, 64, 16, "nhd", "bf16"),    # 4: many requests
    ([701], [5], 8, 64, 16, "hnd", "fp16"),                 # 4: one
    ([1103], [9], 8, 64, 16, "nhd", "bf16"),                # 8
    ([3001, 200], [0, 77], 8, 64, 16, "hnd", "bf16"),       # 16
    ([6199, 1], [3, 16], 8, 64, 16, "nhd", "bf16"),         # a block
    ([40] * 180, [7] * 180, 8, 64, 16, "hnd", "bf16"),      # a block: many requests
    ([3100, 33], [17, 31], 8, 64, 32, "hnd", "fp32"),       # 32
    ([701, 30], [65, 0], 8, 64, 64, "nhd", "bf16"),         # 16 of a block of 64
    ([3001, 90, 3], [63, 64, 1], 8, 64, 64, "hnd", "bf16"),
    ([3001, 130, 5], [127, 0, 130], 8, 64, 128, "nhd", "fp16"),
    ([25001], [100], 1, 64, 128, "hnd", "bf16"),
])
def test_store_at_every_size(gpu, new, held, heads, d, bs, layout, dtype):
    rng = np.random.default_rng(sum(new) + bs)
    tables, blocks = requests_of(new, held, bs, rng)
    cache = Cache(gpu, rng, blocks, heads, d, bs, layout, fill="anything")
    cache.scales[...] = rng.integers(110, 135, cache.scales.shape)
    cache.dev_scales.view(torch.uint8).copy_(torch.from_numpy(cache.scales).to(gpu))
    starts = np.cumsum([0] + new)
    lens = [h + n for h, n in zip(held, new)]
    k, v = (torch.from_numpy(loud(rng, (int(starts[-1]) + 5, heads, d))).to(gpu, DTYPES[dtype])
            for _ in range(2))
    flags = i32([0], gpu)
    store_scaled(cache.dev, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu),
                 error_flags=flags)
    plain.store(cache.codes, cache.scales, k.double().cpu().numpy(), v.double().cpu().numpy(),
                tables, starts.tolist(), lens, bs)
    assert flags.item() == 0
    cache.check()
