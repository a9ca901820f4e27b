"""What a block-scaled cache is made from: tensors that leave no row to write, or whose rows lie
in one another, are refused where the cache is made."""

from __future__ import annotations

import pytest
import torch

from marathon_amd import ScaledCache

pytestmark = pytest.mark.gpu


def fp8(shape, gpu):
    return torch.zeros(shape, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)


def scales_of(blocks, heads, gpu):
    return torch.full((blocks, heads, 2), 127, dtype=torch.uint8, device=gpu).view(
        torch.float8_e8m0fnu)


def test_a_cache_without_heads_is_refused(gpu):
    with pytest.raises(ValueError, match="heads"):
        ScaledCache(fp8((4, 0, 16, 128), gpu), scales_of(4, 0, gpu), "hnd")
    with pytest.raises(ValueError, match="heads"):
        ScaledCache(fp8((4, 16, 0, 64), gpu), scales_of(4, 0, gpu), "nhd",
                    v_cache=fp8((4, 16, 0, 64), gpu))
