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


def test_rows_that_lie_in_one_another_are_refused(gpu):
    flat = fp8((1 << 16,), gpu)
    scales = scales_of(4, 2, gpu)
    for strides in [(2048, 2048, 128, 1),     # both heads of a block one
                    (4096, 1024, 128, 1),     # a head's tokens reach into the next
                    (4096, 2048, 64, 1),      # a token's V is the next one's K
                    (2048, 2048 * 3, 128, 1), # heads between blocks: block 3 of head 0 is 0 of 1
                    (64, 2048, 128, 1)]:
        with pytest.raises(ValueError, match="overlap"):
            ScaledCache(flat.as_strided((4, 2, 16, 128), strides), scales, "hnd")
    with pytest.raises(ValueError, match="overlap"):
        ScaledCache(fp8((4, 1, 1, 128), gpu).expand(4, 16, 2, 128), scales, "nhd")
    kv = fp8((4, 2, 16, 64), gpu)
    wide = fp8((5, 2, 16, 64), gpu)
    for k, v in [(kv, kv), (wide[:4], wide[1:])]:
        with pytest.raises(ValueError, match="share"):
            ScaledCache(k, scales, "hnd", v_cache=v)


def test_interleaved_caches_are_taken(gpu):
    """K and V in one allocation, a block's layers side by side, heads in front of blocks."""
    scales = scales_of(4, 2, gpu)
    both = fp8((4, 2, 16, 2, 64), gpu)
    ScaledCache(both[:, :, :, 0], scales, "hnd", v_cache=both[:, :, :, 1])
    ScaledCache(both[..., 0, :], scales, "hnd", v_cache=both[..., 1, :])
    planes = fp8((2, 4, 16, 2, 64), gpu)
    ScaledCache(planes[0], scales, "nhd", v_cache=planes[1])
    layers = fp8((4, 3, 2, 16, 128), gpu)
    for i in range(3):
        ScaledCache(layers[:, i], scales, "hnd")
    ScaledCache(fp8((2, 4, 16, 128), gpu).transpose(0, 1), scales, "hnd")
    ScaledCache(fp8((4, 2, 16, 160), gpu)[..., 16:144], scales, "hnd")
    ScaledCache(fp8((0, 2, 16, 128), gpu), scales_of(0, 2, gpu), "hnd")
    ScaledCache(fp8((1, 1, 16, 128), gpu), scales_of(1, 1, gpu), "hnd")
