"""Caches that share memory, in a shift and in an attention call: told apart where they merely
interleave, taken where the call's own rows do not meet, and refused where they do."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import ScaledCache, ScaledShifts, _lib, attend_scaled
from marathon_amd.shift_kernels import inv_freq_for
from tests import scaled_plain as plain
from tests.test_gpu_scaled import Cache, i32

pytestmark = pytest.mark.gpu

INV = inv_freq_for(64, 1e4)


def caches(gpu, n, blocks=8, **kw):
    rng = np.random.default_rng(n)
    return [Cache(gpu, rng, blocks, 2, 64, 16, **kw) for _ in range(n)]


def span(n, delta=5):
    return [(3, 0, 0, 0, n, delta, 0, 0)]


def moved(src, dst, rows, st, dt):
    """The host's twins after the shift of each (src, dst) pair."""
    plain.shift(src.codes, src.scales, dst.codes, dst.scales, rows, st, dt, 16, 16, INV.numpy())


def refuses(runner, st, dt, n=40):
    with pytest.raises(_lib.KVShiftError, match="source and a destination|and, .* a source"):
        runner.run(span(n), st, dt)


def test_one_cache_on_both_sides_of_a_later_layer(gpu):
    a, b, c = caches(gpu, 3)
    runner = ScaledShifts([a.dev, c.dev], [b.dev, c.dev], INV)
    refuses(runner, [0, 1, 2], [5, 6, 2])
    for x in (a, b, c):
        x.check()  # nothing was launched
    runner.run(span(40), [0, 1, 2], [5, 6, 7])
    moved(a, b, span(40), [0, 1, 2], [5, 6, 7])
    moved(c, c, span(40), [0, 1, 2], [5, 6, 7])
    for x in (a, b, c):
        x.check()


def test_layers_crosswise(gpu):
    a, b = caches(gpu, 2)
    runner = ScaledShifts([a.dev, b.dev], [b.dev, a.dev], INV)
    refuses(runner, [0, 1, 2], [1, 6, 7])
    runner.run(span(40), [0, 1, 2], [5, 6, 7])
    twin = [x.codes.copy() for x in (a, b)], [x.scales.copy() for x in (a, b)]
    for (dst, i) in ((b, 0), (a, 1)):
        plain.shift(twin[0][i], twin[1][i], dst.codes, dst.scales, span(40), [0, 1, 2], [5, 6, 7], 16,
                    16, INV.numpy())
    a.check()
    b.check()


def test_a_destination_twice(gpu):
    a, b, c = caches(gpu, 3)
    with pytest.raises(ValueError, match="dst share"):
        ScaledShifts([a.dev, b.dev], [c.dev, c.dev], INV)
    again = ScaledCache(c.planes[0], c.dev_scales, "hnd")
    with pytest.raises(ValueError, match="dst share"):
        ScaledShifts([a.dev, b.dev], [c.dev, again], INV)
    # a layer that stands there twice, on both sides, is one
    runner = ScaledShifts([a.dev, b.dev, a.dev], [c.dev, b.dev, again], INV)
    assert runner.layers == 2
    runner.run(span(20), [0, 1], [4, 5])
    moved(a, c, span(20), [0, 1], [4, 5])
    moved(b, b, span(20), [0, 1], [4, 5])
    for x in (a, b, c):
        x.check()


@pytest.mark.parametrize("split", [False, True])
def test_views_of_one_caches_blocks(gpu, split):
    """Block 3 of one view is block 1 of the other."""
    whole, = caches(gpu, 1, split=split)
    planes = whole.planes + [None]

    def view(lo, hi):
        v = planes[1][lo:hi] if split else None
        return ScaledCache(planes[0][lo:hi], whole.dev_scales[lo:hi], "hnd", 16, v)

    runner = ScaledShifts([view(0, 5)], [view(2, 8)], INV)
    refuses(runner, [0, 3, 1], [5, 0, 1])
    refuses(runner, [4, 0, 1], [2, 3, 4])
    whole.check()
    runner.run(span(40), [0, 3, 1], [5, 0, 2])
    moved(whole, whole, span(40), [0, 3, 1], [7, 2, 4])
    whole.check()
    runner = ScaledShifts([view(2, 8)], [view(0, 5)], INV)  # and the other way
    refuses(runner, [1], [3], 10)
    runner.run(span(10), [1], [1])
    moved(whole, whole, span(10), [3], [1])
    whole.check()
    runner = ScaledShifts([view(0, 3)], [whole.dev], INV)  # of fewer blocks
    refuses(runner, [1], [1], 10)
    runner.run(span(10), [1], [6])
    moved(whole, whole, span(10), [1], [6])
    runner = ScaledShifts([view(0, 3)], [view(4, 8)], INV)  # that share nothing
    runner.run(span(10), [1], [1])
    moved(whole, whole, span(10), [1], [5])
    whole.check()
    one = ScaledShifts([view(3, 4)], [whole.dev], INV)  # of one block
    refuses(one, [0], [3], 10)


def test_a_span_without_a_source_meets_nothing(gpu):
    """An id out of range names no block: it is flagged, not refused."""
    whole, = caches(gpu, 1)
    views = [ScaledCache(whole.planes[0][i:j], whole.dev_scales[i:j], "hnd") for i, j in ((0, 4), (2, 8))]
    flags = torch.zeros(1, dtype=torch.int32, device=gpu)
    ScaledShifts(views[:1], views[1:], INV).run(span(40), [-1, 9, -3], [0, 1, 2], error_flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SRC_RANGE
    whole.check()


def test_sharing_that_no_block_number_says_is_refused(gpu):
    whole, = caches(gpu, 1)
    flat = whole.planes[0].view(torch.uint8).view(-1).view(torch.float8_e4m3fn)
    half = flat[2048:2048 + 7 * 4096].view(7, 2, 16, 128)  # half a block on
    scales = whole.dev_scales.clone()
    for kv, sc in [(half, whole.dev_scales[:7]),
                   (whole.planes[0], scales),                       # rows shared, scales apart
                   (whole.planes[0][1:], whole.dev_scales[:7]),     # by different numbers of blocks
                   (whole.planes[0].clone(), whole.dev_scales)]:    # scales alone
        other = ScaledCache(kv, sc, "hnd")
        for pair in ((whole.dev, other), (other, whole.dev)):
            with pytest.raises(ValueError, match="share memory"):
                ScaledShifts([pair[0]], [pair[1]], INV)


def test_layers_that_interleave_share_nothing(gpu):
    """Layers side by side in each block of one allocation: the same block numbers are others."""
    rng = np.random.default_rng(4)
    layers = 4
    pool = torch.from_numpy(rng.integers(0, 0x70, (6, layers, 2, 16, 128), np.uint8)).to(gpu)
    scales = torch.full((layers, 6, 2, 2), 125, dtype=torch.uint8, device=gpu)
    views = [ScaledCache(pool.view(torch.float8_e4m3fn)[:, i], scales.view(torch.float8_e8m0fnu)[i],
                         "hnd") for i in range(layers)]
    runner = ScaledShifts(views[:2], views[2:], None)
    runner.run([(0, 0, 0, 0, 48, 0, 0, 0)], [0, 1, 2], [0, 2, 1])
    for i in range(2):
        x, y = (pool[:, j].view(torch.float8_e4m3fn).double() for j in (i, i + 2))
        e = torch.exp2(scales[i + 2].double() - 127)
        y = y.reshape(6, 2, 16, 2, 64) * e[:, :, None, :, None]
        assert torch.equal(x.reshape(6, 2, 16, 2, 64)[:3] * 0.25, y[[0, 2, 1]])


# ------------------------------------------------------------------------- attention's output


def attend_args(gpu):
    cache, = caches(gpu, 1)
    return cache, (i32([[0, 1], [2, 3]], gpu), i32([0, 2, 3], gpu), i32([20, 30], gpu))


def test_outputs_that_overlap_are_refused(gpu):
    cache, step = attend_args(gpu)
    flat = torch.zeros(8192, dtype=torch.bfloat16, device=gpu)
    q = torch.randn(3, 4, 64, dtype=torch.bfloat16, device=gpu)
    for strides in [(64, 64, 1),      # (token 1, head 0) is (token 0, head 1)
                    (128, 64, 1),     # token 1 begins among token 0's heads
                    (64, 128, 1), (0, 64, 1), (256, 0, 1), (256, 32, 1), (32, 256, 1)]:
        with pytest.raises(_lib.KVShiftError, match="overlap"):
            attend_scaled(cache.dev, q, *step, out=flat.as_strided((3, 4, 64), strides))
    assert not flat.any()
    want = attend_scaled(cache.dev, q, *step)
    for strides in [(256, 64, 1), (64, 192, 1), (320, 72, 1), (64, 256, 1)]:
        out = flat.as_strided((3, 4, 64), strides)
        assert torch.equal(attend_scaled(cache.dev, q, *step, out=out), want)
        flat.zero_()
    one = i32([[0, 1]], gpu), i32([0, 1], gpu), i32([20], gpu)
    out = flat.as_strided((1, 4, 64), (0, 64, 1))  # of one token, whose stride is nobody's
    assert torch.equal(attend_scaled(cache.dev, q[:1], *one, out=out),
                       attend_scaled(cache.dev, q[:1], *one))


def test_an_output_in_the_queries_or_the_cache_is_refused(gpu):
    cache, step = attend_args(gpu)
    flat = torch.randn(8192, device=gpu).to(torch.bfloat16)
    q = flat.as_strided((3, 4, 64), (256, 64, 1))
    before = flat.clone()
    for at, strides in [(0, (256, 64, 1)), (64, (256, 64, 1)), (512, (256, 64, 1)),
                        (8, (256, 64, 1)), (0, (512, 64, 1)), (256, (1024, 256, 1))]:
        with pytest.raises(ValueError, match="memory with q"):
            attend_scaled(cache.dev, q, *step, out=flat.as_strided((3, 4, 64), strides, at))
    assert torch.equal(flat, before)
    inside = cache.planes[0].view(torch.bfloat16).view(-1)[:768].view(3, 4, 64)
    with pytest.raises(ValueError, match="memory with the cache"):
        attend_scaled(cache.dev, q, *step, out=inside)
    cache.check()


def test_an_output_between_the_queries_is_taken(gpu):
    """Queries and outputs in one buffer, a token's beside each other."""
    cache, step = attend_args(gpu)
    both = torch.randn(3, 12, 64, device=gpu).to(torch.bfloat16)
    q, out = both[:, :4], both[:, 4:8]
    rest = both[:, 8:].clone()
    want = attend_scaled(cache.dev, q.clone(), *step)
    assert attend_scaled(cache.dev, q, *step, out=out) is out
    assert torch.equal(out, want) and torch.equal(both[:, 8:], rest)
    wide = torch.randn(3, 4, 128, device=gpu).to(torch.bfloat16)
    want = attend_scaled(cache.dev, wide[..., :64].clone(), *step)
    assert torch.equal(attend_scaled(cache.dev, wide[..., :64], *step, out=wide[..., 64:]), want)
