"""Blocks whose angles fill the memory that a launch has unasked, and more than that."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from marathon_amd import store_rotated
from tests import step_plain as plain
from tests.test_gpu_norm_rotate import freq
from tests.test_gpu_scaled import i32
from tests.test_gpu_store_rotated import make

pytestmark = pytest.mark.gpu

# D, rotary, block: [block][rotary / 2] pairs of 8 bytes are 64 KiB, just below and twice that
SHAPES = [(256, 256, 64), (128, 128, 128), (256, 224, 64), (128, 96, 128), (256, 128, 128), (256, 256, 128)]


@pytest.mark.parametrize("d,rotary,bs", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_equals_the_formula(gpu, d, rotary, bs, dtype):
    rng = np.random.default_rng(d + rotary + bs)
    new, held = [bs + 9, 1, 3], [5, bs - 1, 0]
    cache, tables, starts, lens, (q, k, v), (q64, k64, v64), pos = make(
        gpu, rng, new, held, 4, 2, d, bs, "hnd", dtype, False)
    before, inv = cache.read(), freq(rotary)
    out = store_rotated(cache.dev, q, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), inv.to(gpu))
    plain.check_turned(out, *plain.turned(q64, None, pos, inv.numpy(), 1e-6))
    want, size = plain.turned(k64, None, pos, inv.numpy(), 1e-6)
    plain.check_store(before, *cache.read(), want, size, v64, tables, starts, lens, bs)


def test_threads_that_need_different_amounts(gpu):
    """Calls of one kernel from several threads, on streams of their own, with blocks of each size."""
    rng = np.random.default_rng(7)
    jobs = []
    for bs in (16, 64, 128, 128):
        cache, tables, starts, lens, (q, k, v), _, _ = make(
            gpu, rng, [bs + 3], [2], 4, 2, 256, bs, "hnd", "bf16", False)
        args = (cache.dev, q, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), freq(256).to(gpu))
        jobs.append((args, store_rotated(*args), torch.cuda.Stream(), []))
    torch.cuda.synchronize()

    def work(args, want, stream, out):
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = store_rotated(*args)
            out.append(torch.equal(got, want))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert [j[3] for j in jobs] == [[True]] * len(jobs)
