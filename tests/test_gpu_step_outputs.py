"""A caller's own outputs, told from what a call reads."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import norm_rotate, scaled_step, store_rotated
from tests.test_gpu_norm_rotate import freq
from tests.test_gpu_scaled import Cache, i32, requests_of
from tests.test_gpu_step import Nothing

pytestmark = pytest.mark.gpu


def step_of(gpu, tokens=21, heads=2, d=128):
    rng = np.random.default_rng(tokens)
    tables, blocks = requests_of([tokens], [9], 16, rng, spare=8)
    cache = Cache(gpu, rng, blocks, heads, d, 16)
    return cache, (i32(tables, gpu), i32([0, tokens], gpu), i32([9 + tokens], gpu))


def projection(gpu, tokens=21, parts=(8, 2, 2), d=128):
    g = torch.Generator(device=gpu).manual_seed(1)
    return torch.randn((tokens, sum(parts), d), generator=g, device=gpu).to(torch.bfloat16).split(parts, 1)


@pytest.mark.parametrize("short", [True, False])
def test_outputs_in_what_a_call_reads_are_refused(gpu, short, monkeypatch):
    cache, step = step_of(gpu)
    q, k, v = projection(gpu)
    pos, inv = torch.arange(21, device=gpu), freq(128).to(gpu)
    w = torch.ones(128, dtype=torch.bfloat16, device=gpu)
    if not short:
        monkeypatch.setattr(scaled_step, "_usual", Nothing())

    def refused(match, call, *args, **kw):
        with pytest.raises((ValueError, RuntimeError), match=match):
            call(*args, **kw)

    # a buffer of queries whose first bytes are the positions, the weights, the frequencies, the lengths
    room = torch.zeros((21, 8, 128), dtype=torch.bfloat16, device=gpu)
    flat = room.flatten()
    for there in (dict(positions=flat[:42].view(torch.int32)), dict(positions=flat[:84].view(torch.int64)),
                  dict(q_weight=flat[128:256]), dict(k_weight=flat[-128:]),
                  dict(inv_freq=flat[256:384].view(torch.float32))):
        given = dict(positions=pos, inv_freq=inv, q_weight=w, k_weight=w) | there
        args = given.pop("positions"), given.pop("inv_freq")
        refused("an input", norm_rotate, room, k, *args, out_q=room, out_k=k, **given)
        if "positions" not in there:
            refused("an input", store_rotated, cache.dev, room, k, v, *step, args[1], out_q=room, **given)
    table = flat[:2 * step[0].numel()].view(torch.int32).view(step[0].shape)
    # (rows far apart, the second of them in the queries' buffer)
    far = torch.zeros(2048 + room.numel(), dtype=torch.bfloat16, device=gpu)
    wide = far[1024:].view(torch.int32).as_strided((2, step[0].shape[1]), (1024, 1))
    refused("an input", store_rotated, cache.dev, far[2048:].view(21, 8, 128), k, v, wide, i32([0, 20, 21], gpu),
            i32([20, 1], gpu), inv, out_q=far[2048:].view(21, 8, 128))
    for i, t in enumerate((table, flat[:4].view(torch.int32), flat[8:10].view(torch.int32))):
        mine = [*step]
        mine[i] = t
        refused("an input", store_rotated, cache.dev, room, k, v, *mine, inv, out_q=room)
    # rows that lie in others'
    long = torch.zeros((26, 12, 128), dtype=torch.bfloat16, device=gpu)
    refused("not q itself", norm_rotate, long[:21, :8], k, pos, inv, out_q=long[5:, :8])
    refused("with k", norm_rotate, long[:21, :8], long[:21, 7:9], pos, inv, out_q=long[:21, :8])
    refused("with k", store_rotated, cache.dev, long[:21, :8], long[:21, 7:9], v, *step, inv, out_q=long[:21, :8])
    refused("with v", store_rotated, cache.dev, long[:21, 2:10], k, long[:21, 1:3], *step, inv,
            out_q=long[:21, 2:10])
    mine = v.clone()
    refused("with v", store_rotated, cache.dev, q, k, mine, *step, inv,
            out_q=mine.as_strided((21, 8, 128), (mine.stride(0), 0, 1)))
    refused("with out_k|with k|out_q", norm_rotate, q, k, pos, inv, out_q=long[:21, :8], out_k=long[:21, 6:8])
    inside = cache.planes[0].view(torch.bfloat16).flatten()[:21 * 8 * 128].view(21, 8, 128)
    refused("cache", store_rotated, cache.dev, q, k, v, *step, inv, out_q=inside)
    refused("cache", store_rotated, cache.dev, inside, k, v, *step, inv, out_q=inside)
    refused("backward", store_rotated, cache.dev, q, k, v, *step, inv,
            out_q=torch.empty((21, 8, 128), dtype=torch.bfloat16, device=gpu).requires_grad_())
    torch.cuda.synchronize()
