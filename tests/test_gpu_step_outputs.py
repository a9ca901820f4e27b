"""A caller's own outputs: taken by the calls' short path, told from what a call reads, and alike by
both paths."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import norm_rotate, scaled_step, store_rotated
from tests.test_gpu_norm_rotate import freq
from tests.test_gpu_scaled import Cache, i32, requests_of
from tests.test_gpu_step import Counted, Nothing

pytestmark = pytest.mark.gpu


def step_of(gpu, tokens=21, heads=2, d=128):
    rng = np.random.default_rng(tokens)
    tables, blocks = requests_of([tokens], [9], 16, rng, spare=8)
    cache = Cache(gpu, rng, blocks, heads, d, 16)
    return cache, (i32(tables, gpu), i32([0, tokens], gpu), i32([9 + tokens], gpu))


def projection(gpu, tokens=21, parts=(8, 2, 2), d=128):
    g = torch.Generator(device=gpu).manual_seed(1)
    return torch.randn((tokens, sum(parts), d), generator=g, device=gpu).to(torch.bfloat16).split(parts, 1)


def taken(monkeypatch, short, call):
    """The call by the short path, which has to take it, or by the general one."""
    usual = Counted() if short else Nothing()
    monkeypatch.setattr(scaled_step, "_usual", usual)
    got = call()
    assert not short or (usual.got and usual.got[-1] is not None)
    return got


@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("where", ["views", "apart", "other", "strided"])
@pytest.mark.parametrize("tokens", [1, 21])
def test_queries_of_a_store(gpu, short, where, tokens, monkeypatch):
    cache, step = step_of(gpu, tokens)
    q, k, v = projection(gpu, tokens)
    inv = freq(128).to(gpu)
    want = store_rotated(cache.dev, q, k, v, *step, inv)
    codes = cache.planes[0].view(torch.uint8).clone()
    whole = torch.full((tokens, 12, 128), 7.0, dtype=torch.bfloat16, device=gpu)
    if where == "apart":
        q = q.clone()
    out = {"other": torch.empty(q.shape, dtype=q.dtype, device=gpu), "strided": whole[:, 2:10]}.get(where, q)
    rest = [x.clone() for x in (k, v)]
    got = taken(monkeypatch, short, lambda: store_rotated(cache.dev, q, k, v, *step, inv, out_q=out))
    assert got is out and torch.equal(got, want)
    assert torch.equal(cache.planes[0].view(torch.uint8), codes)
    assert torch.equal(k, rest[0]) and torch.equal(v, rest[1])
    if where == "strided":
        assert (whole[:, :2] == 7).all() and (whole[:, 10:] == 7).all()


@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("where", ["views", "apart", "other", "strided", "one"])
@pytest.mark.parametrize("tokens", [1, 21])
def test_queries_and_keys(gpu, short, where, tokens, monkeypatch):
    q, k, v = projection(gpu, tokens)
    pos, inv = torch.arange(tokens, device=gpu) + 3, freq(64).to(gpu)
    want = norm_rotate(q, k, pos, inv)
    whole = torch.full((tokens, 12, 128), 7.0, dtype=torch.bfloat16, device=gpu)
    if where == "apart":
        q, k = q.clone(), k.clone()
    out = {"other": (torch.empty_like(q), torch.empty_like(k)), "strided": (whole[:, 3:11], whole[:, :2]),
           "one": (None, k)}.get(where, (q, k))
    rest = v.clone()
    got = taken(monkeypatch, short, lambda: norm_rotate(q, k, pos, inv, out_q=out[0], out_k=out[1]))
    for a, b, o in zip(got, want, out):
        assert torch.equal(a, b) and (o is None or a is o)
    assert torch.equal(v, rest)
    if where == "strided":
        assert (whole[:, 2:3] == 7).all() and (whole[:, 11:] == 7).all()


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
