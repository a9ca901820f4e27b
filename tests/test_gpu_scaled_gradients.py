"""The block-scaled cache has no gradients: calls that would lose one are refused."""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from marathon_amd import attend_scaled, store_scaled
from tests.test_gpu_scaled import Cache, i32

pytestmark = pytest.mark.gpu


def parts(gpu):
    cache = Cache(gpu, np.random.default_rng(1), 3, 2, 64, 16)
    k = torch.randn(3, 2, 64, device=gpu, dtype=torch.bfloat16)
    q = torch.randn(3, 4, 64, device=gpu, dtype=torch.bfloat16)
    return cache, k, q, (i32([[0, 1]], gpu), i32([0, 3], gpu), i32([3], gpu))


def test_rows_that_need_a_gradient_are_refused(gpu):
    cache, k, q, step = parts(gpu)
    leaf = k.clone().requires_grad_()
    for rows in ((leaf, k), (k, leaf), (leaf * 2, k)):
        with pytest.raises(RuntimeError, match="no backward"):
            store_scaled(cache.dev, *rows, *step)
    with pytest.raises(RuntimeError, match="no backward"):
        attend_scaled(cache.dev, q.clone().requires_grad_(), *step)
    with pytest.raises(RuntimeError, match="no backward"):
        attend_scaled(cache.dev, q, *step, out=torch.empty_like(q).requires_grad_())
    cache.check()  # nothing was written


def test_without_gradients_the_same_tensors_are_taken(gpu):
    cache, k, q, step = parts(gpu)
    twin = Cache(gpu, np.random.default_rng(1), 3, 2, 64, 16)
    store_scaled(twin.dev, k, k, *step)
    want = attend_scaled(twin.dev, q, *step)
    with torch.no_grad():
        store_scaled(cache.dev, k.clone().requires_grad_(), k.clone().requires_grad_(), *step)
        out = torch.empty_like(q).requires_grad_()
        got = attend_scaled(cache.dev, q.clone().requires_grad_(), *step, out=out)
    assert got is out and torch.equal(got.detach(), want)
    assert torch.equal(cache.planes[0].view(torch.uint8), twin.planes[0].view(torch.uint8))
    with torch.inference_mode():
        assert torch.equal(attend_scaled(cache.dev, q.clone(), *step), want)


def test_forward_mode_tangents_are_refused(gpu):
    cache, k, q, step = parts(gpu)
    with forward_ad.dual_level():
        dual_k = forward_ad.make_dual(k, torch.ones_like(k))
        dual_q = forward_ad.make_dual(q, torch.ones_like(q))
        for rows in ((dual_k, k), (k, dual_k)):
            with pytest.raises(RuntimeError, match="tangent"):
                store_scaled(cache.dev, *rows, *step)
        with pytest.raises(RuntimeError, match="tangent"):
            attend_scaled(cache.dev, dual_q, *step)
        with pytest.raises(RuntimeError, match="tangent"):
            attend_scaled(cache.dev, q, *step, out=forward_ad.make_dual(q.clone(), q))
        cache.check()
        attend_scaled(cache.dev, q, *step)  # a tensor without one is taken within a level
