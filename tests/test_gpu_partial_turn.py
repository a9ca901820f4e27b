"""Heads of which a part is turned: the other values are their own, whatever stands beside them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import norm_rotate, store_rotated
from tests import scaled_plain
from tests.test_gpu_norm_rotate import DTYPES, freq
from tests.test_gpu_scaled import Cache, i32, requests_of

pytestmark = pytest.mark.gpu

SHAPES = [(64, 32), (128, 32), (128, 96), (256, 64), (256, 224)]  # D, rotary


def odd(rng, tokens, heads, d, rotary, dtype, nan=True):
    """Rows with infinities, NaNs and zeros of both signs among the values that are not turned."""
    x = torch.from_numpy(rng.standard_normal((tokens, heads, d))).to(dtype)
    values = [float("inf"), -float("inf"), -0.0, 0.0] + ([float("nan")] if nan else [])
    for t in range(tokens):
        for h in range(heads):
            at = rotary + rng.integers(0, d - rotary, 3)
            x[t, h, at] = torch.tensor(rng.choice(values, 3)).to(dtype)
    return x


def bits(t):
    """Bit for bit but for NaNs, which are one value."""
    t = torch.where(t.isnan(), torch.full_like(t, float("nan")), t)
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("d,rotary", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads", [1, 8])
def test_what_is_not_turned_comes_out_as_it_went_in(gpu, d, rotary, dtype, heads):
    rng = np.random.default_rng(d + rotary + heads)
    q, k = (odd(rng, 40, h, d, rotary, DTYPES[dtype]).to(gpu) for h in (heads, 2))
    pos = torch.arange(40, dtype=torch.int32, device=gpu) + 5
    for out, x in zip(norm_rotate(q, k, pos, freq(rotary).to(gpu), eps=None), (q, k)):
        assert torch.equal(bits(out[..., rotary:].contiguous()), bits(x[..., rotary:].contiguous()))
        assert out[..., :rotary].isfinite().all()


@pytest.mark.parametrize("d,rotary", SHAPES)
def test_an_infinity_under_the_norm_is_nan_alone(gpu, d, rotary):
    """x / sqrt(mean) with an infinite mean: inf / inf there, and zeros elsewhere."""
    rng = np.random.default_rng(d + rotary)
    q = torch.from_numpy(rng.standard_normal((7, 4, d))).to(gpu, torch.float32)
    pos = torch.arange(7, dtype=torch.int32, device=gpu)
    at = rng.integers(rotary, d, 7)
    q[range(7), 2, at] = float("inf")
    out, _ = norm_rotate(q, q.clone(), pos, freq(rotary).to(gpu))
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[range(7), 2, at] = True
    assert torch.equal(out.isnan(), nan)
    assert (out[:, 2].nan_to_num() == 0).all()


@pytest.mark.parametrize("d,rotary", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_keys_on_their_way_into_the_cache(gpu, d, rotary, dtype):
    """Infinities of a key saturate and NaNs stay, in their places alone; the queries as above."""
    rng = np.random.default_rng(3 * d + rotary)
    tables, blocks = requests_of([37], [0], 16, rng)
    cache = Cache(gpu, rng, blocks, 2, d, 16)
    q, k = (odd(rng, 37, h, d, rotary, DTYPES[dtype]) for h in (6, 2))
    v = torch.from_numpy(rng.standard_normal((37, 2, d))).to(DTYPES[dtype])
    out = store_rotated(cache.dev, q.to(gpu), k.to(gpu), v.to(gpu), i32(tables, gpu), i32([0, 37], gpu),
                        i32([37], gpu), freq(rotary).to(gpu), eps=None).cpu()
    assert torch.equal(bits(out[..., rotary:].contiguous()), bits(q[..., rotary:].contiguous()))
    codes, scales = cache.read()
    pos = np.arange(37)
    at = tables[0, pos // 16]
    got, e = codes[at, pos % 16, :, 0, rotary:], scaled_plain.exponents(scales[at, :, 0])
    want = scaled_plain.encode(k.double().numpy()[..., rotary:] * 2.0 ** -e[..., None].astype(np.float64))
    nan = (want & 127) == 127
    assert np.array_equal((got & 127) == 127, nan)
    assert np.array_equal(scaled_plain.decode(got[~nan]), scaled_plain.decode(want[~nan]))
