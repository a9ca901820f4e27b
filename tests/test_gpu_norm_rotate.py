"""Heads normalised and turned on the GPU against the formula in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import norm_rotate
from marathon_amd.shift_kernels import inv_freq_for
from tests import step_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rows(gpu, rng, tokens, heads, d, dtype, spread=4):
    """Heads whose sizes differ by powers of two, and their values in 64 bits."""
    x = rng.standard_normal((tokens, heads, d)) * np.exp2(rng.integers(-spread, spread + 1, (tokens, heads, 1)))
    t = torch.from_numpy(x).to(dtype)
    return t.to(gpu), t.double().numpy()


def freq(rotary):
    return None if not rotary else inv_freq_for(rotary, 1e6).to(torch.float32)


def on(gpu, t):
    return None if t is None else t.to(gpu)


def host(t):
    return None if t is None else t.double().numpy()


def weights(rng, d, dtype):
    return None if dtype is None else torch.from_numpy(1 + 0.3 * rng.standard_normal(d)).to(dtype)


CASES = [  # tokens, query heads, key heads, D, rotary, dtype, weights, eps, positions
    (1, 1, 1, 128, 128, "bf16", "bf16", 1e-6, torch.int32),
    (1, 40, 8, 128, 128, "bf16", "bf16", 1e-6, torch.int64),
    (37, 5, 1, 64, 64, "fp16", "fp16", 1e-6, torch.int32),
    (37, 7, 3, 64, 32, "fp32", "fp32", 1e-5, torch.int64),
    (2, 16, 2, 256, 256, "fp32", "bf16", 1e-6, torch.int32),
    (300, 9, 4, 256, 96, "bf16", "fp32", 1e-6, torch.int32),
    (300, 3, 17, 128, 96, "fp16", "fp32", 0.1, torch.int64),
    (19, 8, 8, 128, 0, "bf16", "bf16", 1e-6, None),      # a layer without positions
    (19, 8, 8, 128, 64, "bf16", None, None, torch.int32),  # a model without the norm
    (64, 4, 4, 64, 64, "fp32", None, 1e-6, torch.int32),  # ones for weights
    (1500, 40, 8, 128, 128, "bf16", "bf16", 1e-6, torch.int32),  # several heads a wave, unevenly
    (5000, 33, 1, 64, 64, "fp16", "fp16", 1e-6, torch.int32),
]


@pytest.mark.parametrize("tokens,qh,kh,d,rotary,dtype,wt,eps,pt", CASES)
def test_equals_the_formula(gpu, tokens, qh, kh, d, rotary, dtype, wt, eps, pt):
    rng = np.random.default_rng(tokens * 31 + qh + d)
    q, q64 = rows(gpu, rng, tokens, qh, d, DTYPES[dtype])
    k, k64 = rows(gpu, rng, tokens, kh, d, DTYPES[dtype])
    pos = rng.integers(0, 40000, tokens)
    inv = freq(rotary)
    wq, wk = (weights(rng, d, DTYPES.get(wt)) for _ in range(2))
    positions = None if pt is None else torch.from_numpy(pos).to(gpu, pt)
    got = norm_rotate(q, k, positions, on(gpu, inv), q_weight=on(gpu, wq), k_weight=on(gpu, wk), eps=eps)
    for out, x, w in zip(got, (q64, k64), (wq, wk)):
        assert out.dtype == DTYPES[dtype] and out.is_contiguous()
        plain.check_turned(out, *plain.turned(x, host(w), pos, None if inv is None else inv.numpy(), eps))
    assert torch.equal(q.cpu().double(), torch.from_numpy(q64))  # the inputs are as they were


@pytest.mark.parametrize("top", [10**6, 2**24 + 1, 2**31 - 1])
@pytest.mark.parametrize("sign", [1, -1])
def test_far_positions_keep_their_angles(gpu, top, sign):
    """In 32 bits a position of 2^24 turns times a frequency has lost its place in the turn."""
    rng = np.random.default_rng(top % 1000)
    pos = sign * (top - rng.integers(0, 1000, 50))
    q, q64 = rows(gpu, rng, 50, 2, 128, torch.float32, 0)
    inv = freq(128)
    out, _ = norm_rotate(q, q.clone(), torch.from_numpy(pos).to(gpu, torch.int32), inv.to(gpu))
    plain.check_turned(out, *plain.turned(q64, None, pos, inv.numpy(), 1e-6))


def test_views_of_one_projection_in_place_and_into_strided_outputs(gpu):
    rng = np.random.default_rng(5)
    tokens, qh, kh, d = 83, 6, 2, 128
    inv = freq(64).to(gpu)
    pos = torch.arange(tokens, dtype=torch.int32, device=gpu) + 777
    both, _ = rows(gpu, rng, tokens, qh + 2 * kh, d, torch.bfloat16)
    w = weights(rng, d, torch.bfloat16).to(gpu)

    def parts(t):
        return t[:, :qh], t[:, qh:qh + kh]

    want = norm_rotate(*(x.contiguous() for x in parts(both)), pos, inv, q_weight=w, k_weight=w)
    got = norm_rotate(*parts(both), pos, inv, q_weight=w, k_weight=w)
    # heads first in memory, with room between
    roomy = [torch.full((h, tokens, d + 8), 7.0, dtype=torch.bfloat16, device=gpu) for h in (qh, kh)]
    views = [t.transpose(0, 1)[..., :d] for t in roomy]
    into = norm_rotate(*parts(both), pos, inv, q_weight=w, k_weight=w, out_q=views[0], out_k=views[1])
    assert into[0] is views[0] and into[1] is views[1]
    for t in roomy:
        assert (t[..., d:] == 7).all()
    rest = both[:, qh + kh:].clone()
    norm_rotate(*parts(both), pos, inv, q_weight=w, k_weight=w, out_q=both[:, :qh], out_k=both[:, qh:qh + kh])
    for a, b, c, e in zip(want, got, into, parts(both)):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, e)
    assert torch.equal(both[:, qh + kh:], rest)


def test_odd_values_stay_in_their_heads(gpu):
    """Zeros, a NaN, an infinity, values whose squares leave fp32, and what eps does with zeros."""
    rng = np.random.default_rng(8)
    q, q64 = rows(gpu, rng, 6, 4, 64, torch.float32, 0)
    inv, pos = freq(64), np.arange(6)
    q[0, 1] = 0
    q[1, 2, 5], q[2, 3, 60] = float("nan"), float("inf")
    q[3, 0] *= 2.0 ** 100
    q64 = q.double().cpu().numpy()
    at = torch.arange(6, dtype=torch.int32, device=gpu)
    out, _ = norm_rotate(q, q.clone(), at, inv.to(gpu))
    clean = np.ones((6, 4), bool)
    clean[1, 2] = clean[2, 3] = clean[3, 0] = False
    want, size = plain.turned(np.where(clean[..., None], q64, 0), None, pos, inv.numpy(), 1e-6)
    got = out.cpu()
    assert got[1, 2].isnan().all() and got[2, 3].isnan().any()
    assert (got[3, 0] == 0).all() and (got[0, 1] == 0).all()
    got[~torch.from_numpy(clean)] = 0
    plain.check_turned(got, want, size)
    out, _ = norm_rotate(q, q.clone(), at, inv.to(gpu), eps=0.0)
    assert out[0, 1].isnan().all() and out[0, 0].isfinite().all()
    # without the norm an infinity stays one; at position 0 its partner adds inf * sin(0), a NaN
    out, _ = norm_rotate(q[2:3], q[2:3].clone(), at[:1], inv.to(gpu), eps=None)
    want = q[2:3].clone()
    want[0, 3, 28] = float("nan")
    assert torch.equal(out.nan_to_num(nan=9.0, posinf=8.0), want.nan_to_num(nan=9.0, posinf=8.0))


def test_no_tokens_and_no_heads(gpu):
    inv = freq(128).to(gpu)
    none = torch.empty((0, 8, 128), dtype=torch.bfloat16, device=gpu)
    out = norm_rotate(none, none[:, :2], torch.empty(0, dtype=torch.int32, device=gpu), inv)
    assert out[0].shape == (0, 8, 128) and out[1].shape == (0, 2, 128)
    x = torch.randn((3, 2, 128), dtype=torch.bfloat16, device=gpu)
    pos = torch.arange(3, dtype=torch.int32, device=gpu)
    a, b = norm_rotate(x, x[:, :0], pos, inv)
    assert b.shape == (3, 0, 128) and torch.equal(a, norm_rotate(x, x.clone(), pos, inv)[1])


def test_on_another_stream_and_from_a_graph(gpu):
    rng = np.random.default_rng(3)
    q, _ = rows(gpu, rng, 40, 8, 128, torch.bfloat16)
    k, _ = rows(gpu, rng, 40, 2, 128, torch.bfloat16)
    inv, pos = freq(128).to(gpu), torch.arange(40, dtype=torch.int32, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = norm_rotate(q, k, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(late, norm_rotate(q, k, pos, inv)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = norm_rotate(q, k, pos, inv)
    for i in range(4):
        q.copy_(rows(gpu, rng, 40, 8, 128, torch.bfloat16)[0])
        pos.add_(i * 1000)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, norm_rotate(q, k, pos, inv)):
            assert torch.equal(a, b)


def test_refusals(gpu):
    q = torch.randn((4, 8, 128), dtype=torch.bfloat16, device=gpu)
    k = torch.randn((4, 2, 128), dtype=torch.bfloat16, device=gpu)
    inv, pos = freq(128).to(gpu), torch.arange(4, dtype=torch.int32, device=gpu)
    w = torch.ones(128, dtype=torch.bfloat16, device=gpu)

    def refused(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            norm_rotate(*args, **kw)

    refused(ValueError, "tokens, heads, D", q[0], k, pos, inv)
    refused(ValueError, "one of", q[..., :96], k[..., :96], pos, inv)
    refused(ValueError, "tokens, heads, D", q, k[:3], pos, inv)
    refused(TypeError, "of one type", q, k.float(), pos, inv)
    refused(TypeError, "of one type", q.double(), k.double(), pos, inv)
    refused(ValueError, "contiguous", q.transpose(1, 2).contiguous().transpose(1, 2), k, pos, inv)
    refused(TypeError, "float32", q, k, pos, inv.double())
    refused(ValueError, "rotary", q, k, pos, inv[:24])
    refused(ValueError, "rotary", q, k, pos, torch.cat((inv, inv)))
    refused(ValueError, "inv_freq", q, k, pos, inv.cpu())
    refused(TypeError, "positions", q, k, None, inv)
    refused(TypeError, "positions", q, k, pos.float(), inv)
    refused(ValueError, "positions", q, k, pos[:3], inv)
    refused(ValueError, "positions", q, k, pos.repeat(2)[::2], inv)
    refused(ValueError, "without a norm", q, k, pos, inv, q_weight=w, eps=None)
    refused(TypeError, "of one type", q, k, pos, inv, q_weight=w, k_weight=w.float())
    refused(ValueError, "k_weight", q, k, pos, inv, k_weight=w[:64])
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(ValueError, "eps", q, k, pos, inv, eps=eps)
    refused(ValueError, "does not fit", q, k, pos, inv, out_q=k)
    refused(ValueError, "shares memory", q, k, pos, inv, out_k=q[:, :2])
    wide = torch.empty((5, 8, 128), dtype=torch.bfloat16, device=gpu)
    refused(ValueError, "does not fit", q, k, pos, inv, out_q=wide[:1, :1, :1].expand(4, 8, 128))
    refused(RuntimeError, "overlap", q, k, pos, inv, out_q=wide[:1, :1].expand(4, 8, 128))
    refused(ValueError, "not q itself", wide[:4], k, pos, inv, out_q=wide[1:])
    refused(ValueError, "shares memory", q, k, pos, inv, out_q=wide[:4], out_k=wide[:4, 6:])
    refused(RuntimeError, "backward", q.clone().requires_grad_(), k, pos, inv)
    refused(RuntimeError, "backward", q, k, pos, inv, k_weight=w.clone().requires_grad_())
    odd = torch.empty(4 * 8 * 128 + 4, dtype=torch.bfloat16, device=gpu)[4:].view(4, 8, 128)
    refused(RuntimeError, "aligned", odd, k, pos, inv)
    with torch.no_grad():
        norm_rotate(q.clone().requires_grad_(), k, pos, inv)
    torch.cuda.synchronize()


def test_frequencies_that_learn_are_refused_without_a_norm_too(gpu):
    x = torch.randn(3, 2, 64, device=gpu)
    pos, inv = torch.arange(3, device=gpu), torch.rand(32, device=gpu)
    for eps in (None, 1e-6):
        with pytest.raises(RuntimeError, match="backward"):
            norm_rotate(x, x.clone(), pos, inv.clone().requires_grad_(), eps=eps)
