"""A step's projections into the block-scaled cache, normalised and turned: against the formula
in 64 bits, and against the two calls that it stands for."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import _lib, norm_rotate, store_rotated, store_scaled
from marathon_amd.shift_kernels import inv_freq_for
from tests import step_plain as plain
from tests.test_gpu_norm_rotate import DTYPES, freq, host, on, rows, weights
from tests.test_gpu_scaled import Cache, i32, requests_of

pytestmark = pytest.mark.gpu

CASES = [  # new, held, query heads, heads, D, rotary, bs, layout, dtype, split planes, weights
    ([1], [0], 4, 1, 128, 128, 16, "hnd", "bf16", False, "bf16"),
    ([1, 1, 1], [15, 16, 33], 32, 8, 128, 128, 16, "hnd", "bf16", False, "bf16"),
    ([5, 0, 40, 1], [3, 9, 0, 31], 6, 3, 64, 32, 16, "nhd", "fp16", False, "fp32"),
    ([33, 2, 100], [31, 62, 7], 4, 2, 256, 256, 32, "hnd", "fp32", True, "fp32"),
    ([70, 1], [63, 64], 5, 5, 128, 64, 64, "nhd", "bf16", True, None),
    ([300, 129], [1, 127], 8, 2, 64, 64, 128, "hnd", "fp32", False, "bf16"),
    ([150, 9], [3, 120], 2, 1, 256, 256, 128, "hnd", "bf16", False, "bf16"),
    ([4200, 37, 1, 900], [5, 0, 77, 15], 1, 1, 64, 64, 16, "nhd", "bf16", False, "bf16"),
    ([17, 16, 15], [16, 0, 1], 16, 4, 256, 96, 16, "hnd", "fp16", False, "fp16"),
    ([2100], [9], 40, 8, 128, 128, 16, "hnd", "bf16", False, "bf16"),
    ([30, 3], [0, 20], 4, 2, 128, 0, 16, "hnd", "bf16", False, "bf16"),
]


def make(gpu, rng, new, held, qh, heads, d, bs, layout, dtype, split, pad=0):
    tables, count = requests_of(new, held, bs, rng)
    cache = Cache(gpu, rng, count, heads, d, bs, layout, split)
    tokens = sum(new) + pad
    starts = np.concatenate(([0], np.cumsum(new)))
    lens = np.array(held) + np.array(new)
    q, q64 = rows(gpu, rng, tokens, qh, d, DTYPES[dtype])
    k, k64 = rows(gpu, rng, tokens, heads, d, DTYPES[dtype])
    v, v64 = rows(gpu, rng, tokens, heads, d, DTYPES[dtype])
    pos = np.concatenate([np.arange(h, h + n) for h, n in zip(held, new)])
    return cache, tables, starts, lens, (q, k, v), (q64, k64, v64), pos


@pytest.mark.parametrize("new,held,qh,heads,d,rotary,bs,layout,dtype,split,wt", CASES)
def test_equals_the_formula(gpu, new, held, qh, heads, d, rotary, bs, layout, dtype, split, wt):
    rng = np.random.default_rng(sum(new) * 7 + d)
    cache, tables, starts, lens, (q, k, v), (q64, k64, v64), pos = make(
        gpu, rng, new, held, qh, heads, d, bs, layout, dtype, split)
    inv = freq(rotary)
    wq, wk = (weights(rng, d, DTYPES.get(wt)) for _ in range(2))
    flags = i32([0], gpu)
    before = cache.read()
    out = store_rotated(cache.dev, q, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu),
                        on(gpu, inv), q_weight=on(gpu, wq), k_weight=on(gpu, wk), error_flags=flags)
    assert flags.item() == 0
    f = None if inv is None else inv.numpy()
    plain.check_turned(out, *plain.turned(q64, host(wq), pos, f, 1e-6))
    want, size = plain.turned(k64, host(wk), pos, f, 1e-6)
    codes, scales = cache.read()
    plain.check_store(before, codes, scales, want, size, v64, tables, starts, lens, bs)


@pytest.mark.parametrize("new,held,qh,heads,d,rotary,bs,layout,dtype,split,wt", CASES)
@pytest.mark.parametrize("eps", [1e-6, None])
def test_equals_the_two_calls(gpu, new, held, qh, heads, d, rotary, bs, layout, dtype, split, wt, eps):
    """norm_rotate of the rows in fp32, whose outputs are not rounded, then store_scaled: the
    same bits; the queries as norm_rotate gives them."""
    rng = np.random.default_rng(sum(new) * 5 + d)
    cache, tables, starts, lens, (q, k, v), _, pos = make(
        gpu, rng, new, held, qh, heads, d, bs, layout, dtype, split)
    inv = on(gpu, freq(rotary))
    kw = {}
    if eps is not None:
        kw = {f"{n}_weight": on(gpu, weights(rng, d, DTYPES.get(wt))) for n in "qk"}
    args = i32(tables, gpu), i32(starts, gpu), i32(lens, gpu)
    planes = [p.view(torch.uint8).clone() for p in cache.planes]
    scales = cache.dev_scales.view(torch.uint8).clone()
    out = store_rotated(cache.dev, q, k, v, *args, inv, eps=eps, **kw)
    got = [p.view(torch.uint8).clone() for p in cache.planes], cache.dev_scales.view(torch.uint8).clone()
    for p, was in zip(cache.planes, planes):
        p.view(torch.uint8).copy_(was)
    cache.dev_scales.view(torch.uint8).copy_(scales)
    at = torch.from_numpy(pos).to(gpu, torch.int32)
    _, wide = norm_rotate(q.float(), k.float(), at, inv, eps=eps, **kw)
    store_scaled(cache.dev, wide, v.float(), *args)
    for a, b in zip(got[0], cache.planes):
        assert torch.equal(a, b.view(torch.uint8))
    assert torch.equal(got[1], cache.dev_scales.view(torch.uint8))
    assert torch.equal(out, norm_rotate(q, k, at, inv, eps=eps, **kw)[0])


def test_padding_in_place_and_views_of_one_projection(gpu):
    """Rows behind the last request and before the first are nobody's; out_q may be q, a part of
    the projection that k and v are parts of."""
    rng = np.random.default_rng(2)
    new, held, heads, d, bs = [3, 0, 20], [30, 4, 1], 2, 128, 16
    cache, tables, starts, lens, (q, k, v), _, pos = make(
        gpu, rng, new, held, 4, heads, d, bs, "hnd", "bf16", False, pad=9)
    starts = starts + 4  # four rows before the first request, five behind the last
    both = torch.cat((q, k, v), 1)
    was = both.clone()
    inv = freq(d).to(gpu)
    out = store_rotated(cache.dev, both[:, :4], both[:, 4:6], both[:, 6:], i32(tables, gpu),
                        i32(starts, gpu), i32(lens, gpu), inv, out_q=both[:, :4])
    assert out.data_ptr() == both.data_ptr()
    at = torch.from_numpy(pos).to(gpu, torch.int32)
    assert torch.equal(both[4:27, :4], norm_rotate(was[4:27, :4], was[4:27, 4:6], at, inv)[0])
    assert torch.equal(both[:4], was[:4]) and torch.equal(both[27:], was[27:])
    assert torch.equal(both[:, 4:], was[:, 4:])
    wide = norm_rotate(was[4:27, :4].float(), was[4:27, 4:6].float(), at, inv)[1].double().cpu().numpy()
    codes, scales = cache.read()
    plain.check_store((cache.codes, cache.scales), codes, scales, wide, np.zeros_like(wide),
                      was[4:27, 6:].double().cpu().numpy(), tables, starts - 4, lens, bs)


@pytest.mark.parametrize("why", ["starts", "short", "id", "table"])
def test_what_does_not_fit_is_left_out_and_flagged(gpu, why):
    rng = np.random.default_rng(4)
    new, held, heads, d, bs = [18, 5], [14, 3], 2, 64, 16
    cache, tables, starts, lens, (q, k, v), _, _ = make(
        gpu, rng, new, held, 4, heads, d, bs, "hnd", "fp16", False)
    width = tables.shape[1]
    flag = _lib.MKV_FLAG_DST_RANGE
    if why == "starts":
        starts[1:] = [40, 23]
        flag = _lib.MKV_FLAG_SPAN
    elif why == "short":
        lens[0] = 17
        flag = _lib.MKV_FLAG_SPAN
    elif why == "id":
        tables[0, :] = [-1, cache.codes.shape[0], 2**31 - 1][:width] + [0] * max(0, width - 3)
    else:
        width = 1
    flags = i32([0], gpu)
    out = torch.full_like(q, 7.0)
    store_rotated(cache.dev, q, k, v, i32(tables[:, :width], gpu), i32(starts, gpu), i32(lens, gpu),
                  freq(d).to(gpu), out_q=out, error_flags=flags)
    assert flags.item() == flag
    codes, _ = cache.read()
    if why in ("starts", "short"):
        assert (out[:18] == 7).all()
    else:
        assert not (out[:18] == 7).any()  # its queries have their positions all the same
    mine = [b for b in tables[1] if 0 <= b < codes.shape[0]][:1]
    others = np.setdiff1d(np.arange(codes.shape[0]), mine if why != "table" else [*mine, tables[0, 0]])
    assert np.array_equal(codes[others], cache.codes[others])


def test_odd_values(gpu):
    """An infinity or a NaN in a key makes NaN codes in its head alone and does not enter the scale."""
    rng = np.random.default_rng(6)
    cache, tables, starts, lens, (q, k, v), _, _ = make(
        gpu, rng, [16], [0], 2, 2, 64, 16, "hnd", "fp32", False)
    k[3, 1, 7], k[9, 0, 1], v[5, 0, 2] = float("nan"), float("inf"), float("inf")
    clean = k.clone()
    clean[3, 1], clean[9, 0] = 0, 0
    args = i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), freq(64).to(gpu)
    store_rotated(cache.dev, q, k, v, *args)
    codes, scales = cache.read()
    b = tables[0, 0]
    assert ((codes[b, 3, 1, 0] & 127) == 127).all()
    assert ((codes[b, 9, 0, 0] & 127) == 127).any()
    assert codes[b, 5, 0, 1, 2] == 0x7E
    store_rotated(cache.dev, q, clean, v, *args)
    again, scales2 = cache.read()
    assert np.array_equal(scales, scales2)
    keep = np.ones((16, 2), bool)
    keep[3, 1] = keep[9, 0] = False
    assert np.array_equal(codes[b][keep], again[b][keep])


def test_a_captured_step_replays_with_the_lengths_of_its_day(gpu):
    rng = np.random.default_rng(12)
    heads, d, bs = 2, 128, 16
    tables = i32(rng.permutation(24).reshape(3, 8), gpu)
    cache = Cache(gpu, rng, 24, heads, d, bs)
    twin = Cache(gpu, rng, 24, heads, d, bs)
    for a, b in zip((*cache.planes, cache.dev_scales), (*twin.planes, twin.dev_scales)):
        b.view(torch.uint8).copy_(a.view(torch.uint8))
    starts, lens = i32([0, 1, 2, 3], gpu), i32([16, 40, 5], gpu)
    q, k, v = (torch.randn((5, h, d), dtype=torch.bfloat16, device=gpu) for h in (8, 2, 2))
    inv = freq(d).to(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = store_rotated(cache.dev, q, k, v, tables, starts, lens, inv)
    for step in range(20):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t) * (1 + step % 3))
        graph.replay()
        torch.cuda.synchronize()
        want = store_rotated(twin.dev, q, k, v, tables, starts, lens, inv)
        assert torch.equal(out[:3], want[:3])
        for a, b in zip((*cache.planes, cache.dev_scales), (*twin.planes, twin.dev_scales)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        lens.add_(1)


def test_refusals(gpu):
    rng = np.random.default_rng(1)
    cache, tables, starts, lens, (q, k, v), _, _ = make(
        gpu, rng, [3], [5], 4, 2, 128, 16, "hnd", "bf16", False)
    step = i32(tables, gpu), i32(starts, gpu), i32(lens, gpu)
    inv = inv_freq_for(128, 1e6).to(gpu, torch.float32)

    def refused(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            store_rotated(cache.dev, *args, **kw)

    refused(ValueError, "heads", q, k[:, :1], v, *step, inv)
    refused(ValueError, r"\[3, heads, 128\]", q, k[:2], v, *step, inv)
    refused(TypeError, "of one type", q, k, v.float(), *step, inv)
    refused(ValueError, "not cuda", q.cpu(), k, v, *step, inv)
    refused(ValueError, "starts", q, k, v, step[0], step[1][:1], step[2], inv)
    refused(ValueError, "block_tables", q, k, v, step[0].long(), *step[1:], inv)
    refused(ValueError, "shares memory with k", q, k, v, *step, inv,
            out_q=k.as_strided((3, 4, 128), (256, 0, 1)))
    refused(ValueError, "among the cache's", q, k, v, *step, inv,
            out_q=cache.planes[0].view(torch.bfloat16).flatten()[:3 * 4 * 128].view(3, 4, 128))
    refused(RuntimeError, "backward", q, k.clone().requires_grad_(), v, *step, inv)
    codes, _ = cache.read()
    assert np.array_equal(codes, cache.codes)
