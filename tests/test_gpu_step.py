"""A step's operators together, as a serving loop calls them, and each through both of its paths."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import (
    ScaledCache,
    ScaledShifts,
    attend_scaled,
    attend_shared,
    norm_rotate,
    scaled_step,
    step_slots,
    store_rotated,
    store_scaled,
)
from marathon_amd import _lib
from tests.step_plain import check_turned, turned
from tests.test_gpu_attend_shared import Batch, case, run
from tests.test_gpu_norm_rotate import freq
from tests.test_gpu_scaled import Cache, i32

pytestmark = pytest.mark.gpu


def fresh_cache(gpu, blocks, heads, d, bs=16):
    kv = torch.zeros((blocks, heads, bs, 2 * d), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    scales = torch.zeros((blocks, heads, 2), dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu)
    return ScaledCache(kv, scales, "hnd", bs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_serving_loop_over_a_shared_prompt(gpu, dtype):
    """One request fills a prompt's blocks, others begin with them: slots, projections into the cache
    and attention, step after step, next to the calls that these stand for, on caches of their own."""
    heads, group, d, bs, prompt, n = 2, 4, 128, 16, 80, 5
    inv = freq(d).to(gpu)
    g = torch.Generator(device=gpu).manual_seed(3)
    weight = 1 + 0.2 * torch.randn(d, generator=g, device=gpu)
    weight = weight.to(dtype)
    a, b = fresh_cache(gpu, 64, heads, d), fresh_cache(gpu, 64, heads, d)

    def projection(tokens):
        x = torch.randn((tokens, heads * (group + 2), d), generator=g, device=gpu).to(dtype)
        return x.split((heads * group, heads, heads), 1)

    def both(q, k, v, tables, step, positions, groups, shared, **hints):
        """The step on cache a, and the separate calls on cache b."""
        out_q = store_rotated(a, q, k, v, tables, step.starts, step.lens, inv, q_weight=weight,
                              k_weight=weight)
        got = attend_shared(a, out_q, tables, step.starts, step.lens, groups, shared, **hints)
        turned_q, _ = norm_rotate(q, k, positions, inv, q_weight=weight, k_weight=weight)
        _, turned_k = norm_rotate(q.float(), k.float(), positions, inv, q_weight=weight, k_weight=weight)
        store_scaled(b, turned_k, v.float(), tables, step.starts, step.lens)
        want = attend_scaled(b, turned_q, tables, step.starts, step.lens)
        total = int(step.starts[-1])
        assert torch.equal(out_q[:total], turned_q[:total])
        # each within p's rounding (2^-8 of it where bf16 queries meet more than 32 rows), in steps
        # of the output: values of about one, of which a row averages some
        off = (got[:total].float() - want[:total].float()).abs()
        assert off.max() <= (2.0 ** -5 if dtype == torch.bfloat16 else 2.0 ** -9)
        assert torch.equal(a.kv.view(torch.uint8), b.kv.view(torch.uint8))
        assert torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))
        return got

    free = torch.randperm(64, generator=g, device=gpu).to(torch.int32)
    none = i32([0], gpu), i32([], gpu)
    tables = torch.zeros((n, 12), dtype=torch.int32, device=gpu)
    first = step_slots(i32([0], gpu), i32([prompt], gpu), tables[:1], free, i32([0], gpu), bs, prompt + 3)
    q, k, v = projection(prompt + 3)  # (three rows of padding)
    both(q, k, v, tables[:1], first, first.positions, *none)
    # all begin with the prompt's whole blocks; what stands behind them each computes for itself
    whole = prompt // bs * bs
    tables[1:, :whole // bs] = tables[0, :whole // bs]
    held, at = i32([prompt] + [whole] * (n - 1), gpu), first.free_at
    groups, shared = i32([0, n], gpu), i32([whole], gpu)
    flags = i32([0], gpu)
    for new in ([1, 7, 20, 1, 0], [1] * n, [1] * n, [3, 1, 1, 2, 40], [1] * n):
        step = step_slots(held, i32(new, gpu), tables, free, at, bs, sum(new) + 2, error_flags=flags)
        q, k, v = projection(sum(new) + 2)
        both(q, k, v, tables, step, step.positions, groups, shared, max_new=max(new), max_shared=whole)
        held, at = step.lens, step.free_at
    assert flags.item() == 0


def test_keys_turned_here_are_the_ones_that_a_shift_moves(gpu):
    """Rows stored at their positions and shifted by delta are the rows stored at the shifted ones, within
    the codes' rounding."""
    heads, d, n, delta = 2, 128, 64, 208
    inv = freq(d)
    a, b, c = (fresh_cache(gpu, 24, heads, d) for _ in range(3))
    q, k, v = (torch.randn((n, heads, d), device=gpu) for _ in range(3))
    table = torch.arange(24, dtype=torch.int32, device=gpu)[None]
    step = i32([0, n], gpu), i32([n], gpu)
    store_rotated(a, q, k, v, table, *step, inv.to(gpu), eps=None)
    store_rotated(b, q, k, v, table, step[0], i32([n + delta], gpu), inv.to(gpu), eps=None)
    ScaledShifts([a], [c], inv).run([(0, delta, 0, 0, n, delta, 0, 0)], np.arange(24, dtype=np.int32),
                                    np.arange(24, dtype=np.int32))

    def values(cache):
        x = cache.kv.view(torch.uint8)[13:17].view(torch.float8_e4m3fn).double().unflatten(-1, (2, d))
        return x * cache.scales.view(torch.uint8)[13:17].view(torch.float8_e8m0fnu).double()[:, :, None, :, None]

    want, got = values(b), values(c)
    assert torch.equal(want[..., 1, :], got[..., 1, :])  # V's codes
    # K was rounded to e4m3 before it was turned, each value of a pair by 2^-4 of itself, and again behind
    pair = want[..., 0, :].abs()
    size = pair + pair.roll(d // 2, -1)
    assert ((want - got)[..., 0, :].abs() <= 3 * 2.0 ** -4 * size + 2.0 ** -6).all()


class Counted:
    """The binding's calls, whose answers are kept."""

    def __init__(self):
        self.got = []

    def __getattr__(self, name):
        call = getattr(_lib.binding(), name)

        def counted(*args):
            self.got.append(call(*args))
            return self.got[-1]
        return counted


class Nothing:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.parametrize("pt", [torch.int32, torch.int64])
@pytest.mark.parametrize("weighted", [True, False])
def test_both_paths_do_the_same(gpu, pt, weighted, monkeypatch):
    rng = np.random.default_rng(17)
    batch = Batch(rng, [(96, [(3, 2), (20, 1)])], [(7, 1)], 16)
    q, k, v = (torch.randn((4, h, 128), device=gpu, dtype=torch.bfloat16) for h in (8, 2, 2))
    w = torch.randn(128, device=gpu, dtype=torch.bfloat16) if weighted else None
    inv, pos = freq(64).to(gpu), torch.arange(4, device=gpu, dtype=pt)
    tables, starts, lens = i32(batch.tables, gpu), i32(batch.starts, gpu), i32(batch.lens, gpu)
    outs = []
    for usual in (Counted(), Nothing()):
        monkeypatch.setattr(scaled_step, "_usual", usual)
        cache = Cache(gpu, np.random.default_rng(1), batch.blocks, 2, 128, 16)
        kw = dict(q_weight=w, k_weight=w)
        x, y = q.clone(), k.clone()
        got = [*norm_rotate(q, k, pos, inv, **kw), *norm_rotate(x, y, pos, inv, out_q=x, out_k=y, eps=None),
               store_rotated(cache.dev, q, k, v, tables, starts, lens, inv, **kw),
               run(gpu, batch, cache, q, max_new=2, softmax_scale=0.1),
               run(gpu, batch, cache, q, torch.empty_like(q), i32([0], gpu)),
               cache.planes[0].view(torch.uint8), cache.dev_scales.view(torch.uint8)]
        outs.append(got)
        if isinstance(usual, Counted):
            assert len(usual.got) == 5 and all(x is not None for x in usual.got)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_more_rows_than_four_waves_each_join(gpu):
    rng = np.random.default_rng(44)
    case(gpu, rng, [(64, [(3, 250), (0, 1), (9, 130)])], [(20, 140)], 1, 16, 64, 16, "hnd", "bf16")


def test_rows_further_apart_than_32_bits(gpu):
    """Token strides that put the last rows beyond 4 GiB."""
    stride = (1 << 30) + 64
    big = torch.empty(2 * stride + 4096, dtype=torch.bfloat16, device=gpu)
    q = big.as_strided((3, 4, 64), (stride, 64, 1))
    x = torch.randn((3, 4, 64), device=gpu).to(torch.bfloat16)
    q.copy_(x)
    pos, inv = torch.arange(3, dtype=torch.int32, device=gpu), freq(64)
    out, _ = norm_rotate(q, x.clone(), pos, inv.to(gpu), out_q=q)
    check_turned(out, *turned(x.double().cpu().numpy(), None, np.arange(3), inv.numpy(), 1e-6))
    q.copy_(x)
    cache = fresh_cache(gpu, 4, 4, 64)
    args = i32([[0, 1]], gpu), i32([0, 3], gpu), i32([20], gpu), inv.to(gpu)
    far = store_rotated(cache, q, q, q, *args)
    codes = cache.kv.view(torch.uint8).clone()
    near = store_rotated(cache, x, x, x, *args)
    assert torch.equal(far, near) and torch.equal(codes, cache.kv.view(torch.uint8))


def test_a_cache_beyond_4_gib(gpu):
    """Blocks whose offsets pass 32 bits, shared and own."""
    heads, d, bs = 8, 256, 16
    blocks = (4 << 30) // (heads * bs * 2 * d) + 64
    kv = torch.zeros((blocks, heads, bs, 2 * d), dtype=torch.uint8, device=gpu)
    scales = torch.full((blocks, heads, 2), 127, dtype=torch.uint8, device=gpu)
    kv[-40:] = torch.randint(0, 0x50, (40, heads, bs, 2 * d), device=gpu, dtype=torch.uint8)
    kv[:40], scales[:40] = kv[-40:], scales[-40:]
    cache = ScaledCache(kv.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), "hnd", bs)
    q = torch.randn((2, heads, d), device=gpu, dtype=torch.bfloat16)
    near = torch.tensor([list(range(12)), list(range(10)) + [12, 13]], dtype=torch.int32, device=gpu)
    args = i32([0, 1, 2], gpu), i32([180, 190], gpu), i32([0, 2], gpu), i32([160], gpu)
    got = [attend_shared(cache, q, t, *args) for t in (near, near + blocks - 40)]
    assert torch.equal(*got)


@pytest.mark.parametrize("qh,kh,d,rotary", [(5, 1, 128, 128), (10, 3, 128, 32), (3, 7, 64, 64), (40, 8, 64, 32),
                                            (1, 1, 64, 64), (5, 2, 256, 256), (1, 3, 256, 64)])
def test_a_large_call_does_what_small_ones_do(gpu, qh, kh, d, rotary):
    """Bit for bit: waves that take several tokens and rounds, against those that take one, and the
    queries of requests whose ends lie within a wave's tokens, beside rows of nobody."""
    rng = np.random.default_rng(qh * d + kh)
    n = 8192 * (1024 // d) // qh + 13
    q, k, v = (torch.randn((n, h, d), device=gpu).to(torch.bfloat16) for h in (qh, kh, kh))
    w = torch.randn(d, device=gpu, dtype=torch.bfloat16)
    inv = freq(rotary).to(gpu)
    new = rng.integers(0, 2 * n // 300, 300)
    new[rng.integers(0, 300, 60)] = 1
    starts = 5 + np.concatenate(([0], np.cumsum(new)))
    assert starts[-1] > n // 2
    new, starts = np.diff(np.minimum(starts, n - 3)), np.minimum(starts, n - 3)
    held = rng.integers(0, 40, 300)
    lens = held + new
    at = np.zeros(n, np.int64)
    for r in range(300):
        at[starts[r]:starts[r + 1]] = held[r] + np.arange(new[r])
    positions = i32(at, gpu)
    all_q, all_k = norm_rotate(q, k, positions, inv, q_weight=w, k_weight=w)
    for first in range(0, n, 997):
        part = slice(first, first + 997)
        some = norm_rotate(q[part], k[part], positions[part], inv, q_weight=w, k_weight=w)
        assert torch.equal(some[0], all_q[part]) and torch.equal(some[1], all_k[part])
    need = -(-lens // 16)
    tables = np.zeros((300, need.max()), np.int32)
    for r, b in enumerate(np.cumsum(need) - need):
        tables[r, :need[r]] = b + np.arange(need[r])
    cache = fresh_cache(gpu, int(need.sum()) + 1, kh, d)
    out = torch.full_like(q, 77.0)
    store_rotated(cache, q, k, v, i32(tables, gpu), i32(starts, gpu), i32(lens, gpu), inv, q_weight=w,
                  k_weight=w, out_q=out)
    a, b = int(starts[0]), int(starts[-1])
    assert torch.equal(out[a:b], all_q[a:b])
    assert (out[:a] == 77.0).all() and (out[b:] == 77.0).all()


def test_outputs_beyond_the_caches_are_the_same(gpu):
    """Bit for bit: outputs that are streamed (150 MiB and more), in place and not, against small calls."""
    n, qh, kh, d = 15500, 40, 8, 128
    q, k, v = (torch.randn((n, h, d), device=gpu).to(torch.bfloat16) for h in (qh, kh, kh))
    inv = freq(d).to(gpu)
    positions = torch.arange(n, dtype=torch.int32, device=gpu) + 3
    all_q, all_k = norm_rotate(q, k, positions, inv)
    for first in range(0, n, 499):
        part = slice(first, first + 499)
        some = norm_rotate(q[part], k[part], positions[part], inv)
        assert torch.equal(some[0], all_q[part]) and torch.equal(some[1], all_k[part])
    cache = fresh_cache(gpu, n // 16 + 2, kh, d)
    table = torch.arange(n // 16 + 2, dtype=torch.int32, device=gpu)[None]
    into = store_rotated(cache, q, k, v, table, i32([0, n], gpu), i32([n + 3], gpu), inv)
    assert torch.equal(into, all_q)
    norm_rotate(q, k, positions, inv, out_q=q, out_k=k)
    assert torch.equal(q, all_q) and torch.equal(k, all_k)
