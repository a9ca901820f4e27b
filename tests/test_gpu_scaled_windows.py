"""Attention whose parts are longer than one lookup of block ids and scales (1,024 tokens in the
kernel of many rows, 8,192 in that of few), and more tiles than run at once: against the
softmax in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import ScaledCache, attend_scaled
from tests import scaled_plain as plain
from tests.test_gpu_scaled import DTYPES, Cache, i32

pytestmark = pytest.mark.gpu


def random_cache(gpu, rng, lengths, heads, d, bs, layout):
    """A cache of codes of every kind but NaN, its shuffled tables, and each request's rows in
    64 bits, [tokens, heads, 2, D]."""
    need = [-(-n // bs) for n in lengths]
    blocks = sum(need) + 3
    codes = torch.from_numpy(rng.integers(0, 0x68, (blocks, bs, heads, 2 * d), np.uint8)).to(gpu)
    codes |= torch.from_numpy(rng.integers(0, 2, codes.shape, np.uint8)).to(gpu) << 7
    scales = torch.from_numpy(rng.integers(120, 125, (blocks, heads, 2), np.uint8)).to(gpu)
    kv = codes if layout == "nhd" else codes.transpose(1, 2).contiguous()
    cache = ScaledCache(kv.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), layout, bs)
    ids = rng.permutation(blocks).astype(np.int32)
    tables = np.full((len(lengths), max(need)), 2**31 - 1, np.int32)
    rows, at = [], 0
    for r, n in enumerate(need):
        mine = tables[r, :n] = ids[at:at + n]
        at += n
        mine = torch.from_numpy(mine.astype(np.int64)).to(gpu)
        x = codes[mine].view(torch.float8_e4m3fn).double().reshape(n * bs, heads, 2, d)
        s = torch.exp2(scales[mine].double() - 127).repeat_interleave(bs, 0)
        rows.append((x * s[..., None])[:lengths[r]])
    return cache, i32(tables, gpu), rows


def check(got, q, rows, new, dtype, whole_p=False):
    """Each entry within the roundings that the definition of the operator allows: of the output
    half a step; of p, in the sum over V alone, half a step of bf16, 2^-8 of each term (2^-17
    where two terms hold it: for fp16, or ``whole_p``); of exponential, sums and quotient 2^-20;
    of a score (D + 4) * 2^-24 of the sizes of its products, a share of p in the sums above and
    below."""
    d, at = q.shape[2], 0
    eps = torch.finfo(dtype).eps / 2
    for x, n in zip(rows, new):
        heads = x.shape[1]
        group = q.shape[1] // heads
        sees = len(x) - n + 1 + torch.arange(n, device=q.device)
        mask = torch.arange(len(x), device=q.device)[None] >= sees[:, None]
        for h in range(q.shape[1]):
            k, v = x[:, h // group, 0].contiguous(), x[:, h // group, 1].contiguous()
            qh = q[at:at + n, h].double()
            p = torch.softmax((qh @ k.T * d ** -0.5).masked_fill(mask, -torch.inf), 1)
            size = (qh.abs() @ k.T.abs() * d ** -0.5).masked_fill(mask, 0.0).amax(1, keepdim=True)
            want = p @ v
            rounded = 2.0 ** -8 if dtype == torch.bfloat16 and not whole_p else 2.0 ** -17
            share = 2 * (2.0 ** -20 + (d + 4) * 2.0 ** -24 * size) + rounded
            tol = share * (p @ v.abs())
            tol = tol + eps * (want.abs() + tol) + 1e-30
            off = (got[at:at + n, h].double() - want).abs()
            assert (off <= tol).all(), (h, float((off / tol).max()))
        at += n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,new,heads,group,d,bs,layout", [
    ([20011, 8192, 8193], [1, 1, 1], 2, 4, 128, 16, "hnd"),  # 16 rows a tile, three lookups
    ([16385, 40], [4, 3], 1, 8, 64, 64, "nhd"),              # 32
    ([9001], [1], 1, 16, 256, 32, "hnd"),
])
def test_few_rows_look_up_again(gpu, lengths, new, heads, group, d, bs, layout, dtype):
    """A short ``max_len`` leaves a request one part."""
    rng = np.random.default_rng(sum(lengths) + d)
    cache, tables, rows = random_cache(gpu, rng, lengths, heads, d, bs, layout)
    q = torch.randn(sum(new), heads * group, d, device=gpu).to(DTYPES[dtype])
    got = attend_scaled(cache, q, tables, i32(np.cumsum([0] + new), gpu), i32(lengths, gpu),
                        max_new=max(new), max_len=16)
    check(got, q, rows, new, q.dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,new,heads,group,d,bs,layout", [
    ([5003, 1024, 1025], [40, 30, 33], 2, 4, 128, 16, "hnd"),
    ([2113, 3000], [300, 1], 1, 2, 64, 128, "nhd"),
    ([2500], [70], 1, 4, 256, 32, "hnd"),
])
def test_many_rows_look_up_again(gpu, lengths, new, heads, group, d, bs, layout, dtype):
    rng = np.random.default_rng(sum(lengths) + d)
    cache, tables, rows = random_cache(gpu, rng, lengths, heads, d, bs, layout)
    q = torch.randn(sum(new), heads * group, d, device=gpu).to(DTYPES[dtype])
    got = attend_scaled(cache, q, tables, i32(np.cumsum([0] + new), gpu), i32(lengths, gpu),
                        max_new=max(new), max_len=16)
    check(got, q, rows, new, q.dtype)


@pytest.mark.parametrize("lengths,new,heads,group,d,dtype", [
    ([5001], [2100], 8, 4, 64, "bf16"),             # 528 tiles of one request
    ([3007, 2500, 1900], [900, 1100, 700], 4, 6, 128, "bf16"),
    ([2600, 1500], [1000, 1300], 4, 8, 64, "fp16"),
    ([4100], [1100], 4, 8, 256, "bf16"),            # 276
])
def test_more_tiles_than_run_at_once(gpu, lengths, new, heads, group, d, dtype):
    rng = np.random.default_rng(sum(lengths) + d)
    cache, tables, rows = random_cache(gpu, rng, lengths, heads, d, 16, "hnd")
    q = torch.randn(sum(new), heads * group, d, device=gpu).to(DTYPES[dtype])
    got = attend_scaled(cache, q, tables, i32(np.cumsum([0] + new), gpu), i32(lengths, gpu),
                        max_new=max(new))
    check(got, q, rows, new, q.dtype)


def test_a_row_that_sees_one_token_is_its_value(gpu):
    """Of two new rows whose request holds one token, the first stands before it and is zeros,
    the second is V, which its rounding keeps: a code times a power of two."""
    rng = np.random.default_rng(9)
    cache = Cache(gpu, rng, 4, 2, 128, 16)
    q = torch.randn(2, 4, 128, device=gpu, dtype=torch.bfloat16)
    out = attend_scaled(cache.dev, q, i32([[1, 2]], gpu), i32([0, 2], gpu), i32([1], gpu))
    want = plain.rows(cache.codes, cache.scales, [1], 1, 16)[0, :, 1]
    assert (out[0] == 0).all()
    assert np.array_equal(out[1].double().cpu().numpy(), np.repeat(want, 2, 0))


@pytest.mark.parametrize("tokens,new,lengths,most", [
    (6000, [1], [20000], 1),             # a padded array
    (6000, [1, 2], [9000, 40], 1),       # and a hint that is too small
    (3000, [2900, 1], [2900, 4000], 1),  # a wrong hint
])
def test_a_small_hint_for_a_large_array(gpu, tokens, new, lengths, most):
    rng = np.random.default_rng(tokens + len(new))
    cache, tables, rows = random_cache(gpu, rng, lengths, 4, 64, 16, "hnd")
    tables = torch.nn.functional.pad(tables, (0, 3000), value=-1)
    q = torch.randn(tokens, 16, 64, device=gpu, dtype=torch.bfloat16)
    out = torch.full_like(q, 3.0)
    attend_scaled(cache, q, tables, i32(np.cumsum([0] + new), gpu), i32(lengths, gpu), out=out,
                  max_new=most)
    check(out, q, rows, new, q.dtype)
    assert (out[sum(new):] == 3.0).all()


@pytest.mark.parametrize("most", [2**31 - 1, 2**31, 2**32 + 1, 2**40])
def test_hints_of_any_size(gpu, most):
    rng = np.random.default_rng(5)
    cache, tables, rows = random_cache(gpu, rng, [300], 2, 64, 16, "hnd")
    q = torch.randn(2, 8, 64, device=gpu, dtype=torch.bfloat16)
    step = tables, i32([0, 2], gpu), i32([300], gpu)
    check(attend_scaled(cache, q, *step, max_new=most, max_len=most), q, rows, [2], q.dtype)
    with pytest.raises(Exception, match="max_len"):
        attend_scaled(cache, q, *step, max_len=-most)


@pytest.mark.parametrize("lengths,new,heads,group,d", [
    ([5000, 700, 17], [1, 1, 1], 2, 4, 128), ([3000, 90], [2, 1], 1, 8, 64), ([2000], [1], 2, 16, 256),
    ([4000, 33], [4, 1], 2, 8, 128), ([1500], [8], 1, 4, 256)])
def test_few_rows_keep_their_probabilities(gpu, lengths, new, heads, group, d):
    """Up to 32 rows: p in two bf16 terms for bf16 queries too."""
    rng = np.random.default_rng(sum(lengths) + d)
    cache, tables, rows = random_cache(gpu, rng, lengths, heads, d, 16, "hnd")
    q = torch.randn(sum(new), heads * group, d, device=gpu).to(torch.bfloat16)
    got = attend_scaled(cache, q, tables, i32(np.cumsum([0] + new), gpu), i32(lengths, gpu),
                        max_new=max(new))
    check(got, q, rows, new, q.dtype, whole_p=True)
