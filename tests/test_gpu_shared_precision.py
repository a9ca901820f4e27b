"""How far attention over a shared prefix may be from 64 bits, by the rows that a request brings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import scaled_plain as plain
from tests.step_plain import LEAST
from tests.test_gpu_attend_shared import Batch, run
from tests.test_gpu_scaled import Cache

pytestmark = pytest.mark.gpu


def within(cache, q, tables, starts, lens, bs, got, p_rounding, requests=None):
    """Whether outputs are within the roundings of the exact ones, entry by entry.

    Of p where it meets V: ``p_rounding`` of each term.  Of a score: fp32 sums of D products and the
    scaling, (D + 4) * 2^-24 of the sum of the products' sizes, which multiplies p; of the
    exponential, the sums, the join and the quotient: 2^-20 in all at these lengths.  Each moves the
    output by at most that share of sum(p |v|), twice with the denominator.  Of the output itself half
    a step, eps / 2 of it."""
    qh, d, scale = q.double().cpu().numpy(), q.shape[2], q.shape[2] ** -0.5
    group = q.shape[1] // cache.codes.shape[2]
    out, half = got.double().cpu().numpy(), torch.finfo(got.dtype).eps / 2
    worst = 0.0
    for r, last in enumerate(lens):
        if requests is not None and r not in requests:
            continue
        x = plain.rows(cache.codes, cache.scales, tables[r], last, bs)
        for t in range(starts[r], starts[r + 1]):
            sees = last - (starts[r + 1] - t) + 1
            for h in range(q.shape[1]):
                k, v = x[:sees, h // group, 0], x[:sees, h // group, 1]
                s = k @ qh[t, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                share = p_rounding + 2.0 ** -20
                share += (d + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(qh[t, h]) * scale).max()
                want, slack = p @ v, 2 * share * (p @ np.abs(v))
                tolerance = slack + half * (np.abs(want) + slack) + LEAST[got.dtype]
                worst = max(worst, (np.abs(out[t, h] - want) / tolerance).max())
    return worst <= 1


def batch_of(gpu, requests, new, heads, group, d, seed, more=()):
    rng = np.random.default_rng(seed)
    batch = Batch(rng, [(512, [(int(n), new) for n in rng.integers(0, 60, requests)] + list(more))], [], 16)
    cache = Cache(gpu, rng, batch.blocks, heads, d, 16, fill="any")
    # values of about one and scores of about a half: p's rounding stands out from the scores'
    cache.codes[:] = plain.encode(rng.standard_normal(cache.codes.shape) * 2.0 ** 4)
    cache.scales[:] = 127 - 4
    x = cache.codes.transpose(0, 2, 1, 3, 4)
    cache.planes[0].view(torch.uint8).copy_(torch.from_numpy(x.reshape(*x.shape[:3], 2 * d).copy()))
    cache.dev_scales.view(torch.uint8).fill_(127 - 4)
    tokens = requests * new + sum(n for _, n in more)
    q = torch.from_numpy(rng.standard_normal((tokens, heads * group, d)) / 2).to(gpu, torch.bfloat16)
    return batch, cache, q


SHAPES = [  # requests, new tokens of each, KV heads, query heads of each, D
    (40, 1, 2, 4, 128),   # a decode step: 160 rows of 4
    (12, 3, 1, 8, 128),   # drafts: 288 rows of 24
    (24, 1, 1, 8, 64),
    (9, 1, 1, 16, 256),
]


@pytest.mark.parametrize("requests,new,heads,group,d", SHAPES)
@pytest.mark.parametrize("known", ["all", "new"])
def test_rows_of_decode_steps_keep_two_terms_of_p(gpu, requests, new, heads, group, d, known):
    """At most 32 rows a request: 2^-17 of p over both ranges, however many rows share."""
    batch, cache, q = batch_of(gpu, requests, new, heads, group, d, requests + d)
    kw = dict(max_new=new)
    if known == "all":
        kw.update(max_shared=512, max_own=60 + new)
    got = run(gpu, batch, cache, q, **kw)
    assert within(cache, q, batch.tables, batch.starts, batch.lens, 16, got, 2.0 ** -17)


@pytest.mark.parametrize("requests,new,heads,group,d", SHAPES)
def test_without_hints_p_may_be_one_term(gpu, requests, new, heads, group, d):
    """The tokens count for one request's: half a step of bf16, 2^-8, of p."""
    batch, cache, q = batch_of(gpu, requests, new, heads, group, d, requests + d)
    got = run(gpu, batch, cache, q)
    assert within(cache, q, batch.tables, batch.starts, batch.lens, 16, got, 2.0 ** -8)


@pytest.mark.parametrize("group,d", [(16, 128), (16, 64), (8, 256)])
def test_decoding_requests_beside_a_long_chunk_keep_them_too(gpu, group, d):
    """2,048 rows and more beside requests of up to 16: these have a launch of their own over their own
    tokens, as in attend_scaled, and lose nothing over what is shared."""
    chunk = 2048 // group
    batch, cache, q = batch_of(gpu, 5, 1, 1, group, d, group + d, more=[(9, chunk)])
    got = run(gpu, batch, cache, q, max_new=chunk, max_shared=512)
    args = cache, q, batch.tables, batch.starts, batch.lens, 16, got
    assert within(*args, 2.0 ** -17, requests=range(5))
    assert within(*args, 2.0 ** -8, requests=[5])
