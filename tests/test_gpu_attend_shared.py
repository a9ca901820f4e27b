"""Attention of requests that begin, in groups, with the same tokens: against the definition in
64 bits, and against each request's own attention."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from marathon_amd import _lib, attend_scaled, attend_shared
from tests import scaled_plain as plain
from tests.step_plain import LEAST
from tests.test_gpu_scaled import DTYPES, Cache, i32
from tests.test_gpu_scaled import bound_of as bound_of_normal

pytestmark = pytest.mark.gpu


def bound_of(*args):
    """As for each request alone, and half the smallest step of the output's type: an fp16 output
    below 2^-14 is a multiple of 2^-24, off by up to 2^-25 whatever its size."""
    return bound_of_normal(*args) + LEAST[args[-1]]


class Batch:
    """Requests in groups: [(shared, [(own, new), ...]), ...], and ``alone`` [(held, new), ...] in no
    group.  ``tables`` are whole; ``given`` has ids out of range wherever no entry may be read."""

    def __init__(self, rng, groups, alone, bs, gap=1):
        self.shared = [s for s, _ in groups]
        self.groups = np.cumsum([0] + [len(r) for _, r in groups])
        self.new = [n for _, rs in groups for _, n in rs] + [n for _, n in alone]
        self.held = [s + own for s, rs in groups for own, _ in rs] + [h for h, _ in alone]
        self.lens = [h + n for h, n in zip(self.held, self.new)]
        self.starts = np.cumsum([0] + self.new)
        need = [-(-n // bs) for n in self.lens]
        width = max(max(need, default=0), 1) + gap
        self.tables = np.full((len(need), width), -7, np.int64)
        at = r = 0
        for s, rs in groups:
            common = np.arange(at, at + s // bs)
            at += s // bs
            for i in range(len(rs)):
                mine = max(need[r] - s // bs, 0)
                self.tables[r, :s // bs] = common
                self.tables[r, s // bs:s // bs + mine] = np.arange(at, at + mine)
                at += mine
                r += 1
        for r in range(r, len(need)):
            self.tables[r, :need[r]] = np.arange(at, at + need[r])
            at += need[r]
        self.blocks = at + 3
        ids = rng.permutation(self.blocks)
        self.tables = np.where(self.tables >= 0, ids[np.maximum(self.tables, 0)], 2**31 - 1).astype(np.int32)
        self.given = self.tables.copy()
        for g, (s, rs) in enumerate(groups):
            self.given[self.groups[g] + 1:self.groups[g + 1], :s // bs] = 2**31 - 1


def run(gpu, batch, cache, q, out=None, flags=None, **kw):
    return attend_shared(cache.dev, q, i32(batch.given, gpu), i32(batch.starts, gpu), i32(batch.lens, gpu),
                         i32(batch.groups, gpu), i32(batch.shared, gpu), out=out, error_flags=flags, **kw)


CASES = [  # groups, alone, heads, query heads of each, D, bs, layout, dtype
    ([(16, [(0, 1)])], [], 1, 1, 64, 16, "hnd", "bf16"),
    ([(160, [(0, 1), (5, 1), (40, 1)])], [], 2, 4, 128, 16, "hnd", "bf16"),
    ([(700, [(3, 1)] * 5), (40, [(9, 1), (0, 1)])], [(33, 1), (0, 1)], 2, 5, 128, 16, "nhd", "bf16"),
    # the shared tokens end inside a block: its rows are read from each request's own
    ([(75, [(0, 1), (5, 2)]), (15, [(9, 1), (70, 3)])], [], 1, 8, 64, 16, "hnd", "fp16"),
    ([(256, [(1, 2), (90, 5), (0, 1)])], [(3, 4)], 2, 2, 256, 64, "hnd", "bf16"),
    ([(300, [(17, 1)] * 20)], [], 1, 7, 128, 32, "nhd", "fp16"),   # 140 rows: two tiles
    ([(512, [(30, 40), (2, 33), (0, 1)])], [(100, 7)], 1, 3, 128, 128, "hnd", "bf16"),
    ([(200, [(8, 60), (0, 3)]), (64, [(1, 130)])], [], 1, 2, 256, 16, "nhd", "fp16"),
    # a long chunk beside decoding requests: a launch of its own over the own tokens
    ([(160, [(700, 1), (3, 300), (15, 2)]), (0, [(50, 1), (8, 0)])], [(90, 2), (0, 1)], 2, 8, 128, 16,
     "hnd", "bf16"),
    ([(1700, [(9, 1)] * 9)], [], 1, 2, 64, 16, "nhd", "fp16"),  # 18 rows in parts
    ([(2100, [(700, 1), (0, 1)])], [], 1, 40, 128, 16, "hnd", "bf16"),
    # no new tokens in a group, a group of no requests
    ([(48, [(9, 0), (5, 0)]), (32, []), (32, [(1, 1)])], [], 1, 4, 64, 16, "hnd", "bf16"),
]


def case(gpu, rng, groups, alone, heads, group, d, bs, layout, dtype, scale=None, loud=1.0, **kw):
    batch = Batch(rng, groups, alone, bs)
    cache = Cache(gpu, rng, batch.blocks, heads, d, bs, layout, split=d == 256)
    raw = [p.view(torch.uint8) for p in cache.planes]
    for r, n in enumerate(batch.lens):  # rows behind a request's last one hold NaNs, on the GPU alone
        if n % bs:
            b = int(batch.tables[r, n // bs])
            for p in raw:
                (p[b, n % bs:] if layout == "nhd" else p[b, :, n % bs:]).fill_(0x7F)
    total, pad = int(batch.starts[-1]), 2
    q = torch.from_numpy(rng.standard_normal((total + pad, heads * group, d)) * loud).to(gpu, DTYPES[dtype])
    out, flags = torch.full_like(q, 77.0), i32([0], gpu)
    got = run(gpu, batch, cache, q, out, flags, softmax_scale=scale, **kw)
    assert got is out and flags.item() == 0
    assert (out[total:] == 77.0).all()
    qh, s = q.double().cpu().numpy(), scale or d ** -0.5
    want = plain.attend(cache.codes, cache.scales, qh, batch.tables, batch.starts, batch.lens, bs, s)[:total]
    tol = bound_of(cache, qh, batch.tables, batch.starts, batch.lens, bs, s, want, q.dtype)
    off = np.abs(out.double().cpu().numpy()[:total] - want)
    assert (off <= tol).all(), float((off / tol).max())
    return batch, cache, q, out


@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("groups,alone,heads,group,d,bs,layout,dtype", CASES)
def test_matches_the_plain_one(gpu, groups, alone, heads, group, d, bs, layout, dtype, known):
    rng = np.random.default_rng(len(groups) * 100 + d + bs + group)
    kw = {}
    if known:
        own = [(o, n) for _, rs in groups for o, n in rs]
        kw = dict(max_new=max(n for _, n in [*own, *alone]), max_shared=max(s for s, _ in groups),
                  max_own=max([o + n + bs for o, n in own] + [h + n for h, n in alone]))
    case(gpu, rng, groups, alone, heads, group, d, bs, layout, dtype, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_sharp_scores(gpu, dtype):
    """Scores that spread over hundreds: the running largest moves often, in either range."""
    rng = np.random.default_rng(4)
    case(gpu, rng, [(900, [(200, 1), (3, 30)])], [], 2, 4, 128, 16, "hnd", dtype, loud=4.0)


def test_hints_change_nothing_but_the_order(gpu):
    rng = np.random.default_rng(6)
    case(gpu, rng, [(2000, [(10, 1), (500, 50)])], [(40, 3)], 1, 4, 128, 16, "hnd", "bf16", max_new=1,
         max_shared=16, max_own=16)


def test_rows_that_stand_inside_what_is_shared(gpu):
    """A request that computes a part of its group's tokens again sees those before its own; one
    whose rows all stand there has nothing of its own; rows before position 0 see nothing."""
    rng = np.random.default_rng(9)
    batch = Batch(rng, [(320, [(0, 1), (0, 40), (0, 100), (0, 9)])], [], 16)
    batch.lens[1] = 330   # its first rows stand inside
    batch.lens[2] = 200   # all of them
    batch.lens[3] = 5     # and before position 0
    for heads, group, d, dtype in ((1, 2, 128, "bf16"), (2, 1, 64, "fp16")):
        cache = Cache(gpu, rng, batch.blocks, heads, d, 16)
        q = torch.from_numpy(rng.standard_normal((150, heads * group, d))).to(gpu, DTYPES[dtype])
        out = run(gpu, batch, cache, q)
        qh = q.double().cpu().numpy()
        want = plain.attend(cache.codes, cache.scales, qh, batch.tables, batch.starts, batch.lens, 16, d ** -0.5)
        tol = bound_of(cache, qh, batch.tables, batch.starts, batch.lens, 16, d ** -0.5, want, q.dtype)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
        assert (out[141:145] == 0).all()


def test_without_groups_and_with_groups_that_share_nothing(gpu):
    rng = np.random.default_rng(2)
    batch = Batch(rng, [], [(40, 1), (700, 3), (0, 50)], 16)
    cache = Cache(gpu, rng, batch.blocks, 2, 64, 16)
    q = torch.randn(54, 6, 64, device=gpu, dtype=torch.float16)
    args = i32(batch.tables, gpu), i32(batch.starts, gpu), i32(batch.lens, gpu)
    none = attend_shared(cache.dev, q, *args, i32([0], gpu), i32([], gpu))
    zero = attend_shared(cache.dev, q, *args, i32([0, 2, 3], gpu), i32([0, 15], gpu))
    assert torch.equal(none, zero)
    want = attend_scaled(cache.dev, q, *args)
    # One sum in two orders, each rounded to fp16 once: where a tie lies between them, a step apart.
    # A value in [2^e, 2^(e+1)) has steps of 2^(e-10), at most 2^-10 of itself (2^-7 from 8 on, which
    # rows that see few tokens reach: an absolute 2^-8 is too little there); subnormals of 2^-24.
    apart = (none.double() - want.double()).abs()
    assert (apart <= 2.0 ** -10 * torch.maximum(none.abs(), want.abs()).double() + 2.0 ** -24).all()


@pytest.mark.parametrize("n,group,d", [(1, 4, 128), (40, 4, 128), (40, 1, 64), (6, 8, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_nan_reaches_only_the_rows_that_see_it(gpu, n, group, d, dtype):
    """In V of a shared token: every row of the group.  Of an own token: its request alone."""
    rng = np.random.default_rng(d + n)
    batch = Batch(rng, [(80, [(9, 1)] * n)], [(90, 1)], 16)
    cache = Cache(gpu, rng, batch.blocks, 1, d, 16)
    q = torch.randn(n + 1, group, d, device=gpu).to(DTYPES[dtype])
    clean = run(gpu, batch, cache, q)
    raw = cache.planes[0].view(torch.uint8)
    own = int(batch.tables[0, 5])
    raw[own, 0, 3, 2 * d - 3] = 0x7F
    got = run(gpu, batch, cache, q)
    assert torch.equal(got[1:], clean[1:]) and got[0, :, d - 3].isnan().all()
    keep = [i for i in range(d) if i != d - 3]
    assert torch.equal(got[0][:, keep], clean[0][:, keep])
    raw[int(batch.tables[0, 2]), 0, 7, 2 * d - 5] = 0xFF
    got = run(gpu, batch, cache, q)
    assert got[:n, :, d - 5].isnan().all() and torch.equal(got[n], clean[n])
    raw[int(batch.tables[0, 1]), 0, 0, 4] = 0x7F  # and K: whole scores
    got = run(gpu, batch, cache, q)
    assert got[:n].isnan().all() and torch.equal(got[n], clean[n])


@pytest.mark.parametrize("why", ["order", "behind", "before", "negative", "room", "id", "starts"])
def test_what_does_not_fit_is_flagged_and_harms_nobody_else(gpu, why):
    rng = np.random.default_rng(5)
    batch = Batch(rng, [(64, [(5, 1), (9, 1)]), (48, [(3, 2), (70, 1)])], [(20, 1)], 16)
    cache = Cache(gpu, rng, batch.blocks, 1, 64, 16)
    q = torch.randn(6, 2, 64, device=gpu, dtype=torch.bfloat16)
    batch.given = batch.tables.copy()
    clean = run(gpu, batch, cache, q)
    flag, good = _lib.MKV_FLAG_SPAN, [0, 1, 5]
    if why == "order":
        batch.groups = np.array([0, 4, 2])
        good = [5]
    elif why == "behind":
        batch.groups = np.array([0, 2, 9])
    elif why == "before":
        batch.groups = np.array([-1, 2, 4])
        good = [2, 3, 4, 5]
    elif why == "negative":
        batch.shared[1] = -5
    elif why == "room":
        batch.shared[1] = 10**6
        flag, good = _lib.MKV_FLAG_SRC_RANGE, [0, 1, 5]
    elif why == "id":
        batch.given[2, 1] = batch.blocks
        flag = _lib.MKV_FLAG_SRC_RANGE
    else:
        batch.starts = np.array([0, 1, 2, 9, 5, 6])
        good = [0, 1, 5]
    flags = i32([0], gpu)
    got = run(gpu, batch, cache, q, torch.full_like(q, 7.0), flags)
    assert flags.item() == flag
    size = clean.float().abs().max()
    assert (got[good].float() - clean[good].float()).abs().max() <= 2.0 ** -6 * size
    if why in ("behind", "negative", "before"):  # they share nothing, and read it all themselves
        assert (got.float() - clean.float()).abs().max() <= 2.0 ** -6 * size


@pytest.mark.parametrize("bad", [[0, 2, 9, 9], [0, 2, 9, 4], [0, 2, 2, 9]])
def test_groups_behind_the_requests_leave_the_others_theirs(gpu, bad):
    rng = np.random.default_rng(6)
    batch = Batch(rng, [(64, [(5, 1), (9, 1)]), (48, [(3, 2), (70, 1)])], [(20, 1)], 16)
    cache = Cache(gpu, rng, batch.blocks, 1, 64, 16)
    q = torch.randn(6, 2, 64, device=gpu, dtype=torch.bfloat16)
    clean = run(gpu, batch, cache, q)
    batch.given = batch.tables  # whole: who shares nothing reads all of its own
    batch.groups, batch.shared = np.array(bad), np.array([64, 48, 48])
    flags = i32([0], gpu)
    got = run(gpu, batch, cache, q, flags=flags)
    assert flags.item() == _lib.MKV_FLAG_SPAN
    # one rounding of p (2^-8) and of the output (2^-8) on either side, as above
    assert (got.float() - clean.float()).abs().max() <= 2.0 ** -6 * clean.float().abs().max()


def test_strides_scale_and_another_stream(gpu):
    rng = np.random.default_rng(21)
    batch = Batch(rng, [(100, [(4, 4), (30, 1)])], [], 16)
    cache = Cache(gpu, rng, batch.blocks, 2, 64, 16)
    wide = torch.randn(5, 4, 3 * 64, device=gpu, dtype=torch.bfloat16)
    q = wide[:, :, 64:128]
    out = torch.zeros(5, 4, 128, device=gpu, dtype=torch.bfloat16)
    run(gpu, batch, cache, q, out[..., 64:], softmax_scale=0.3)
    want = run(gpu, batch, cache, q.contiguous(), softmax_scale=0.3)
    assert torch.equal(out[..., 64:], want) and (out[..., :64] == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = run(gpu, batch, cache, q, softmax_scale=0.3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(late, want)


def test_a_captured_call_replays_with_the_groups_of_its_day(gpu):
    rng = np.random.default_rng(33)
    batch = Batch(rng, [(640, [(90, 1)] * 6), (320, [(64, 1)] * 3)], [(50, 1)], 16)
    cache = Cache(gpu, rng, batch.blocks, 2, 128, 16)
    q = torch.randn(10, 8, 128, device=gpu, dtype=torch.bfloat16)
    tables, starts, lens = i32(batch.tables, gpu), i32(batch.starts, gpu), i32(batch.lens, gpu)
    groups, shared = i32(batch.groups, gpu), i32(batch.shared, gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend_shared(cache.dev, q, tables, starts, lens, groups, shared, max_new=1)
    for step in range(5):
        q.copy_(torch.randn_like(q))
        lens.sub_(step)
        shared.copy_(i32([640 - 160 * step, 16 * step], gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attend_shared(cache.dev, q, tables, starts, lens, groups, shared, max_new=1))


def test_refusals(gpu):
    rng = np.random.default_rng(1)
    batch = Batch(rng, [(32, [(4, 1), (3, 1)])], [], 16)
    cache = Cache(gpu, rng, batch.blocks, 2, 64, 16)
    q = torch.randn(2, 4, 64, device=gpu, dtype=torch.bfloat16)
    step = i32(batch.tables, gpu), i32(batch.starts, gpu), i32(batch.lens, gpu)
    groups, shared = i32([0, 2], gpu), i32([32], gpu)

    def refused(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            attend_shared(cache.dev, *args, **kw)

    refused(ValueError, "groups", q, *step, i32([0, 1, 2], gpu), shared)
    refused(ValueError, "groups", q, *step, groups.long(), shared)
    refused(ValueError, "shared", q, *step, groups, shared.cpu())
    refused(ValueError, "shared", q, *step, groups, shared[:, None])
    refused(TypeError, "one of", q.float(), *step, groups, shared)
    refused(ValueError, "multiple", q[:, :3], *step, groups, shared)
    refused(ValueError, "shares memory with q", q, *step, groups, shared, out=q)
    refused(RuntimeError, "backward", q.clone().requires_grad_(), *step, groups, shared)
    refused(RuntimeError, "max_shared", q, *step, groups, shared, max_shared=-1)
    refused(RuntimeError, "softmax_scale", q, *step, groups, shared, softmax_scale=0.0)
    torch.cuda.synchronize()
