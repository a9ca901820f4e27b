"""The serving step between the projections and the output, measured: rotate, put, shared.

Three operators stand around the block-scaled 8-bit KV cache (``x = code * 2 ** e``, e4m3 codes
with one power of two for the K rows and one for the V rows of each block and KV head):

* ``rotate`` -- every query and key head normalised (root mean square over the head, a weight
  for each of its values) and turned to its token's position (rotate-half pairs, all of the
  head or its first part), in one pass;
* ``put``    -- the same for a step's projections with the keys and values written straight into
  the cache, each block under the scale of the rows that it receives; the queries come back;
* ``shared`` -- causal grouped-query attention of a batch whose requests begin, in groups, with
  the same cached tokens (a system prompt, a document, one history that several drafts
  continue): what a group shares is read once for all of its rows.

``run`` computes each in elementary torch operations, or, with ``own`` set, through the
package's entry points.  Sizes and lengths come from the case alone, values and block tables
from the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
THETA = 1e6
EPS = 1e-6
TOP = 448.0  # the largest e4m3 value
LOW, HIGH = -100, 100  # the exponents that a scale may have
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rotate_case(**kw):
    return {"op": "rotate", "tokens": 1, "context": 4096, "heads": 8, "group": 4, "head": 128,
            "rotary": 128, "dtype": "bf16", **kw}


def _put_case(**kw):
    return {"op": "put", "requests": 1, "tokens": 1, "context": 4096, "heads": 8, "group": 4,
            "head": 128, "rotary": 128, "block": BLOCK, "dtype": "bf16", "layout": "hnd", **kw}


def _shared_case(**kw):
    return {"op": "shared", "requests": 8, "groups": 1, "tokens": 8, "shared": 4096, "own": 256,
            "heads": 8, "group": 4, "head": 128, "block": BLOCK, "dtype": "bf16",
            "layout": "hnd", **kw}


def listed() -> list:
    """Geometry of the repository's workloads: 8 KV heads of 128 (4 or 5 query heads each),
    blocks of 16 tokens, 32 sessions, 22,141 and 30,720 tokens of history."""
    return [
        # a decode step of a batch of sessions, one layer's heads: the smallest call
        _rotate_case(name="rotate_decode_32", tokens=32, context=16000),
        # one layer of a long prompt's prefill
        _rotate_case(name="rotate_chunk_22k", tokens=22141, context=0, group=5),
        # a ragged chunk far into a history, small heads of which half is turned
        _rotate_case(name="rotate_part_fp16", tokens=5003, context=700000, heads=4, group=2,
                     head=64, rotary=32, dtype="fp16"),
        # projections kept in fp32, large heads
        _rotate_case(name="rotate_fp32_256", tokens=1999, context=30000, heads=2, group=8,
                     head=256, rotary=256, dtype="fp32"),
        # a decode step's projections, one layer
        _put_case(name="put_decode_32", requests=32, tokens=32, context=16000),
        # one layer of a long prompt's prefill
        _put_case(name="put_chunk_22k", requests=1, tokens=22141, context=0, group=5),
        # ragged prefill chunks that continue half-filled blocks, half of each head turned, NHD
        _put_case(name="put_ragged_fp16", requests=13, tokens=5003, context=3000, heads=4,
                  group=2, head=64, rotary=32, dtype="fp16", layout="nhd"),
        # a few requests' next tokens behind a short system prompt
        _shared_case(name="shared_decode_4", requests=4, tokens=4, shared=2000, own=100),
        # a batch of sessions over one long document, a token each
        _shared_case(name="shared_decode_32", requests=32, tokens=32, shared=16000, own=1000),
        # several documents, a few drafted tokens a request, small heads, NHD, fp16
        _shared_case(name="shared_drafts_fp16", requests=24, groups=3, tokens=96, shared=30000,
                     own=500, heads=2, group=8, head=64, dtype="fp16", layout="nhd"),
        # one history that many drafts continue: more rows than one tile holds
        _shared_case(name="shared_decode_96", requests=96, tokens=96, shared=30720, own=64,
                     group=5),
        # prompts behind one long prefix, their ragged chunks
        _shared_case(name="shared_chunk_2k", requests=7, tokens=1801, shared=22141, own=16,
                     group=5),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        op = rng.choice(["rotate", "put", "shared", "shared"])
        head = rng.choice([64, 128, 128, 256])
        geometry = {"heads": rng.choice([1, 2, 4, 8, 8]), "head": head,
                    "group": rng.choice([1, 2, 4, 5, 8])}
        paged = {"layout": rng.choice(["hnd", "hnd", "nhd"]),
                 "block": rng.choice([16, 16, 16, 32, 64])}
        turned = {"rotary": head // rng.choice([1, 1, 2]),
                  "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if op == "rotate":
            case = _rotate_case(tokens=_log(rng, 1, 22141), context=_log(rng, 1, 1000000),
                                **geometry, **turned)
        elif op == "put":
            n = _log(rng, 1, 64)
            case = _put_case(requests=n, tokens=rng.choice([n, max(n, _log(rng, 16, 22141))]),
                             context=_log(rng, 16, 16000), **geometry, **turned, **paged)
        else:
            n = _log(rng, 2, 96)
            case = _shared_case(requests=n, groups=rng.randint(1, max(1, min(4, n // 2))),
                                tokens=rng.choice([n, n, n * rng.randint(2, 6),
                                                   max(n, _log(rng, 16, 1800))]),
                                shared=_log(rng, 64, 30720), own=_log(rng, 16, 2000),
                                dtype=rng.choice(["bf16", "bf16", "fp16"]), **geometry, **paged)
        if _cost(case) <= 1.0:
            return case


# ------------------------------------------------------------------ sizes of a case


def _parts(total: int, n: int, rng) -> list:
    """`total` cut into `n` positive parts of unequal sizes."""
    weights = [rng.uniform(0.2, 1.0) for _ in range(n)]
    spare = total - n
    parts = [1 + int(spare * w / sum(weights)) for w in weights]
    parts[-1] += total - sum(parts)
    return parts


def _new(n: int, tokens: int, rng) -> list:
    """New tokens of each request: alike where they are few."""
    if tokens < 8 * n:
        return [tokens // n + (i < tokens % n) for i in range(n)]
    return _parts(tokens, n, rng)


def _groups(case) -> tuple:
    """The groups' first requests (and the number of requests), and the tokens each shares."""
    rng = random.Random(case["requests"] * 31 + case["groups"])
    sizes = _parts(case["requests"], case["groups"], rng)
    bounds = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    shares = [case["shared"]] + [int(case["shared"] * rng.uniform(0.3, 1.0)) for _ in sizes[1:]]
    return bounds, shares


def _lengths(case) -> tuple:
    """Tokens that each request holds before the step, and its new ones."""
    rng = random.Random(case["requests"] * 7919 + case["tokens"])
    n, tokens = case["requests"], case["tokens"]
    if case["op"] == "shared":
        bounds, shares = _groups(case)
        held = [share + int(case["own"] * rng.uniform(0.1, 1.0))
                for i, share in enumerate(shares) for _ in range(bounds[i], bounds[i + 1])]
    elif n == 1:
        held = [case["context"]]
    else:
        held = [int(case["context"] * rng.uniform(0.1, 1.0)) for _ in range(n)]
    return held, _new(n, tokens, rng)


def _blocks(n: int, block: int) -> int:
    return -(-n // block)


def _prefixes(case) -> list:
    """The shared tokens of each group that fill whole blocks."""
    return [share // case["block"] * case["block"] for share in _groups(case)[1]]


def _own_most(case) -> int:
    """The most tokens that a request has behind its group's."""
    held, new = _lengths(case)
    bounds, _ = _groups(case)
    return max(held[r] + new[r] - p for g, p in enumerate(_prefixes(case))
               for r in range(bounds[g], bounds[g + 1]))


def _pairs(case) -> int:
    """(query, key) pairs of one head."""
    held, new = _lengths(case)
    return sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))


def _cost(case) -> float:
    """A case's size as a share of the largest that is worth measuring."""
    heads = case["heads"] * case["group"]
    if case["op"] != "shared":
        size = case["tokens"] * (heads + 2 * case["heads"]) * case["head"] * BYTES[case["dtype"]]
        return size / (22141 * 56 * 128 * 2)
    held, new = _lengths(case)
    # the plain form's scores over the shared tokens and the padded ones over the rest, the
    # cache, and the work itself
    padded = case["requests"] * max(new) * _own_most(case) * heads
    rows = (sum(case["shared"] for _ in range(case["groups"]))
            + case["requests"] * _own_most(case)) * case["heads"] * case["head"]
    return max(case["tokens"] * case["shared"] * heads / (1801 * 22141 * 40),
               padded / (1801 * 22141 * 10), rows / (32 * 8000 * 8 * 128),
               _pairs(case) * heads * case["head"] / (1801 * 22500 * 40 * 128))


def work(case) -> dict:
    heads, group, d = case["heads"], case["group"], case["head"]
    size = BYTES[case["dtype"]] if "dtype" in case else 0
    if case["op"] == "rotate":
        rows = case["tokens"] * heads * (group + 1)
        # rows in and out, a position each token; a square and its sum, two scalings a value
        # and the turn's three operations
        return {"bytes": 2 * rows * d * size + 4 * case["tokens"],
                "flops": rows * (4 * d + 3 * case["rotary"])}
    if case["op"] == "put":
        held, new = _lengths(case)
        touched = sum(_blocks(h + n, case["block"]) - h // case["block"]
                      for h, n in zip(held, new))
        # queries in and out, keys and values in, their codes out
        return {"bytes": case["tokens"] * heads * d * (2 * group * size + 2 * (size + 1))
                + touched * heads * 2,
                "flops": case["tokens"] * heads * (group + 1) * (4 * d + 3 * case["rotary"])}
    held, new = _lengths(case)
    bounds, _ = _groups(case)
    keys = sum(p + sum(held[r] + new[r] - p for r in range(bounds[g], bounds[g + 1]))
               for g, p in enumerate(_prefixes(case)))
    return {"bytes": keys * heads * 2 * d + _blocks(keys, case["block"]) * heads * 2
            + 2 * case["tokens"] * heads * group * d * size,
            "flops": 4 * d * heads * group * _pairs(case)}


# ------------------------------------------------------------------ inputs


def _tables(case, held, new, gen, device, spare):
    """Shuffled block tables wide enough for every request, a group's requests beginning with
    the same blocks, and how many blocks there are."""
    block = case["block"]
    need = [_blocks(h + n, block) for h, n in zip(held, new)]
    first, common, count = [], [], 0  # of a request: its own blocks, its group's, how many
    if case["op"] == "shared":
        bounds, prefixes = _groups(case)[0], _prefixes(case)
        for g, p in enumerate(prefixes):
            at, count = count, count + p // block
            for r in range(bounds[g], bounds[g + 1]):
                common.append((at, p // block))
                first.append(count)
                count += need[r] - p // block
    else:
        for n in need:
            common.append((0, 0))
            first.append(count)
            count += n
    count += spare
    order = torch.randperm(count, generator=gen, device=device, dtype=torch.int64).to(torch.int32)
    at = np.zeros((len(need), max(need)), np.int64)
    for r, n in enumerate(need):
        a, c = common[r]
        at[r, :c] = np.arange(a, a + c)
        at[r, c:n] = np.arange(first[r], first[r] + n - c)
    short = torch.from_numpy(np.arange(max(need)) >= np.array(need)[:, None]).to(device)
    return order[torch.from_numpy(at).to(device)].masked_fill(short, 0), count


def _cache(case, blocks, gen, device):
    """A cache whose rows are filled: keys with the uneven channels that real ones have,
    values of about one, encoded block by block."""
    block, heads, d = case["block"], case["heads"], case["head"]
    shape = ((blocks, heads, block, 2 * d) if case["layout"] == "hnd"
             else (blocks, block, heads, 2 * d))
    kv = torch.zeros(shape, dtype=torch.uint8, device=device)
    channel = torch.exp(0.7 * torch.randn(2 * d, generator=gen, device=device))
    channel[d:] = 1.0
    x = torch.randn((blocks, block, heads, 2, d), generator=gen, device=device)
    x *= channel.view(2, d)
    e = _exponent(x.abs().amax((1, 4)))
    scales = (e + 127).to(torch.uint8)
    x = (x * _power(-e)[:, None, :, :, None]).to(torch.float8_e4m3fn)
    _by_token(kv, case["layout"]).copy_(x.view(torch.uint8).view(blocks, block, heads, 2 * d))
    return kv.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    device = torch.device("cuda", 0)
    gen = torch.Generator(device=device).manual_seed(int(seed))

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    s = dict(case)
    heads, d, dtype = case["heads"], case["head"], DTYPES[case["dtype"]]
    q_heads, tokens = heads * case["group"], case["tokens"]
    if case["op"] != "shared":
        # one product's output, cut into heads: uneven channels, rows of different size
        parts = [q_heads, heads, heads] if case["op"] == "put" else [q_heads, heads]
        x = normal(tokens, sum(parts), d) * torch.exp(0.5 * normal(d))
        x *= torch.exp(0.5 * normal(tokens, sum(parts), 1))
        s["q"], s["k"], *rest = x.to(dtype).split(parts, 1)
        s["v"] = rest[0] if rest else None
        s["wq"], s["wk"] = ((1 + 0.2 * normal(d)).to(dtype) for _ in range(2))
        r = case["rotary"]
        s["inv_freq"] = 1.0 / THETA ** (torch.arange(0, r, 2, device=device).float() / r)
    if case["op"] == "rotate":
        if tokens <= 64:  # a batch of sessions
            rng = random.Random(tokens * 7919)
            s["positions"] = ints([int(case["context"] * rng.uniform(0.1, 1.0))
                                   for _ in range(tokens)])
        else:
            s["positions"] = ints(range(case["context"], case["context"] + tokens))
        return s
    held, new = _lengths(case)
    s["tables"], count = _tables(case, held, new, gen, device, spare=8)
    s["max_new"] = max(new)
    s["starts"] = ints(np.cumsum([0] + new).tolist())
    s["lens"] = ints([h + n for h, n in zip(held, new)])
    s["kv"], s["scales"] = _cache(case, count, gen, device)
    if case["op"] == "shared":
        bounds, shares = _groups(case)
        s["groups"], s["shares"] = ints(bounds), ints(shares)
        s["max_shared"], s["max_own"] = max(shares), _own_most(case)
        s["bounds"], s["prefixes"] = bounds, _prefixes(case)
        s["rows"] = [sum(new[:b]) for b in bounds]  # the groups' first rows
        s["q"] = (normal(tokens, q_heads, d) * 1.5).to(dtype)
    if own:
        from marathon_amd import ScaledCache

        s["cache"] = ScaledCache(s["kv"], s["scales"], case["layout"], case["block"])
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    return {"rotate": _rotate, "put": _put, "shared": _shared}[s["op"]](s)


def _by_token(kv, layout):
    """The cache with its dimensions in the order block, token, head, value."""
    return kv if layout == "nhd" else kv.transpose(-3, -2)


def _exponent(most):
    """The smallest exponent e with most <= 448 * 2 ** e, for finite fp32 values."""
    m, e = torch.frexp(most)  # most = m * 2 ** e, 0.5 <= m < 1; 448 = 0.875 * 2 ** 9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(most > 0, e, LOW).clamp(LOW, HIGH).to(torch.int32)


def _power(e):
    """2 ** e in fp32, from its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _encode(x, e):
    return (x * _power(-e)).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(torch.uint8)


def _exponents(scales):
    return scales.view(torch.uint8).to(torch.int32) - 127


def _owners(starts, tokens, device):
    """The request of each of the step's rows, and the rows' numbers."""
    t = torch.arange(tokens, device=device)
    r = torch.searchsorted(starts[1:], t, right=True, out_int32=True).long()
    return r.clamp_(max=starts.numel() - 2), t


def _turned(x, weight, cos, sin):
    """Heads normalised, weighted and turned, in fp32; the angles were taken in 64 bits."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)


def _angles(positions, inv_freq):
    angle = positions.double()[:, None] * inv_freq.double()
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _rotate(s):
    if own:
        from marathon_amd import norm_rotate

        return norm_rotate(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["wq"],
                           k_weight=s["wk"], eps=EPS)
    turn = _angles(s["positions"], s["inv_freq"])
    return (_turned(s["q"], s["wq"], *turn).to(s["q"].dtype),
            _turned(s["k"], s["wk"], *turn).to(s["k"].dtype))


def _put(s):
    if own:
        from marathon_amd import store_rotated

        q = store_rotated(s["cache"], s["q"], s["k"], s["v"], s["tables"], s["starts"], s["lens"],
                          s["inv_freq"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS)
        return {"q": q, "kv": s["kv"], "scales": s["scales"]}
    block, d = s["block"], s["head"]
    starts, lens = s["starts"].long(), s["lens"].long()
    held = lens - (starts[1:] - starts[:-1])
    r, t = _owners(starts, s["k"].shape[0], s["k"].device)
    pos = held[r] + t - starts[r]
    turn = _angles(pos, s["inv_freq"])
    q = _turned(s["q"], s["wq"], *turn).to(s["q"].dtype)
    x = torch.stack((_turned(s["k"], s["wk"], *turn), s["v"].float()), 2)
    blocks = s["tables"][r, pos // block].long()
    most = x.abs().amax(-1)
    at = blocks[:, None, None].expand_as(most)
    e = _exponent(most.new_zeros((s["kv"].shape[0], *most.shape[1:]))
                  .scatter_reduce_(0, at, most, "amax"))
    # a block that a request had begun keeps its rows, and its scale where that is larger
    begun = s["tables"].gather(1, (held // block)[:, None].clamp(max=s["tables"].shape[1] - 1))
    begun = begun[:, 0].long()
    keeps = (held % block > 0) & (lens > held)
    old = _exponents(s["scales"])[begun]
    e[begun] = torch.where(keeps[:, None, None], torch.maximum(e[begun], old), e[begun])
    codes = _by_token(s["kv"].view(torch.uint8), s["layout"])
    rows = codes[begun]  # request, token, head, values of K then V
    was = rows.view(torch.float8_e4m3fn).float().unflatten(-1, (2, d))
    again = _encode(was, (e[begun] - old)[:, None, :, :, None]).flatten(-2)
    kept = torch.arange(block, device=x.device) < (held % block)[:, None]
    kept = (kept & keeps[:, None])[:, :, None, None]
    codes[begun] = torch.where(kept, again, rows)
    codes[blocks, pos % block] = _encode(x, e[blocks][..., None]).flatten(2)
    scales = s["scales"].view(torch.uint8)
    scales[blocks] = (e[blocks] + 127).to(torch.uint8)
    return {"q": q, "kv": s["kv"], "scales": s["scales"]}


def _rows(s, table):
    """Keys and values of the tokens behind block tables [..., width], in fp32: each
    [..., heads, tokens, value]."""
    codes = _by_token(s["kv"].view(torch.uint8), s["layout"])[table.long()]
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (2, s["head"]))
    x = x * _power(_exponents(s["scales"]))[table.long()][..., None, :, :, None]
    x = x.flatten(-5, -4)  # tokens, heads, K or V, value
    return x[..., 0, :].transpose(-3, -2), x[..., 1, :].transpose(-3, -2)


def _softmax_parts(score, values):
    """Largest score, sum and unnormalised output of rows over one part of their tokens."""
    most = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(most.isfinite(), most, 0)).exp_()
    return most, p.sum(-1, keepdim=True), torch.matmul(p, values)


def _shared(s):
    if own:
        from marathon_amd import attend_shared

        return attend_shared(s["cache"], s["q"], s["tables"], s["starts"], s["lens"], s["groups"],
                             s["shares"], max_new=s["max_new"], max_shared=s["max_shared"],
                             max_own=s["max_own"])
    block, d, heads, group, device = s["block"], s["head"], s["heads"], s["group"], s["q"].device
    q = s["q"].float().view(-1, heads, group, d)
    starts, lens = s["starts"].long(), s["lens"].long()
    bounds, prefixes = s["bounds"], s["prefixes"]
    n, width, most_new = lens.numel(), s["tables"].shape[1], s["max_new"]
    prefix = torch.tensor(prefixes, device=device).repeat_interleave(
        s["groups"][1:].long() - s["groups"][:-1].long(), output_size=n)
    # every request's own tokens, padded: request, head, group * new, tokens
    cols = torch.arange(_blocks(s["max_own"], block), device=device)
    table = s["tables"].gather(1, (prefix[:, None] // block + cols).clamp(max=width - 1))
    keys, values = _rows(s, table)
    i = torch.arange(most_new, device=device)
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    mine = q[rows].permute(0, 2, 3, 1, 4).reshape(n, heads, group * most_new, d)
    score = torch.matmul(mine, keys.transpose(-1, -2).contiguous()) * d ** -0.5
    new = starts[1:] - starts[:-1]
    reach = (lens - new - prefix)[:, None] + i
    sees = torch.arange(keys.shape[2], device=device) <= reach[..., None]
    sees = (sees & (i < new[:, None])[..., None]).repeat(1, group, 1)[:, None]
    parts = _softmax_parts(score.masked_fill_(~sees, -math.inf), values.contiguous())
    # back to the step's rows: token, head, group, value
    r, t = _owners(starts, q.shape[0], device)
    at = (t - starts[r]).clamp(max=most_new - 1)
    most, total, out = (x.unflatten(2, (group, most_new)).permute(0, 3, 1, 2, 4)[r, at]
                        for x in parts)
    # what each group shares, once for all of its rows
    done = []
    for g, p in enumerate(prefixes):
        lo, hi = s["rows"][g], s["rows"][g + 1]
        a, b, c = most[lo:hi], total[lo:hi], out[lo:hi]
        if p > 0 and hi > lo:
            keys, values = _rows(s, s["tables"][bounds[g], :p // block])
            theirs = q[lo:hi].permute(1, 0, 2, 3).reshape(heads, (hi - lo) * group, d)
            score = torch.matmul(theirs, keys.transpose(-1, -2).contiguous()) * d ** -0.5
            x, y, z = (w.view(heads, hi - lo, group, -1).transpose(0, 1)
                       for w in _softmax_parts(score, values.contiguous()))
            top = torch.maximum(a, x)
            f, h = (a - top).exp(), (x - top).exp()
            b, c = b * f + y * h, c * f + z * h
        done.append(c / torch.where(b > 0, b, 1))
    return torch.cat(done).flatten(1, 2).to(s["q"].dtype)


# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _rotate64, "put": _put64, "shared": _shared64}[case["op"]](s)


def _turned64(x, weight, positions, inv_freq):
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
    half = inv_freq.numel()
    z = torch.complex(x[..., :half], x[..., half:2 * half])
    angle = positions.double()[:, None, None] * inv_freq.double()
    z = z * torch.polar(torch.ones_like(angle), angle)
    x[..., :half], x[..., half:2 * half] = z.real, z.imag
    return x


def _rotate64(s):
    return tuple(_turned64(s[name], s[w], s["positions"], s["inv_freq"])
                 for name, w in (("q", "wq"), ("k", "wk")))


def _scale64(most):
    """2 ** e for the smallest e with most <= 448 * 2 ** e, from the logarithm."""
    def power(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    e = torch.ceil(torch.log2(most / TOP)).clamp(-200, 200)
    e = torch.where(most > TOP * power(e), e + 1, e)  # the logarithm's own rounding
    e = torch.where(most <= TOP * power(e - 1), e - 1, e)
    return power(torch.where(most > 0, e, LOW).clamp(LOW, HIGH))


def _put64(s):
    """The queries; the codes before their rounding, and the scales."""
    block, layout = s["block"], s["layout"]
    x = _by_token(s["kv"], layout).double()
    x = x.unflatten(-1, (2, s["head"]))
    scales = s["scales"].double()
    starts, lens, tables = s["starts"].tolist(), s["lens"].tolist(), s["tables"].cpu()
    pos = torch.cat([torch.arange(last - starts[r + 1] + starts[r], last)
                     for r, last in enumerate(lens)]).to(x.device)
    q = _turned64(s["q"], s["wq"], pos, s["inv_freq"])
    k, v = _turned64(s["k"], s["wk"], pos, s["inv_freq"]), s["v"].double()
    for r, last in enumerate(lens):
        t, n = starts[r], starts[r + 1] - starts[r]
        pos, begun = last - n, (last - n) % block
        fresh = torch.stack((k[t:t + n], v[t:t + n]), 2)
        table = tables[r, pos // block:-(-last // block)].long().to(x.device)
        room = torch.zeros((table.numel() * block, *fresh.shape[1:]), dtype=torch.float64,
                           device=x.device)
        room[begun:begun + n] = fresh
        room = room.unflatten(0, (-1, block))
        scale = _scale64(room.abs().amax((1, 4)))
        if begun:
            first = table[0]
            grown = torch.maximum(scale[0], scales[first])
            x[first, :begun] *= (scales[first] / grown)[..., None]
            scale[0] = grown
        codes = (room / scale[:, None, :, :, None]).flatten(0, 1)[begun:begun + n]
        p = torch.arange(pos, last, device=x.device)
        x[table[p // block - pos // block], p % block] = codes
        scales[table] = scale
    x = x.flatten(-2)
    x = x if layout == "nhd" else x.transpose(-3, -2)
    return {"q": q, "kv": x.contiguous(), "scales": scales}


def _shared64(s):
    """Every request for itself, over its own table from its first token on."""
    block, group, d = s["block"], s["group"], s["head"]
    starts, lens, tables = s["starts"].tolist(), s["lens"].tolist(), s["tables"].long()
    q = s["q"].double()
    out = torch.zeros_like(q)
    kv = _by_token(s["kv"], s["layout"])
    for r, last in enumerate(lens):
        lo, hi = starts[r], starts[r + 1]
        table = tables[r, :-(-last // block)]
        x = kv.view(torch.uint8)[table].view(torch.float8_e4m3fn).double().unflatten(-1, (2, d))
        scale = s["scales"].view(torch.uint8)[table].view(s["scales"].dtype).double()
        x = (x * scale[:, None, :, :, None]).flatten(0, 1)[:last]
        future = (torch.arange(last, device=q.device)[None]
                  > torch.arange(last - (hi - lo), last, device=q.device)[:, None])
        for h in range(x.shape[1]):
            theirs = q[lo:hi, h * group:(h + 1) * group].transpose(0, 1)
            score = theirs @ x[:, h, 0].T / math.sqrt(d)
            p = torch.softmax(score.masked_fill(future, -math.inf), -1)
            out[lo:hi, h * group:(h + 1) * group] = (p @ x[:, h, 1]).transpose(0, 1)
    return out
