"""The block-scaled 8-bit KV cache's operators, measured: slots, store, attention, shift.

A paged cache holds K and V as e4m3 codes, with one power of two for each (block of tokens,
KV head) and for K and V apart: ``x = code * 2 ** e``, the smallest exponent under which the
block's largest value fits 448.  Four operators work on it:

* ``slots``  -- block tables and slot maps of an engine step, built on the GPU from the
  requests' lengths;
* ``store``  -- new K and V rows into their blocks: a block's scale grows with its rows, and
  the rows that it held are encoded again where it did;
* ``attend`` -- causal grouped-query attention of the step's queries over the cache, from
  one token a request to long chunks;
* ``shift``  -- reused spans moved into other blocks, K re-rotated by the span's offset,
  every layer in one call.

``run`` computes each in elementary torch operations, or, with ``own`` set, through the
package's entry points.  Sizes, lengths and deltas come from the case alone, values and
block tables from the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
THETA = 1e6
TOP = 448.0  # the largest e4m3 value
LOW, HIGH = -100, 100  # the exponents that a scale may have
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _slots_case(**kw):
    return {"op": "slots", "requests": 1, "tokens": 1, "context": 4096, "block": BLOCK, **kw}


def _store_case(**kw):
    return {"op": "store", "requests": 1, "tokens": 1, "context": 4096, "heads": 8, "head": 128,
            "block": BLOCK, "dtype": "bf16", "layout": "hnd", **kw}


def _attend_case(**kw):
    return {"op": "attend", "requests": 1, "tokens": 1, "context": 4096, "heads": 8, "group": 4,
            "head": 128, "block": BLOCK, "dtype": "bf16", "layout": "hnd", **kw}


def _shift_case(**kw):
    return {"op": "shift", "tokens": 512, "spans": 1, "layers": 40, "heads": 8, "head": 128,
            "rotary": 128, "block": BLOCK, "layout": "hnd", **kw}


def listed() -> list:
    """Geometry of the repository's workloads: 8 KV heads of 128 (4 or 5 query heads each),
    28 to 40 layers, blocks of 16 tokens, 32 sessions, 22,141 tokens in 8 spans."""
    return [
        # a decode step of a batch of sessions: one token each, now and then a new block
        _slots_case(name="slots_decode_32", requests=32, tokens=32, context=16000),
        # a step that prefills several long prompts beside many decoding requests
        _slots_case(name="slots_mixed_256", requests=256, tokens=50021, context=30000),
        # a decode step's new rows, one layer: the smallest store
        _store_case(name="store_decode_32", requests=32, tokens=32, context=16000),
        # one layer of a long prompt's prefill
        _store_case(name="store_chunk_22k", requests=1, tokens=22141, context=0),
        # ragged prefill chunks that continue half-filled blocks, small heads, NHD
        _store_case(name="store_ragged_fp16", requests=13, tokens=5003, context=3000, heads=4,
                    head=64, dtype="fp16", layout="nhd"),
        # one session's next token over a long edited history
        _attend_case(name="attend_decode_1_30k", requests=1, tokens=1, context=30720, group=5),
        # a batch's next tokens, ragged histories
        _attend_case(name="attend_decode_32", requests=32, tokens=32, context=16000),
        # the edited part of a history recomputed against the spans that were reused
        _attend_case(name="attend_chunk_2k", requests=1, tokens=2048, context=22141, group=5),
        # short ragged chunks of several requests, one GPU's share of the heads, NHD, fp16
        _attend_case(name="attend_ragged_fp16", requests=7, tokens=1501, context=4000, heads=2,
                     group=8, head=64, dtype="fp16", layout="nhd"),
        # a short span moved by an edit, every layer: the smallest shift
        _shift_case(name="shift_512", tokens=512),
        # the whole edited history of a long session, 8 spans
        _shift_case(name="shift_22k_8spans", tokens=22141, spans=8),
        # one GPU's share of the heads, half of each head rotated, NHD
        _shift_case(name="shift_6k_2heads", tokens=6007, spans=3, layers=28, heads=2, rotary=64,
                    layout="nhd"),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        op = rng.choice(["slots", "store", "attend", "attend", "attend", "shift"])
        geometry = {"heads": rng.choice([1, 2, 4, 8, 8]), "head": rng.choice([64, 128, 128, 256]),
                    "layout": rng.choice(["hnd", "hnd", "nhd"]),
                    "block": rng.choice([16, 16, 16, 32, 64])}
        if op == "slots":
            n = _log(rng, 1, 512)
            case = _slots_case(requests=n, tokens=rng.choice([n, max(n, _log(rng, 16, 50000))]),
                               context=_log(rng, 16, 30000), block=geometry["block"])
        elif op == "store":
            n = _log(rng, 1, 64)
            case = _store_case(requests=n, tokens=rng.choice([n, max(n, _log(rng, 16, 22000))]),
                               context=_log(rng, 16, 16000),
                               dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), **geometry)
        elif op == "attend":
            n = _log(rng, 1, 32)
            case = _attend_case(requests=n, tokens=rng.choice([n, max(n, _log(rng, 16, 2048))]),
                                context=_log(rng, 16, 30000), group=rng.choice([1, 2, 4, 5, 8]),
                                dtype=rng.choice(["bf16", "bf16", "fp16"]), **geometry)
        else:
            tokens = _log(rng, 16, 22000)
            case = _shift_case(tokens=tokens, spans=rng.randint(1, max(1, min(8, tokens // 64))),
                               layers=rng.randint(24, 40),
                               rotary=geometry["head"] // rng.choice([1, 1, 2]), **geometry)
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


def _lengths(case) -> tuple:
    """Tokens that each request holds before the step, and its new ones."""
    rng = random.Random(case["requests"] * 7919 + case["tokens"])
    n, tokens, context = case["requests"], case["tokens"], case["context"]
    if n == 1:
        return [context], [tokens]
    held = [int(context * rng.uniform(0.1, 1.0)) for _ in range(n)]
    if tokens < 4 * n:  # a decode step; what is over goes to its last request
        new = [1] * n
        new[-1] += tokens - n
    elif case["op"] == "slots":  # most requests decode, an eighth of them prefill
        many = max(1, n // 8)
        new = [1] * (n - many) + _parts(tokens - (n - many), many, rng)
    else:
        new = _parts(tokens, n, rng)
    return held, new


def _blocks(n: int, block: int) -> int:
    return -(-n // block)


def _rows_of(case) -> list:
    """A shift's spans: (source position, destination position, tokens, delta); each starts
    at a block of its destination, as loads do, and anywhere in its source."""
    rng = random.Random(case["tokens"] * 31 + case["spans"])
    rows, src, dst = [], 0, 0
    for n in _parts(case["tokens"], case["spans"], rng):
        src += rng.randint(0, 40)
        dst += case["block"] * rng.randint(0, 3)
        rows.append((src, dst, n, dst - src))
        src += n
        dst += _blocks(n, case["block"]) * case["block"]
    return rows


def _pairs(case) -> int:
    """(query, key) pairs of one head."""
    held, new = _lengths(case)
    return sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))


def _cost(case) -> float:
    """A case's size as a share of the largest that is worth measuring."""
    if case["op"] == "slots":
        return case["tokens"] / 50021
    if case["op"] == "store":
        return case["tokens"] * case["heads"] * case["head"] / (22141 * 8 * 128)
    if case["op"] == "shift":
        return (case["tokens"] * case["layers"] * case["heads"] * case["head"]
                / (22141 * 40 * 8 * 128))
    held, new = _lengths(case)
    longest = max(h + n for h, n in zip(held, new))
    heads = case["heads"] * case["group"]
    # the plain form's padded scores, its padded cache, and the work itself
    return max(case["requests"] * max(new) * longest * heads / (2048 * 24189 * 40),
               case["requests"] * longest * case["heads"] * case["head"] / (32 * 16000 * 8 * 128),
               _pairs(case) * heads * case["head"] / (2048 * 23165 * 40 * 128))


def work(case) -> dict:
    if case["op"] == "slots":
        held, new = _lengths(case)
        fresh = sum(_blocks(h + n, case["block"]) - _blocks(h, case["block"])
                    for h, n in zip(held, new))
        # lengths in, starts and lengths out, a free block read and entered, a slot and a
        # position for each token
        return {"bytes": case["requests"] * 16 + fresh * 8 + case["tokens"] * 12, "flops": 0}
    rows = case["heads"] * 2 * case["head"]
    if case["op"] == "store":
        held, new = _lengths(case)
        touched = sum(_blocks(h + n, case["block"]) - h // case["block"] for h, n in zip(held, new))
        return {"bytes": case["tokens"] * rows * (BYTES[case["dtype"]] + 1)
                + touched * case["heads"] * 2, "flops": 0}
    if case["op"] == "shift":
        blocks = _blocks(case["tokens"], case["block"])
        return {"bytes": 2 * case["layers"] * (case["tokens"] * rows + blocks * case["heads"] * 2),
                "flops": 3 * case["layers"] * case["tokens"] * case["heads"] * case["rotary"]}
    held, new = _lengths(case)
    keys = sum(h + n for h, n in zip(held, new))
    heads = case["heads"] * case["group"]
    return {"bytes": keys * rows + _blocks(keys, case["block"]) * case["heads"] * 2
            + 2 * case["tokens"] * heads * case["head"] * BYTES[case["dtype"]],
            "flops": 4 * case["head"] * heads * _pairs(case)}


# ------------------------------------------------------------------ inputs


def _tables(held, new, block, gen, device, spare=0):
    """Shuffled block tables wide enough for every request, and how many blocks there are."""
    need = [_blocks(h + n, block) for h, n in zip(held, new)]
    count = sum(need) + spare
    order = torch.randperm(count, generator=gen, device=device, dtype=torch.int64).to(torch.int32)
    starts = torch.tensor([0] + need[:-1], device=device).cumsum(0)
    cols = torch.arange(max(need), device=device)
    at = (starts[:, None] + cols).clamp_(max=count - 1)
    short = cols >= torch.tensor(need, device=device)[:, None]
    return order[at].masked_fill(short, 0), count


def _empty(case, blocks, device, layers):
    block, heads, d = case["block"], case["heads"], case["head"]
    shape = ((blocks, heads, block, 2 * d) if case["layout"] == "hnd"
             else (blocks, block, heads, 2 * d))
    kv = torch.zeros((layers, *shape), dtype=torch.uint8, device=device)
    scales = torch.zeros((layers, blocks, heads, 2), dtype=torch.uint8, device=device)
    return kv.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def _cache(case, blocks, gen, device, layers=None):
    """A cache whose rows are filled: keys with the uneven channels that real ones have,
    values of about one, encoded block by block."""
    block, heads, d = case["block"], case["heads"], case["head"]
    kv, scales = _empty(case, blocks, device, layers or 1)
    channel = torch.exp(0.7 * torch.randn(2 * d, generator=gen, device=device))
    channel[d:] = 1.0
    for layer in range(layers or 1):
        x = torch.randn((blocks, block, heads, 2, d), generator=gen, device=device)
        x *= channel.view(2, d)
        e = _exponent(x.abs().amax((1, 4)))
        scales[layer].view(torch.uint8).copy_(e + 127)
        x = (x * _power(-e)[:, None, :, :, None]).to(torch.float8_e4m3fn)
        _by_token(kv[layer].view(torch.uint8), case["layout"]).copy_(
            x.view(torch.uint8).view(blocks, block, heads, 2 * d))
    return (kv, scales) if layers else (kv[0], scales[0])


def prepare(case, seed):
    device = torch.device("cuda", 0)
    gen = torch.Generator(device=device).manual_seed(int(seed))

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    s = dict(case)
    if case["op"] == "shift":
        rows = _rows_of(case)
        src_end, dst_end = rows[-1][0] + rows[-1][2], rows[-1][1] + rows[-1][2]
        src_blocks = _blocks(src_end, case["block"])
        dst_blocks = _blocks(dst_end, case["block"])
        s["src"] = _cache({**case, "layout": "nhd"}, src_blocks, gen, device, case["layers"])
        s["dst"] = _empty(case, dst_blocks, device, case["layers"])
        host = torch.Generator().manual_seed(int(seed))
        s["src_table"] = torch.randperm(src_blocks, generator=host).numpy().astype(np.int32)
        s["dst_table"] = torch.randperm(dst_blocks, generator=host).numpy().astype(np.int32)
        s["rows"] = [(a, b, 0, 0, n, delta, 0, 0) for a, b, n, delta in rows]
        r = case["rotary"]
        s["inv_freq"] = 1.0 / THETA ** (torch.arange(0, r, 2, dtype=torch.float32) / r)
        if own:
            from marathon_amd import ScaledCache, ScaledShifts

            s["shifts"] = ScaledShifts(
                [ScaledCache(a, b, "nhd", case["block"]) for a, b in zip(*s["src"])],
                [ScaledCache(a, b, case["layout"], case["block"]) for a, b in zip(*s["dst"])],
                s["inv_freq"])
        return s
    held, new = _lengths(case)
    s["tables"], count = _tables(held, new, case["block"], gen, device, spare=8)
    s["max_new"] = max(new)
    s["max_len"] = max(h + n for h, n in zip(held, new))
    if case["op"] == "slots":
        s["held"], s["new"] = ints(held), ints(new)
        s["free"] = torch.randperm(2 * count, generator=gen, device=device).to(torch.int32)
        s["free_at"] = torch.randint(0, count // 2, (1,), generator=gen, device=device,
                                     dtype=torch.int32)
        return s
    s["starts"] = ints(np.cumsum([0] + new).tolist())
    s["lens"] = ints([h + n for h, n in zip(held, new)])
    s["kv"], s["scales"] = _cache(case, count, gen, device)
    dtype, d = DTYPES[case["dtype"]], case["head"]
    if case["op"] == "store":
        shape = (case["tokens"], case["heads"], d)
        # now and then a row is larger than what its block held: the scale grows
        loud = 1 + 7 * (torch.rand(shape[:2], generator=gen, device=device) < 0.05).float()
        for name in ("k", "v"):
            x = torch.randn(shape, generator=gen, device=device) * loud[..., None]
            s[name] = x.to(dtype)
    else:
        s["q"] = (torch.randn((case["tokens"], case["heads"] * case["group"], d), generator=gen,
                              device=device) * 1.5).to(dtype)
    if own:
        from marathon_amd import ScaledCache

        s["cache"] = ScaledCache(s["kv"], s["scales"], case["layout"], case["block"])
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    return {"slots": _slots, "store": _store, "attend": _attend, "shift": _shift}[s["op"]](s)


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


def _slots(s):
    if own:
        from marathon_amd import step_slots

        step = step_slots(s["held"], s["new"], s["tables"], s["free"], s["free_at"], s["block"],
                          s["tokens"])
        return {"tables": s["tables"], "starts": step.starts, "lens": step.lens,
                "slots": step.slots, "positions": step.positions, "free_at": step.free_at}
    held, new, block = s["held"].long(), s["new"].long(), s["block"]
    lens = held + new
    before, after = (held + block - 1) // block, (lens + block - 1) // block
    need = after - before
    first = need.cumsum(0) - need + s["free_at"]
    cols = torch.arange(s["tables"].shape[1], device=held.device)
    fresh = (cols >= before[:, None]) & (cols < after[:, None])
    at = ((first - before)[:, None] + cols).clamp(0, s["free"].numel() - 1)
    s["tables"].copy_(torch.where(fresh, s["free"][at], s["tables"]))
    starts = torch.cat((new.new_zeros(1), new.cumsum(0)))
    r, t = _owners(starts, s["tokens"], held.device)
    there = t < starts[-1]
    pos = held[r] + t - starts[r]
    slots = s["tables"][r, pos // block].long() * block + pos % block
    return {"tables": s["tables"], "starts": starts.int(), "lens": lens.int(),
            "slots": torch.where(there, slots, -1), "positions": torch.where(there, pos, 0).int(),
            "free_at": (s["free_at"] + need.sum()).int()}


def _store(s):
    if own:
        from marathon_amd import store_scaled

        store_scaled(s["cache"], s["k"], s["v"], s["tables"], s["starts"], s["lens"])
        return {"kv": s["kv"], "scales": s["scales"]}
    block, d = s["block"], s["head"]
    starts, lens = s["starts"].long(), s["lens"].long()
    held = lens - (starts[1:] - starts[:-1])
    x = torch.stack((s["k"], s["v"]), 2).float()  # token, head, K or V, value
    r, t = _owners(starts, x.shape[0], x.device)
    pos = held[r] + t - starts[r]
    blocks = s["tables"][r, pos // block].long()
    most = torch.where(x.isfinite(), x.abs(), 0).amax(-1)
    count = s["kv"].shape[0]
    at = blocks[:, None, None].expand_as(most)
    e = _exponent(most.new_zeros((count, *most.shape[1:])).scatter_reduce_(0, at, most, "amax"))
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
    return {"kv": s["kv"], "scales": s["scales"]}


def _attend(s):
    if own:
        from marathon_amd import attend_scaled

        return attend_scaled(s["cache"], s["q"], s["tables"], s["starts"], s["lens"],
                             max_new=s["max_new"], max_len=s["max_len"])
    block, d, heads, group = s["block"], s["head"], s["heads"], s["group"]
    starts, lens = s["starts"].long(), s["lens"].long()
    n, width = lens.numel(), s["tables"].shape[1]
    new = starts[1:] - starts[:-1]
    codes = _by_token(s["kv"].view(torch.uint8), s["layout"])[s["tables"].long()]
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (2, d))
    x = x * _power(_exponents(s["scales"]))[s["tables"].long()][:, :, None, :, :, None]
    x = x.flatten(1, 2)  # request, token, head, K or V, value
    keys = x[..., 0, :].permute(0, 2, 3, 1).contiguous()  # request, KV head, value, token
    values = x[..., 1, :].transpose(1, 2).contiguous()
    i = torch.arange(s["max_new"], device=x.device)
    rows = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(n, s["max_new"], heads, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, heads, group * s["max_new"], d)
    score = torch.matmul(q, keys) * d ** -0.5
    reach = (lens - new)[:, None] + i  # a query's own position
    sees = torch.arange(width * block, device=x.device) <= reach[..., None]
    sees = (sees & (i < new[:, None])[..., None]).repeat(1, group, 1)[:, None]
    score = score.masked_fill_(~sees, -math.inf)
    most = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(most.isfinite(), most, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total > 0, total, 1)
    out = out.view(n, heads, group, s["max_new"], d).permute(0, 3, 1, 2, 4).flatten(2, 3)
    r, t = _owners(starts, s["q"].shape[0], x.device)
    return out[r, (t - starts[r]).clamp(max=s["max_new"] - 1)].to(s["q"].dtype)


def _moves(s, device):
    """Per token of a shift: source block and row, destination block and row, the number of
    its destination block among those written, and its span; as tensors on the GPU."""
    rows = np.array([(a, b, n) for a, b, _, _, n, _, _, _ in s["rows"]], dtype=np.int64)
    n, block = rows[:, 2], s["block"]
    span = np.repeat(np.arange(len(n)), n)
    i = np.arange(n.sum()) - np.repeat(np.cumsum(n) - n, n)
    src, dst = rows[span, 0] + i, rows[span, 1] + i
    written = -(-n // block)
    unit = (np.cumsum(written) - written)[span] + i // block
    cols = (s["src_table"][src // block], src % block, s["dst_table"][dst // block], dst % block,
            unit, span)
    return torch.from_numpy(np.stack(cols).astype(np.int64)).to(device)


def _shift(s):
    if own:
        s["shifts"].run(s["rows"], s["src_table"], s["dst_table"])
        return {"kv": s["dst"][0], "scales": s["dst"][1]}
    d, rotary, half = s["head"], s["rotary"], s["rotary"] // 2
    (src_kv, src_scales), (dst_kv, dst_scales) = s["src"], s["dst"]
    device, layers, heads = src_kv.device, s["layers"], s["heads"]
    sb, so, db, do, unit, span = _moves(s, device)
    delta = torch.tensor([float(row[5]) for row in s["rows"]], device=device)
    angle = (delta[:, None] * s["inv_freq"].to(device)).double()
    cos, sin = angle.cos().float()[span][:, None], angle.sin().float()[span][:, None]
    codes = src_kv.view(torch.uint8)[:, sb, so]  # layer, token, head, values of K then V
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (2, d))
    x = x * _power(_exponents(src_scales))[:, sb][..., None]
    a, b = x[..., 0, :half], x[..., 0, half:rotary]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    x[..., 0, :rotary] = torch.where(delta[span][:, None, None] != 0, turned, x[..., 0, :rotary])
    most = x.abs().amax(-1)
    units = sum(-(-row[4] // s["block"]) for row in s["rows"])
    at = unit[None, :, None, None].expand_as(most)
    e = _exponent(most.new_zeros((layers, units, heads, 2)).scatter_reduce_(1, at, most, "amax"))
    e = e[:, unit]
    out = _by_token(dst_kv.view(torch.uint8), s["layout"])
    out[:, db, do] = _encode(x, e[..., None]).flatten(3)
    dst_scales.view(torch.uint8)[:, db] = (e + 127).to(torch.uint8)
    return {"kv": dst_kv, "scales": dst_scales}


# ------------------------------------------------------------------ in 64 bits


def _scale64(most):
    """2 ** e for the smallest e with most <= 448 * 2 ** e, from the logarithm."""
    def power(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    e = torch.ceil(torch.log2(most / TOP)).clamp(-200, 200)
    e = torch.where(most > TOP * power(e), e + 1, e)  # the logarithm's own rounding
    e = torch.where(most <= TOP * power(e - 1), e - 1, e)
    return power(torch.where(most > 0, e, LOW).clamp(LOW, HIGH))


def _values64(kv, scales, layout):
    """(codes, scales) as numbers: block, token, head, K or V, value; block, head, K or V."""
    x = (kv if layout == "nhd" else kv.transpose(-3, -2)).double()
    return x.unflatten(-1, (2, x.shape[-1] // 2)), scales.double()


def _laid_out(x, layout):
    x = x.flatten(-2)
    return (x if layout == "nhd" else x.transpose(-3, -2)).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    return {"slots": _slots64, "store": _store64, "attend": _attend64, "shift": _shift64}[
        case["op"]](s)


def _slots64(s):
    held, new, tables = s["held"].tolist(), s["new"].tolist(), s["tables"].cpu().numpy()
    free, at, block = s["free"].tolist(), int(s["free_at"]), s["block"]
    starts, slots, positions = [0], [], []
    for r, (h, n) in enumerate(zip(held, new)):
        for b in range(-(-h // block), -(-(h + n) // block)):
            tables[r, b] = free[at]
            at += 1
        pos = np.arange(h, h + n)
        slots.append(tables[r, pos // block].astype(np.int64) * block + pos % block)
        positions.append(pos)
        starts.append(starts[-1] + n)

    def i32(a):
        return torch.from_numpy(np.asarray(a).astype(np.int32))

    return {"tables": i32(tables), "starts": i32(starts),
            "lens": i32([h + n for h, n in zip(held, new)]),
            "slots": torch.from_numpy(np.concatenate(slots)),
            "positions": i32(np.concatenate(positions)), "free_at": i32([at])}


def _store64(s):
    """The codes before their rounding, and the scales."""
    block, layout = s["block"], s["layout"]
    x, scales = _values64(s["kv"], s["scales"], layout)
    k, v = s["k"].double(), s["v"].double()
    starts, lens, tables = s["starts"].tolist(), s["lens"].tolist(), s["tables"].cpu()
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
        q = (room / scale[:, None, :, :, None]).flatten(0, 1)[begun:begun + n]
        p = torch.arange(pos, last, device=x.device)
        x[table[p // block - pos // block], p % block] = q
        scales[table] = scale
    return {"kv": _laid_out(x, layout), "scales": scales}


def _attend64(s):
    block, group, d = s["block"], s["group"], s["head"]
    if s["requests"] * s["max_new"] * s["max_len"] * s["heads"] * group > 4e9:
        return None
    starts, lens, tables = s["starts"].tolist(), s["lens"].tolist(), s["tables"].long()
    q = s["q"].double()
    out = torch.zeros_like(q)
    kv = s["kv"] if s["layout"] == "nhd" else s["kv"].transpose(1, 2)
    for r, last in enumerate(lens):
        lo, hi = starts[r], starts[r + 1]
        table = tables[r, :-(-last // block)]
        x = kv.view(torch.uint8)[table].view(torch.float8_e4m3fn).double().unflatten(-1, (2, d))
        scale = s["scales"].view(torch.uint8)[table].view(s["scales"].dtype).double()
        x = (x * scale[:, None, :, :, None]).flatten(0, 1)[:last]
        future = (torch.arange(last, device=q.device)[None]
                  > torch.arange(last - (hi - lo), last, device=q.device)[:, None])
        for h in range(q.shape[1]):
            score = q[lo:hi, h] @ x[:, h // group, 0].T / math.sqrt(d)
            p = torch.softmax(score.masked_fill(future, -math.inf), -1)
            out[lo:hi, h] = p @ x[:, h // group, 1]
    return out


def _shift64(s):
    """The codes before their rounding, and the scales."""
    d, half, block, layers = s["head"], s["rotary"] // 2, s["block"], s["layers"]
    out = torch.zeros(s["dst"][0].shape, dtype=torch.float64, device=s["dst"][0].device)
    out = _by_token(out, s["layout"]).unflatten(-1, (2, d))
    scales = s["dst"][1].double()
    src, src_scales = s["src"]
    for a, b, _, _, n, delta, _, _ in s["rows"]:
        p = np.arange(a, a + n)
        blocks = torch.from_numpy(s["src_table"][p // block].astype(np.int64)).to(src.device)
        offset = torch.from_numpy(p % block).to(src.device)
        x = src.view(torch.uint8)[:, blocks, offset].view(src.dtype).double().unflatten(-1, (2, d))
        x = x * src_scales.view(torch.uint8)[:, blocks].view(src_scales.dtype).double()[..., None]
        # the angle is the product in 32 bits, as the cache's own rotation takes it
        angle = (torch.tensor(float(delta)) * s["inv_freq"]).double().to(src.device)
        z = torch.complex(x[..., 0, :half], x[..., 0, half:2 * half])
        z = z * torch.polar(torch.ones_like(angle), angle)
        x[..., 0, :half], x[..., 0, half:2 * half] = z.real, z.imag
        room = x.new_zeros((layers, -(-n // block) * block, *x.shape[2:]))
        room[:, :n] = x
        scale = _scale64(room.unflatten(1, (-1, block)).abs().amax((2, 5)))
        q = (room.unflatten(1, (-1, block)) / scale[:, :, None, :, :, None]).flatten(1, 2)[:, :n]
        p = np.arange(b, b + n)
        blocks = torch.from_numpy(s["dst_table"][p // block].astype(np.int64)).to(src.device)
        out[:, blocks, torch.from_numpy(p % block).to(src.device)] = q
        first = torch.from_numpy(s["dst_table"][b // block:-(-(b + n) // block)].astype(np.int64))
        scales[:, first.to(src.device)] = scale
    return {"kv": _laid_out(out, s["layout"]), "scales": scales}
