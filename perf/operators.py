"""The operators of an 8-bit KV cache in blocks, as cases to be measured: plain torch forms and this package's calls.

The cache of one layer: ``k`` and ``v`` are e4m3 codes ``[blocks, kv_heads, block, head_dim]``,
``k_scale`` and ``v_scale`` fp32 ``[blocks, kv_heads]``: a value is its code times the scale of its block
and head.  Token ``p`` of request ``r`` lives in block ``block_table[r, p // block]``, at offset
``p % block``; its slot is ``block number * block + offset``.

Five operators:

* ``plan``    blocks handed out to the requests of a step, the slots of their new tokens (and the
              ``req_to_token`` rows that the page selection reads), then the blocks behind the kept
              tokens handed back;
* ``append``  new keys and values quantised into their slots (a block's scale grows with its largest
              value), then the rows of the touched blocks read back as bf16 or fp32;
* ``decode``  attention of one token per request over its whole cached sequence;
* ``select``  the same over listed rows (pages chosen by a selection, then the most recent tokens);
* ``extend``  causal attention of the new tokens of a batch over prefix and new tokens.

``own`` is set by the program that measures: false, ``run`` computes the plain forms; true, it makes the
calls of this package.
"""

import math
import random

import torch

own = False

BLOCK = 64  # tokens per block of the listed cases: the page of the page selection
E4M3_MAX = 448.0


# ---------------------------------------------------------------- cases


def listed():
    heads = {"heads": 32, "kv": 4, "dim": 128, "block": BLOCK, "dtype": "bf16"}
    small = {"heads": 8, "kv": 2, "dim": 64, "block": 16, "dtype": "f32"}
    return [
        # four drafted tokens for each of 64 running requests, three of them taken back after the check
        {"name": "plan_drafts_64", "op": "plan", "bs": 64, "lo": 16384, "hi": 32764, "new": 4, "keep": 1, "block": BLOCK,
         "map": False, "ragged": 1},
        # a batch of prompts admitted and, at the end of the pass, all of it handed back
        {"name": "plan_prompts_16", "op": "plan", "bs": 16, "lo": 100, "hi": 8192, "new": 0, "keep": 0, "block": BLOCK,
         "map": True, "ragged": 2},
        # one layer of a decode step: one token for each of 64 requests
        {"name": "append_step_64", "op": "append", "bs": 64, "lo": 500, "hi": 4000, "new": 1, "ragged": 3, **heads},
        # one layer of a prefill of ragged prompts
        {"name": "append_prompts_6", "op": "append", "bs": 6, "lo": 33, "hi": 8192, "new": 0, "ragged": 4, **heads},
        # one request of 8192 tokens: the latency of a lone decode
        {"name": "decode_1x8k", "op": "decode", "bs": 1, "lo": 8192, "hi": 8192, "ragged": 5, **heads},
        # one request of 131072 tokens: one long axis split over the whole GPU
        {"name": "decode_1x128k", "op": "decode", "bs": 1, "lo": 131071, "hi": 131071, "ragged": 6, **heads},
        # a full batch of long contexts, the bandwidth-bound serving step
        {"name": "decode_64x32k", "op": "decode", "bs": 64, "lo": 16384, "hi": 32768, "ragged": 7, **heads},
        # fp32 activations of a small model in short blocks
        {"name": "decode_f32_5", "op": "decode", "bs": 5, "lo": 1, "hi": 2500, "ragged": 8, **small},
        # 2048 selected rows of each of 64 long requests: a layer of sparse decoding
        {"name": "select_64x2048", "op": "select", "bs": 64, "lo": 8192, "hi": 32768, "top": 2048, "ragged": 9, **heads},
        # a few requests, some of them shorter than the selection
        {"name": "select_3x2048", "op": "select", "bs": 3, "lo": 65, "hi": 5000, "top": 2048, "ragged": 10, **heads},
        # chunks of new tokens behind cached prefixes
        {"name": "extend_chunks_4", "op": "extend", "bs": 4, "lo": 1000, "hi": 6000, "new": 509, "ragged": 11, **heads},
        # one whole prompt
        {"name": "extend_prompt_8k", "op": "extend", "bs": 1, "lo": 8192, "hi": 8192, "new": 8192, "ragged": 12, **heads},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "decode", "decode", "select", "select", "extend", "extend"])
    ragged = rng.randrange(1 << 30)
    if op == "plan":
        if rng.random() < 0.5:
            hi = _log_uniform(rng, 200, 32000)
            return {"op": op, "bs": _log_uniform(rng, 1, 200), "lo": max(1, hi // 3), "hi": hi, "new": rng.randint(1, 9),
                    "keep": rng.randint(0, 1), "block": rng.choice([16, 32, 64, 128]), "map": rng.random() < 0.5,
                    "ragged": ragged}
        return {"op": op, "bs": _log_uniform(rng, 1, 40), "lo": 1, "hi": _log_uniform(rng, 20, 6000), "new": 0, "keep": 0,
                "block": rng.choice([16, 32, 64, 128]), "map": rng.random() < 0.5, "ragged": ragged}
    if rng.random() < 0.75:
        heads = {"heads": 4 * rng.choice([2, 4, 6, 8]), "kv": 4, "dim": 128,
                 "block": rng.choice([16, 32, 64, 64, 64, 128]), "dtype": "bf16"}
        big = 1.0
    else:
        kv = rng.choice([1, 2, 3])
        heads = {"heads": kv * rng.choice([1, 3, 4]), "kv": kv, "dim": rng.choice([16, 32, 64, 128]),
                 "block": rng.choice([16, 32, 64]), "dtype": rng.choice(["f32", "f32", "bf16"])}
        big = 0.1
    if op == "append":
        if rng.random() < 0.5:
            hi = _log_uniform(rng, 10, 4000)
            return {"op": op, "bs": _log_uniform(rng, 1, 200), "lo": max(1, hi // 4), "hi": hi, "new": rng.randint(1, 5),
                    "ragged": ragged, **heads}
        return {"op": op, "bs": _log_uniform(rng, 1, 8), "lo": 1, "hi": _log_uniform(rng, 16, 8000), "new": 0,
                "ragged": ragged, **heads}
    if op == "decode":
        total = _log_uniform(rng, 64, 1000000 * big)
        bs = _log_uniform(rng, 1, max(1, min(64, total // 32)))
        hi = max(1, min(131072, total // bs))
        return {"op": op, "bs": bs, "lo": max(1, hi // rng.choice([1, 2, 100])), "hi": hi, "ragged": ragged, **heads}
    if op == "select":
        top = heads["block"] * rng.randint(2, max(2, 2048 // heads["block"]))
        hi = _log_uniform(rng, 100, 30000 * big)
        return {"op": op, "bs": _log_uniform(rng, 1, 64), "lo": max(1, hi // rng.choice([1, 3, 50])), "hi": hi, "top": top,
                "ragged": ragged, **heads}
    new = _log_uniform(rng, 1, 2500 if big == 1.0 else 300)
    hi = max(new, _log_uniform(rng, 16, 6000 if big == 1.0 else 1000))
    return {"op": op, "bs": rng.randint(1, 4), "lo": max(1, hi // 4), "hi": hi, "new": new, "ragged": ragged, **heads}


def _lengths(case):
    """(sequence lengths, new tokens of each): the ragged batch of a case, the first request the longest."""
    r = random.Random(case["ragged"])
    seq = [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["bs"] - 1)]
    new = case.get("new", 1)
    if case["op"] == "plan" and new:  # the tokens before the drafts, then the drafts
        return [s + new for s in seq], [new] * len(seq)
    if not new:  # whole prompts
        return seq, list(seq)
    if case["op"] == "extend":
        return seq, [min(s, n) for s, n in zip(seq, [new] + [r.randint(1, new) for _ in seq[1:]])]
    return seq, [min(s, new) for s in seq]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _blocks(n, block):
    return -(-n // block)


def work(case):
    seq, new = _lengths(case)
    total = sum(new)
    if case["op"] == "plan":
        blocks = sum(_blocks(s, case["block"]) - (_blocks(s - n, case["block"]) if s > n else 0) for s, n in zip(seq, new))
        # lengths and requests in, slots and offsets out, each new block's number out of the free list and into the
        # table, and back; the rows of the token map
        return {"bytes": 24 * len(seq) + 8 * (total + len(seq)) + 16 * blocks + (4 * total if case["map"] else 0), "flops": total}
    kv, dim, size = case["kv"], case["dim"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "append":
        rows = sum(s - (s - n) // case["block"] * case["block"] for s, n in zip(seq, new))
        put = 2 * total * kv * dim * (size + 1) + 8 * total
        return {"bytes": put + 2 * rows * kv * dim * (1 + size) + 8 * rows, "flops": 4 * total * kv * dim}
    q = case["heads"] * dim * size
    if case["op"] == "decode":
        return {"bytes": 2 * sum(seq) * kv * dim + 2 * len(seq) * q, "flops": 4 * sum(seq) * case["heads"] * dim}
    if case["op"] == "select":
        rows = sum(min(s, case["top"]) for s in seq)
        return {"bytes": 2 * rows * kv * dim + 4 * rows + 2 * len(seq) * q, "flops": 4 * rows * case["heads"] * dim}
    pairs = sum(n * (s - n) + n * (n + 1) // 2 for s, n in zip(seq, new))
    return {"bytes": 2 * sum(seq) * kv * dim + 2 * total * q, "flops": 4 * pairs * case["heads"] * dim}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _tables(case, seq, g):
    """A block table over scattered blocks (a few of the pool stay free) and the pool's size."""
    width = max(_blocks(s, case["block"]) for s in seq)
    need = sum(_blocks(s, case["block"]) for s in seq)
    total = need + 1 + need // 8
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["bs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, s in enumerate(seq):
        n = _blocks(s, case["block"])
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _codes(shape, g):
    """Codes of normally distributed values, the largest of a block near the top of the type."""
    flat = torch.empty(math.prod(shape), dtype=torch.float8_e4m3fn, device="cuda")
    for part in flat.split(1 << 27):
        x = torch.randn(part.numel(), generator=g, device="cuda", dtype=torch.float32)
        part.copy_((x * 90.0).clamp_(-E4M3_MAX, E4M3_MAX))
    return flat.view(shape)


def _scales(shape, g):
    """Powers of two around the step that puts the values near one."""
    return torch.exp2(torch.randint(-8, -5, shape, generator=g, device="cuda").float())


def _int64(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def _inputs(case, seed):
    g = _gen(seed)
    seq, new = _lengths(case)
    bs, block = case["bs"], case["block"]
    s = {"case": case}
    # a request's row of the tables is not its place in the batch
    rows = torch.randperm(bs, generator=g, device="cuda")
    s["reqs"], s["seq"] = rows, _int64(seq)
    s["prefix"] = s["seq"] - _int64(new)
    s["tokens"] = sum(new)
    if case["op"] == "plan":
        held = [_blocks(a - n, block) if a > n else 0 for a, n in zip(seq, new)]
        width = max(_blocks(a, block) for a in seq) + 1
        total = sum(_blocks(a, block) for a in seq) + 5
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = torch.full((bs, width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(held):
            table[rows[i], :n] = order[at:at + n]
            at += n
        s["table"] = table
        s["held"] = torch.zeros(bs, dtype=torch.int32, device="cuda")
        s["held"][rows] = torch.tensor(held, dtype=torch.int32, device="cuda")
        s["free"] = order.roll(-at).contiguous()  # the free blocks first; the others' places are filled as they come back
        s["ring"] = _int64([0, total - at])
        s["keep"] = s["prefix"] + case["keep"]
        s["map"] = torch.zeros(bs, width * block, dtype=torch.int32, device="cuda") if case["map"] else None
        return s
    kv, dim, dtype = case["kv"], case["dim"], _dtype(case)
    table, total = _tables(case, seq, g)
    s["table"] = torch.empty_like(table)
    s["table"][rows] = table
    shape = (total, kv, block, dim)
    if case["op"] == "append":
        # channels of different size, and now and then a token that makes its block's scale grow
        size = torch.exp(0.5 * torch.randn(kv, dim, generator=g, device="cuda"))
        grow = 1 + 7 * (torch.rand(s["tokens"], 1, 1, generator=g, device="cuda") < 0.05)
        s["k_new"], s["v_new"] = ((torch.randn(s["tokens"], kv, dim, generator=g, device="cuda") * size * grow).to(dtype)
                                  for _ in range(2))
        slots, touched = [], []
        for i, (a, n) in enumerate(zip(seq, new)):
            for out, first in ((slots, a - n), (touched, (a - n) // block * block)):
                p = torch.arange(first, a, device="cuda")
                out.append(table[i, p // block].long() * block + p % block)
        s["slots"], s["touched"] = torch.cat(slots), torch.cat(touched)
    s["k"], s["v"] = _codes(shape, g), _codes(shape, g)
    s["k_scale"], s["v_scale"] = _scales((total, kv), g), _scales((total, kv), g)
    if case["op"] == "append":
        return s
    tokens = s["tokens"] if case["op"] == "extend" else bs
    s["q"] = (torch.randn(tokens, case["heads"], dim, generator=g, device="cuda") * 1.5).to(dtype)
    s["scaling"] = dim ** -0.5
    if case["op"] == "select":
        top, recent = case["top"], block
        s["rows"] = torch.zeros(bs, top, dtype=torch.int32, device="cuda")
        for i, a in enumerate(seq):
            if a <= top:
                p = torch.arange(a, device="cuda")
            else:  # whole pages in the order of their scores, then the most recent tokens
                pages = torch.randperm(a // block, generator=g, device="cuda")[:top // block - 1]
                p = torch.cat([(pages[:, None] * block + torch.arange(block, device="cuda")).flatten(),
                               torch.arange(a - recent, a, device="cuda")])
            s["rows"][i, :p.numel()] = (table[i, p // block].long() * block + p % block).to(torch.int32)
        s["lens"] = s["seq"].clamp(max=top).to(torch.int32)
    if case["op"] == "extend":
        s["offsets"] = torch.cat([_int64([0]), _int64(new).cumsum(0)])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handles that a program keeps, around the same tensors
        from qwenquest_b200.kv8 import BlockTables, KV8Cache

        if case["op"] == "plan":
            s["tables"] = BlockTables.from_tensors(s["table"], s["held"], s["free"], s["ring"], case["block"])
        else:
            s["cache"] = KV8Cache.from_tensors([s["k"]], [s["v"]], [s["k_scale"]], [s["v_scale"]])
    return s


# ---------------------------------------------------------------- plain forms


def _plain_plan(s):
    case, table, held, free, ring = s["case"], s["table"], s["held"], s["free"], s["ring"]
    block, width, cap, reqs = case["block"], s["table"].shape[1], s["free"].numel(), s["reqs"]
    page = torch.arange(width, device="cuda")
    # blocks for the pages that a request does not hold yet, in batch order, from the head of the ring
    have, want = held[reqs].long(), (s["seq"] + block - 1) // block
    fresh = (page >= have[:, None]) & (page < want[:, None])
    nth = fresh.flatten().cumsum(0).view_as(fresh)
    table[reqs] = torch.where(fresh, free[(ring[0] + nth - 1) % cap], table[reqs])
    held[reqs] = torch.maximum(have, want).to(torch.int32)
    ring[0] += nth[-1, -1]
    # the slots of the new tokens
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), (s["seq"] - s["prefix"]).cumsum(0)])
    t = torch.arange(s["tokens"], device="cuda")
    entry = torch.searchsorted(offsets, t, right=True) - 1
    pos = s["prefix"][entry] + t - offsets[entry]
    slots = table[reqs[entry], pos // block].long() * block + pos % block
    if s["map"] is not None:
        s["map"][reqs[entry], pos] = slots.to(torch.int32)
    # the blocks behind the kept tokens, to the ring's tail
    have, keep = held[reqs].long(), (s["keep"] + block - 1) // block
    back = (page >= keep[:, None]) & (page < have[:, None])
    nth = back.flatten().cumsum(0).view_as(back)
    grown = torch.cat([free, free.new_zeros(1)])
    grown[torch.where(back, (ring[1] + nth - 1) % cap, cap)] = table[reqs]
    grown[cap] = 0
    free.copy_(grown[:cap])
    table[reqs] = torch.where(back, -1, table[reqs])
    held[reqs] = torch.minimum(have, keep).to(torch.int32)
    ring[1] += nth[-1, -1]
    return {"slots": slots, "offsets": offsets, "table": table, "held": held, "free": free, "ring": ring,
            "map": s["map"]}


def _plain_append_one(codes, scale, x, slots, block):
    at, off = slots // block, slots % block
    touched, inverse = torch.unique(at, return_inverse=True)
    x = x.float()
    kv = x.shape[1]
    most = torch.zeros(touched.numel(), kv, device="cuda").scatter_reduce(
        0, inverse[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
    # the smallest power of two that brings the largest value to 448 or below
    m, e = torch.frexp(most)
    e = torch.where(most > 0, e - 9 + (m > 0.875).int(), -126).clamp(min=-126)
    wanted = torch.ldexp(torch.ones_like(most), e)
    begun = torch.zeros(touched.numel(), device="cuda").scatter_reduce(0, inverse, (off == 0).float(), "amax") > 0
    old = scale[touched]
    now = torch.where(begun[:, None], wanted, torch.maximum(old, wanted))
    # what the block holds already, in steps of the new scale; a block written from its first token on starts anew
    before = codes[touched].float()
    ratio = torch.where(begun[:, None], torch.ones_like(now), old / now)
    codes[touched] = (before * ratio[:, :, None, None]).to(torch.float8_e4m3fn)
    scale[touched] = now
    y = (x / now[inverse][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    codes.view(torch.uint8)[at, :, off] = y.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_rows(codes, scale, slots, block):
    at, off = slots // block, slots % block
    return codes.view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn).float() * scale[at][:, :, None]


def _plain_append(s):
    block, dtype = s["case"]["block"], _dtype(s["case"])
    _plain_append_one(s["k"], s["k_scale"], s["k_new"], s["slots"], block)
    _plain_append_one(s["v"], s["v_scale"], s["v_new"], s["slots"], block)
    return {"k": _plain_rows(s["k"], s["k_scale"], s["touched"], block).to(dtype),
            "v": _plain_rows(s["v"], s["v_scale"], s["touched"], block).to(dtype),
            "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attend(q, k, v, seen, scaling):
    """q [b, n, heads, d], k and v [b, L, kv, d], seen [b, n, L]; a query that sees nothing gives zeros."""
    b, n, heads, d = q.shape
    kv = k.shape[2]
    qg = q.float().view(b, n, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    scores = torch.matmul(qg, k.permute(0, 2, 3, 1)).mul_(scaling).view(b, kv, heads // kv, n, -1)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(most > -math.inf, most, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, kv, -1, p.shape[-1]), v.transpose(1, 2)).view(b, kv, heads // kv, n, d)
    out = out / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, heads * d).to(q.dtype)


def _plain_cached(codes, scale, table):
    """The fp32 values of the blocks in `table` [b, pages] as [b, pages * block, kv, d]."""
    at = table.long().clamp(min=0)
    x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at][..., None, None]
    return x.transpose(2, 3).flatten(1, 2)


def _plain_decode(s):
    table = s["table"][s["reqs"]]
    k, v = _plain_cached(s["k"], s["k_scale"], table), _plain_cached(s["v"], s["v_scale"], table)
    seen = torch.arange(k.shape[1], device="cuda") < s["seq"][:, None]
    return _plain_attend(s["q"][:, None], k, v, seen[:, None], s["scaling"])[:, 0]


def _plain_select(s):
    block = s["case"]["block"]
    rows = s["rows"].long()
    k, v = (_plain_rows(c, x, rows.flatten(), block).view(*rows.shape, *c.shape[1::2])
            for c, x in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
    seen = torch.arange(rows.shape[1], device="cuda") < s["lens"][:, None]
    return _plain_attend(s["q"][:, None], k, v, seen[:, None], s["scaling"])[:, 0]


def _plain_extend(s):
    table = s["table"][s["reqs"]]
    k, v = _plain_cached(s["k"], s["k_scale"], table), _plain_cached(s["v"], s["v_scale"], table)
    t = torch.arange(s["tokens"], device="cuda")
    entry = torch.searchsorted(s["offsets"], t, right=True) - 1
    nth = t - s["offsets"][entry]
    widest = max(_lengths(s["case"])[1])
    q = s["q"].new_zeros(s["case"]["bs"], widest, *s["q"].shape[1:])
    q[entry, nth] = s["q"]
    pos = s["prefix"][:, None] + torch.arange(widest, device="cuda")
    seen = torch.arange(k.shape[1], device="cuda") <= pos[:, :, None]
    return _plain_attend(q, k, v, seen, s["scaling"])[entry, nth]


# ---------------------------------------------------------------- one pass


def _own(s):
    op = s["case"]["op"]
    if op == "plan":
        tables = s["tables"]
        slots, offsets = tables.plan(s["reqs"], s["seq"], s["prefix"], s["tokens"], req_to_token=s["map"])
        tables.trim(s["reqs"], s["keep"])
        return {"slots": slots, "offsets": offsets, "table": s["table"], "held": s["held"], "free": s["free"],
                "ring": s["ring"], "map": s["map"]}
    cache = s["cache"]
    if op == "append":
        cache.append(0, s["k_new"], s["v_new"], s["slots"])
        k, v = cache.gather(0, s["touched"], dtype=s["k_new"].dtype)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "decode":
        return cache.decode_attention(0, s["q"], s["table"], s["reqs"], s["seq"], s["scaling"])
    if op == "select":
        return cache.sparse_decode_attention(0, s["q"], s["rows"], s["lens"], s["scaling"])
    return cache.extend_attention(0, s["q"], s["table"], s["reqs"], s["seq"], s["prefix"], s["offsets"], s["scaling"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "plan":
        return _plain_plan(state)
    if op == "append":
        return _plain_append(state)
    if op == "decode":
        return _plain_decode(state)
    if op == "select":
        return _plain_select(state)
    return _plain_extend(state)


# ---------------------------------------------------------------- the definition in 64 bits


def _e4m3_of(x):
    """The e4m3 value nearest to each x (|x| <= 448), ties to even: steps of 2^(exponent - 3), 2^-9 at least."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return torch.round(x / step) * step


def _exact_append(s):
    block, out = s["case"]["block"], {}
    for name in ("k", "v"):
        values = s[name].double() * 1.0
        scale = s[name + "_scale"].double()
        x = s[name + "_new"].double()
        first = torch.nonzero(torch.diff(s["slots"] // block, prepend=s["slots"].new_full((1,), -1))).flatten().tolist()
        slots = s["slots"].tolist()
        for a, b in zip(first, first[1:] + [len(slots)]):  # the tokens a .. b - 1 go to one block
            at, off = slots[a] // block, slots[a] % block
            need = torch.ceil(torch.log2(x[a:b].abs().amax((0, 2)) / E4M3_MAX) - 1e-12).clamp(min=-126)
            step = torch.exp2(need)
            if off:
                step = torch.maximum(step, scale[at])
                values[at] = _e4m3_of(values[at] * (scale[at] / step)[:, None, None])
            scale[at] = step
            values[at, :, off:off + b - a] = _e4m3_of(x[a:b] / step[:, None]).transpose(0, 1)
        at, off = s["touched"] // block, s["touched"] % block
        out[name] = values[at, :, off] * scale[at][:, :, None]
        out[name + "_scale"] = scale
    return {n: out[n] for n in ("k", "v", "k_scale", "v_scale")}


def _exact_rows(s, i, slots, q, limit):
    """Attention of q [n, heads, d] over the listed slots, query j seeing the first limit[j] of them."""
    block, kv = s["case"]["block"], s["case"]["kv"]
    at, off = slots // block, slots % block
    k, v = (s[n].view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn).double() * s[n + "_scale"].double()[at][:, :, None]
            for n in ("k", "v"))
    n, heads, d = q.shape
    out = torch.empty(n, heads, d, dtype=torch.float64, device="cuda")
    hidden = torch.arange(slots.numel(), device="cuda") >= limit[:, None]
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        scores = (q[:, h].double() @ kh.T * s["scaling"]).masked_fill(hidden, -math.inf)
        out[:, h] = torch.softmax(scores, -1) @ vh
    return out.reshape(n, -1)


def exact(case, seed):
    """What `run` returns, from the definition in 64 bits; the plan's outputs are whole numbers and have no such value."""
    if case["op"] == "plan":
        return None
    s = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(s) if s["tokens"] < 40000 else None
    block, seq = case["block"], s["seq"].tolist()
    parts = []
    for i, n in enumerate(seq):
        p = torch.arange(n, device="cuda")
        slots = s["table"][s["reqs"][i]][p // block].long() * block + p % block
        if case["op"] == "decode":
            parts.append(_exact_rows(s, i, slots, s["q"][i:i + 1], _int64([n])))
        elif case["op"] == "select":
            m = min(n, case["top"])
            parts.append(_exact_rows(s, i, s["rows"][i, :m].long(), s["q"][i:i + 1], _int64([m])))
        else:
            a, b = s["offsets"][i].item(), s["offsets"][i + 1].item()
            parts.append(_exact_rows(s, i, slots, s["q"][a:b], s["prefix"][i] + torch.arange(1, b - a + 1, device="cuda")))
    return torch.cat(parts)
