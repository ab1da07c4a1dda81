"""The 8-bit block KV cache against its numpy restatement in 64 bits (``oracle/kv8.py``).

Tables, codes and scales are compared bit for bit.  Attention: with the weights w_j of one query,
W = sum_j w_j |v_j| and S the largest sum_d |q_d k_jd| * scaling of its keys,

* a score is a sum of head_dim products in fp32, then two multiplications: off by at most
  (head_dim + 8) 2^-24 S, which moves a weight by at most twice that, relatively (its own and the sum's),
  and 2^x itself by 2^-22 (2 ulp), also twice;
* n products are summed in fp32: n 2^-24 W at most, and the row sum the same relative to itself;
* on the tensor cores the weights (times the scale of V) are held as two e4m3 numbers: half a step 2^-4 of half a
  step 2^-4, that is 2^-8 relatively, or where the second falls below the type's normal range a fixed part of the row's
  largest: 2^-10 / 16 of 128 at least, 2^-21; the row's sum keeps the fp32 weights.  An extend batch holds them in
  fp16 instead, 2^-11, or 2^-25 of 1 at least, and its queries too: off by 2^-25 of 112 at least (2^-31 of the row's
  largest) where bf16's 8 bits leave the normal range, which the first bound covers: both bounds below cover both;
* the result is rounded once: half a step, 2^-8 in bf16 and 2^-24 in fp32.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8 as oracle
from qwenquest_b200.kv8 import BlockTables, KV8Cache

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _dev(x, dtype=torch.int64):
    return torch.tensor(np.asarray(x), dtype=dtype, device=DEV)


# ---------------------------------------------------------------- tables


def _assert_tables(tables: BlockTables, ref: oracle.Tables):
    assert tables.block_table.cpu().numpy().tolist() == ref.table.tolist()
    assert tables.held.cpu().numpy().tolist() == ref.held.tolist()
    taken, given = tables.ring.tolist()
    cap = tables.free_blocks.numel()
    free = tables.free_blocks.cpu().numpy()
    assert [int(free[i % cap]) for i in range(taken, given)] == ref.free
    assert tables._claim.count_nonzero().item() == 0


@pytest.mark.parametrize(("block", "max_reqs", "ctx", "top"), [
    (16, 5, 200, 3), (64, 9, 1000, 70), (128, 40, 900, 300), (32, 100, 4000, 900)])
def test_plan_and_trim_follow_the_oracle_over_many_steps(block, max_reqs, ctx, top):
    """Prompts, decode steps, drafts taken back and requests that finish, until the ring has gone round."""
    rng = np.random.default_rng(block + max_reqs)
    width = -(-ctx // block)
    total = max_reqs * width
    tables = BlockTables(total, max_reqs, width, DEV, block_size=block)
    ref = oracle.Tables(total, max_reqs, width, block)
    mapped = torch.zeros(max_reqs, ctx, dtype=torch.int32, device=DEV)
    want_map = np.zeros((max_reqs, ctx), dtype=np.int64)
    length = np.zeros(max_reqs, dtype=np.int64)
    for step in range(30):
        bs = int(rng.integers(1, max_reqs + 1))
        reqs = rng.permutation(max_reqs)[:bs]
        prefix = length[reqs]
        seq = np.minimum(prefix + np.where(prefix == 0, rng.integers(0, top + 1, bs), rng.integers(0, 6, bs)), ctx)
        n = int((seq - prefix).sum())
        pad = int(rng.integers(0, 4))
        slots, offsets = tables.plan(_dev(reqs), _dev(seq), _dev(prefix), n + pad, req_to_token=mapped)
        w_slots, w_offsets, failed = ref.plan(reqs, seq, prefix, n + pad)
        tables.synchronize()
        assert not failed
        assert slots.cpu().numpy().tolist() == w_slots.tolist()
        assert offsets.cpu().numpy().tolist() == w_offsets.tolist()
        for r, p, s, at in zip(reqs, prefix, seq, w_offsets):
            want_map[r, p:s] = w_slots[at:at + s - p]
        assert torch.equal(mapped.cpu().long(), torch.from_numpy(want_map))
        _assert_tables(tables, ref)
        length[reqs] = seq
        back = rng.permutation(max_reqs)[:int(rng.integers(0, max_reqs + 1))]
        keep = np.where(rng.random(len(back)) < 0.3, 0, np.maximum(length[back] - rng.integers(0, 3, len(back)), 0))
        tables.trim(_dev(back), _dev(keep))
        ref.trim(back, keep)
        length[back] = np.minimum(length[back], keep)
        _assert_tables(tables, ref)
    tables.trim(torch.arange(max_reqs, device=DEV))  # all finished
    tables.synchronize()
    assert tables.available() == total and int(tables.held.sum()) == 0


@pytest.mark.parametrize("bs", [1, 700, 1025, 4096])
def test_plan_of_large_batches(bs):
    """One token each, and 20 each: the slots of one CTA, and of a grid of their own."""
    block, width = 16, 4
    for new in (1, 20):
        tables = BlockTables(bs * width, bs, width, DEV, block_size=block)
        ref = oracle.Tables(bs * width, bs, width, block)
        reqs = np.random.default_rng(bs).permutation(bs)
        for at in range(2):
            seq, prefix = np.full(bs, (at + 1) * new), np.full(bs, at * new)
            slots, offsets = tables.plan(_dev(reqs), _dev(seq), _dev(prefix), bs * new)
            w_slots, w_offsets, _ = ref.plan(reqs, seq, prefix, bs * new)
            tables.synchronize()
            assert slots.cpu().numpy().tolist() == w_slots.tolist()
            assert offsets.cpu().numpy().tolist() == w_offsets.tolist()
        _assert_tables(tables, ref)


@pytest.mark.parametrize("bs", [1735, 1745, 1754, 1755, 1760])
def test_plan_and_trim_where_shared_memory_passes_48_kib(bs):
    """The kernel's own shared arrays count towards the default limit as well."""
    for new in (1, 3):
        tables = BlockTables(bs, bs, 1, DEV, block_size=16)
        slots, _ = tables.plan(torch.arange(bs), torch.full((bs,), new), torch.zeros(bs, dtype=torch.int64), bs * new)
        assert slots.view(bs, new)[:, 0].tolist() == [16 * i for i in range(bs)]
        tables.trim(torch.arange(bs))
        tables.synchronize()
        assert tables.available() == bs


@pytest.mark.parametrize("big", [False, True])
def test_plan_short_of_blocks_leaves_the_rest_as_it_was(big):
    """The entries behind the last free block get nothing, an entry that needs none is served."""
    block, grow = 16, 2000 if big else 20
    need = -(-grow // block)
    tables = BlockTables(2 * need + 1, 6, 200, DEV, block_size=block)
    ref = oracle.Tables(2 * need + 1, 6, 200, block)
    for reqs, seq, prefix in (([4], [3], [0]), ([1, 2, 3, 4], [grow, grow, grow, 9], [0, 0, 0, 3])):
        n = sum(seq) - sum(prefix)
        slots, _ = tables.plan(reqs, seq, prefix, n)
        w_slots, _, failed = ref.plan(reqs, seq, prefix, n)
        torch.cuda.synchronize()
        assert slots.cpu().numpy().tolist() == w_slots.tolist()
    assert failed == [2]
    with pytest.raises(RuntimeError, match="no free block"):
        tables.check_errors()
    tables.check_errors()  # reported once
    _assert_tables(tables, ref)


@pytest.mark.parametrize(("reqs", "seq", "prefix"), [
    ([0, 7, 1], [5, 5, 5], [0, 0, 0]),        # a request out of range
    ([0, -1, 1], [5, 5, 5], [0, 0, 0]),
    ([0, 2, 1], [5, 4, 5], [0, 5, 0]),        # a prefix past the length
    ([0, 2, 1], [5, 4, 5], [0, -1, 0]),
    ([0, 2, 1], [5, 65, 5], [0, 60, 0]),      # past the table's width
    ([1, 1, 0], [20, 40, 5], [0, 20, 0]),     # a request named twice: the first entry counts
])
def test_plan_refuses_bad_entries_and_serves_the_others(reqs, seq, prefix):
    tables = BlockTables(20, 3, 4, DEV, block_size=16)
    ref = oracle.Tables(20, 3, 4, 16)
    n = 64
    slots, offsets = tables.plan(reqs, seq, prefix, n)
    w_slots, w_offsets, failed = ref.plan(reqs, seq, prefix, n)
    torch.cuda.synchronize()
    assert failed
    assert slots.cpu().numpy().tolist() == w_slots.tolist()
    assert offsets.cpu().numpy().tolist() == w_offsets.tolist()
    with pytest.raises(RuntimeError):
        tables.check_errors()
    _assert_tables(tables, ref)


def test_padding_entries_are_not_looked_at():
    tables = BlockTables(20, 3, 4, DEV, block_size=16)
    slots, offsets = tables.plan([2, 99, -5, 0], [3, 0, 0, 2], [0, 7, -1, 0], 8)
    tables.trim([-1, 2, -1], [4, 1, 9])
    tables.synchronize()
    assert offsets.tolist() == [0, 3, 3, 3, 5]
    assert slots.tolist() == [0, 1, 2, 16, 17, -1, -1, -1]
    slots, offsets = tables.plan([], [], [], 2)
    tables.trim([])
    tables.synchronize()
    assert slots.tolist() == [-1, -1] and offsets.tolist() == [0]


def test_trim_refuses_bad_entries():
    tables = BlockTables(20, 3, 4, DEV, block_size=16)
    tables.plan([0, 1], [60, 60], [0, 0], 120)
    for reqs, keep in (([3], [0]), ([0], [-1]), ([1, 1], [40, 0])):
        tables.trim(reqs, keep)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError):
            tables.check_errors()
    assert tables.held.tolist() == [4, 3, 0]  # the first entry of a request counts
    # a table whose blocks the ring has already: nothing is given back
    bad = BlockTables.from_tensors(tables.block_table, tables.held, tables.free_blocks,
                                   torch.tensor([0, 20], device=DEV), 16)
    bad.trim([0])
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        bad.check_errors()
    assert tables.held.tolist() == [4, 3, 0]


# ---------------------------------------------------------------- append and gather


def _cache(blocks, kv, block, dim, seed, layers=1, scales=None):
    """A cache of random codes (no NaN) and power-of-two scales, and its numpy twin per layer."""
    rng = np.random.default_rng(seed)
    k, v, ks, vs = [], [], [], []
    for _ in range(layers):
        for codes, sc in ((k, ks), (v, vs)):
            c = rng.integers(0, 256, (blocks, kv, block, dim), dtype=np.uint8)
            c[(c & 0x7F) == 0x7F] ^= 1
            codes.append(c)
            sc.append(np.ldexp(1.0, rng.integers(-9, -5, (blocks, kv))).astype(np.float32)
                      if scales is None else scales(rng, (blocks, kv)))
    cache = KV8Cache.from_tensors(
        [torch.from_numpy(c.copy()).to(DEV).view(torch.float8_e4m3fn) for c in k],
        [torch.from_numpy(c.copy()).to(DEV).view(torch.float8_e4m3fn) for c in v],
        [torch.from_numpy(s.copy()).to(DEV) for s in ks], [torch.from_numpy(s.copy()).to(DEV) for s in vs])
    return cache, k, v, ks, vs


def _assert_cache(cache, layer, k, v, ks, vs):
    for got, want in ((cache.k, k), (cache.v, v)):
        g = got[layer].view(torch.uint8).cpu().numpy()
        nan = (g & 0x7F) == 0x7F
        assert np.array_equal(nan, (want & 0x7F) == 0x7F)
        assert np.array_equal(np.where(nan, 0, g), np.where(nan, 0, want))
    assert np.array_equal(cache.k_scale[layer].cpu().numpy(), ks)
    assert np.array_equal(cache.v_scale[layer].cpu().numpy(), vs)


def _runs(rng, blocks, block, count, longest):
    """Runs of consecutive slots in distinct blocks, with padding between them now and then."""
    out = []
    for b in rng.permutation(blocks)[:count]:
        off = int(rng.integers(0, block)) if rng.random() < 0.6 else 0
        n = int(rng.integers(1, min(longest, block - off) + 1))
        out += list(range(b * block + off, b * block + off + n))
        if rng.random() < 0.2:
            out += [-1] * int(rng.integers(1, 4))
    return np.array(out, dtype=np.int64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("block", "kv", "dim", "count", "longest"), [
    (64, 4, 128, 1, 1), (64, 4, 128, 70, 1), (64, 4, 128, 30, 64), (16, 1, 8, 40, 16), (32, 3, 24, 40, 5),
    (128, 2, 256, 9, 128), (16, 9, 64, 120, 16)])
def test_append_writes_the_oracles_codes_and_scales(dtype, block, kv, dim, count, longest):
    blocks = count + 3
    cache, k, v, ks, vs = _cache(blocks, kv, block, dim, seed=block + dim)
    rng = np.random.default_rng(7 * block + kv)
    for step in range(2):
        slots = _runs(rng, blocks, block, count, longest)
        grow = np.where(rng.random((len(slots), 1, 1)) < 0.3, 40.0, 1.0) * np.exp2(rng.integers(-30, 3, (1, kv, 1)))
        x = [torch.from_numpy(rng.standard_normal((len(slots), kv, dim)) * grow).to(dtype) for _ in range(2)]
        x[1][:, 0] = 0  # a head of zeros
        cache.append(0, x[0].to(DEV), x[1].to(DEV), _dev(slots))
        cache.synchronize()
        oracle.append(k[0], ks[0], x[0].double().numpy(), slots)
        oracle.append(v[0], vs[0], x[1].double().numpy(), slots)
        _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])
    for out in (torch.bfloat16, torch.float32):
        probe = np.concatenate([rng.integers(0, blocks * block, 200), [-1, 0, blocks * block - 1]])
        got = cache.gather(0, _dev(probe), dtype=out)
        cache.synchronize()
        for g, c, s in zip(got, (k[0], v[0]), (ks[0], vs[0])):
            want = torch.from_numpy(oracle.rows(c, s, probe)).to(out)  # four bits times a power of two: exact
            assert torch.equal(g.cpu(), want)


def test_append_of_a_long_prompt_crosses_its_windows():
    """20,000 tokens in blocks of 64 at every alignment of run and window; slots of one block in one run."""
    block, kv, dim = 64, 1, 16
    slots, b = [], 0
    rng = np.random.default_rng(3)
    while len(slots) < 20000:
        off = int(rng.integers(0, block)) if rng.random() < 0.3 else 0
        n = block - off if rng.random() < 0.8 else int(rng.integers(1, block - off + 1))
        slots += list(range(b * block + off, b * block + off + n))
        b += 1
    slots = np.array(slots, dtype=np.int64)
    cache, k, v, ks, vs = _cache(b, kv, block, dim, seed=1)
    x = [torch.from_numpy(rng.standard_normal((len(slots), kv, dim))).to(torch.bfloat16) for _ in range(2)]
    cache.append(0, x[0].to(DEV), x[1].to(DEV), _dev(slots))
    cache.synchronize()
    oracle.append(k[0], ks[0], x[0].double().numpy(), slots)
    oracle.append(v[0], vs[0], x[1].double().numpy(), slots)
    _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])


def test_append_keeps_a_callers_scales_and_the_ends_of_the_range():
    """Scales that are no powers of two; zeros, subnormals, the largest fp32, infinities and NaN."""
    cache, k, v, ks, vs = _cache(4, 1, 16, 8, seed=2, scales=lambda r, s: (0.01 + r.random(s)).astype(np.float32))
    rows = np.zeros((12, 1, 8), dtype=np.float32)
    rows[0, 0, :3] = [1e-40, -1e-42, 0.0]
    rows[1, 0, :4] = [3.4028235e38, -3.4028235e38, 1.0, 448.0]
    rows[2, 0, :4] = [np.inf, -np.inf, np.nan, 0.5]
    rows[3, 0, :5] = [np.nan] * 5
    rows[4, 0, :6] = [448, -449, 464, 463.9, 480, 2.0 ** -9]
    rows[5:, 0] = np.random.default_rng(0).standard_normal((7, 8))
    slots = np.array([0, 16, 32, 48, 5, 6, 7, 20, 21, 36, 37, 38])
    for a, b in ((0, 4), (4, 12)):
        cache.append(0, torch.from_numpy(rows[a:b]).to(DEV), torch.from_numpy(-rows[a:b]).to(DEV), _dev(slots[a:b]))
        oracle.append(k[0], ks[0], rows[a:b], slots[a:b])
        oracle.append(v[0], vs[0], -rows[a:b], slots[a:b])
        cache.synchronize()
        _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])


def test_append_takes_strided_rows_and_other_layers_stay():
    cache, k, v, ks, vs = _cache(6, 2, 32, 64, seed=4, layers=3)
    rng = np.random.default_rng(5)
    qkv = torch.from_numpy(rng.standard_normal((40, 2 + 2 + 4, 64))).to(torch.bfloat16).to(DEV)
    slots = np.concatenate([np.arange(64, 96), np.arange(130, 138)])
    spread = torch.empty(80, dtype=torch.int64, device=DEV)
    spread[::2] = _dev(slots)
    cache.append(1, qkv[:, 4:6], qkv[:, 6:8], spread[::2])           # heads of a fused projection
    oracle.append(k[1], ks[1], qkv[:, 4:6].double().cpu().numpy(), slots)
    oracle.append(v[1], vs[1], qkv[:, 6:8].double().cpu().numpy(), slots)
    flipped = qkv[:, :2].transpose(0, 2).contiguous().transpose(0, 2)  # no dense rows
    cache.append(2, flipped, qkv[:, 1:3], _dev(slots))
    oracle.append(k[2], ks[2], qkv[:, :2].double().cpu().numpy(), slots)
    oracle.append(v[2], vs[2], qkv[:, 1:3].double().cpu().numpy(), slots)
    cache.synchronize()
    for layer in range(3):
        _assert_cache(cache, layer, k[layer], v[layer], ks[layer], vs[layer])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_takes_values_off_the_16_byte_grid(dtype):
    """Contiguous rows at an odd element: the kernel's wide loads get an aligned copy."""
    cache, k, v, ks, vs = _cache(4, 2, 16, 24, seed=8)
    x = torch.randn(20 * 48 + 3, dtype=dtype, device=DEV)
    slots = np.arange(16, 36)
    rows = [x[i:i + 20 * 48].view(20, 2, 24) for i in (1, 3)]
    assert all(r.data_ptr() % 16 for r in rows)
    cache.append(0, *rows, _dev(slots))
    cache.synchronize()
    oracle.append(k[0], ks[0], rows[0].double().cpu().numpy(), slots)
    oracle.append(v[0], vs[0], rows[1].double().cpu().numpy(), slots)
    _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])


def test_appends_of_two_streams_into_one_layer():
    """Calls of few and of many thread blocks that overlap, in blocks of their own; afterwards a block met twice is
    found as before, so no call's count was lost."""
    block, kv, dim, blocks = 16, 4, 32, 800
    cache, k, v, ks, vs = _cache(blocks, kv, block, dim, seed=9)
    rng = np.random.default_rng(10)
    streams = [torch.cuda.Stream() for _ in range(2)]
    todo = [[], []]
    for i in range(2):
        own = rng.permutation(np.arange(i * blocks // 2, (i + 1) * blocks // 2))
        for n in (1, 3, 40, 300, 30, 2, 350) * 3:  # blocks: 8 to 2800 thread blocks
            slots = np.concatenate([b * block + np.arange(rng.integers(1, 4)) for b in rng.permutation(own)[:n]])
            x = torch.from_numpy(rng.standard_normal((len(slots), kv, dim))).to(torch.bfloat16)
            todo[i].append((x.to(DEV), _dev(slots), x.double().numpy(), slots))
    torch.cuda.synchronize()
    for a, b in zip(*todo):
        for s, (x, slots, _, _) in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                cache.append(0, x, x, slots)
    torch.cuda.synchronize()
    cache.check_errors()
    for calls in todo:
        for _, _, x, slots in calls:
            oracle.append(k[0], ks[0], x, slots)
            oracle.append(v[0], vs[0], x, slots)
    _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])
    words = cache._state[0, :2].tolist()  # 64 bits: whole calls, none left in parts
    assert words == [0, sum(len(calls) for calls in todo)]
    x = torch.randn(2, kv, dim, device=DEV)
    for _ in range(2):
        cache.append(0, x, x, _dev([3, 3]))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError):
            cache.check_errors()
        cache.append(0, x[:1], x[:1], _dev([3]))
        cache.synchronize()


@pytest.mark.parametrize("slots", [
    [3, 3],              # a slot twice
    [3, 5],              # a block in two stretches
    [5, 4],              # descending
    [0, 1, 16, 17, 2],   # a block met again later
    list(range(48, 64)) + list(range(16, 32)) + [50],
])
def test_append_reports_a_block_met_twice(slots):
    """Each stretch claims its block; all other blocks keep their codes, and the next call is clean."""
    cache, k, v, ks, vs = _cache(4, 1, 16, 16, seed=6)
    x = torch.randn(len(slots), 1, 16, device=DEV)
    cache.append(0, x, x, _dev(slots))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        cache.check_errors()
    untouched = [b for b in range(4) if b not in {s // 16 for s in slots}]
    assert np.array_equal(cache.k[0].view(torch.uint8).cpu().numpy()[untouched], k[0][untouched])
    cache.append(0, x[:1], x[:1], _dev(slots[:1]))
    cache.synchronize()


def test_append_and_gather_report_slots_out_of_range():
    cache, k, v, ks, vs = _cache(4, 1, 16, 16, seed=6)
    x = torch.randn(3, 1, 16, device=DEV)
    cache.append(0, x, x, _dev([64, 10, 1 << 40]))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        cache.check_errors()
    xs = x.double().cpu().numpy()
    oracle.append(k[0], ks[0], xs[1:2], np.array([10]))
    oracle.append(v[0], vs[0], xs[1:2], np.array([10]))
    _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])
    got, _ = cache.gather(0, _dev([64, 10, -2]), dtype=torch.float32)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        cache.check_errors()
    assert got[0].count_nonzero() == 0 and got[2].count_nonzero() == 0
    assert torch.equal(got[1].cpu().double(), torch.from_numpy(oracle.rows(k[0], ks[0], np.array([10])))[0])


def test_no_tokens_is_no_work():
    cache, k, v, ks, vs = _cache(2, 1, 16, 16, seed=1)
    none = torch.empty(0, 1, 16, device=DEV)
    cache.append(0, none, none, _dev([]))
    a, b = cache.gather(0, _dev([]))
    out = cache.decode_attention(0, none.view(0, 1, 16), torch.zeros(1, 1, dtype=torch.int32, device=DEV), [], [], 1.0)
    cache.synchronize()
    assert a.shape == b.shape == (0, 1, 16) and out.shape == (0, 16)
    _assert_cache(cache, 0, k[0], v[0], ks[0], vs[0])


# ---------------------------------------------------------------- attention


SMALL_DECODE = 2.0 ** -21
SMALL_EXTEND = SMALL_DECODE


def _tolerance(dtype, n, dim, out, weight, spread, small, part):
    rel = 2 * (dim + 8) * 2.0 ** -24 * spread[:, None] + 2 * 2.0 ** -22 + 2 * n * 2.0 ** -24
    err = rel * weight
    if dtype == torch.bfloat16:
        err = err + 2.0 ** -8 * weight + part * small
    step = torch.finfo(dtype).eps / 2
    return step * np.abs(out) + (1 + step) * err + 1e-37


class _Batch:
    """Requests over scattered blocks, with NaN codes and NaN scales wherever no live token is."""

    def __init__(self, seq, kv, dim, block, seed, heads, dtype, spare=2, scales=None, width=None):
        rng = np.random.default_rng(seed)
        pages = [-(-s // block) for s in seq]
        blocks = sum(pages) + spare
        self.cache, self.k, self.v, self.ks, self.vs = _cache(blocks, kv, block, dim, seed, scales=scales)
        order = rng.permutation(blocks)
        self.reqs = rng.permutation(len(seq) + 2)[:len(seq)]
        table = np.full((len(seq) + 2, width or max(pages + [1])), -1, dtype=np.int64)
        live = np.zeros((blocks, block), dtype=bool)
        at = 0
        for r, s, p in zip(self.reqs, seq, pages):
            table[r, :p] = order[at:at + p]
            at += p
            pos = np.arange(s)
            live[table[r, pos // block], pos % block] = True
        for c in (self.k[0], self.v[0]):
            c[np.broadcast_to(~live[:, None, :, None], c.shape)] = 0x7F
        for s in (self.ks[0], self.vs[0]):
            s[~live.any(1)] = np.nan
        for got, want in ((self.cache.k, self.k), (self.cache.v, self.v)):
            got[0].view(torch.uint8).copy_(torch.from_numpy(want[0]))
        self.cache.k_scale[0].copy_(torch.from_numpy(self.ks[0]))
        self.cache.v_scale[0].copy_(torch.from_numpy(self.vs[0]))
        self.seq, self.table, self.block, self.dtype, self.dim = list(seq), table, block, dtype, dim
        self.table_dev = _dev(table, torch.int32)
        self.scaling = dim ** -0.5
        self.rng, self.heads = rng, heads

    def queries(self, n):
        return torch.from_numpy(self.rng.standard_normal((n, self.heads, self.dim)) * 1.5).to(self.dtype)

    def slots(self, i, positions):
        p = np.asarray(positions)
        return self.table[self.reqs[i], p // self.block] * self.block + p % self.block

    def check(self, got, q, slots, part=SMALL_DECODE):
        k, v = (oracle.rows(c, s, slots) for c, s in ((self.k[0], self.ks[0]), (self.v[0], self.vs[0])))
        q = q.double().numpy()
        scale = self.vs[0][slots // self.block]
        out, weight, spread, small = oracle.attend(q, k, v, self.scaling, scale)
        err = np.abs(got.double().cpu().numpy().reshape(out.shape) - out)
        tol = _tolerance(self.dtype, len(slots), self.dim, out, weight, spread, small, part)
        assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


#: (kv heads, heads, head_dim, block, dtype): the tensor-core geometry, and what goes to the fp32 kernel
GEOMETRIES = [
    (4, 32, 128, 64, torch.bfloat16),
    (2, 2, 128, 16, torch.bfloat16),
    (1, 7, 128, 32, torch.bfloat16),
    (1, 16, 128, 128, torch.bfloat16),
    (2, 40, 128, 64, torch.bfloat16),
    (2, 8, 64, 16, torch.float32),
    (1, 3, 8, 32, torch.float32),
    (3, 3, 256, 64, torch.float32),
    (4, 32, 128, 64, torch.float32),
    (2, 36, 24, 16, torch.bfloat16),
]


@pytest.mark.parametrize(("kv", "heads", "dim", "block", "dtype"), GEOMETRIES)
@pytest.mark.parametrize("seq", [[1], [2, 0, 63, 64, 65], [127, 128, 129, 191, 256, 257], [1000, 3, 5001, 0]])
def test_decode_attention_matches_64_bits(kv, heads, dim, block, dtype, seq):
    b = _Batch(seq, kv, dim, block, seed=sum(seq) + dim, heads=heads, dtype=dtype)
    q = b.queries(len(seq))
    out = b.cache.decode_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), b.scaling)
    b.cache.synchronize()
    for i, s in enumerate(seq):
        if s == 0:
            assert out[i].count_nonzero() == 0
        b.check(out[i], q[i], b.slots(i, np.arange(s)))


@pytest.mark.parametrize(("kv", "heads", "dim", "block", "dtype"), GEOMETRIES)
def test_sparse_decode_attention_matches_64_bits(kv, heads, dim, block, dtype):
    """Pages and recent tokens, single rows in any order, duplicates, padding rows, an entry with none."""
    seq = [3000, 700, 40, 129, 513, 64]
    b = _Batch(seq, kv, dim, block, seed=dim + heads, heads=heads, dtype=dtype)
    top = 8 * max(block, 64)
    rows = np.full((len(seq), top), -7, dtype=np.int64)
    lens = [top, 0, 40, 129, 300, 64]
    rows[0] = b.slots(0, np.concatenate([(b.rng.permutation(3000 // block)[:top // block - 1, None] * block
                                          + np.arange(block)).ravel(), np.arange(3000 - block, 3000)]))
    rows[2, :40] = b.slots(2, np.arange(40))
    rows[3, :129] = b.slots(3, b.rng.integers(0, 129, 129))
    rows[4, :300] = np.where(b.rng.random(300) < 0.3, -1, b.slots(4, b.rng.integers(0, 513, 300)))
    rows[5, :64] = -1  # every row masked: zeros
    q = b.queries(len(seq))
    out = b.cache.sparse_decode_attention(0, q.to(DEV), _dev(rows, torch.int32), _dev(lens, torch.int32), b.scaling)
    b.cache.synchronize()
    for i, n in enumerate(lens):
        r = rows[i, :n]
        b.check(out[i], q[i], r[r >= 0])
    assert out[1].count_nonzero() == 0 and out[5].count_nonzero() == 0


@pytest.mark.parametrize(("kv", "heads", "dim", "block", "dtype"), GEOMETRIES)
@pytest.mark.parametrize(("seq", "new"), [
    ([1], [1]), ([70, 5, 200], [70, 1, 130]), ([300, 0, 129, 1000], [4, 0, 1, 260]), ([640], [515])])
def test_extend_attention_matches_64_bits(kv, heads, dim, block, dtype, seq, new):
    """Whole prompts, chunks behind a prefix, single tokens; rows behind the last sequence stay as they were."""
    b = _Batch(seq, kv, dim, block, seed=sum(seq) + heads, heads=heads, dtype=dtype)
    offsets = np.concatenate([[0], np.cumsum(new)])
    n = int(offsets[-1])
    q = b.queries(n + 3)
    out = torch.full((n + 3, heads * dim), 7.0, dtype=dtype, device=DEV)
    got = b.cache.extend_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), _dev(np.subtract(seq, new)),
                                   _dev(offsets), b.scaling, out=out)
    b.cache.synchronize()
    assert got is out and bool((out[n:] == 7.0).all())
    probe = set(b.rng.integers(0, max(n, 1), 40).tolist()) | {0, 1, n - 1, n - 2}
    for i, (s, m) in enumerate(zip(seq, new)):
        for t in range(m):
            if n > 64 and offsets[i] + t not in probe and t not in (0, m - 1):
                continue
            row = offsets[i] + t
            b.check(out[row], q[row], b.slots(i, np.arange(s - m + t + 1)), SMALL_EXTEND)


@pytest.mark.parametrize(("heads", "dim", "dtype"), [
    (4, 128, torch.bfloat16), (32, 128, torch.bfloat16), (48, 128, torch.bfloat16), (8, 64, torch.float32),
    (24, 40, torch.bfloat16), (64, 256, torch.float32)])
@pytest.mark.parametrize("bs", [1, 2, 3, 6, 12])
@pytest.mark.parametrize("width", [16, 100, 400])
def test_decode_by_clusters_and_by_shares(heads, dim, dtype, bs, width):
    """The table's width and the number of requests decide which form takes a call: a cluster of CTAs to a (request,
    KV head) pair, of three sizes, or equal shares of all tiles."""
    rng = np.random.default_rng(bs + width)
    seq = [1000, 0, 1, 129, 1024, 640, 128, 2, 900, 511, 512, 513][:bs]
    b = _Batch(seq, 4, dim, 64, seed=heads + bs, heads=heads, dtype=dtype, width=width)
    q = b.queries(bs)
    reqs, lens = _dev(b.reqs), _dev(seq)
    out = b.cache.decode_attention(0, q.to(DEV), b.table_dev, reqs, lens, b.scaling)
    again = b.cache.decode_attention(0, q.to(DEV), b.table_dev, reqs, lens, b.scaling)
    top = 16 * width
    rows = np.full((bs, top), -1, dtype=np.int64)
    for i, s in enumerate(seq):
        rows[i, :min(s, top)] = b.slots(i, rng.permutation(s)[:top])
    few = np.minimum(seq, top)
    sparse = b.cache.sparse_decode_attention(0, q.to(DEV), _dev(rows, torch.int32), _dev(few, torch.int32), b.scaling)
    b.cache.synchronize()
    assert torch.equal(out, again)
    for i, s in enumerate(seq):
        if s == 0:
            assert not out[i].count_nonzero() and not sparse[i].count_nonzero()
            continue
        b.check(out[i], q[i], b.slots(i, np.arange(s)))
        b.check(sparse[i], q[i], rows[i, :few[i]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_with_scales_far_apart(dtype):
    """Scales over 2^40 between blocks, and no powers of two: the block with the large values need not be the
    one with the large weights."""
    def scales(rng, shape):
        return (np.exp2(rng.integers(-20, 20, shape)) * (1 + rng.random(shape))).astype(np.float32)

    def k_scales(rng, shape):
        return (0.002 * (1 + rng.random(shape))).astype(np.float32)

    seq = [900, 130]
    b = _Batch(seq, 4, 128, 64, seed=11, heads=32, dtype=dtype, scales=scales)
    b.ks[0] = np.where(np.isnan(b.ks[0]), b.ks[0], k_scales(b.rng, b.ks[0].shape)).astype(np.float32)
    b.cache.k_scale[0].copy_(torch.from_numpy(b.ks[0]))
    q = b.queries(2)
    out = b.cache.decode_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), b.scaling)
    rows = np.stack([b.slots(i, np.arange(130)) for i in range(2)])
    sparse = b.cache.sparse_decode_attention(0, q.to(DEV), _dev(rows, torch.int32), _dev([130, 77], torch.int32),
                                             b.scaling)
    ext = b.cache.extend_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), _dev([899, 129]), _dev([0, 1]),
                                   b.scaling)
    b.cache.synchronize()
    for i, s in enumerate(seq):
        b.check(out[i], q[i], b.slots(i, np.arange(s)))
        b.check(ext[i], q[i], b.slots(i, np.arange(s)), SMALL_EXTEND)
        b.check(sparse[i], q[i], rows[i, :(130, 77)[i]])


@pytest.mark.parametrize(("dtype", "heads"), [(torch.bfloat16, 32), (torch.float32, 32)])
def test_attention_of_unequal_queries(dtype, heads):
    """Query rows from 2^-60 to 2^20, a row of zeros, one dominant key: nothing overflows or vanishes."""
    seq = [400]
    b = _Batch(seq, 4, 128, 64, seed=5, heads=heads, dtype=dtype)
    q = b.queries(1) * torch.exp2(torch.arange(heads) - 28.0)[None, :, None].clamp(max=8.0)
    q[0, 3] = 0
    q = q.to(dtype)
    out = b.cache.decode_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), b.scaling)
    ext = b.cache.extend_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), _dev([399]), _dev([0]), b.scaling)
    b.cache.synchronize()
    b.check(out[0], q[0], b.slots(0, np.arange(400)))
    b.check(ext[0], q[0], b.slots(0, np.arange(400)), SMALL_EXTEND)


def test_a_nan_reaches_the_heads_that_see_it_and_no_others():
    seq = [200, 200]
    for dtype in (torch.bfloat16, torch.float32):
        b = _Batch(seq, 2, 128, 64, seed=8, heads=8, dtype=dtype)
        at = int(b.slots(0, [150])[0])
        b.cache.k[0].view(torch.uint8)[at // 64, 1, at % 64, 5] = 0x7F
        q = b.queries(2)
        q[1, 2, 0] = float("nan")
        args = (b.table_dev, _dev(b.reqs), _dev(seq))
        out = b.cache.decode_attention(0, q.to(DEV), *args, b.scaling).view(2, 8, 128)
        ext = b.cache.extend_attention(0, q.to(DEV), *args, _dev([199, 199]), _dev([0, 1]), b.scaling).view(2, 8, 128)
        b.cache.synchronize()
        for o in (out, ext):
            bad = o.isnan()
            assert bad[0, 4:].all() and not bad[0, :4].any()
            assert bad[1, 2].all() and not bad[1, :2].any() and not bad[1, 3:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_nan_of_a_later_token_stays_behind_the_mask(dtype):
    """Keys and values of token 150 are NaN: the rows up to 149 are what they would be without it."""
    seq = [200]
    b = _Batch(seq, 2, 128, 64, seed=12, heads=8, dtype=dtype)
    at = int(b.slots(0, [150])[0])
    q = b.queries(200)
    args = (_dev(b.reqs), _dev(seq), _dev([0]), _dev([0]), b.scaling)
    want = b.cache.extend_attention(0, q.to(DEV), b.table_dev, *args)
    for codes in (b.cache.k, b.cache.v):
        saved = codes[0].clone()
        codes[0].view(torch.uint8)[at // 64, 1, at % 64, 5] = 0xFF
        got = b.cache.extend_attention(0, q.to(DEV), b.table_dev, *args).view(200, 8, 128)
        b.cache.synchronize()
        assert torch.equal(got[:150].reshape(150, -1), want[:150]) and torch.equal(got[:, :4], want.view(200, 8, 128)[:, :4])
        assert got[150:, 4:, 5].isnan().all()
        codes[0].view(torch.uint8).copy_(saved.view(torch.uint8))


def test_attention_reports_bad_entries_and_serves_the_others():
    seq = [100, 70, 90]
    for dtype in (torch.bfloat16, torch.float32):
        b = _Batch(seq, 4, 128, 64, seed=9, heads=32, dtype=dtype, width=2)
        q = b.queries(3)
        for reqs, lens in (([b.reqs[0], 99, b.reqs[2]], seq), ([b.reqs[0], -1, b.reqs[2]], seq),
                           (b.reqs, [100, 129, 90]), (b.reqs, [100, -3, 90])):
            out = b.cache.decode_attention(0, q.to(DEV), b.table_dev, _dev(reqs), _dev(lens), b.scaling)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError):
                b.cache.check_errors()
            assert out[1].count_nonzero() == 0
            ext = torch.full((3, 32 * 128), 7.0, dtype=dtype, device=DEV)
            b.cache.extend_attention(0, q.to(DEV), b.table_dev, _dev(reqs), _dev(lens), _dev(np.array(lens) - 1),
                                     _dev([0, 1, 2]), b.scaling, out=ext)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError):
                b.cache.check_errors()
            assert bool((ext[1] == 7.0).all())
            for i in (0, 2):
                b.check(out[i], q[i], b.slots(i, np.arange(seq[i])))
                b.check(ext[i], q[i], b.slots(i, np.arange(seq[i])), SMALL_EXTEND)
        # a block out of range takes no part
        broken = b.table_dev.clone()
        broken[b.reqs[1], 0] = 1 << 20
        out = b.cache.decode_attention(0, q.to(DEV), broken, _dev(b.reqs), _dev(seq), b.scaling)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError):
            b.cache.check_errors()
        ext = b.cache.extend_attention(0, q.to(DEV), broken, _dev(b.reqs), _dev(seq), _dev(np.array(seq) - 1),
                                       _dev([0, 1, 2]), b.scaling)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError):
            b.cache.check_errors()
        for i in range(3):
            left = np.arange(64 if i == 1 else 0, seq[i])
            b.check(out[i], q[i], b.slots(i, left))
            b.check(ext[i], q[i], b.slots(i, left), SMALL_EXTEND)
        rows = np.stack([b.slots(i, np.arange(64)) for i in range(3)])
        rows[1, 10] = 1 << 30
        out = b.cache.sparse_decode_attention(0, q.to(DEV), _dev(rows, torch.int32), _dev([64, 64, 65], torch.int32),
                                              b.scaling)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError):
            b.cache.check_errors()
        b.check(out[0], q[0], rows[0])
        b.check(out[1], q[1], np.delete(rows[1], 10))
        assert out[2].count_nonzero() == 0  # more rows than the list has


def test_attention_takes_strided_queries_tables_and_outputs():
    seq = [333, 64]
    for dtype in (torch.bfloat16, torch.float32):
        b = _Batch(seq, 2, 128, 32, seed=10, heads=8, dtype=dtype)
        qkv = torch.from_numpy(b.rng.standard_normal((2, 12, 128))).to(dtype).to(DEV)
        q = qkv[:, :8]
        wide = torch.zeros(b.table_dev.shape[0], 2 * b.table_dev.shape[1], dtype=torch.int32, device=DEV)
        wide[:, ::2] = b.table_dev
        want = b.cache.decode_attention(0, q.contiguous(), b.table_dev, _dev(b.reqs), _dev(seq), b.scaling)
        room = torch.zeros(2, 8 * 128 + 256, dtype=dtype, device=DEV)
        out = b.cache.decode_attention(0, q, wide[:, ::2], b.reqs.tolist(), seq, b.scaling, out=room[:, 128:-128])
        odd = torch.empty(2 * 8 * 128 + 1, dtype=dtype, device=DEV)[1:].view(2, 8, 128)
        odd.copy_(q)
        odd_out = torch.empty(2 * 8 * 128 + 1, dtype=dtype, device=DEV)[1:].view(2, 8 * 128)
        b.cache.decode_attention(0, odd, b.table_dev, _dev(b.reqs), _dev(seq), b.scaling, out=odd_out)
        b.cache.synchronize()
        assert torch.equal(out, want)
        for i, n in enumerate(seq):  # an unaligned result is another kernel's
            b.check(odd_out[i], q[i].cpu(), b.slots(i, np.arange(n)))
        assert room[:, :128].count_nonzero() == 0 and room[:, -128:].count_nonzero() == 0


def test_results_do_not_depend_on_the_batch_or_the_call():
    """Run twice: bit-identical."""
    seq = [5000, 1, 777, 64, 4097]
    b = _Batch(seq, 4, 128, 64, seed=21, heads=32, dtype=torch.bfloat16)
    q = b.queries(5).to(DEV)
    args = (b.table_dev, _dev(b.reqs), _dev(seq))
    first = b.cache.decode_attention(0, q, *args, b.scaling)
    again = b.cache.decode_attention(0, q, *args, b.scaling)
    assert torch.equal(first, again)


@pytest.mark.parametrize("dim", [128, 136, 144])
@pytest.mark.parametrize("heads", [3, 7, 12])
def test_fp32_kernel_where_shared_memory_passes_48_kib(dim, heads):
    seq, new = [70, 5], [20, 5]
    b = _Batch(seq, 1, dim, 16, seed=dim + heads, heads=heads, dtype=torch.float32)
    q = b.queries(25)
    lens = _dev(b.reqs), _dev(seq)
    out = b.cache.extend_attention(0, q.to(DEV), b.table_dev, *lens, _dev([50, 0]), _dev([0, 20]), b.scaling)
    one = b.cache.decode_attention(0, q[:2].to(DEV), b.table_dev, *lens, b.scaling)
    b.cache.synchronize()
    b.check(out[19], q[19], b.slots(0, np.arange(70)), SMALL_EXTEND)
    b.check(out[24], q[24], b.slots(1, np.arange(5)), SMALL_EXTEND)
    for i in range(2):
        b.check(one[i], q[i], b.slots(i, np.arange(seq[i])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extend_of_ragged_chunks_in_every_cut(dtype):
    """From fewer query tiles than SMs, all of whose keys are cut, to whole tiles with a cut rest (bf16: 256 rows)."""
    kv, heads, dim, block = 4, 32, 128, 64
    for seq, new in (([2600], [3]), ([700, 2000], [300, 600]), ([900, 1500, 1300], [900, 500, 10])):
        if dtype == torch.float32 and len(seq) == 3:
            continue
        b = _Batch(seq, kv, dim, block, seed=sum(new), heads=heads, dtype=dtype)
        offsets = np.concatenate([[0], np.cumsum(new)])
        q = b.queries(int(offsets[-1]))
        out = b.cache.extend_attention(0, q.to(DEV), b.table_dev, _dev(b.reqs), _dev(seq), _dev(np.subtract(seq, new)),
                                       _dev(offsets), b.scaling)
        b.cache.synchronize()
        for i, (s, m) in enumerate(zip(seq, new)):
            for t in sorted({0, 1, m // 2, m - 2, m - 1} & set(range(m))):
                row = offsets[i] + t
                b.check(out[row], q[row], b.slots(i, np.arange(s - m + t + 1)), SMALL_EXTEND)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extend_reports_entries_that_share_rows(dtype):
    n = 512
    b = _Batch([n, n, n], 4, 128, 64, seed=41, heads=32, dtype=dtype)
    q = b.queries(n).to(DEV)
    lens = _dev([n, n, n]), _dev([0, 0, 0])
    b.cache.extend_attention(0, q, b.table_dev, _dev(b.reqs), *lens, _dev([0, 0, 0]), b.scaling)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        b.cache.check_errors()
    one = b.cache.extend_attention(0, q, b.table_dev, _dev(b.reqs[:1]), lens[0][:1], lens[1][:1], _dev([0]), b.scaling)
    b.cache.synchronize()
    b.check(one[n - 1], q[n - 1].cpu(), b.slots(0, np.arange(n)), SMALL_EXTEND)


@pytest.mark.parametrize(("kv", "heads", "dim", "dtype"), [(4, 8, 128, torch.bfloat16), (2, 4, 32, torch.float32)])
def test_attention_of_the_largest_batch(kv, heads, dim, dtype):
    bs = 4096
    rng = np.random.default_rng(2)
    seq = rng.integers(0, 40, bs)
    b = _Batch(seq, kv, dim, 16, seed=43, heads=heads, dtype=dtype)
    q = b.queries(bs)
    reqs, lens = _dev(b.reqs), _dev(seq)
    out = b.cache.decode_attention(0, q.to(DEV), b.table_dev, reqs, lens, b.scaling)
    prefix = np.maximum(seq - 1, 0)
    offsets = np.concatenate([[0], np.cumsum(seq - prefix)])
    few = q[:offsets[-1]]
    ext = b.cache.extend_attention(0, few.to(DEV), b.table_dev, reqs, lens, _dev(prefix), _dev(offsets), b.scaling)
    b.cache.synchronize()
    for i in [*range(0, bs, 97), bs - 1]:
        if seq[i] == 0:
            assert not out[i].count_nonzero()
            continue
        b.check(out[i], q[i], b.slots(i, np.arange(seq[i])))
        b.check(ext[offsets[i]], few[offsets[i]], b.slots(i, np.arange(seq[i])), SMALL_EXTEND)


def test_a_cache_past_32_bits_of_codes():
    """Blocks whose codes lie beyond 2^32 bytes: written, read back and attended to."""
    kv, heads, dim, block = 4, 32, 128, 64
    blocks = 2 ** 32 // (kv * block * dim) + 40
    cache = KV8Cache(1, blocks, kv, dim, DEV, block_size=block)
    n = 10 * block + 5
    chosen = [blocks - 1 - 3 * i for i in range(11)]
    slots = np.concatenate([b * block + np.arange(block) for b in chosen])[:n]
    rng = np.random.default_rng(12)
    k, v = (torch.from_numpy(rng.standard_normal((n, kv, dim))).to(torch.bfloat16) for _ in range(2))
    cache.append(0, k.to(DEV), v.to(DEV), _dev(slots))
    q = torch.from_numpy(rng.standard_normal((1, heads, dim))).to(torch.bfloat16)
    table = _dev([chosen], torch.int32)
    outs = [cache.decode_attention(0, q.to(DEV), table, [0], [n], dim ** -0.5),
            cache.sparse_decode_attention(0, q.to(DEV), _dev([slots], torch.int32), [n], dim ** -0.5),
            cache.extend_attention(0, q.to(DEV), table, [0], [n], [n - 1], [0], dim ** -0.5)]
    wide = cache.decode_attention(0, q.float().to(DEV), table, [0], [n], dim ** -0.5)
    got = cache.gather(0, _dev(slots), dtype=torch.float32)
    cache.synchronize()
    small = [np.zeros((11, kv, block, dim), dtype=np.uint8) for _ in range(2)]
    scales = [np.zeros((11, kv), dtype=np.float32) for _ in range(2)]
    place = np.arange(n)
    rows = []
    for c, s, x in zip(small, scales, (k, v)):
        oracle.append(c, s, x.double().numpy(), place)
        rows.append(oracle.rows(c, s, place))
    for g, want in zip(got, rows):
        assert np.array_equal(g.double().cpu().numpy(), want)
    out, *bounds = oracle.attend(q[0].double().numpy(), *rows, dim ** -0.5, scales[1][place // block])
    for o, dtype in [(x, torch.bfloat16) for x in outs] + [(wide, torch.float32)]:
        tol = _tolerance(dtype, n, dim, out, *bounds, SMALL_DECODE)
        assert (np.abs(o[0].double().cpu().numpy().reshape(out.shape) - out) <= tol).all()


# ---------------------------------------------------------------- streams, graphs, the step as a whole


def test_a_captured_step_replays_over_new_lengths():
    """Plan, append, decode and trim captured once; every replay reads the lengths of its step, and two graphs
    and an eager call in between share nothing."""
    kv, heads, dim, block, bs = 4, 32, 128, 64, 6
    tables = BlockTables(80, bs, 10, DEV, block_size=block)
    cache = KV8Cache(1, 80, kv, dim, DEV, block_size=block)
    k_ref, v_ref = (np.zeros((80, kv, block, dim), dtype=np.uint8) for _ in range(2))
    ks_ref, vs_ref = (np.zeros((80, kv), dtype=np.float32) for _ in range(2))
    ref = oracle.Tables(80, bs, 10, block)
    rng = np.random.default_rng(0)
    seq = np.array([60, 1, 63, 128, 200, 64])
    reqs = np.arange(bs)
    reqs_dev, seq_dev, prefix_dev = _dev(reqs), _dev(seq), _dev(np.zeros(bs))

    def put(slots, k, v):
        oracle.append(k_ref, ks_ref, k.double().cpu().numpy(), slots)
        oracle.append(v_ref, vs_ref, v.double().cpu().numpy(), slots)

    def rand(n, h):
        return torch.from_numpy(rng.standard_normal((n, h, dim))).to(torch.bfloat16).to(DEV)

    n = int(seq.sum())
    slots, _ = tables.plan(reqs_dev, seq_dev, prefix_dev, n)
    k, v = rand(n, kv), rand(n, kv)
    cache.append(0, k, v, slots)
    w_slots, _, _ = ref.plan(reqs, seq, 0 * seq, n)
    put(w_slots, k, v)
    k, v, q = rand(bs, kv), rand(bs, kv), rand(bs, heads)

    def step():
        slots, offsets = tables.plan(reqs_dev, seq_dev, prefix_dev, bs)
        cache.append(0, k, v, slots)
        one = cache.decode_attention(0, q, tables.block_table, reqs_dev, seq_dev, dim ** -0.5)
        two = cache.extend_attention(0, q, tables.block_table, reqs_dev, seq_dev, prefix_dev, offsets, dim ** -0.5)
        return one, two

    graphs = []
    keep = (tables.block_table.clone(), tables.held.clone(), tables.free_blocks.clone(), tables.ring.clone())
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for a, t in zip(keep, (tables.block_table, tables.held, tables.free_blocks, tables.ring)):
        assert torch.equal(a, t)  # capturing ran nothing
    for i in range(8):
        prefix, seq = seq.copy(), seq + 1
        seq_dev.copy_(_dev(seq)), prefix_dev.copy_(_dev(prefix))
        for t in (k, v):
            t.copy_(rand(bs, kv))
        q.copy_(rand(bs, heads))
        if i == 3:
            one, two = step()
        else:
            g, (one, two) = graphs[i % 2]
            g.replay()
        w_slots, _, _ = ref.plan(reqs, seq, prefix, bs)
        put(w_slots, k, v)
        tables.synchronize()
        cache.check_errors()
        _assert_cache(cache, 0, k_ref, v_ref, ks_ref, vs_ref)
        for r in range(bs):
            pos = np.arange(seq[r])
            at = ref.table[r, pos // block] * block + pos % block
            kk, vv = oracle.rows(k_ref, ks_ref, at), oracle.rows(v_ref, vs_ref, at)
            out, *bounds = oracle.attend(q[r].double().cpu().numpy(), kk, vv, dim ** -0.5, vs_ref[at // block])
            for got, part in ((one, SMALL_DECODE), (two, SMALL_EXTEND)):
                tol = _tolerance(torch.bfloat16, len(at), dim, out, *bounds, part)
                assert (np.abs(got[r].double().cpu().numpy().reshape(out.shape) - out) <= tol).all()


def test_two_streams_read_one_cache_at_once():
    seq = [3000, 500, 64, 4000]
    b = _Batch(seq, 4, 128, 64, seed=31, heads=32, dtype=torch.bfloat16)
    q = [b.queries(4).to(DEV) for _ in range(2)]
    args = (b.table_dev, _dev(b.reqs), _dev(seq))
    want = [b.cache.decode_attention(0, x, *args, b.scaling) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(b.cache.decode_attention(0, q[i], *args, b.scaling))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_selection_over_the_8_bit_cache():
    """The page selection's own kernels next to the cache: bounds from the new keys, pages selected, their positions
    translated through the map that the plan filled, attention over exactly those rows."""
    from qwenquest_b200 import _lib

    lib = _lib.load()
    kv, heads, dim, page, top, ctx = 4, 32, 128, 64, 256, 1500
    lens = [1500, 700, 200]
    bs = len(lens)
    tables = BlockTables(60, bs, -(-ctx // page), DEV, block_size=page)
    cache = KV8Cache(1, 60, kv, dim, DEV, block_size=page)
    mapped = torch.zeros(bs, ctx, dtype=torch.int32, device=DEV)
    reqs, seq = _dev(range(bs)), _dev(lens)
    n = sum(lens)
    slots, offsets = tables.plan(reqs, seq, [0] * bs, n, req_to_token=mapped)
    g = torch.Generator().manual_seed(0)
    k = torch.randn(n, kv, dim, generator=g).to(torch.bfloat16).to(DEV)
    v = torch.randn(n, kv, dim, generator=g).to(torch.bfloat16).to(DEV)
    q = torch.randn(bs, heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    cache.append(0, k, v, slots)
    pages = -(-ctx // page)
    i32 = dict(dtype=torch.int32, device=DEV)
    bounds = torch.empty(1, bs, pages, kv, dim, 2, dtype=torch.bfloat16, device=DEV)
    low, high = (torch.empty(1, bs, kv, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    count, index = torch.zeros(bs, **i32), torch.zeros(bs, **i32)
    st = _lib.QQQuestState(bounds.data_ptr(), low.data_ptr(), high.data_ptr(), count.data_ptr(), index.data_ptr(),
                           1, bs, pages, kv, dim, page, top, 0)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.qq_quest_init_storage(st, stream) == 0
    for i, m in enumerate(lens):  # the bounds need no bf16 pool: the new keys are rows of their own
        rows = torch.arange(int(offsets[i]), int(offsets[i]) + m, **i32)
        arr, keep = _lib.ptr_array([k.data_ptr()])
        assert lib.qq_quest_bounds_prefill(st, 0, 1, arr, 0, k.stride(0), rows.data_ptr(), m, i, 1, stream) == 0
    ws = torch.zeros(int(lib.qq_workspace_bytes(bs, top, heads, dim)), dtype=torch.uint8, device=DEV)
    positions, rows = torch.empty(bs, top, **i32), torch.empty(bs, top, **i32)
    actual = torch.empty(bs, **i32)
    scores = torch.empty(bs, pages, dtype=torch.float32, device=DEV)
    batch = _lib.QQBatch(reqs.data_ptr(), seq.data_ptr(), bs)
    table = _lib.QQTokenTable(mapped.data_ptr(), mapped.stride(0), bs)
    assert lib.qq_quest_retrieve_topk(st, 0, batch, q.data_ptr(), 0, heads, q.stride(0), positions.data_ptr(),
                                      actual.data_ptr(), scores.data_ptr(), table, rows.data_ptr(), None,
                                      ws.data_ptr(), ws.numel(), stream) == 0
    out = cache.sparse_decode_attention(0, q, rows, actual, dim ** -0.5)
    cache.synchronize()
    codes = [t.view(torch.uint8).cpu().numpy() for t in (cache.k[0], cache.v[0])]
    scales = [t.cpu().numpy() for t in (cache.k_scale[0], cache.v_scale[0])]
    for i, m in enumerate(lens):
        pos = positions[i, :min(m, top)].cpu().numpy()
        at = mapped[i].cpu().numpy()[pos]
        assert at.tolist() == rows[i, :len(pos)].tolist()
        kk, vv = (oracle.rows(c, s, at.astype(np.int64)) for c, s in zip(codes, scales))
        want, *bounds = oracle.attend(q[i].double().cpu().numpy(), kk, vv, dim ** -0.5, scales[1][at // page])
        tol = _tolerance(torch.bfloat16, len(at), dim, want, *bounds, SMALL_DECODE)
        assert (np.abs(out[i].double().cpu().numpy().reshape(want.shape) - want) <= tol).all()
