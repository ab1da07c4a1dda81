"""The 8-bit cache's tables, writes and arguments at their edges, against the numpy restatement (``oracle/kv8.py``)."""

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


@pytest.mark.parametrize("grow", [5, 5000])
@pytest.mark.parametrize(("reqs", "live"), [([0, 0], [0, 1]), ([2, 0, 2, 1, 2], [0, 0, 0, 1, 1]), ([1, 1], [1, 0])])
def test_a_padding_entry_may_name_a_live_request(reqs, live, grow):
    """An entry of length 0 is not looked at: a finished slot of a fixed batch keeps its old request number."""
    tables = BlockTables(700, 3, 350, DEV, block_size=16)
    ref = oracle.Tables(700, 3, 350, 16)
    seq = np.array(live) * grow
    n = int(seq.sum())
    slots, offsets = tables.plan(_dev(reqs), _dev(seq), _dev(np.zeros(len(reqs))), n)
    w_slots, w_offsets, failed = ref.plan(reqs, seq, [0] * len(reqs), n)
    tables.synchronize()
    assert not failed
    assert slots.tolist() == w_slots.tolist() and offsets.tolist() == w_offsets.tolist()
    assert tables.block_table.tolist() == ref.table.tolist() and tables.held.tolist() == ref.held.tolist()
    assert not tables._claim.any()


def test_a_map_of_some_columns_keeps_the_others():
    """Columns of a wider map: refused where a request may outgrow them, else filled without a word beside them."""
    tables = BlockTables(20, 3, 4, DEV, block_size=16)
    big = torch.full((4, 200), -9, dtype=torch.int32, device=DEV)
    args = [0, 2], [40, 64], [0, 0], 104
    for narrow in (big[:3, 8:48], big[:3, 150:], big[:, :63], big[:1].expand(3, -1), big[:, ::2]):
        with pytest.raises(ValueError, match="req_to_token"):
            tables.plan(*args, req_to_token=narrow)
    assert (big == -9).all() and tables.available() == 20
    slots, _ = tables.plan(*args, req_to_token=big[:3, 8:72])
    tables.synchronize()
    assert big[0, 8:48].tolist() == slots[:40].tolist() and big[2, 8:72].tolist() == slots[40:].tolist()
    big[0, 8:48], big[2, 8:72] = -9, -9
    assert (big == -9).all()
    # a map of its own that is shorter than the tables: what fits is written, the rest reported
    short = torch.full((3, 50), -9, dtype=torch.int32, device=DEV)
    again, _ = tables.plan([2], [64], [30], 34, req_to_token=short)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        tables.check_errors()
    assert again.tolist() == slots[70:].tolist() and short[2, 30:].tolist() == again[:20].tolist()
    short[2, 30:] = -9
    assert (short == -9).all()


def test_a_map_of_one_row():
    """The distance between the rows of one row is any number."""
    big = torch.full((100,), -9, dtype=torch.int32, device=DEV)
    for stride in (0, 1, 64, 1000):
        tables = BlockTables(20, 1, 4, DEV, block_size=16)
        one = big.as_strided((1, 64), (stride, 1))
        slots, _ = tables.plan([0], [64], [0], 64, req_to_token=one)
        tables.synchronize()
        assert one[0].tolist() == slots.tolist()
    assert (big[64:] == -9).all()


@pytest.mark.parametrize("stride", [0, 1, 7])
def test_tables_of_one_row_or_one_column(stride):
    """What a tensor says of the stride of a dimension of size 1 is any number."""
    for shape, strides, grow in (((1, 4), (stride, 1), 60), ((3, 1), (1, stride), 10)):
        table = torch.full((9,), -1, dtype=torch.int32, device=DEV)
        held = torch.zeros(shape[0], dtype=torch.int32, device=DEV)
        tables = BlockTables.from_tensors(table.as_strided(shape, strides), held, torch.arange(8, dtype=torch.int32, device=DEV),
                                          torch.tensor([0, 8], device=DEV), 16)
        n = shape[0]
        slots, _ = tables.plan(list(range(n)), [grow] * n, [0] * n, n * grow)
        tables.synchronize()
        pages = -(-grow // 16)
        assert table[:n * pages].tolist() == list(range(n * pages)) and (table[n * pages:] == -1).all()
        assert slots.tolist() == [i * pages * 16 + t for i in range(n) for t in range(grow)]
        tables.trim(list(range(n)))
        tables.synchronize()
        assert (table == -1).all() and tables.available() == 8
    wide = torch.zeros(1, 4, dtype=torch.int32, device=DEV).expand(3, -1)
    with pytest.raises(ValueError, match="block_table"):
        BlockTables.from_tensors(wide, held, torch.arange(8, dtype=torch.int32, device=DEV), torch.tensor([0, 8], device=DEV), 16)


@pytest.mark.parametrize("stride", [0, 1, 1000])
def test_selected_rows_of_one_request(stride):
    """The same of the rows of one request, and of one row of each."""
    cache = KV8Cache(1, 8, 2, 128, DEV, block_size=16)
    x = torch.randn(100, 2, 128, device=DEV).to(torch.bfloat16)
    cache.append(0, x, x, torch.arange(100, device=DEV))
    q = torch.randn(3, 8, 128, device=DEV).to(torch.bfloat16)
    rows = torch.arange(100, dtype=torch.int32, device=DEV)
    want = cache.sparse_decode_attention(0, q[:1], rows.view(1, 100), [90], 0.1)
    got = cache.sparse_decode_attention(0, q[:1], rows.as_strided((1, 100), (stride, 1)), [90], 0.1)
    assert torch.equal(got, want)
    want = cache.sparse_decode_attention(0, q, rows[:3].view(3, 1).clone(), [1] * 3, 0.1)
    got = cache.sparse_decode_attention(0, q, rows.as_strided((3, 1), (1, stride)), [1] * 3, 0.1)
    assert torch.equal(got, want)
    cache.synchronize()


def test_a_plan_that_asks_for_more_than_31_bits_of_blocks():
    """Each request may hold 2^29 blocks; five of them want 2^31 and more between them, and the ring has 20."""
    width = 1 << 29
    i32 = dict(dtype=torch.int32, device=DEV)
    table, held, free = torch.empty(6, width, **i32), torch.zeros(6, **i32), torch.arange(100, 120, **i32)
    tables = BlockTables.from_tensors(table, held, free, torch.tensor([0, 20], device=DEV), 16)
    for first in (0, 5000):  # the slots by one thread block, and by a grid
        reqs, seq = [5, 0, 1, 2, 3, 4], [first + 20] + [width * 16] * 5
        prefix = [0] + [width * 16 - 1] * 5
        if first:
            seq[0], prefix[0] = 40, 20
        n = first + 25
        slots, offsets = tables.plan(reqs, seq, prefix, n)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="no free block"):
            tables.check_errors()
        at = prefix[0]
        assert slots[:20].tolist() == [(100 + p // 16) * 16 + p % 16 for p in range(at, at + 20)]
        assert (slots[20:] == -1).all() and offsets.tolist() == [0, 20, 21, 22, 23, 24, 25]
        pages = -(-seq[0] // 16)
        assert held.tolist() == [0, 0, 0, 0, 0, pages] and tables.ring.tolist() == [pages, 20]
        assert table[5, :pages].tolist() == list(range(100, 100 + pages))
    # lengths the table never had: nothing goes back to the ring
    held[:5] = width
    tables.trim([5, 0, 1, 2, 3, 4])
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        tables.check_errors()
    assert held.tolist() == [width] * 5 + [3] and tables.ring.tolist() == [3, 20] and free.tolist() == list(range(100, 120))


def test_selected_rows_past_32_bits_are_reported():
    """int64 rows and lengths: what lies past 32 bits takes no part and is reported, and is not cut off to a valid row."""
    cache = KV8Cache(1, 8, 2, 128, DEV, block_size=16)
    x = torch.randn(100, 2, 128, device=DEV).to(torch.bfloat16)
    cache.append(0, x, x, torch.arange(100, device=DEV))
    q = torch.randn(2, 8, 128, device=DEV).to(torch.bfloat16)
    rows = torch.arange(60, device=DEV).view(2, 30)
    want = cache.sparse_decode_attention(0, q, rows.to(torch.int32), [30, 30], 0.1)
    assert torch.equal(cache.sparse_decode_attention(0, q, rows, _dev([30, 30]), 0.1), want)
    cache.synchronize()
    few = torch.cat([rows[:, :5], torch.full((2, 1), -1, device=DEV), rows[:, 6:]], 1)
    want = cache.sparse_decode_attention(0, q, few, [30, 30], 0.1)
    far = rows.clone()
    far[:, 5] = 2 ** 32 + 99
    got = cache.sparse_decode_attention(0, q, far, [30, 30], 0.1)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        cache.check_errors()
    assert torch.equal(got, want)
    got = cache.sparse_decode_attention(0, q, rows, _dev([30, 2 ** 32 + 3]), 0.1)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):
        cache.check_errors()
    assert not got[1].any()
    with pytest.raises(ValueError, match="integers are wanted"):
        cache.sparse_decode_attention(0, q, rows.float(), [30, 30], 0.1)


# ---------------------------------------------------------------- append


class _Twin:
    """An empty cache and its numpy twin."""

    def __init__(self, blocks, kv, block, dim):
        self.cache = KV8Cache(1, blocks, kv, dim, DEV, block_size=block)
        self.codes = [np.zeros((blocks, kv, block, dim), dtype=np.uint8) for _ in range(2)]
        self.scales = [np.zeros((blocks, kv), dtype=np.float32) for _ in range(2)]

    def put(self, x, slots):
        for c, s in zip(self.codes, self.scales):
            oracle.append(c, s, x.double().cpu().numpy(), np.asarray(slots))

    def check(self):
        got = (self.cache.k[0], self.cache.v[0]), (self.cache.k_scale[0], self.cache.v_scale[0])
        for g, want in zip(got[0], self.codes):
            assert np.array_equal(g.view(torch.uint8).cpu().numpy(), want)
        for g, want in zip(got[1], self.scales):
            assert np.array_equal(g.cpu().numpy(), want)
        assert not self.cache._state[0, 2:].any()  # no claim is left


def test_appends_that_continue_their_blocks_beside_a_long_one():
    """A call of slow thread blocks, more than fit at a time (64 tokens each, a block per token), and on another stream
    calls of more blocks than the first one leaves room for: each continues the blocks of the one before it."""
    block, kv, dim, long, mine, steps = 16, 1, 32, 1 << 16, 1024, 14
    rng = np.random.default_rng(0)
    twin = _Twin(long + mine, kv, block, dim)
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(slots):
        x = torch.from_numpy(rng.standard_normal((len(slots), kv, dim))).to(torch.bfloat16)
        return x, slots, x.to(DEV), _dev(slots)

    calls = [[call(mine * block + np.arange(long) * block)],
             [call(rng.permutation(mine) * block + step) for step in range(steps)]]
    graphs = []
    for todo, stream in zip(calls, streams):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            for _, _, x, slots in todo:
                twin.cache.append(0, x, x, slots)
    for _ in range(10):  # each replay starts its blocks anew
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    twin.cache.check_errors()
    for x, slots, _, _ in calls[1]:
        twin.put(x, slots)
    x, slots, _, _ = calls[0][0]
    for part in np.split(np.arange(long), 1 << 6)[::9]:
        twin.put(x[torch.from_numpy(part)], slots[part])
    seen = np.concatenate([np.arange(mine), mine + np.concatenate(np.split(np.arange(long), 1 << 6)[::9])])
    for got, want in zip((twin.cache.k[0], twin.cache.v[0]), twin.codes):
        assert np.array_equal(got.view(torch.uint8).cpu().numpy()[seen], want[seen])


@pytest.mark.parametrize("n", [2, 511, 512, 513, 3000])
def test_the_first_stretch_of_a_block_is_written(n):
    """Blocks met again at every distance, in calls that look for them and in calls that claim them."""
    block, kv, dim, blocks = 16, 2, 16, n + 4
    rng = np.random.default_rng(n)
    twin = _Twin(blocks, kv, block, dim)
    slots = rng.permutation(blocks)[:n] * block + 3
    again = np.sort(rng.permutation(n - 1)[:max(1, n // 20)]) + 1
    for t in again:  # at another offset of a block met before, which may be that of a skipped token
        slots[t] = slots[rng.integers(0, t)] // block * block + rng.integers(0, block)
    kept, seen = [], set()
    for t, s in enumerate(slots):
        run_on = t > 0 and s % block and slots[t - 1] == s - 1
        if run_on:
            kept.append(kept[-1])
            continue
        kept.append(s // block not in seen)
        seen.add(s // block)
    kept = np.array(kept)
    x = torch.from_numpy(rng.standard_normal((n, kv, dim))).to(torch.bfloat16)
    for _ in range(2):
        twin.cache.append(0, x.to(DEV), x.to(DEV), _dev(slots))
        torch.cuda.synchronize()
        if not kept.all():
            with pytest.raises(RuntimeError):
                twin.cache.check_errors()
        twin.put(x[torch.from_numpy(kept)], slots[kept])
        twin.check()


def test_a_captured_append_replays_beside_eager_ones():
    """Replays in which a block is met twice, or not, of few and of many tokens, with a call of another stream between."""
    block, kv, dim, blocks = 16, 2, 16, 2000
    rng = np.random.default_rng(3)
    for n in (40, 900):
        twin = _Twin(blocks, kv, block, dim)
        x = torch.from_numpy(rng.standard_normal((n, kv, dim))).to(torch.bfloat16).to(DEV)
        slots = torch.zeros(n, dtype=torch.int64, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            twin.cache.append(0, x, x, slots)
        other = torch.cuda.Stream()
        for step in range(5):
            mine = rng.permutation(900)[:n] * block + step
            if step == 2:
                mine[n - 1] = mine[0] + 1 + block // 2
            slots.copy_(_dev(mine))
            theirs = (1000 + rng.permutation(900)[:n]) * block + step
            y = torch.from_numpy(rng.standard_normal((n, kv, dim))).to(torch.bfloat16).to(DEV)
            theirs_dev = _dev(theirs)
            torch.cuda.synchronize()
            with torch.cuda.stream(other):
                twin.cache.append(0, y, y, theirs_dev)
            graph.replay()
            torch.cuda.synchronize()
            if step == 2:
                with pytest.raises(RuntimeError):
                    twin.cache.check_errors()
                mine = mine[:-1]
            twin.cache.check_errors()
            twin.put(x[:len(mine)], mine)
            twin.put(y, theirs)
            twin.check()


@pytest.mark.parametrize("n", [4, 700])
def test_append_reports_a_negative_slot_that_is_no_padding(n):
    """-1 skips a token; -2 and below are out of range, the other tokens are written."""
    for bad in (-2, -5, -(1 << 40)):
        twin = _Twin(n, 1, 16, 16)
        slots = np.arange(n) * 16
        slots[1], slots[n - 1] = -1, bad
        x = torch.randn(n, 1, 16, generator=torch.Generator().manual_seed(n))
        twin.cache.append(0, x.to(DEV), x.to(DEV), _dev(slots))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError):
            twin.cache.check_errors()
        twin.put(x[: n - 1], slots[: n - 1])
        twin.check()
