"""The 8-bit block KV cache without a GPU: the oracle's own arithmetic, and the refusals of the C ABI and the classes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8 as oracle
from qwenquest_b200 import _lib
from qwenquest_b200.kv8 import BlockTables, KV8Cache

OK, INV, UNS, WS = _lib.QQ_OK, _lib.QQ_ERR_INVALID, _lib.QQ_ERR_UNSUPPORTED, _lib.QQ_ERR_WORKSPACE


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        import __graft_entry__

        __graft_entry__.build()
    return _lib.load()


def test_oracle_codes_are_torchs():
    """e4m3 rounding against torch's conversion, on every code, every midpoint and random values."""
    values = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.isnan(values), np.isnan(oracle.E4M3))
    assert np.array_equal(values[~np.isnan(values)], oracle.E4M3[~np.isnan(values)].astype(np.float32))
    pos = oracle.E4M3[:0x7F]
    x = np.concatenate([pos, (pos[1:] + pos[:-1]) / 2, np.random.default_rng(0).standard_normal(5000) * 60,
                        np.exp2(np.random.default_rng(1).uniform(-14, 8.8, 5000))]).astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(oracle.to_e4m3(x), want)


@pytest.mark.parametrize("amax", [448.0, 448.1, 447.9, 1.0, 1.75, 1.7500001, 3.4e38, 1e-38, 1e-45, 0.0])
def test_oracle_scale_is_the_smallest_that_fits(amax):
    s = float(oracle.scale_for(np.float64(amax)))
    assert amax <= 448 * s and np.log2(s) == int(np.log2(s))
    assert s == 2.0 ** -126 or amax > 448 * s / 2


def test_table_calls_check_their_arguments_without_a_device(lib):
    def tables(**kw):
        base = dict(block_table=0x1000, table_stride=8, held=0x2000, claim=0x3000, free_blocks=0x4000, ring=0x5000,
                    capacity=10, max_reqs=4, max_blocks=8, block_size=64)
        base.update(kw)
        return _lib.QQBlockTables(*base.values())

    def plan(t, reqs=0x10, seq=0x20, prefix=0x30, bs=1, slots=0x40, n=1, offsets=0x50, mapped=None, stride=0, rows=0):
        return lib.qq_block_plan(t, reqs, seq, prefix, bs, slots, n, offsets, mapped, stride, rows, None, None)

    for name in ("block_table", "held", "claim", "free_blocks", "ring", "capacity", "max_reqs", "max_blocks"):
        assert plan(tables(**{name: 0})) == INV, name
    assert plan(None) == INV
    assert plan(tables(table_stride=7)) == INV
    assert plan(tables(block_size=48)) == UNS
    assert plan(tables(), bs=_lib.QQ_MAX_BS + 1) == UNS
    assert plan(tables(), bs=-1) == INV
    assert plan(tables(), reqs=None) == INV and plan(tables(), seq=None) == INV and plan(tables(), prefix=None) == INV
    assert plan(tables(), slots=None) == INV and plan(tables(), offsets=None) == INV and plan(tables(), n=-1) == INV
    assert plan(tables(), mapped=0x60) == INV
    assert lib.qq_block_trim(None, 0x10, 0x20, 1, None, None) == INV
    assert lib.qq_block_trim(tables(), None, 0x20, 1, None, None) == INV
    assert lib.qq_block_trim(tables(), None, None, 0, None, None) == OK


def _cache(**kw):
    base = dict(k=0x1000, v=0x2000, k_scale=0x3000, v_scale=0x4000, state=0x5000, num_blocks=10, kv_heads=4,
                head_dim=128, block_size=64)
    base.update(kw)
    return _lib.QQKv8Cache(*base.values())


def test_cache_calls_check_their_arguments_without_a_device(lib):
    def append(c, k=0x10000, v=0x20000, dtype=_lib.QQ_BF16, ks=512, vs=512, slots=0x30, n=1):
        return lib.qq_kv8_append(c, k, v, dtype, ks, vs, slots, n, None, None)

    def gather(c, slots=0x30, n=1, k=0x10000, v=0x20000, dtype=_lib.QQ_BF16):
        return lib.qq_kv8_gather(c, slots, n, k, v, dtype, None, None)

    bad = [(dict(k=0), INV), (dict(v=0), INV), (dict(k_scale=0), INV), (dict(v_scale=0), INV),
           (dict(num_blocks=0), INV), (dict(kv_heads=0), INV), (dict(head_dim=0), INV), (dict(block_size=8), UNS),
           (dict(block_size=256), UNS), (dict(head_dim=12), UNS), (dict(head_dim=264), UNS), (dict(k=0x1008), UNS),
           (dict(num_blocks=1 << 25), UNS), (dict(num_blocks=1 << 23), UNS)]
    for kw, rc in bad:
        assert append(_cache(**kw)) == rc and gather(_cache(**kw)) == rc, kw
    assert append(None) == INV and gather(None) == INV
    assert append(_cache(state=0)) == INV
    assert append(_cache(), n=0) == OK and gather(_cache(), n=0) == OK
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(dtype=2), dict(ks=511), dict(vs=0), dict(n=-1)):
        assert append(_cache(), **kw) == INV, kw
    for kw in (dict(k=0x10008), dict(v=0x20002), dict(ks=516), dict(vs=513)):
        assert append(_cache(), **kw) == UNS, kw
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(dtype=5), dict(n=-1)):
        assert gather(_cache(), **kw) == INV, kw
    assert gather(_cache(), k=0x10008) == UNS


def test_attention_calls_check_their_arguments_without_a_device(lib):
    b = _lib.QQBatch(0x100, 0x200, 1)

    def decode(c=None, batch=b, table=0x300, stride=4, rows=2, q=0x10000, dtype=_lib.QQ_BF16, heads=32, q_stride=4096,
               out=0x20000, out_stride=4096, ws=0x30000, size=1 << 30):
        return lib.qq_kv8_decode_attention(c or _cache(), batch, table, stride, rows, q, dtype, heads, q_stride, 0.1,
                                           out, out_stride, None, ws, size, None)

    assert decode(batch=None) == INV and decode(batch=_lib.QQBatch(0, 0, -1)) == INV
    assert decode(batch=_lib.QQBatch(0, 0, 0)) == OK
    assert decode(batch=_lib.QQBatch(0, 0x200, 1)) == INV and decode(batch=_lib.QQBatch(0x100, 0, 1)) == INV
    for kw in (dict(table=None), dict(stride=0), dict(rows=0), dict(q=None), dict(out=None), dict(dtype=3),
               dict(heads=0), dict(heads=30), dict(q_stride=4095), dict(out_stride=1)):
        assert decode(**kw) == INV, kw
    assert decode(batch=_lib.QQBatch(0x100, 0x200, _lib.QQ_MAX_BS + 1)) == UNS
    assert decode(ws=0x30004) == UNS
    assert decode(c=_cache(block_size=24)) == UNS
    # one request over long tables is split: the records need room
    need = lib.qq_kv8_workspace_bytes(_cache(), 32, _lib.QQ_BF16, 1, 1, 1 << 16, 0)
    assert need > 0
    assert decode(stride=1024, ws=None, size=0) == WS
    assert decode(stride=1024, size=need - 4) == WS

    def sparse(c=None, bs=1, rows=0x300, stride=256, top=256, lens=0x400, q=0x10000):
        return lib.qq_kv8_sparse_attention(c or _cache(), bs, rows, stride, top, lens, q, _lib.QQ_BF16, 32, 4096, 0.1,
                                           0x20000, 4096, None, 0x30000, 1 << 30, None)

    assert sparse(bs=-1) == INV and sparse(bs=0) == OK
    for kw in (dict(rows=None), dict(lens=None), dict(top=0), dict(stride=255), dict(q=None)):
        assert sparse(**kw) == INV, kw
    assert sparse(bs=_lib.QQ_MAX_BS + 1) == UNS

    e = _lib.QQExtendBatch(0x1, 0x2, 0x3, 0x4, 0, 8, 1, 0)

    def extend(batch=e, table=0x300, stride=4, rows=2):
        return lib.qq_kv8_extend_attention(_cache(), batch, table, stride, rows, 0x10000, _lib.QQ_BF16, 32, 4096, 0.1,
                                           0x20000, 4096, None, 0x30000, 1 << 30, None)

    assert extend(batch=None) == INV
    assert extend(batch=_lib.QQExtendBatch(0x1, 0x2, 0x3, 0x4, 0, 0, 1, 0)) == OK
    assert extend(batch=_lib.QQExtendBatch(0x1, 0x2, 0x3, 0x4, 0, 8, 0, 0)) == OK
    for i in range(4):
        p = [0x1, 0x2, 0x3, 0x4]
        p[i] = 0
        assert extend(batch=_lib.QQExtendBatch(*p, 0, 8, 1, 0)) == INV
    assert extend(table=None) == INV and extend(stride=0) == INV and extend(rows=0) == INV
    assert lib.qq_kv8_workspace_bytes(None, 32, 0, 1, 1, 64, 0) == 0
    assert lib.qq_kv8_workspace_bytes(_cache(), 30, 0, 1, 1, 64, 0) == 0


def test_classes_refuse_the_cpu_and_bad_shapes():
    i32 = torch.int32
    with pytest.raises(ValueError, match="CUDA device"):
        KV8Cache(1, 4, 2, 64, "cpu")
    with pytest.raises(ValueError, match="CUDA device"):
        BlockTables(4, 2, 2, "cpu")
    codes = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.zeros(4, 2)
    with pytest.raises(ValueError, match="CUDA device"):
        KV8Cache.from_tensors([codes], [codes], [scale], [scale])
    with pytest.raises(ValueError, match="one tensor per layer"):
        KV8Cache.from_tensors([codes], [codes], [scale], [])
    with pytest.raises(ValueError, match="codes must be"):
        KV8Cache.from_tensors([codes.view(torch.uint8)], [codes], [scale], [scale])
    with pytest.raises(ValueError, match="scales must be"):
        KV8Cache.from_tensors([codes], [codes], [scale[:3]], [scale])
    with pytest.raises(ValueError, match="block_size"):
        KV8Cache.from_tensors([codes[:, :, :8].contiguous()], [codes], [scale], [scale])
    with pytest.raises(ValueError, match="head_dim"):
        KV8Cache.from_tensors([codes[..., :4].contiguous()], [codes], [scale], [scale])
    table, held = torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32)
    free, ring = torch.arange(4, dtype=i32), torch.tensor([0, 4])
    with pytest.raises(ValueError, match="CUDA device"):
        BlockTables.from_tensors(table, held, free, ring, 64)
    for args in ((table.long(), held, free, ring, 64), (table, held[:1], free, ring, 64),
                 (table, held, free.long(), ring, 64), (table, held, free, ring.int(), 64),
                 (table, held, free, ring, 48), (table.T, held, free, ring, 64)):
        with pytest.raises(ValueError):
            BlockTables.from_tensors(*args)
