"""The 8-bit cache's arguments without a GPU."""

from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from qwenquest_b200 import _lib, kv8
from qwenquest_b200._device import DeviceError

HOST = SimpleNamespace(device=torch.device("cpu"), _index=-1)


def test_integers_past_32_bits_stay_out_of_range():
    """2^32 + 5 must not become 5."""
    wide = [5, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, -2 ** 32 + 5, 2 ** 62]
    want = [5, -1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, -2 ** 31, 2 ** 31 - 1]
    for given in (wide, torch.tensor(wide)):
        got = kv8._OnDevice._ints(HOST, given, torch.int32, "lens")
        assert got.dtype == torch.int32 and got.tolist() == want
    got = kv8._as_int(torch.tensor(wide).view(2, 4), torch.int32, "rows", HOST.device)
    assert got.dtype == torch.int32 and got.flatten().tolist() == want
    unsigned = torch.tensor([5, 2 ** 32 - 1]).to(torch.uint32)
    assert kv8._OnDevice._ints(HOST, unsigned, torch.int32, "lens").tolist() == [5, 2 ** 31 - 1]
    assert kv8._OnDevice._ints(HOST, wide, torch.int64, "seq_lens").tolist() == wide


@pytest.mark.parametrize("small", [torch.int8, torch.uint8, torch.int16])
def test_narrower_integers_are_widened(small):
    assert kv8._OnDevice._ints(HOST, torch.tensor([3, 7], dtype=small), torch.int32, "lens").tolist() == [3, 7]


@pytest.mark.parametrize("other", [torch.float32, torch.bfloat16, torch.bool, torch.complex64])
def test_what_is_no_integer_is_refused(other):
    for dtype in (torch.int32, torch.int64):
        with pytest.raises(ValueError, match="integers are wanted"):
            kv8._OnDevice._ints(HOST, torch.ones(2, dtype=other), dtype, "lens")


def test_errors_beside_a_full_ring_are_named_too():
    """One batch may run out of blocks and name a bad request: both are raised, once."""
    tables = kv8.BlockTables.__new__(kv8.BlockTables)
    tables._err = DeviceError(torch.zeros(1, dtype=torch.int32))
    tables._err_word = ctypes.c_int32.from_address(tables._err.word.data_ptr())
    tables._what = "(block tables)"
    full, bounds = _lib.QQ_DEV_ERR_CAPACITY, _lib.QQ_DEV_ERR_BOUNDS
    for bits, said in ((full, ["no free block"]), (full | bounds, ["no free block", "out of range"]), (bounds, ["out of range"])):
        tables._err.word[0] = bits
        with pytest.raises(RuntimeError) as raised:
            tables.check_errors()
        assert all(text in str(raised.value) for text in said)
        assert ("no free block" in str(raised.value)) == bool(bits & full)
        tables.check_errors()


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        import __graft_entry__

        __graft_entry__.build()
    return _lib.load()


def test_extend_refuses_a_table_whose_positions_near_31_bits(lib):
    """The kernel holds the positions of key tiles behind the last one in 32 bits too: 2^31 - 2^17 tokens at most."""
    cache = _lib.QQKv8Cache(0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 100, 4, 128, 128)
    batch = _lib.QQExtendBatch(0x100, 0x200, 0x300, 0x400, None, 10, 1, 0)

    def extend(stride, workspace=None):
        return lib.qq_kv8_extend_attention(cache, batch, 0x300, stride, 2, 0x10000, _lib.QQ_BF16, 32, 4096, 0.1, 0x20000, 4096,
                                           None, workspace, 0, None)

    most = (2 ** 31 - 2 ** 17) // 128
    for stride in (2 ** 24 - 1, 2 ** 24 - 2, most + 1):
        assert extend(stride) == _lib.QQ_ERR_UNSUPPORTED
    assert extend(most - 1) == _lib.QQ_ERR_WORKSPACE  # within the limit: the next check refuses


def test_decode_refuses_more_tiles_than_31_bits_count(lib):
    """All heads of one request's row: 2^24 tiles of 128 keys times 128 heads."""
    def calls(kv, block, stride, top):
        cache = _lib.QQKv8Cache(0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 100, kv, 128, block)
        tail = (0x10000, _lib.QQ_BF16, kv, kv * 128, 0.1, 0x20000, kv * 128, None, None, 0, None)
        return (lib.qq_kv8_decode_attention(cache, _lib.QQBatch(0x100, 0x200, 1), 0x300, stride, 2, *tail),
                lib.qq_kv8_sparse_attention(cache, 1, 0x300, top, top, 0x400, *tail))

    assert calls(129, 128, 2 ** 24 - 1, 2 ** 31 - 1) == (_lib.QQ_ERR_UNSUPPORTED,) * 2
    assert calls(127, 128, 2 ** 24 - 1, 2 ** 31 - 1) == (_lib.QQ_ERR_WORKSPACE,) * 2
