"""The 8-bit cache's arguments without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from qwenquest_b200 import kv8

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
