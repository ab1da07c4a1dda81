"""The 8-bit cache's tables, writes and arguments at their edges, against the numpy restatement (``oracle/kv8.py``)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8 as oracle
from qwenquest_b200.kv8 import BlockTables

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
