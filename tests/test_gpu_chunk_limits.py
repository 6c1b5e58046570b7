"""Attention of runs of new tokens at the limits of its arguments, against the definition in 64 bits
(tests/chunk_cases.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.chunk_cases import check_attention, device_args, make_case
from tests.gpu_util import need_gpu

pytestmark = [pytest.mark.gpu, need_gpu]

MOST = 2**31 - 1

# A window of (nearly) every position there is hides nothing, wherever the run starts; key tiles that lie behind a query
# tile's first row are the ones whose distance to the window's start does not fit 32 bits.
WIDE_WINDOWS = {
    "unaligned_first": dict(counts=[200], firsts=[100]),
    "tile_behind_the_first_row": dict(counts=[170], firsts=[131]),
    "sinks": dict(counts=[200, 3], firsts=[100, 7], sinks=5),
    "own_rows": dict(counts=[190, 66], firsts=[77, 0], own_rows=True),
    "group1": dict(counts=[310], firsts=[130], heads=4, group=1),
    "page5": dict(counts=[170], firsts=[131], page=5),
    "dim512": dict(counts=[90, 100], firsts=[131, 67], heads=1, group=16, dim=512, page=64),
    "few_rows": dict(counts=[5], firsts=[61]),
}


@pytest.mark.parametrize("window", [MOST, MOST - 100, MOST - 1024, MOST - 1200])
@pytest.mark.parametrize("name", list(WIDE_WINDOWS))
def test_a_window_of_all_positions_hides_nothing(kv, name, window):
    case = make_case(21, window=window, **WIDE_WINDOWS[name])
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


@pytest.mark.parametrize("own", [False, True])
def test_a_ring_with_a_window_of_all_positions(kv, own):
    """Its page table is as long as that takes; the pages that the run's positions need are mapped."""
    case = make_case(22, [200], [100], page=64, own_rows=own)
    slots = (MOST + 200) // 64 + 1
    table = np.full((1, slots), -1, dtype=np.int32)
    table[:, :case.table.shape[1]] = case.table
    case.table = table
    case.cfg = (*case.cfg[:3], slots, *case.cfg[4:7], MOST)
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)
