"""Attention of runs of new tokens at the limits of its arguments, against the definition in 64 bits
(tests/chunk_cases.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.chunk_cases import check_attention, device_args, make_case
from tests.gpu_util import need_gpu
from tests.test_gpu_chunk_attention import CASES as ATTENTION_CASES

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


# --------------------------------------------------------------------------------------------- the write
def check_write(kv, case, run_count=None, **over):
    """The runs' rows are where they belong, every other row of the cache as it was."""
    from tests.test_gpu_chunk_append import stored

    a, t = device_args(kv, case)
    if run_count is not None:                    # runs without rows behind the case's own
        for n in ("seq_batch", "first_position", "row_count", "row_start"):
            t[n] = torch.cat([t[n], torch.zeros(run_count - t[n].numel(), dtype=torch.int32, device="cuda")])
            setattr(a, n, t[n].data_ptr())
        a.run_count = run_count
    for name, value in over.items():
        setattr(a, name, value)
    bits = lambda x: x.view(torch.int16).reshape(-1)  # noqa: E731
    want = [bits(stored(case, t[c], t[r])) for c, r in (("cache_k", "k_rows"), ("cache_v", "v_rows"))]
    kv.chunk_write(a)
    torch.cuda.synchronize()
    assert torch.equal(bits(t["cache_k"]), want[0]) and torch.equal(bits(t["cache_v"]), want[1])


WRITES = {
    "ragged": dict(counts=[1, 33, 70, 2], firsts=[100, 0, 15, 300], own_rows=True, gap=2),
    "ring": dict(counts=[200, 3, 64, 1], firsts=[10, 1000, 0, 70], ring=True, window=64, gap=1),
    "ring_page5": dict(counts=[140, 7], firsts=[33, 9], ring=True, window=61, page=5),
    "odd_heads": dict(counts=[9, 40], firsts=[7, 64], heads=3, group=1, own_rows=True),
    "dim512": dict(counts=[9, 40], firsts=[7, 64], heads=1, group=16, dim=512, page=64, own_rows=True),
    "layer": dict(counts=[21, 3], firsts=[7, 30], layers=3, layer=1, own_rows=True),
    "unmapped": dict(counts=[40], firsts=[0], unmap=[(0, 1)], own_rows=True),
    # several rows to a CTA
    "long": dict(counts=[1500, 1, 650, 90, 2, 33], firsts=[3, 500, 0, 41, 7, 15], heads=2, gap=3, own_rows=True),
    "long_ring": dict(counts=[1700, 3, 640, 1], firsts=[10, 1000, 0, 63], heads=2, ring=True, window=64),
    "many_runs": dict(counts=[1 + i % 40 for i in range(100)], firsts=[i * 7 for i in range(100)], heads=2, page=5, gap=1,
                      own_rows=True),
}


@pytest.mark.parametrize("name", list(WRITES))
def test_write_of_runs(kv, name):
    check_write(kv, make_case(23, **WRITES[name]))


@pytest.mark.parametrize("name", ["ragged", "ring"])
@pytest.mark.parametrize("bound", [100 * 70, 2**31 - 1])
def test_a_generous_bound_of_the_run_length(kv, name, bound):
    """The grid is cut to the rows there are and to a fixed size: max_row_count x run_count is 2^41 here."""
    check_write(kv, make_case(24, **WRITES[name]), run_count=1024, max_row_count=bound)


@pytest.mark.parametrize("name", ["long", "long_ring", "many_runs"])
def test_a_cta_writes_every_so_manyth_row(kv, name):
    """1024 runs leave a run 32 CTAs."""
    check_write(kv, make_case(25, **WRITES[name]), run_count=1024)


# --------------------------------------------------------------------------------------------- waits that run out
GIVE_UPS = {
    "first_tile": (0, dict(counts=[4], firsts=[1500], ring=True, window=1024)),
    "next_tile_on_its_way": (0, dict(counts=[3], firsts=[3000])),
    "second_tile": (1, dict(counts=[3], firsts=[3000])),
    "page5": (0, dict(counts=[4], firsts=[3000], page=5)),
    "dim512": (1, dict(counts=[1, 1], firsts=[1900, 2000], heads=1, group=16, dim=512, page=64)),
}


@pytest.mark.parametrize("name", list(GIVE_UPS))
def test_rows_of_a_call_that_gives_up_are_nan(kv, name):
    """Not an average over the keys that came in time. The context stays usable: the same call afterwards is right."""
    tile, over = GIVE_UPS[name]
    case = make_case(26, **over)
    a, t = device_args(kv, case)
    kv.chunk_attention_give_up_selftest(a, tile)
    torch.cuda.synchronize()
    assert t["status"][0].item() == kv.STATUS_WAIT_TIMEOUT
    assert bool(t["out"].isnan().all()) and bool(t["lse"].isnan().all())
    t["status"].zero_()
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


@pytest.mark.parametrize("window", [0, MOST])
def test_give_up_selftest_of_a_tile_that_no_cta_has(kv, window):
    case = make_case(27, [4], [500], window=window)
    a, t = device_args(kv, case)
    kv.chunk_attention_give_up_selftest(a, 1000)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_give_up_selftest_refuses(kv):
    a, t = device_args(kv, make_case(28, [4], [500]))
    assert kv.chunk_attention_give_up_selftest(a, -1, check=False) == 1
    a.status = None
    assert kv.chunk_attention_give_up_selftest(a, 0, check=False) == 1
    large, _ = device_args(kv, make_case(28, [1, 2], [6000, 5200], heads=1, group=16, dim=512, page=64))
    assert kv.chunk_attention_give_up_selftest(large, 0, check=False) == 1


# --------------------------------------------------------------------------------------------- which kernel, and what is refused
@pytest.mark.parametrize("name", [n for n in ATTENTION_CASES if n.startswith(("few_", "large_"))])
def test_the_cases_of_each_kernel_reach_it(kv, name):
    a, _ = device_args(kv, make_case(len(name) * 7 + 1, **ATTENTION_CASES[name]))
    assert kv.chunk_attention_launches(a) == (1 if name.startswith("few_") else 2)


SIZE_RULE = {
    # a row sees no more than the table has, however wide the window
    "window_wider_than_the_table": (1, dict(counts=[3], firsts=[500], window=100000)),
    "window_of_all_positions": (1, dict(counts=[3], firsts=[500], window=MOST, sinks=3)),
    # the run's own rows are keys too: 1600 of them in 100 tiles for a CTA each
    "own_rows_behind_a_short_table": (2, dict(counts=[1600], firsts=[10], heads=1, group=1, own_rows=True)),
    "own_rows_in_a_window": (1, dict(counts=[1600], firsts=[10], heads=1, group=1, own_rows=True, window=64)),
}


@pytest.mark.parametrize("name", list(SIZE_RULE))
def test_small_calls_go_by_what_a_row_can_see(kv, name):
    launches, over = SIZE_RULE[name]
    case = make_case(29, **over)
    a, t = device_args(kv, case)
    assert kv.chunk_attention_launches(a) == launches
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


@pytest.mark.parametrize("own", [False, True])
def test_a_window_over_a_table_of_all_positions_is_not_refused(kv, own):
    """The limit of a call's key tiles goes by the window, as documented, not by the table."""
    case = make_case(30, [520, 3], [300, 40], page=64, window=100, sinks=3, own_rows=own)
    slots = 2**31 // 64
    table = np.full((2, slots), -1, dtype=np.int32)
    table[:, :case.table.shape[1]] = case.table
    case.table = table
    case.cfg = (*case.cfg[:3], slots, *case.cfg[4:])
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)
    a.window_size = a.sink_tokens = 0           # without a window it goes by the table
    assert kv.chunk_attention_launches(a) == 0 and kv.chunk_attention(a, check=False) == 1


# --------------------------------------------------------------------------------------------- page copies
@pytest.mark.parametrize("partial", [False, True])
@pytest.mark.parametrize("pages,ps,heads,dim,count", [(30, 8, 1, 8, 11), (30, 16, 3, 8, 11), (40, 24, 5, 72, 13)])
def test_copies_of_8_bit_rows_of_an_odd_number_of_eights(kv, pages, ps, heads, dim, count, partial):
    """A row is a multiple of 8 elements, of an 8-bit cache as little as 8 bytes."""
    from tests.test_gpu_chunk_append import copy_case

    cfg, caches, scales = copy_case(kv, 2, pages, ps, heads, dim, True, 4)
    rng = np.random.default_rng(5)
    pick = rng.permutation(pages).astype(np.int32)
    src, dst = pick[:count].copy(), pick[count:2 * count].copy()
    rows = rng.integers(0, ps + 3, count).astype(np.int32) if partial else None
    want, want_scales = [c.clone() for c in caches], [s.clone() for s in scales]
    for i in range(count):
        n = ps if rows is None else -(-min(int(rows[i]), ps) // 8) * 8
        for c, s in zip(want, want_scales):
            c[:, dst[i], :n] = c[:, src[i], :n]
            if n:
                s[:, dst[i]] = s[:, src[i]]
    up = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
    kv.copy_pages_fp8(*caches, *scales, cfg, up(src), up(dst), up(rows), count)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(caches + scales, want + want_scales))
