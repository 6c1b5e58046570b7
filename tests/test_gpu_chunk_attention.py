"""Attention of runs of new tokens over the paged cache, against the definition in 64 bits (tests/chunk_cases.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.chunk_cases import attention_f64, check_attention, device_args, make_case
from tests.gpu_util import need_gpu

pytestmark = [pytest.mark.gpu, need_gpu]

CASES = {
    "one_token": dict(counts=[1], firsts=[37]),
    "first_token_of_all": dict(counts=[1], firsts=[0]),
    "four_tokens": dict(counts=[4], firsts=[500]),
    "prompt_from_zero": dict(counts=[200], firsts=[0]),
    "tile_edges": dict(counts=[64, 65, 63, 128, 1], firsts=[64, 63, 65, 0, 127]),
    "ragged": dict(counts=[1, 130, 7, 33, 300], firsts=[900, 0, 255, 1000, 77], gap=3),
    "long_keys_few_rows": dict(counts=[3, 1], firsts=[6000, 4097]),
    "many_runs": dict(counts=[1 + i % 5 for i in range(70)], firsts=[(i * 53) % 400 for i in range(70)]),
    "heads4": dict(counts=[40, 2], firsts=[300, 10], heads=4),
    "heads1": dict(counts=[100, 5], firsts=[700, 2000], heads=1),
    "group1": dict(counts=[70, 3], firsts=[130, 64], heads=4, group=1),
    "group3": dict(counts=[50, 3], firsts=[130, 64], heads=2, group=3),
    "group64": dict(counts=[5, 3], firsts=[130, 64], heads=1, group=64),
    "dim512": dict(counts=[40, 1, 3], firsts=[300, 1000, 0], heads=1, group=16, dim=512, page=64),
    "dim512_two_heads": dict(counts=[70], firsts=[90], heads=2, group=2, dim=512),
    "dim512_ring": dict(counts=[90, 3], firsts=[300, 1000], heads=1, group=16, dim=512, ring=True, window=128),
    "page1": dict(counts=[30, 2], firsts=[60, 100], page=1),
    "page5": dict(counts=[70, 2], firsts=[131, 100], page=5),
    "page8": dict(counts=[70, 2], firsts=[131, 100], page=8),
    "page24": dict(counts=[70, 2], firsts=[131, 100], page=24),
    "page64": dict(counts=[70, 2], firsts=[131, 1000], page=64),
    "page200": dict(counts=[70, 2], firsts=[131, 1000], page=200),
    "layer": dict(counts=[20], firsts=[100], layers=3, layer=1),
    "ring_tight": dict(counts=[4, 1, 200, 30], firsts=[1500, 256, 100, 0], ring=True, window=256),
    "ring_run_longer_than_window": dict(counts=[500, 20], firsts=[300, 64], ring=True, window=64),
    "ring_slack": dict(counts=[16, 1, 9], firsts=[1000, 40, 64], ring=True, window=64, ring_slots=5, own_rows=False),
    "ring_window1": dict(counts=[20, 1], firsts=[50, 0], ring=True, window=1),
    "ring_page5": dict(counts=[40, 3], firsts=[333, 64], ring=True, window=61, page=5),
    "own_rows_linear": dict(counts=[100, 3, 65], firsts=[333, 64, 0], own_rows=True),
    "own_rows_page5": dict(counts=[100, 3, 65], firsts=[333, 64, 0], own_rows=True, page=5),
    "window_linear": dict(counts=[100, 3], firsts=[333, 700], window=90),
    "sinks": dict(counts=[1, 1, 1], firsts=[1000, 5, 70], window=64, sinks=4, free_middle=True),
    "sinks_chunk": dict(counts=[150, 33], firsts=[700, 0], window=100, sinks=70, free_middle=True),
    "sinks_beyond_run": dict(counts=[10], firsts=[3], window=4, sinks=200),
    "sinks_own_rows": dict(counts=[150, 33], firsts=[700, 20], window=100, sinks=30, free_middle=True, own_rows=True),
    "hole": dict(counts=[40], firsts=[200], unmap=[(0, 3), (0, 14)]),
    "no_key_at_all": dict(counts=[2, 5], firsts=[14, 100], unmap=[(0, 0)]),
    # the same geometries in calls that are not small
    "large_heads1": dict(counts=[1200, 5], firsts=[700, 2000], heads=1),
    "large_heads4": dict(counts=[310, 2], firsts=[300, 10], heads=4),
    "large_group1": dict(counts=[310, 3], firsts=[130, 64], heads=4, group=1),
    "large_group3": dict(counts=[300, 3], firsts=[130, 64], heads=2, group=3),
    "large_512_two_heads": dict(counts=[650], firsts=[90], heads=2, group=2, dim=512),
    "large_512_single": dict(counts=[1, 2], firsts=[6000, 5200], heads=1, group=16, dim=512, page=64),
    "large_512_own": dict(counts=[100, 60], firsts=[6000, 20], heads=1, group=16, dim=512, page=64, own_rows=True),
    "large_page8": dict(counts=[170, 2], firsts=[131, 100], page=8),
    "large_page24": dict(counts=[170, 2], firsts=[131, 100], page=24),
    "large_page64": dict(counts=[170, 2], firsts=[131, 1000], page=64),
    "large_sinks_single": dict(counts=[1] * 20, firsts=[(i * 97) % 1200 for i in range(20)], window=64, sinks=4,
                               free_middle=True),
    "large_ring_single": dict(counts=[1] * 20, firsts=[(i * 97) % 1200 for i in range(20)], ring=True, window=128),
    "large_hole": dict(counts=[300], firsts=[200], unmap=[(0, 3), (0, 14)]),
    "large_no_key": dict(counts=[300, 5], firsts=[14, 100], unmap=[(0, 0)]),
    "large_peaked": dict(counts=[200, 3], firsts=[500, 800], q_scale=30.0),
    # small calls (a kernel of their own)
    "few_ring": dict(counts=[4], firsts=[1500], ring=True, window=1024),
    "few_ring_runs": dict(counts=[4, 8], firsts=[300, 64], ring=True, window=256),
    "few_ring_uneven": dict(counts=[8, 1, 3], firsts=[1000, 0, 250], ring=True, window=250, page=8, gap=1),
    "few_slack": dict(counts=[5], firsts=[777], ring=True, window=200, page=8, ring_slots=30, own_rows=False),
    "few_linear": dict(counts=[7], firsts=[1333]),
    "few_page24": dict(counts=[3, 2], firsts=[131, 700], page=24),
    "few_page64": dict(counts=[8], firsts=[1190], page=64),
    "few_page200": dict(counts=[6], firsts=[1190], page=200),
    "few_sinks": dict(counts=[1], firsts=[3000], window=500, sinks=4, free_middle=True),
    "few_sinks_own": dict(counts=[8], firsts=[700], window=100, sinks=37, free_middle=True, own_rows=True),
    "few_window_inside_run": dict(counts=[8], firsts=[40], window=3),
    "few_hole": dict(counts=[5], firsts=[300], unmap=[(0, 2), (0, 3), (0, 18)]),
    "few_no_key": dict(counts=[3], firsts=[12], unmap=[(0, 0)]),
    "few_group16": dict(counts=[1], firsts=[900], heads=2, group=16),
    "few_group3": dict(counts=[5], firsts=[200], heads=2, group=3),
    "few_group1": dict(counts=[16], firsts=[350], heads=3, group=1),
    "few_512": dict(counts=[1, 1], firsts=[2000, 5], heads=1, group=16, dim=512, page=64),
    "few_512_tokens": dict(counts=[5], firsts=[900], heads=4, group=2, dim=512, page=8),
    "few_512_ring": dict(counts=[7, 8], firsts=[1000, 40], heads=1, group=2, dim=512, ring=True, window=512),
    "few_many": dict(counts=[1 + 3 * i % 8 for i in range(8)], firsts=[(i * 331) % 1200 for i in range(8)], gap=1),
    "few_many_512": dict(counts=[1] * 12, firsts=[(i * 331) % 1500 for i in range(12)], heads=2, group=8, dim=512, page=16),
    "few_layer": dict(counts=[3], firsts=[200], layers=3, layer=2),
    # more than one query tile of 16 rows
    "few_tiles": dict(counts=[40], firsts=[300]),
    "few_tiles_ring": dict(counts=[61], firsts=[500], ring=True, window=128),
    "few_tiles_short_window": dict(counts=[70], firsts=[90], ring=True, window=16),
    "few_tiles_slack": dict(counts=[33, 5], firsts=[400, 10], ring=True, window=64, ring_slots=8, own_rows=False),
    "few_tiles_own_sinks": dict(counts=[90], firsts=[10], window=20, sinks=37, own_rows=True, heads=2),
    "few_tiles_sinks": dict(counts=[50], firsts=[333], window=40, sinks=20, free_middle=True, page=8),
    "few_tiles_uneven": dict(counts=[30, 1, 17], firsts=[0, 200, 64], heads=2, group=3, gap=2),
    "few_tiles_group16": dict(counts=[9, 3], firsts=[100, 30], heads=2, group=16),
    "few_tiles_group1": dict(counts=[100], firsts=[200], heads=3, group=1),
    "few_tiles_512": dict(counts=[20, 3], firsts=[300, 0], heads=1, group=16, dim=512, page=64),
    "few_tiles_512_own": dict(counts=[24], firsts=[200], heads=2, group=2, dim=512, own_rows=True),
    "few_page5": dict(counts=[4], firsts=[777], page=5),
    "few_page5_ring": dict(counts=[8, 3], firsts=[333, 64], ring=True, window=61, page=5),
    "few_page3_tiles": dict(counts=[37, 2], firsts=[100, 9], page=3, heads=4, gap=1),
    "few_page5_hole": dict(counts=[40], firsts=[120], unmap=[(0, 3), (0, 19)], heads=4, page=5),
    "few_page5_512": dict(counts=[9, 1], firsts=[200, 3], heads=1, group=16, dim=512, page=5),
    "few_page7_512_own": dict(counts=[24], firsts=[200], heads=2, group=2, dim=512, own_rows=True, page=7),
    "few_page5_sinks": dict(counts=[50], firsts=[333], window=40, sinks=18, free_middle=True, page=5),
    "large_page5": dict(counts=[170, 2], firsts=[131, 100], page=5),
    "large_page5_own": dict(counts=[170, 2], firsts=[131, 100], page=5, own_rows=True),
    "large_page5_512": dict(counts=[60, 100], firsts=[131, 100], heads=1, group=16, dim=512, page=5),
    "large_page1": dict(counts=[170, 2], firsts=[60, 100], page=1),
    "few_tiles_hole": dict(counts=[40], firsts=[120], unmap=[(0, 3), (0, 9)], heads=4),
    "few_peaked": dict(counts=[8], firsts=[900], q_scale=30.0),
    "peaked": dict(counts=[64, 3], firsts=[500, 800], q_scale=30.0),
}


@pytest.mark.parametrize("name", list(CASES))
def test_attention_of_runs(kv, name):
    case = make_case(len(name) * 7 + 1, **CASES[name])
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_attention_without_lse(kv):
    case = make_case(5, [3, 70], [100, 400])
    a, t = device_args(kv, case, lse=False)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_runs_that_make_no_sense_are_skipped(kv):
    case = make_case(6, [5, 6, 7, 8, 9, 10], [50, 60, 70, 80, 90, 100], gap=1)
    case.seq[1] = 6          # not a sequence
    case.first[2] = -1
    case.count[3] = 0
    case.start[4] = case.rows - 3
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_few_rows_of_runs_that_make_no_sense_are_skipped(kv):
    case = make_case(6, [5, 6, 7], [50, 60, 70], gap=1)
    case.seq[1] = 3          # not a sequence
    case.count[2] = 0
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_pages_outside_the_cache_count_as_unmapped(kv):
    case = make_case(7, [30], [100])
    a, t = device_args(kv, case)
    case.table[0, 2] = -1
    t["page_table"][0, 2] = case.cfg[1]
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_repeated_and_replayed_calls_give_the_same_bits(kv):
    """A captured call (on its own stream, workspace of its own) and eager calls between its replays."""
    case = make_case(8, [1, 130, 7, 300], [3000, 100, 255, 77])
    a, t = device_args(kv, case)
    b, tb = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    want, want_lse = t["out"].clone(), t["lse"].clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        kv.chunk_attention(b, stream=torch.cuda.current_stream())
    for _ in range(5):
        t["out"].fill_(0)
        tb["out"].fill_(0)
        graph.replay()
        kv.chunk_attention(a)
        torch.cuda.synchronize()
        assert torch.equal(t["out"], want) and torch.equal(tb["out"], want)
        assert torch.equal(t["lse"], want_lse) and torch.equal(tb["lse"], want_lse)
    check_attention(case, t)


def test_a_replayed_call_reads_the_lengths_of_the_moment(kv):
    case = make_case(9, [20, 30], [500, 100])
    a, t = device_args(kv, case)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.chunk_attention(a, stream=torch.cuda.current_stream())
    case.count[:] = [3, 11]
    case.first[:] = [480, 40]
    t["row_count"].copy_(torch.from_numpy(case.count))
    t["first_position"].copy_(torch.from_numpy(case.first))
    graph.replay()
    torch.cuda.synchronize()
    check_attention(case, t)


@pytest.mark.parametrize("over", [dict(ring=True, window=256), dict(heads=1, group=8, dim=512), dict()])
def test_few_rows_captured_and_replayed(kv, over):
    """The small call's kernel in a graph, between eager calls on the same and on another stream; lengths change."""
    case = make_case(19, [2, 1], [700, 90], **over)
    case.count[:], case.first[:] = [1, 1], [650, 60]
    (a, t), (b, tb) = device_args(kv, case), device_args(kv, case)
    a.max_row_count = b.max_row_count = 2
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        for _ in range(3):
            kv.chunk_attention(b, stream=torch.cuda.current_stream())
    case.count[:], case.first[:] = [2, 1], [700, 90]
    for x in (t, tb):
        x["row_count"].copy_(torch.from_numpy(case.count))
        x["first_position"].copy_(torch.from_numpy(case.first))
    torch.cuda.synchronize()
    for _ in range(5):
        graph.replay()
        kv.chunk_attention(a, stream=side)
        kv.chunk_attention(a, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(t["out"], tb["out"]) and torch.equal(t["lse"], tb["lse"])
    check_attention(case, t)


@pytest.mark.parametrize("count", [40, 170])
@pytest.mark.parametrize("page,own", [(16, True), (64, True), (64, False), (5, True)])
def test_the_last_positions_there_are(kv, page, own, count):
    """A ring at the end of the positions: nothing beyond them is looked up."""
    end = 2**31 - 1024
    window = 128 if page != 5 else 125
    case = make_case(12, [count, 1], [end - 1 - count, end - 1 - 1], ring=True, window=window, page=page,
                     own_rows=own, ring_slots=None if own else 5)
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_rows_of_no_run_are_not_used(kv):
    """Rows between the runs hold NaN, and key tiles of 64 own rows reach into them and into the next run's."""
    case = make_case(13, [70, 3, 65, 1], [100, 64, 0, 7], own_rows=True, gap=2)
    free = torch.ones(case.rows, dtype=torch.bool)
    for s, c in zip(case.start, case.count):
        free[s:s + c] = False
    for x in (case.q, case.k_rows, case.v_rows):
        x[free] = float("nan")
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


@pytest.mark.parametrize("where", ["cache_k", "cache_v"])
@pytest.mark.parametrize("first", [40, 4000, 40000])      # few keys to a cluster's CTA, many; one launch more
def test_a_nan_that_a_row_sees_is_in_its_result(kv, where, first):
    case = make_case(14, [3], [first])
    page = int(case.table[0, 1])                         # position 20
    getattr(case, where)[0, page * 16 + 4, 5] = float("nan")
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    out, lse = t["out"].cpu().view(3, 8, 2, 256), t["lse"].cpu().view(3, 8, 2)
    assert bool(out[:, 5].isnan().all())
    assert bool(lse[:, 5].isnan().all()) == (where == "cache_k")
    want, want_lse, tol, tol_lse = (x.view(3, 8, 2, -1) for x in attention_f64(case)[0])
    rest = [h for h in range(8) if h != 5]
    assert bool(((out.double() - want).abs() <= tol)[:, rest].all())
    assert bool(((lse.double()[..., None] - want_lse).abs() <= tol_lse)[:, rest].all())


@pytest.mark.parametrize("ctas", [1, 2, 7])
def test_a_small_workspace_means_fewer_ctas(kv, ctas):
    case = make_case(15, [1, 130, 7], [900, 0, 255])
    a, t = device_args(kv, case)
    a.workspace_bytes = kv.chunk_workspace_bytes(16, 8, 256, 3, 130, sm_count=ctas)
    t["workspace"][a.workspace_bytes:].fill_(77)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)
    assert bool((t["workspace"][a.workspace_bytes:] == 77).all())


def test_calls_on_two_streams_at_once(kv):
    """Each with its own workspace, on streams of their own; the bits are those of the call alone."""
    case = make_case(16, [1, 130, 7, 300], [3000, 100, 255, 77])
    calls = [device_args(kv, case) for _ in range(3)]
    kv.chunk_attention(calls[0][0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for (a, _t), s in zip(calls[1:], streams):
            kv.chunk_attention(a, stream=s)
    torch.cuda.synchronize()
    for _a, t in calls[1:]:
        assert torch.equal(t["out"], calls[0][1]["out"]) and torch.equal(t["lse"], calls[0][1]["lse"])
    check_attention(case, calls[0][1])


def test_calls_one_behind_the_other_share_a_workspace(kv):
    """On one stream: the second call's partial results come after the first one's have been joined."""
    one, two = make_case(17, [3, 1], [6000, 4097]), make_case(18, [1, 130, 7], [2000, 0, 255])
    (a, ta), (b, tb) = device_args(kv, one), device_args(kv, two)
    work = torch.empty(max(a.workspace_bytes, b.workspace_bytes), dtype=torch.uint8, device="cuda")
    a.workspace = b.workspace = work.data_ptr()
    for _ in range(5):
        kv.chunk_attention(a)
        kv.chunk_attention(b)
    torch.cuda.synchronize()
    check_attention(one, ta)
    check_attention(two, tb)


@pytest.mark.parametrize("count", [20, 170])
def test_cache_offsets_beyond_32_bits(kv, count):
    """A cache of more than 2^32 bytes a tensor: the run's pages are its last ones."""
    case = make_case(10, [count, 1], [200, 70], page=64)
    a, t = device_args(kv, case)
    page_elems = 64 * 8 * 256
    pages = (1 << 32) // (page_elems * 2) + case.cfg[1] + 7
    shift = pages - case.cfg[1]
    for n in ("cache_k", "cache_v"):
        big = torch.zeros(pages, page_elems, dtype=torch.bfloat16, device="cuda")
        big[shift:] = t[n].view(-1, page_elems)
        t[n] = big
        setattr(a, n, big.data_ptr())
    t["page_table"][t["page_table"] >= 0] += shift
    a.cache_config.num_pages = pages
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)


def test_long_run_against_prompt_attention(kv):
    """The same prompt in one piece by the prompt attention and in chunks of odd length over the cache."""
    rng = np.random.default_rng(11)
    n, H, G, D, ps = 1500, 8, 2, 256, 16
    q, k, v = (torch.from_numpy(rng.standard_normal((n, h, D), dtype=np.float32)).to(torch.bfloat16).cuda()
               for h in (H * G, H, H))
    whole = torch.empty_like(q)
    kv.prefill_attention(whole, q, k, v, 1, n, H * G, H, D, 0, 1 / 16.0)
    slots = -(-n // ps)
    cfg = kv.make_kv_config(1, slots, ps, slots, 1, H, D, 0)
    table = torch.from_numpy(rng.permutation(slots).astype(np.int32)).cuda()
    ck, cv = (torch.full((slots * ps, H, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    done = 0
    for step in (1, 333, 64, 500, n):
        m = min(step, n - done)
        at = torch.arange(done, done + m, device="cuda")
        place = table[at // ps].long() * ps + at % ps
        ck[place], cv[place] = k[done:done + m], v[done:done + m]
        a = kv.ChunkArgs()
        ints = [torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, done, m, done)]
        a.seq_batch, a.first_position, a.row_count, a.row_start = (x.data_ptr() for x in ints)
        a.q, a.out, a.cache_k, a.cache_v, a.page_table = (x.data_ptr() for x in (q, out, ck, cv, table))
        size = kv.chunk_workspace_bytes(H * G, H, D, 1, m)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes, a.cache_config = ws.data_ptr(), size, cfg
        a.run_count, a.max_row_count, a.rows, a.q_heads, a.softmax_scale = 1, m, n, H * G, 1 / 16.0
        kv.chunk_attention(a)
        torch.cuda.synchronize()
        done += m
    # two results, each off by what chunk_cases.py derives: 2 (2^-8 (A + |out|)) with A <= max |v| of the row's average
    err = (out.float() - whole.float()).abs()
    assert err.max().item() <= 4 * 2.0 ** -8 * float(v.float().abs().max())
    assert err.mean().item() <= 2.0 ** -8 * float(whole.float().abs().mean()) * 2
