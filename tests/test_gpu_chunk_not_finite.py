"""NaN and infinities in V of runs of new tokens: they are in the results of the rows that see them and in no other,
whichever rows share a tile. Against the definition in 64 bits (tests/chunk_cases.py)."""
from __future__ import annotations

import copy
import math

import pytest
import torch

from tests.chunk_cases import attention_f64, check_attention, device_args, make_case
from tests.gpu_util import need_gpu

pytestmark = [pytest.mark.gpu, need_gpu]

NAN, INF = math.nan, math.inf


def places(case, i, position):
    """The row of (cache_v or v_rows) that position of run i is in."""
    _, _, ps, slots, _, _, _, _ = case.cfg
    if case.v_rows is not None and position >= int(case.first[i]):
        return case.v_rows, int(case.start[i]) + position - int(case.first[i])
    page = int(case.table[case.seq[i], (position // ps) % slots])
    return case.cache_v[case.layer], page * ps + position % ps


def spoil(case, spots):
    """spots: (run, position, KV head, dim, value). Returns the same case with zeros in their places."""
    clean = copy.copy(case)
    clean.cache_v = case.cache_v.clone()
    clean.v_rows = None if case.v_rows is None else case.v_rows.clone()
    for i, p, h, d, value in spots:
        for c, x in ((case, value), (clean, 0.0)):
            rows, at = places(c, i, p)
            rows[at, h, d] = x
    return clean


def check(kv, case, spots, args=None):
    clean = spoil(case, spots)
    a, t = device_args(kv, case) if args is None else args
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    assert t["status"].cpu().tolist()[0] == 0
    out, lse, w = t["out"].cpu().double(), t["lse"].cpu().double(), case.eff_window
    untouched = torch.ones(case.rows, dtype=torch.bool)
    for i, (want, want_lse, tol, tol_lse) in attention_f64(clean).items():
        first, count = int(case.first[i]), int(case.count[i])
        rows = slice(int(case.start[i]), int(case.start[i]) + count)
        untouched[rows] = False
        spoiled = torch.zeros_like(want, dtype=torch.bool)
        want = want.clone()
        for _i, p, h, d, value in (s for s in spots if s[0] == i):
            for t_row in range(count):
                t_at = first + t_row
                if p <= t_at and (not w or p > t_at - w or p < case.sinks):
                    at = (t_row, slice(h * case.group, (h + 1) * case.group), d)
                    spoiled[at] = True
                    want[at] = want[at] + value      # inf - inf: NaN
        got = out[rows]
        assert torch.equal(got[spoiled].isnan(), want[spoiled].isnan())
        inf = spoiled & want.isinf()
        assert torch.equal(got[inf], want[inf])
        worst = ((got - want).abs() / tol)[~spoiled].max().item()
        assert worst <= 1.0, f"run {i}: out {worst:.2f} times its tolerance"
        seen = ~want_lse.isinf()
        assert torch.equal(lse[rows][~seen], want_lse[~seen])
        assert bool(((lse[rows] - want_lse).abs() <= tol_lse)[seen].all())
    assert bool((out[untouched] == 7.0).all())


# (case, spots, kernels)
CASES = {
    # a drafted token whose row is bad: the tokens before it do not see it
    "few_cache": (dict(counts=[4], firsts=[500]), [(0, 502, 3, 17, NAN)], 1),
    "few_own": (dict(counts=[4], firsts=[1500], ring=True, window=1024), [(0, 1503, 0, slice(0, 256), NAN)], 1),
    "few_last_dims": (dict(counts=[8], firsts=[100]), [(0, 107, 7, slice(250, 256), INF)], 1),
    # a key that leaves the window: the rows behind the first do not see it
    "few_window_start": (dict(counts=[6], firsts=[400], window=100), [(0, 301, 2, 5, NAN), (0, 303, 2, 6, INF)], 1),
    "few_ring_start": (dict(counts=[6], firsts=[400], ring=True, window=96), [(0, 305, 2, 5, NAN), (0, 404, 1, 9, NAN)], 1),
    "few_tiles": (dict(counts=[61], firsts=[300]), [(0, 320, 1, 30, NAN), (0, 355, 4, 31, INF), (0, 355, 4, 32, -INF)], 1),
    "few_page5": (dict(counts=[30], firsts=[300], page=5), [(0, 320, 1, 30, NAN), (0, 329, 4, 31, NAN)], 1),
    "few_512": (dict(counts=[3], firsts=[900], heads=1, group=16, dim=512, page=64),
                [(0, 901, 0, 3, NAN), (0, 902, 0, slice(300, 512), INF)], 1),
    "few_sinks": (dict(counts=[8], firsts=[700], window=100, sinks=37, free_middle=True),
                  [(0, 2, 1, 1, INF), (0, 602, 1, 2, NAN), (0, 705, 0, 3, NAN)], 1),
    "few_tiny_window": (dict(counts=[8], firsts=[40], window=3), [(0, 41, 5, 100, NAN), (0, 39, 5, 101, NAN)], 1),
    "few_row_without_a_key": (dict(counts=[5], firsts=[13], unmap=[(0, 0)]), [(0, 16, 2, 8, NAN), (0, 17, 0, 0, INF)], 1),
    # both signs, and a NaN behind an infinity
    "few_signs": (dict(counts=[6], firsts=[50]), [(0, 10, 0, 0, INF), (0, 53, 0, 0, -INF), (0, 11, 1, 1, INF), (0, 54, 1, 1, NAN)], 1),
    # whole items (several query tiles of one CTA) and items that CTAs share
    "whole": (dict(counts=[1300, 1200, 900], firsts=[10, 0, 130], heads=2, ring=True, window=96),
              [(0, 700, 0, 7, NAN), (1, 5, 1, 255, INF), (2, 130 + 899, 0, 128, NAN), (0, 12, 1, 127, NAN)], 2),
    "shared": (dict(counts=[200, 3], firsts=[700, 800]), [(0, 750, 3, 7, NAN), (0, 899, 6, slice(0, 256), INF), (1, 801, 1, 200, NAN)], 2),
    "shared_by_many": (dict(counts=[3], firsts=[40000]), [(0, 40001, 3, 7, NAN), (0, 40002, 6, slice(0, 256), INF)], 2),
    "window": (dict(counts=[500, 33], firsts=[300, 700], window=90), [(0, 215, 3, 7, NAN), (0, 640, 1, 9, INF), (1, 612, 0, 0, NAN)], 2),
    "sinks": (dict(counts=[350, 33], firsts=[700, 0], window=100, sinks=70, free_middle=True),
              [(0, 1, 3, 7, NAN), (0, 605, 1, 9, INF), (1, 30, 0, 0, NAN)], 2),
    "own_rows": (dict(counts=[300, 130], firsts=[333, 0], own_rows=True), [(0, 500, 3, 7, NAN), (1, 64, 2, 2, NAN)], 2),
    "page5": (dict(counts=[200, 130], firsts=[333, 0], page=5), [(0, 500, 3, 7, NAN), (1, 64, 2, 2, NAN)], 2),
    "group64": (dict(counts=[50, 30], firsts=[130, 64], heads=1, group=64), [(0, 140, 0, 7, NAN), (1, 93, 0, 2, INF)], 2),
    "row_without_a_key": (dict(counts=[300, 5], firsts=[13, 100], unmap=[(0, 0)]), [(0, 16, 2, 8, NAN), (0, 17, 0, 0, INF)], 2),
    "dim512": (dict(counts=[100, 60], firsts=[6000, 20], heads=1, group=16, dim=512, page=64),
               [(0, 6050, 0, 3, NAN), (1, 79, 0, slice(250, 270), INF)], 2),
    "dim512_ring": (dict(counts=[400, 300], firsts=[300, 1000], heads=1, group=16, dim=512, ring=True, window=128),
                    [(0, 500, 0, 3, NAN), (1, 874, 0, 300, NAN)], 2),
}


@pytest.mark.parametrize("name", list(CASES))
def test_only_rows_that_see_it_have_it(kv, name):
    over, spots, launches = CASES[name]
    case = make_case(31, **over)
    args = device_args(kv, case)
    if launches != kv.chunk_attention_launches(args[0]):
        pytest.fail("the case is another kernel's")
    check(kv, case, spots)


@pytest.mark.parametrize("over", [dict(counts=[6, 1], firsts=[200, 50]), dict(counts=[700, 300], firsts=[200, 0], heads=2),
                                  dict(counts=[40, 90], firsts=[300, 2000], heads=1, group=16, dim=512, page=64)])
@pytest.mark.parametrize("value", [NAN, INF])
def test_every_value_of_a_head(kv, over, value):
    """A model whose V is broken throughout: every row of the head is, and the rows of the other heads are not."""
    case = make_case(32, **over)
    spots = [(i, p, 0, slice(None), value) for i in range(2) for p in range(int(case.first[i] + case.count[i]))]
    H, D = case.cfg[5:7]
    for i, p, h, d, x in spots:
        rows, at = places(case, i, p)
        rows[at, h, d] = x
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    out = t["out"].cpu().view(case.rows, H, case.group, D).double()
    assert bool((out[:, 0].isnan() if math.isnan(value) else out[:, 0] == value).all())
    for i, (want, _lse, tol, _tol_lse) in attention_f64(case).items():
        rows = slice(int(case.start[i]), int(case.start[i] + case.count[i]))
        shape = (-1, H, case.group, D)
        assert bool(((out[rows] - want.view(shape)).abs() <= tol.view(shape))[:, 1:].all())


def test_a_nan_in_the_scores_stays(kv):
    """Of K or of q: the whole row, and nothing that the other rows' values could repair."""
    for over in (dict(counts=[5], firsts=[300]), dict(counts=[300], firsts=[300])):
        case = make_case(33, **over)
        case.q[2, 3] = NAN
        a, t = device_args(kv, case)
        kv.chunk_attention(a)
        torch.cuda.synchronize()
        out, lse = t["out"].cpu(), t["lse"].cpu()
        assert bool(out[2, 3].isnan().all()) and bool(lse[2, 3].isnan())
        out[2, 3] = lse[2, 3] = 0.0
        assert not bool(out.isnan().any()) and not bool(lse.isnan().any())


@pytest.mark.parametrize("over", [dict(counts=[6], firsts=[400], window=100), dict(counts=[300, 80], firsts=[400, 30], window=100)])
def test_captured_and_repeated_calls_give_the_same_bits(kv, over):
    case = make_case(34, **over)
    spoil(case, [(0, 302, 2, 5, NAN), (0, 403, 1, slice(0, 9), INF)])
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    want = t["out"].view(torch.int16).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.chunk_attention(a, stream=torch.cuda.current_stream())
    for _ in range(10):
        t["out"].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t["out"].view(torch.int16), want)


@pytest.mark.parametrize("over", [dict(counts=[6, 1], firsts=[200, 50]), dict(counts=[300, 130], firsts=[200, 0])])
def test_an_average_of_the_largest_values_is_finite(kv, over):
    case = make_case(35, **over)
    most = torch.finfo(torch.bfloat16).max
    for i in range(2):
        for p in range(int(case.first[i] + case.count[i])):
            rows, at = places(case, i, p)
            rows[at, 0, :128] = most
            rows[at, 1, 5] = -most if p % 2 else most / 2
    a, t = device_args(kv, case)
    kv.chunk_attention(a)
    torch.cuda.synchronize()
    check_attention(case, t)
