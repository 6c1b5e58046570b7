"""Append and write of runs of new tokens, page copies, and the operators together as a serving loop uses them."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.chunk_cases import attention_f64, check_attention, device_args, make_case
from tests.gpu_util import need_gpu

pytestmark = [pytest.mark.gpu, need_gpu]


def raw_inputs(kv, case, rotary, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, D = case.cfg[5], case.cfg[6]
    normal = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)  # noqa: E731
    w = torch.empty(2, D, device="cuda").normal_(1.0, 0.05, generator=gen).bfloat16()
    cos, sin = kv.fill_rope_tables(int((case.first.astype(np.int64) + case.count).max()), rotary // 2, 10000.0, D)
    return {"raw_q": normal(case.rows, case.q_heads, D), "raw_k": normal(case.rows, H, D),
            "raw_v": normal(case.rows, H, D), "q_norm_weight": w[0].contiguous(), "k_norm_weight": w[1].contiguous(),
            "cos": torch.from_numpy(cos).cuda(), "sin": torch.from_numpy(sin).cuda()}


def fill(a, tensors):
    for name, x in tensors.items():
        setattr(a, name, None if x is None else x.data_ptr())


def prepared(kv, case, raw, rotary, norm_mode, has_v=True):
    """Prepared rows of every run by the whole-prompt prep, whose bits the append has to have."""
    H, D = case.cfg[5], case.cfg[6]
    position = torch.full((case.rows,), -1, dtype=torch.int32)
    for s, f, c in zip(case.start, case.first, case.count):
        position[s:s + c] = torch.arange(f, f + c, dtype=torch.int32)
    position = position.cuda()
    q = torch.full((case.rows, case.q_heads, D), 7.0, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.full((case.rows, H, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv.prefill_prep(q, k, v, raw["raw_q"], raw["raw_k"], raw["raw_v"] if has_v else None, raw["q_norm_weight"],
                    raw["k_norm_weight"], raw["cos"], raw["sin"], position, case.rows, case.q_heads, H, D, rotary,
                    norm_mode)
    return q, k, v


def stored(case, cache, rows):
    """The cache with the runs' rows where they belong: later rows of a run over earlier ones, unmapped ones nowhere."""
    layers, pages, ps, slots, _, H, D, ring = case.cfg
    want = cache.clone().view(layers, pages * ps, H, D)
    for i in range(case.count.size):
        for r in range(int(case.count[i])):
            p = int(case.first[i]) + r
            if not ring and p // ps >= slots:
                continue
            page = int(case.table[case.seq[i], (p // ps) % slots])
            if 0 <= page < pages:
                want[case.layer, page * ps + p % ps] = rows[int(case.start[i]) + r]
    return want


APPENDS = {
    "ragged": dict(counts=[1, 33, 70, 2], firsts=[100, 0, 15, 300], gap=2),
    "page5": dict(counts=[21, 3], firsts=[7, 300], page=5),
    "layer": dict(counts=[21, 3], firsts=[7, 30], layers=2, layer=1),
    "dim512": dict(counts=[9, 40], firsts=[7, 64], heads=1, group=16, dim=512, page=64),
    "odd_heads": dict(counts=[9, 4], firsts=[7, 64], heads=3, group=1),
    "ring": dict(counts=[200, 3, 64], firsts=[10, 1000, 0], ring=True, window=64, own_rows=False),
    "unmapped": dict(counts=[40], firsts=[0], unmap=[(0, 1)]),
    "many_runs": dict(counts=[1 + i % 3 for i in range(70)], firsts=[i * 3 for i in range(70)]),
    # several rows to a CTA: runs that begin and end inside its share, gaps, pages of the ring it comes to again
    "shares": dict(counts=[700, 1, 650, 90, 2, 33], firsts=[3, 500, 0, 41, 7, 15], gap=3),
    "shares_ring": dict(counts=[700, 3, 640, 1], firsts=[10, 1000, 0, 63], ring=True, window=64, own_rows=False),
    "shares_many": dict(counts=[1 + i % 40 for i in range(100)], firsts=[i * 7 for i in range(100)], page=5, gap=1),
    "shares512": dict(counts=[300, 290, 5], firsts=[7, 64, 0], heads=1, group=16, dim=512, page=64, gap=2),
    "shares_odd": dict(counts=[900, 301], firsts=[7, 64], heads=3, group=1),
}


@pytest.mark.parametrize("norm_mode", [0, 1])
@pytest.mark.parametrize("name", list(APPENDS))
def test_append_has_the_prompt_preps_bits(kv, name, norm_mode):
    case = make_case(3, **APPENDS[name])
    rotary = 128 if case.cfg[6] == 512 else 256
    has_v = case.cfg[6] == 256
    raw = raw_inputs(kv, case, rotary, 1)
    q, k, v = prepared(kv, case, raw, rotary, norm_mode, has_v)
    a, t = device_args(kv, case)
    fill(a, raw)
    if not has_v:
        a.raw_v = None
    a.rotary_dim, a.norm_mode = rotary, norm_mode
    t["q"].fill_(7.0)
    want_k, want_v = stored(case, t["cache_k"], k), stored(case, t["cache_v"], v)
    kv.chunk_append(a)
    torch.cuda.synchronize()
    bits = lambda x: x.view(torch.int16).reshape(-1)  # noqa: E731
    assert torch.equal(bits(t["q"]), bits(q))
    assert torch.equal(bits(t["cache_k"]), bits(want_k)) and torch.equal(bits(t["cache_v"]), bits(want_v))


def test_append_beside_the_cache_then_write(kv):
    case = make_case(4, [200, 3, 64, 1], [10, 1000, 0, 70], ring=True, window=64, gap=1)
    raw = raw_inputs(kv, case, 256, 2)
    q, k, v = prepared(kv, case, raw, 256, 0)
    a, t = device_args(kv, case)
    fill(a, raw)
    a.rotary_dim = 256
    for n in ("q", "k_rows", "v_rows"):
        t[n].fill_(7.0)
    before = [t[n].clone() for n in ("cache_k", "cache_v")]
    kv.chunk_append(a)
    torch.cuda.synchronize()
    bits = lambda x: x.view(torch.int16).reshape(-1)  # noqa: E731
    assert all(torch.equal(bits(x), bits(y)) for x, y in ((t["q"], q), (t["k_rows"], k), (t["v_rows"], v),
                                                          (t["cache_k"], before[0]), (t["cache_v"], before[1])))
    kv.chunk_write(a)
    torch.cuda.synchronize()
    assert torch.equal(bits(t["cache_k"]), bits(stored(case, before[0], k)))
    assert torch.equal(bits(t["cache_v"]), bits(stored(case, before[1], v)))


@pytest.mark.parametrize("ring", [False, True])
def test_layer_step(kv, ring):
    """Append, attention and write in one call: the attention is that of the prepared rows, the cache ends with them."""
    case = make_case(5, [90, 1, 17], [120, 300, 0], ring=ring, window=64 if ring else 0)
    raw = raw_inputs(kv, case, 256, 3)
    q, k, v = prepared(kv, case, raw, 256, 0)
    a, t = device_args(kv, case)
    fill(a, raw)
    a.rotary_dim = 256
    want_k, want_v = stored(case, t["cache_k"], k), stored(case, t["cache_v"], v)
    kv.chunk_layer_step(a)
    torch.cuda.synchronize()
    bits = lambda x: x.view(torch.int16).reshape(-1)  # noqa: E731
    assert torch.equal(bits(t["cache_k"]), bits(want_k)) and torch.equal(bits(t["cache_v"]), bits(want_v))
    case.q = q.cpu()
    if ring:
        case.k_rows, case.v_rows = k.cpu(), v.cpu()
    else:
        case.cache_k, case.cache_v = (x.cpu().view(case.cache_k.shape) for x in (want_k, want_v))
    check_attention(case, t)


def test_a_captured_layer_step(kv):
    """Append, attention and write captured once, replayed on rows and lengths of the moment."""
    case = make_case(6, [90, 1, 17], [120, 300, 0], ring=True, window=64)
    raw = raw_inputs(kv, case, 256, 4)
    a, t = device_args(kv, case)
    fill(a, raw)
    a.rotary_dim = 256
    before = [t[n].clone() for n in ("cache_k", "cache_v")]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.chunk_layer_step(a, stream=torch.cuda.current_stream())
    case.count[:], case.first[:] = [33, 1, 16], [100, 290, 3]
    case.cache_k, case.cache_v = (torch.from_numpy(np.random.default_rng(8 + i).standard_normal(
        case.cache_k.shape, dtype=np.float32)).bfloat16() for i in range(2))
    for n in ("cache_k", "cache_v"):
        t[n].copy_(getattr(case, n))
    t["row_count"].copy_(torch.from_numpy(case.count))
    t["first_position"].copy_(torch.from_numpy(case.first))
    raw["raw_q"].mul_(0.5)
    q, k, v = prepared(kv, case, raw, 256, 0)
    want_k, want_v = stored(case, t["cache_k"], k), stored(case, t["cache_v"], v)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(before[0], t["cache_k"])
    bits = lambda x: x.view(torch.int16).reshape(-1)  # noqa: E731
    assert torch.equal(bits(t["cache_k"]), bits(want_k)) and torch.equal(bits(t["cache_v"]), bits(want_v))
    case.q, case.k_rows, case.v_rows = q.cpu(), k.cpu(), v.cpu()
    check_attention(case, t)


# --------------------------------------------------------------------------------------------- page copies
def copy_case(kv, layers, pages, ps, heads, dim, fp8, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    cfg = kv.make_kv_config(layers, pages, ps, pages, 1, heads, dim, 0)
    kind = torch.uint8 if fp8 else torch.int16
    caches = [torch.randint(0, 255 if fp8 else 32767, (layers, pages, ps, heads, dim), generator=gen, device="cuda",
                            dtype=torch.int32).to(kind) for _ in range(2)]
    scales = [torch.rand(layers, pages, heads, generator=gen, device="cuda") for _ in range(2)]
    return cfg, caches, scales


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layers,pages,ps,heads,dim,count", [
    (1, 10, 16, 8, 256, 1), (3, 40, 16, 8, 256, 13), (2, 9, 64, 8, 256, 4), (2, 30, 8, 1, 512, 9), (1, 400, 8, 3, 256, 150)])
@pytest.mark.parametrize("partial", [False, True])
def test_copy_pages(kv, fp8, layers, pages, ps, heads, dim, count, partial):
    cfg, caches, scales = copy_case(kv, layers, pages, ps, heads, dim, fp8, 1)
    rng = np.random.default_rng(2)
    pick = rng.permutation(pages).astype(np.int32)
    src, dst = pick[:count].copy(), pick[count:2 * count].copy()
    src[count // 2:] = src[0]                        # a fork: one source, several destinations
    rows = rng.integers(0, ps + 3, count).astype(np.int32) if partial else None
    want, want_scales = [c.clone() for c in caches], [s.clone() for s in scales]
    for i in range(count):
        n = ps if rows is None else min(int(rows[i]), ps)
        n = -(-n // 8) * 8 if fp8 else n
        for c in want:
            c[:, dst[i], :n] = c[:, src[i], :n]
        for s in want_scales:
            if n:
                s[:, dst[i]] = s[:, src[i]]
    up = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
    if fp8:
        kv.copy_pages_fp8(*caches, *scales, cfg, up(src), up(dst), up(rows), count)
    else:
        kv.copy_pages(*caches, cfg, up(src), up(dst), up(rows), count)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    if fp8:
        assert all(torch.equal(a, b) for a, b in zip(scales, want_scales))


def test_copy_pages_odd_page_and_pairs_that_make_no_sense(kv):
    cfg, caches, _ = copy_case(kv, 2, 20, 3, 1, 256, False, 3)
    src = torch.tensor([0, -1, 20, 4, 5, 6], dtype=torch.int32, device="cuda")
    dst = torch.tensor([10, 11, 12, 4, -7, 20], dtype=torch.int32, device="cuda")
    rows = torch.tensor([2, 3, 3, 3, 3, 3], dtype=torch.int32, device="cuda")
    want = [c.clone() for c in caches]
    for c in want:
        c[:, 10, :2] = c[:, 0, :2]
    kv.copy_pages(*caches, cfg, src, dst, rows, 6)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


# --------------------------------------------------------------------------------------------- all of it together
def test_fork_append_attend_release_compact(kv):
    """A prompt, two continuations that share its pages (copy-on-write of the partial page), the parent released, the
    pool compacted: each continuation's attention is that of its own tokens throughout."""
    H, G, D, ps, slots, pool = 8, 2, 256, 16, 20, 64
    cfg = kv.make_kv_config(1, pool, ps, slots, 3, H, D, 0)
    table, refs = np.full((3, slots), -1, dtype=np.int32), np.zeros(pool, dtype=np.int32)
    copies = kv.PageCopies(64)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    normal = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)  # noqa: E731
    ck, cv = (torch.full((1, pool * ps, H, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    weights = [normal(D) for _ in range(2)]
    cos, sin = (torch.from_numpy(x).cuda() for x in kv.fill_rope_tables(slots * ps, D // 2, 10000.0, D))
    history = {b: [] for b in range(3)}              # prepared (k, v) rows of each sequence, by position

    def make_copies():
        src, dst, rows = (torch.from_numpy(x[:copies.count].copy()).cuda() for x in (copies.src, copies.dst, copies.rows))
        kv.copy_pages(ck, cv, cfg, src, dst, rows, copies.count)
        copies.clear()

    def step(batches, firsts, counts):
        for b, f, c in zip(batches, firsts, counts):
            assert kv.pages_ensure(table, refs, cfg, b, f, c, copies) == 0
        make_copies()
        rows = sum(counts)
        starts = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(np.int32)
        t = {"raw_q": normal(rows, H * G, D), "raw_k": normal(rows, H, D), "raw_v": normal(rows, H, D),
             "q": torch.empty(rows, H * G, D, dtype=torch.bfloat16, device="cuda"),
             "out": torch.empty(rows, H * G, D, dtype=torch.bfloat16, device="cuda"),
             "lse": torch.empty(rows, H * G, device="cuda"), "q_norm_weight": weights[0], "k_norm_weight": weights[1],
             "cos": cos, "sin": sin, "cache_k": ck, "cache_v": cv}
        up = lambda x: torch.from_numpy(np.asarray(x, dtype=np.int32)).cuda()  # noqa: E731
        t.update(page_table=up(table), seq_batch=up(batches), first_position=up(firsts), row_count=up(counts),
                 row_start=up(starts))
        a = kv.ChunkArgs()
        fill(a, t)
        size = kv.chunk_workspace_bytes(H * G, H, D, len(counts), max(counts))
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes, a.cache_config = ws.data_ptr(), size, cfg
        a.run_count, a.max_row_count, a.rows, a.q_heads = len(counts), max(counts), rows, H * G
        a.rotary_dim, a.softmax_scale = 256, 1 / 16.0
        kv.chunk_layer_step(a)
        torch.cuda.synchronize()
        position = up(np.concatenate([np.arange(f, f + c) for f, c in zip(firsts, counts)]))
        q, k, v = (torch.empty(rows, h, D, dtype=torch.bfloat16, device="cuda") for h in (H * G, H, H))
        kv.prefill_prep(q, k, v, t["raw_q"], t["raw_k"], t["raw_v"], *weights, cos, sin, position, rows, H * G, H, D, 256)
        for b, f, c, s in zip(batches, firsts, counts, starts):
            assert len(history[b]) == f
            history[b] += list(zip(k[s:s + c].double(), v[s:s + c].double()))
            kk, vv = (torch.stack([h[n] for h in history[b]]) for n in (0, 1))
            scores = torch.einsum("thgd,khd->thgk", q[s:s + c].double().view(c, H, G, D), kk) / 16.0
            later = torch.arange(f + c, device="cuda")[None] > torch.arange(f, f + c, device="cuda")[:, None]
            scores = scores.masked_fill(later[:, None, None], -math.inf)
            p = scores.softmax(-1)
            want = torch.einsum("thgk,khd->thgd", p, vv).reshape(c, H * G, D)
            spread = torch.einsum("thgk,khd->thgd", p, vv.abs()).reshape(c, H * G, D)
            # tests/chunk_cases.py: weights and result rounded to bf16, scores of at most 2^6 in fp32
            tol = 2.0 ** -8 * (spread + want.abs()) + 2 * 1.5 * 256 * 2.0 ** -24 * 64 * spread
            assert ((t["out"][s:s + c].double() - want).abs() <= tol).all()

    step([0], [0], [75])
    assert kv.pages_fork(table, refs, cfg, 0, 1, 75) == 0 and kv.pages_fork(table, refs, cfg, 0, 2, 64) == 0
    history[1], history[2] = list(history[0]), list(history[0][:64])
    step([1, 2], [75, 64], [5, 30])                  # 1 copies the partial page, 2 starts a fresh one
    step([0, 2, 1], [75, 94, 80], [1, 1, 60])
    assert kv.pages_release(table, refs, cfg, 0, 0, slots) == 0
    history[0] = []
    code, used = kv.pages_compact(table, refs, cfg, copies)
    assert code == 0 and used == int((refs > 0).sum()) and int(table.max()) < used
    make_copies()
    step([1, 2], [140, 95], [3, 40])
    step([0], [0], [20])


@pytest.mark.parametrize("counts", [[4, 3], [70, 200]])
def test_two_runs_of_one_sequence_in_a_layer_step(kv, counts):
    """Over a linear cache, without rows beside it: the later run sees the earlier one's rows."""
    case = make_case(7, [sum(counts)], [90])
    b, tb = device_args(kv, case)
    raw = raw_inputs(kv, case, 256, 5)
    fill(b, raw)
    b.rotary_dim = 256
    kv.chunk_layer_step(b)
    a, t = device_args(kv, case)
    fill(a, raw)
    a.rotary_dim = 256
    runs = {"seq_batch": [0, 0], "first_position": [90, 90 + counts[0]], "row_count": counts, "row_start": [0, counts[0]]}
    for name, x in runs.items():
        t[name] = torch.tensor(x, dtype=torch.int32, device="cuda")
        setattr(a, name, t[name].data_ptr())
    a.run_count, a.max_row_count = 2, max(counts)
    size = kv.chunk_workspace_bytes(16, 8, 256, 2, max(counts))
    t["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = t["workspace"].data_ptr(), size
    kv.chunk_layer_step(a)
    torch.cuda.synchronize()
    bits = lambda x: x.view(torch.int16).reshape(-1)  # noqa: E731
    for name in ("q", "cache_k", "cache_v"):
        assert torch.equal(bits(t[name]), bits(tb[name]))
    case.q, case.cache_k, case.cache_v = t["q"].cpu(), t["cache_k"].cpu(), t["cache_v"].cpu()
    check_attention(case, t)
