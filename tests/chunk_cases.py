"""Seeded cases and 64-bit definitions for runs of new tokens over the paged cache.

A case is plain data: a cache (numpy bf16 bits), a page table, runs, and the same tensors as float64 for the definitions.
Places of the cache that no row of the call may see hold NaN."""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import numpy as np
import torch

BF16_HALF_STEP = 2.0 ** -8      # a rounding to bf16, relative
FP32_HALF_STEP = 2.0 ** -24


def bf16(rng: np.random.Generator, *shape) -> torch.Tensor:
    return torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).to(torch.bfloat16)


@dataclass
class ChunkCase:
    cfg: tuple
    layer: int
    q_heads: int
    table: np.ndarray
    seq: np.ndarray
    first: np.ndarray
    count: np.ndarray
    start: np.ndarray
    rows: int
    window: int          # as passed: 0 for a ring (its own) or none
    sinks: int
    scale: float
    q: torch.Tensor
    cache_k: torch.Tensor
    cache_v: torch.Tensor
    k_rows: torch.Tensor = None
    v_rows: torch.Tensor = None
    extra: dict = field(default_factory=dict)

    @property
    def group(self):
        return self.q_heads // self.cfg[5]

    @property
    def eff_window(self):
        return self.window or self.cfg[7]

    @property
    def max_rows(self):
        return int(self.count.max())


def visible_positions(case: ChunkCase, i: int):
    """Positions some row of run i sees (mapped or in its own rows), ascending, and where each lies."""
    _, num_pages, ps, slots, _, _, _, ring = case.cfg
    first, count, w = int(case.first[i]), int(case.count[i]), case.eff_window
    lo = max(0, first - w + 1) if w else 0
    wanted = [*range(min(case.sinks, lo, first + count)), *range(lo, first + count)]
    found = []
    for p in wanted:
        if case.k_rows is not None and p >= first:
            found.append((p, -1))
            continue
        page = p // ps
        if not ring and page >= slots:
            continue
        physical = int(case.table[case.seq[i], page % slots])
        if 0 <= physical < num_pages:
            found.append((p, physical * ps + p % ps))
    return found


def run_is_valid(case: ChunkCase, i: int) -> bool:
    return (0 <= case.seq[i] < case.cfg[4] and case.first[i] >= 0 and 0 < case.count[i]
            and case.start[i] >= 0 and case.start[i] + case.count[i] <= case.rows)


def make_case(seed, counts, firsts, *, heads=8, group=2, dim=256, page=16, window=0, ring=False, sinks=0, layers=1,
              layer=0, own_rows=None, gap=0, free_middle=False, unmap=(), spare_pages=3, ring_slots=None,
              q_scale=1.0) -> ChunkCase:
    """counts / firsts per run; `gap`: packed rows left between runs; `free_middle`: pages between the sinks and the
    first row's window are not mapped; `unmap`: (run, slot) entries set to -1."""
    rng = np.random.default_rng(seed)
    counts, firsts = np.asarray(counts, dtype=np.int32), np.asarray(firsts, dtype=np.int32)
    runs = counts.size
    own_rows = ring if own_rows is None else own_rows
    starts = np.concatenate([[0], np.cumsum(counts + gap)[:-1]]).astype(np.int32) + gap
    rows = int((counts + gap).sum()) + gap
    if ring:
        slots = ring_slots or -(-window // page)
    else:
        slots = max(1, max(-(-int(f + c) // page) for f, c in zip(firsts, counts)))
    need = np.zeros((runs, slots), dtype=bool)
    for i in range(runs):
        last = int(firsts[i]) + (0 if own_rows else int(counts[i]))
        pages = np.arange(-(-last // page)) if not ring else np.arange(max(0, last - slots * page) // page, -(-max(last, 1) // page))
        if free_middle and not ring:
            lo = max(0, int(firsts[i]) - window + 1) // page
            pages = pages[(pages >= lo) | (pages < -(-sinks // page))]
        need[i, pages % slots] = True
        if ring:
            need[i] = True
    total = int(need.sum()) + spare_pages
    pool = rng.permutation(total).astype(np.int32)
    table = np.full((runs, slots), -1, dtype=np.int32)
    table[need] = pool[:int(need.sum())]
    for i, s in unmap:
        table[i, s] = -1
    seq = rng.permutation(runs).astype(np.int32)
    table = table[np.argsort(seq)]          # run i is sequence seq[i]
    cfg = (layers, total, page, slots, runs, heads, dim, window if ring else 0)
    case = ChunkCase(cfg, layer, heads * group, table, seq, firsts, counts, starts, rows, 0 if ring else window, sinks,
                     q_scale / math.sqrt(dim), bf16(rng, rows, heads * group, dim), None, None)
    if own_rows:
        case.k_rows, case.v_rows = bf16(rng, rows, heads, dim), bf16(rng, rows, heads, dim)
    live = np.zeros((layers, total * page), dtype=bool)
    for i in range(runs):
        if run_is_valid(case, i):
            live[layer, [at for _, at in visible_positions(case, i) if at >= 0]] = True
    for name in ("cache_k", "cache_v"):
        cache = bf16(rng, layers, total * page, heads, dim)
        cache[torch.from_numpy(~live)] = float("nan")
        setattr(case, name, cache)
    return case


def attention_f64(case: ChunkCase):
    """{run: (out, lse, tolerance of out, tolerance of lse)} in 64 bits.

    Tolerances, per element. The weights are rounded to bf16 before they meet V: each is off by 2^-8 of itself, so the sum
    by 2^-8 A with A = sum w |v|. The result is rounded to bf16: 2^-8 |out|. A score is a sum of D products in fp32, off
    by at most D 2^-24 B with B = max over the keys of sum |q_i k_i| scale (half as much again for the scale and the
    accumulation in the tensor cores); a weight is exp of it, off by that much relative (twice: numerator and
    denominator), plus 2^-20 for the exponential. The log-sum-exp takes the scores' error and the sum's, n 2^-24."""
    H, D, G = case.cfg[5], case.cfg[6], case.group
    result = {}
    for i in range(case.count.size):
        if not run_is_valid(case, i):
            continue
        first, count, start, w = int(case.first[i]), int(case.count[i]), int(case.start[i]), case.eff_window
        seen = visible_positions(case, i)
        pos = torch.tensor([p for p, _ in seen], dtype=torch.long)

        def rows_of(cache, own):
            parts = [cache[case.layer, at] if at >= 0 else own[start + p - first] for p, at in seen]
            return torch.stack(parts).double() if parts else torch.zeros(0, H, D, dtype=torch.float64)

        k, v = rows_of(case.cache_k, case.k_rows), rows_of(case.cache_v, case.v_rows)
        q = case.q[start:start + count].double().view(count, H, G, D)
        t = (first + torch.arange(count))[:, None]
        sees = pos[None] <= t
        if w:
            sees &= (pos[None] > t - w) | (pos[None] < case.sinks)
        s = torch.einsum("thgd,khd->thgk", q, k) * case.scale
        size = torch.einsum("thgd,khd->thgk", q.abs(), k.abs()) * case.scale
        s = s.masked_fill(~sees[:, None, None], -math.inf)
        lse = torch.logsumexp(s, -1) if len(seen) else torch.full((count, H, G), -math.inf, dtype=torch.float64)
        p = torch.exp(s - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
        out = torch.einsum("thgk,khd->thgd", p, v)
        spread = torch.einsum("thgk,khd->thgd", p, v.abs())
        b = (size * sees[:, None, None]).amax(-1) if len(seen) else torch.zeros(count, H, G, dtype=torch.float64)
        score = 1.5 * D * FP32_HALF_STEP * b
        tol = BF16_HALF_STEP * (spread + out.abs()) + (2 * score + 2.0 ** -20)[..., None] * spread + 1e-30
        tol_lse = score + len(seen) * FP32_HALF_STEP + 2.0 ** -20 * (1 + torch.where(torch.isfinite(lse), lse.abs(), 0.0))
        shape = (count, H * G)
        result[i] = (out.reshape(*shape, D), lse.reshape(shape), tol.reshape(*shape, D), tol_lse.reshape(shape))
    return result


def device_args(kv, case: ChunkCase, lse=True, workspace=None):
    """A filled ChunkArgs for the attention and the tensors it points to."""
    def up(x):
        if x is None:
            return None
        return (torch.from_numpy(np.ascontiguousarray(x)) if isinstance(x, np.ndarray) else x).cuda()

    t = {n: up(getattr(case, n)) for n in ("q", "cache_k", "cache_v", "k_rows", "v_rows")}
    t.update(page_table=up(case.table), seq_batch=up(case.seq), first_position=up(case.first),
             row_count=up(case.count), row_start=up(case.start))
    t["out"] = torch.full((case.rows, case.q_heads, case.cfg[6]), 7.0, dtype=torch.bfloat16, device="cuda")
    t["lse"] = torch.full((case.rows, case.q_heads), 7.0, device="cuda") if lse else None
    t["status"] = torch.zeros(4, dtype=torch.int32, device="cuda")
    size = kv.chunk_workspace_bytes(case.q_heads, case.cfg[5], case.cfg[6], case.count.size, case.max_rows)
    t["workspace"] = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    a = kv.ChunkArgs()
    for name, x in t.items():
        if x is not None:
            setattr(a, name, x.data_ptr())
    a.cache_config = kv.make_kv_config(*case.cfg)
    a.workspace_bytes = size
    a.run_count, a.max_row_count, a.rows = case.count.size, case.max_rows, case.rows
    a.cache_layer, a.q_heads = case.layer, case.q_heads
    a.window_size, a.sink_tokens, a.softmax_scale = case.window, case.sinks, case.scale
    return a, t


def check_attention(case: ChunkCase, t):
    """Every run's rows within the derived tolerances, every other row as it was."""
    out, lse = t["out"].cpu().double(), None if t["lse"] is None else t["lse"].cpu().double()
    untouched = torch.ones(case.rows, dtype=torch.bool)
    for i, (want, want_lse, tol, tol_lse) in attention_f64(case).items():
        rows = slice(int(case.start[i]), int(case.start[i]) + int(case.count[i]))
        untouched[rows] = False
        worst = ((out[rows] - want).abs() / tol).max().item()
        assert worst <= 1.0, f"run {i}: out {worst:.2f} times its tolerance"
        if lse is not None:
            empty = torch.isinf(want_lse)
            assert torch.equal(lse[rows][empty], want_lse[empty])
            bad = ((lse[rows] - want_lse).abs() / tol_lse)[~empty]
            assert bad.numel() == 0 or bad.max().item() <= 1.0, f"run {i}: lse {bad.max().item():.2f} times its tolerance"
    assert bool((out[untouched] == 7.0).all())
    if lse is not None:
        assert bool((lse[untouched] == 7.0).all())
    assert t["status"].cpu().tolist()[0] == 0
