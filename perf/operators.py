"""What the paged-cache operators of chunks cost: the cases, their plain forms and their 64-bit values.

Four operators that work on runs of new tokens (a chunk of a prompt, the drafted tokens of a speculative step, a single
token) of sequences that already have rows in the paged K/V cache:

- ``append``: RMSNorm and rotary embedding of the runs' projections, K and V rows straight into the pages;
- ``attention``: the runs' queries over the cache (and, for a sliding ring, over the run's own rows), causal, with the
  log-sum-exp of every row;
- ``attention`` with a window and sinks over a linear cache whose middle pages are already given back;
- ``pages``: copies of pages inside a cache (the copy behind a fork, a copy-on-write, a compaction).

``run`` computes them in elementary torch operations in 32 bits, or, with ``own`` true, calls the library.
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

WINDOW = 1024          # the sliding layers' window
EPS = 1.0e-6


# ------------------------------------------------------------------------------------------------ cases
def listed():
    sliding = {"heads": 8, "group": 2, "dim": 256, "rotary": 256}
    return [
        # four drafted tokens of one sequence on a sliding layer: the ring holds exactly the window, so the run's own
        # rows are not in it yet; the smallest call there is, latency is all of it
        {"name": "verify_one_ring", "op": "attention", **sliding, "runs": 1, "count_lo": 4, "count_hi": 4,
         "first_lo": 1500, "first_hi": 1500, "page": 16, "window": WINDOW, "ring": 1, "sinks": 0, "lengths": 1},
        # a speculative step of a batch: one to eight drafted tokens a sequence over long linear caches
        {"name": "verify_batch", "op": "attention", **sliding, "runs": 32, "count_lo": 1, "count_hi": 8,
         "first_lo": 512, "first_hi": 12000, "page": 16, "window": 0, "ring": 0, "sinks": 0, "lengths": 2},
        # a chunk of a long prompt behind what earlier chunks left in the cache of a global layer
        {"name": "prompt_chunk", "op": "attention", **sliding, "runs": 1, "count_lo": 4096, "count_hi": 4096,
         "first_lo": 12288, "first_hi": 12288, "page": 16, "window": 0, "ring": 0, "sinks": 0, "lengths": 3},
        # prompts of several sequences that go through a sliding layer in one packed batch of chunks, odd lengths
        {"name": "prompt_ragged_ring", "op": "attention", **sliding, "runs": 8, "count_lo": 65, "count_hi": 1500,
         "first_lo": 0, "first_hi": 5000, "page": 16, "window": WINDOW, "ring": 1, "sinks": 0, "lengths": 4},
        # the global layers' other geometry: sixteen query heads on one KV head of 512 dims, pages of 64
        {"name": "global_chunk", "op": "attention", "heads": 1, "group": 16, "dim": 512, "rotary": 128, "runs": 3,
         "count_lo": 200, "count_hi": 700, "first_lo": 1000, "first_hi": 6000, "page": 64, "window": 0, "ring": 0,
         "sinks": 0, "lengths": 5},
        # streaming decode: one token of each of 64 long sequences, four first tokens kept, the middle pages freed
        {"name": "sink_decode", "op": "attention", **sliding, "runs": 64, "count_lo": 1, "count_hi": 1,
         "first_lo": 300, "first_hi": 32000, "page": 16, "window": 2048, "ring": 0, "sinks": 4, "lengths": 6},
        # the same cache while a prompt still comes in by chunks
        {"name": "sink_chunk", "op": "attention", **sliding, "runs": 4, "count_lo": 700, "count_hi": 1100,
         "first_lo": 0, "first_hi": 20000, "page": 32, "window": 2048, "ring": 0, "sinks": 64, "lengths": 7},
        # the rows of a small speculative step
        {"name": "append_few", "op": "append", **sliding, "runs": 4, "count_lo": 1, "count_hi": 5, "first_lo": 100,
         "first_hi": 4000, "page": 16, "lengths": 8},
        # the rows of a packed batch of prompt chunks
        {"name": "append_prompts", "op": "append", **sliding, "runs": 9, "count_lo": 33, "count_hi": 2000,
         "first_lo": 0, "first_hi": 6000, "page": 16, "lengths": 9},
        # copy-on-write of the last, partly filled page of sixteen forked sequences, all layers of a small cache
        {"name": "fork_tails", "op": "pages", "heads": 8, "dim": 256, "layers": 4, "page": 16, "pages": 600,
         "copies": 16, "partial": True, "fp8": False, "lengths": 10},
        # compaction of a cache after sequences have left: two thousand whole pages move down
        {"name": "compact", "op": "pages", "heads": 8, "dim": 256, "layers": 4, "page": 16, "pages": 6000,
         "copies": 2000, "partial": False, "fp8": False, "lengths": 11},
        # a fork of a whole sequence's pages in an 8-bit cache, scales with them
        {"name": "fork_fp8", "op": "pages", "heads": 8, "dim": 256, "layers": 2, "page": 16, "pages": 2000,
         "copies": 500, "partial": False, "fp8": True, "lengths": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    cap = max(_cost(c) for c in listed() if c["op"] == "attention")
    while True:
        kind = rng.choice(["linear", "linear", "ring", "global", "sinks", "append", "pages"])
        seed = rng.randrange(1 << 20)
        if kind == "pages":
            copies = _log(rng, 1, 1500)
            fp8 = rng.random() < 0.4
            return {"op": "pages", "heads": 8 if fp8 else rng.choice([8, 8, 4, 1]), "dim": 256,
                    "layers": rng.randint(1, 4), "page": rng.choice([8, 16, 32] if fp8 else [3, 8, 16, 16, 64]),
                    "pages": 2 * copies + rng.randint(1, 500), "copies": copies, "partial": rng.random() < 0.5,
                    "fp8": fp8, "lengths": seed}
        if kind == "append":
            case = {"op": "append", "heads": rng.choice([8, 8, 4, 2, 1]), "group": 2, "dim": 256, "rotary": 256}
            if rng.random() < 0.25:
                case.update(heads=1, group=16, dim=512, rotary=128)
            hi = _log(rng, 1, 2000)
            case.update(runs=rng.randint(1, 10), count_lo=max(1, hi // rng.randint(1, 8)), count_hi=hi,
                        first_lo=rng.randint(0, 50), first_hi=rng.randint(50, 6000),
                        page=rng.choice([5, 8, 16, 16, 64]), lengths=seed)
            return case
        case = {"op": "attention", "heads": rng.choice([8, 8, 8, 4, 2, 1]), "group": 2, "dim": 256, "rotary": 256,
                "page": rng.choice([8, 16, 16, 32, 64, 24, 5]), "window": 0, "ring": 0, "sinks": 0}
        if kind == "global":
            case.update(heads=1, group=16, dim=512, rotary=128)
        hi = _log(rng, 1, 3000)
        first = _log(rng, 1, 16000)
        case.update(runs=_log(rng, 1, 48), count_lo=max(1, hi // rng.randint(1, 10)), count_hi=hi,
                    first_lo=rng.randint(0, first), first_hi=first, lengths=seed)
        if kind == "ring":
            case.update(window=rng.choice([WINDOW, WINDOW, 512, 100]), ring=1)
        if kind == "sinks":
            case.update(window=_log(rng, 64, 5000), sinks=rng.choice([1, 4, 16, 100]))
        if _cost(case) <= cap:
            return case


# ------------------------------------------------------------------------------------------------ sizes
def _runs(case):
    """Lengths of the runs and positions of their first tokens: spread over the case's ranges, the same for every seed."""
    rs = np.random.RandomState(case["lengths"])
    n = case["runs"]
    counts = rs.randint(case["count_lo"], case["count_hi"] + 1, n)
    firsts = rs.randint(case["first_lo"], case["first_hi"] + 1, n)
    return counts.astype(np.int64), firsts.astype(np.int64)


def _visible(case, first, count):
    """(keys that any row of the run sees, sum over its rows of the keys each sees)."""
    w, s = case["window"], case["sinks"]
    t = np.arange(first, first + count)
    lo = np.maximum(0, t - w + 1) if w else np.zeros_like(t)
    pairs = int((t - lo + 1 + np.minimum(s, lo)).sum())
    keys = first + count - int(lo[0]) + min(s, int(lo[0]))
    return keys, pairs


def _cost(case):
    """Values of the largest intermediate of the plain form and its multiplications, as one number to stay under."""
    counts, firsts = _runs(case)
    span = max(int(f + c) - (max(0, int(f) - case["window"] + 1) if case["window"] else 0)
               for c, f in zip(counts, firsts)) + case["sinks"]
    rows = case["runs"] * int(counts.max())
    heads = case["heads"] * case["group"]
    return max(rows * span * heads * case["dim"] / 256, 2 * case["runs"] * span * case["heads"] * case["dim"])


def work(case):
    if case["op"] == "pages":
        rows = int(_rows_to_copy(case).sum())
        row = case["heads"] * case["dim"] * (1 if case["fp8"] else 2)
        scales = case["copies"] * case["heads"] * 4 if case["fp8"] else 0
        return {"bytes": 2 * case["layers"] * 2 * (rows * row + scales), "flops": 0}
    counts, firsts = _runs(case)
    rows, hq = int(counts.sum()), case["heads"] * case["group"]
    if case["op"] == "append":
        tables = len(set().union(*(range(f, f + c) for c, f in zip(counts, firsts)))) * case["rotary"] * 4
        raw = case["group"] + (1 if case["dim"] == 512 else 2)
        return {"bytes": rows * case["heads"] * case["dim"] * 2 * (raw + case["group"] + 2) + tables,
                "flops": rows * case["heads"] * case["dim"] * (case["group"] + 2) * 7}
    keys, pairs = (sum(v) for v in zip(*(_visible(case, int(f), int(c)) for c, f in zip(counts, firsts))))
    return {"bytes": keys * case["heads"] * case["dim"] * 4 + rows * hq * (case["dim"] * 4 + 4),
            "flops": 4 * pairs * hq * case["dim"]}


def _rows_to_copy(case):
    rs = np.random.RandomState(case["lengths"])
    n = rs.randint(1, case["page"] + 1, case["copies"]) if case["partial"] else np.full(case["copies"], case["page"])
    return (n + 7) // 8 * 8 if case["fp8"] else n      # an 8-bit cache keeps blocks of eight rows


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))

    def normal(*shape):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    H, D, ps = case["heads"], case["dim"], case["page"]
    if case["op"] == "pages":
        L, P = case["layers"], case["pages"]
        st = {"case": case, "config": (L, P, ps, P, 1, H, D, 0)}
        for name in ("cache_k", "cache_v"):
            rows = normal(L, P, ps, H, D)
            if case["fp8"]:
                rows = rows.mul_(100).clamp_(-440, 440).to(torch.float8_e4m3fn).view(torch.uint8)
                st["scale" + name[5:]] = torch.rand(L, P, H, generator=gen, device="cuda")
            st[name] = rows
        pick = rs.permutation(P)[:2 * case["copies"]]
        st["src"], st["dst"] = ints(pick[:case["copies"]]), ints(pick[case["copies"]:])
        st["row_count"] = ints(_rows_to_copy(case)) if case["partial"] else None
        return st

    counts, firsts = _runs(case)
    R, rows, hq = case["runs"], int(counts.sum()), H * case["group"]
    starts = np.concatenate([[0], np.cumsum(counts)[:-1]])
    window = case.get("window", 0)
    ring = case.get("ring", 0)
    if ring:      # the ring holds the window and nothing else: the run's own rows come in beside it
        slots = -(-window // ps)
        table = np.arange(R * slots).reshape(R, slots)
    else:
        slots = int(max(-(-int(f + c) // ps) for c, f in zip(counts, firsts)))
        table = np.full((R, slots), -1)
        used = 0
        for i in range(R):
            keep = np.arange(-(-int(firsts[i] + counts[i]) // ps))
            if window:      # pages between the sinks and the window of the first row are given back
                lo = max(0, int(firsts[i]) - window + 1)
                keep = keep[(keep < -(-case["sinks"] // ps)) | (keep >= lo // ps)]
            table[i, keep] = np.arange(used, used + keep.size)
            used += keep.size
    pages = int(table.max()) + 1
    table = np.where(table >= 0, rs.permutation(pages)[np.maximum(table, 0)], -1)
    st = {"case": case, "config": (1, pages, ps, slots, R, H, D, window if ring else 0),
          "table": ints(table), "seq": ints(np.arange(R)), "first": ints(firsts), "count": ints(counts),
          "start": ints(starts), "rows": rows, "longest": int(counts.max()),
          "span": int(max(f + c - (max(0, f - window + 1) if window else 0) for c, f in zip(counts, firsts))),
          "cache_k": normal(pages, ps, H, D), "cache_v": normal(pages, ps, H, D),
          "q": normal(rows, hq, D)}
    if case["op"] == "append":
        weights = torch.empty(2, D, device="cuda").normal_(1.0, 0.05, generator=gen).bfloat16()
        st["q_weight"], st["k_weight"] = weights[0].contiguous(), weights[1].contiguous()
        half = case["rotary"] // 2
        angle = torch.outer(torch.arange(int((firsts + counts).max()), dtype=torch.float64),
                            10000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / D))
        st["cos"], st["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
        st["raw_q"] = normal(rows, hq, D)
        st["raw_k"] = normal(rows, H, D)
        st["raw_v"] = normal(rows, H, D) if D == 256 else None
        return st
    st["k_rows"] = normal(rows, H, D) if ring else None
    st["v_rows"] = normal(rows, H, D) if ring else None
    st["out"] = torch.zeros(rows, hq, D, dtype=torch.bfloat16, device="cuda")
    st["lse"] = torch.zeros(rows, hq, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _own(st)
    return {"attention": _plain_attention, "append": _plain_append, "pages": _plain_pages}[st["case"]["op"]](st)


def _library():
    name = "gemma_c_b200"
    if name not in sys.modules:
        pkg = Path(__file__).resolve().parent.parent / "gemma.c_b200"
        spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _own(st):
    kv, case = _library(), st["case"]
    if case["op"] == "pages":
        if "cfg" not in st:
            st["cfg"] = kv.make_kv_config(*st["config"])
        if case["fp8"]:
            kv.copy_pages_fp8(st["cache_k"], st["cache_v"], st["scale_k"], st["scale_v"], st["cfg"], st["src"],
                              st["dst"], st["row_count"], case["copies"])
        else:
            kv.copy_pages(st["cache_k"], st["cache_v"], st["cfg"], st["src"], st["dst"], st["row_count"],
                          case["copies"])
        return _pages_of(st)
    if "args" not in st:      # the filled argument block a caller keeps from call to call
        a = kv.ChunkArgs()
        a.cache_config = kv.make_kv_config(*st["config"])
        pointers = {"q": "q", "cache_k": "cache_k", "cache_v": "cache_v", "page_table": "table", "seq_batch": "seq",
                    "first_position": "first", "row_count": "count", "row_start": "start", "out": "out", "lse": "lse",
                    "k_rows": "k_rows", "v_rows": "v_rows", "raw_q": "raw_q", "raw_k": "raw_k", "raw_v": "raw_v",
                    "q_norm_weight": "q_weight", "k_norm_weight": "k_weight", "cos": "cos", "sin": "sin"}
        for field, key in pointers.items():
            if st.get(key) is not None:
                setattr(a, field, st[key].data_ptr())
        a.run_count, a.max_row_count, a.rows = case["runs"], st["longest"], st["rows"]
        a.cache_layer, a.q_heads = 0, case["heads"] * case["group"]
        if case["op"] == "attention":
            a.window_size = 0 if case["ring"] else case["window"]
            a.sink_tokens, a.softmax_scale = case["sinks"], 1.0 / math.sqrt(case["dim"])
            size = kv.chunk_workspace_bytes(a.q_heads, case["heads"], case["dim"], case["runs"], st["longest"])
            st["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
            a.workspace, a.workspace_bytes = st["workspace"].data_ptr(), size
        else:
            a.rotary_dim, a.norm_mode = case["rotary"], kv.NORM_RSQRT_APPROX
        st["args"] = a
    if case["op"] == "attention":
        kv.chunk_attention(st["args"])
        return {"out": st["out"], "lse": st["lse"]}
    kv.chunk_append(st["args"])
    return {"q": st["q"], "cache_k": st["cache_k"], "cache_v": st["cache_v"]}


def _cache_rows(st, positions, valid):
    """Row of the flattened cache that holds each position [runs, n] of each run's sequence, and whether there is one."""
    _, _, ps, slots, _, _, _, window = st["config"]
    page = torch.where(valid, positions, 0) // ps
    slot = page % slots if window else page.clamp(max=slots - 1)
    physical = torch.gather(st["table"].long()[st["seq"].long()], 1, slot)
    return physical.clamp(min=0) * ps + positions.clamp(min=0) % ps, valid & (physical >= 0)


def _plain_attention(st):
    case = st["case"]
    H, G, D, w, sinks = case["heads"], case["group"], case["dim"], case["window"], case["sinks"]
    R, M = case["runs"], st["longest"]
    first, count, start = st["first"].long()[:, None], st["count"].long()[:, None], st["start"].long()[:, None]
    dev = first.device
    # every key position that a row of the run may see: the first `sinks`, then from the first row's window on
    lo = (first - w + 1).clamp(min=0) if w else torch.zeros_like(first)
    tail = lo + torch.arange(st["span"], device=dev)
    head = torch.arange(sinks, device=dev).expand(R, sinks)
    pos = torch.cat([head, tail], 1)
    valid = torch.cat([head < lo, tail < first + count], 1)
    fresh = valid & (pos >= first) if st["k_rows"] is not None else torch.zeros_like(valid)
    at, mapped = _cache_rows(st, pos, valid & ~fresh)
    valid = mapped | fresh
    own_row = (start + (pos - first).clamp(min=0)).clamp(max=st["rows"] - 1)

    def keys(cache, rows):
        x = cache.view(-1, H, D)[at]
        if rows is not None:
            x = torch.where(fresh[:, :, None, None], rows[own_row], x)
        return x.float().transpose(1, 2)                                   # [runs, kv heads, keys, dims]

    row = torch.arange(M, device=dev)[None]
    live = row < count
    at_row = torch.where(live, start + row, 0)
    q = st["q"][at_row].float().view(R, M, H, G, D).permute(0, 2, 3, 1, 4).reshape(R, H, G * M, D)
    s = (q @ keys(st["cache_k"], st["k_rows"]).transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(R, H, G, M, -1)
    t = (first + row)[:, :, None]
    sees = valid[:, None] & (pos[:, None] <= t)
    if w:
        sees &= (pos[:, None] > t - w) | (pos[:, None] < sinks)
    s.masked_fill_(~sees[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(R, H, G * M, -1) @ keys(st["cache_v"], st["v_rows"])).view(R, H, G, M, D)
    out = out / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    pick = live.view(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(R * M, H * G, D)[pick]
    lse = lse.permute(0, 3, 1, 2).reshape(R * M, H * G)[pick]
    target = at_row.view(-1)[pick]
    st["out"][target] = out.to(torch.bfloat16)
    st["lse"][target] = lse
    return {"out": st["out"], "lse": st["lse"]}


def _plain_append(st):
    case = st["case"]
    half = case["rotary"] // 2
    row = torch.arange(st["longest"], device="cuda")[None]
    count, start, first = st["count"].long()[:, None], st["start"].long()[:, None], st["first"].long()[:, None]
    live = row < count
    at, mapped = _cache_rows(st, first + row, live)
    order = (start + row)[mapped]                 # source row of each row that has a place in the cache
    position = torch.zeros(st["rows"], dtype=torch.long, device="cuda")
    position[(start + row)[live]] = (first + row)[live]
    cos, sin = st["cos"][position][:, None], st["sin"][position][:, None]

    def norm(x):
        x = x.float()
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)

    def rotated(x, weight):
        x = norm(x) * weight.float()
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(torch.bfloat16)

    st["q"].copy_(rotated(st["raw_q"], st["q_weight"]))
    k = rotated(st["raw_k"], st["k_weight"])
    v = norm(st["raw_k"] if st["raw_v"] is None else st["raw_v"]).to(torch.bfloat16)
    st["cache_k"].view(-1, *k.shape[1:])[at[mapped]] = k[order]
    st["cache_v"].view(-1, *v.shape[1:])[at[mapped]] = v[order]
    return {"q": st["q"], "cache_k": st["cache_k"], "cache_v": st["cache_v"]}


def _plain_pages(st):
    case = st["case"]
    src, dst = st["src"].long(), st["dst"].long()
    if st["row_count"] is None:
        st["cache_k"][:, dst] = st["cache_k"][:, src]
        st["cache_v"][:, dst] = st["cache_v"][:, src]
    else:
        keep = torch.arange(case["page"], device="cuda")[None] < st["row_count"][:, None]
        if case["fp8"]:      # K pages are blocks of eight rows, head by head: whole blocks either way
            keep = keep.view(case["copies"], -1, 8).any(-1, keepdim=True).expand(-1, -1, 8).reshape(keep.shape)
        keep = keep[None, :, :, None, None]
        st["cache_k"][:, dst] = torch.where(keep, st["cache_k"][:, src], st["cache_k"][:, dst])
        st["cache_v"][:, dst] = torch.where(keep, st["cache_v"][:, src], st["cache_v"][:, dst])
    if case["fp8"]:
        st["scale_k"][:, dst] = st["scale_k"][:, src]
        st["scale_v"][:, dst] = st["scale_v"][:, src]
    return _pages_of(st)


def _pages_of(st):
    if not st["case"]["fp8"]:
        return {"cache_k": st["cache_k"], "cache_v": st["cache_v"]}
    return {"cache_k": st["cache_k"].view(torch.float8_e4m3fn), "cache_v": st["cache_v"].view(torch.float8_e4m3fn),
            "scale_k": st["scale_k"], "scale_v": st["scale_v"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The definitions run by run and head by head in 64 bits."""
    if case["op"] == "pages":
        return None      # nothing is computed: the copies are equal or they are not
    st = prepare(case, seed)
    counts, firsts = _runs(case)
    starts = np.concatenate([[0], np.cumsum(counts)])
    H, G, D, ps = case["heads"], case["group"], case["dim"], case["page"]
    table = st["table"].cpu().numpy()
    ring = case.get("ring", 0)

    def place(i, positions):
        page = positions // ps
        return table[i, page % table.shape[1]].astype(np.int64) * ps + positions % ps

    if case["op"] == "append":
        half = case["rotary"] // 2
        flat = {n: st["cache_" + n].double().view(-1, H, D) for n in "kv"}
        q_out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")

        def unit(x):
            x = x.double()
            return x / ((x * x).sum(-1, keepdim=True) / D + EPS).sqrt()

        for i in range(case["runs"]):
            rows = slice(int(starts[i]), int(starts[i + 1]))
            at = np.arange(firsts[i], firsts[i] + counts[i])
            c, s = (st[n][torch.from_numpy(at).cuda()].double()[:, None] for n in ("cos", "sin"))
            for name, weight in (("raw_q", "q_weight"), ("raw_k", "k_weight")):
                y = unit(st[name][rows]) * st[weight].double()
                a, b = y[..., :half].clone(), y[..., half:2 * half].clone()
                y[..., :half], y[..., half:2 * half] = a * c - b * s, a * s + b * c
                if name == "raw_q":
                    q_out[rows] = y
                else:
                    flat["k"][torch.from_numpy(place(i, at)).cuda()] = y
            v = st["raw_v"] if st["raw_v"] is not None else st["raw_k"]
            flat["v"][torch.from_numpy(place(i, at)).cuda()] = unit(v[rows])
        return {"q": q_out, "cache_k": flat["k"].view(st["cache_k"].shape), "cache_v": flat["v"].view(st["cache_v"].shape)}

    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["lse"].shape, dtype=torch.float64, device="cuda")
    w, sinks = case["window"], case["sinks"]
    for i in range(case["runs"]):
        first, count, start = int(firsts[i]), int(counts[i]), int(starts[i])
        lo = max(0, first - w + 1) if w else 0
        positions = np.unique(np.concatenate([np.arange(min(sinks, first + count)), np.arange(lo, first + count)]))
        old = positions[positions < first] if ring else positions
        where = torch.from_numpy(place(i, old)).cuda()
        kpos = torch.from_numpy(positions).cuda()
        for h in range(H):
            k, v = (st["cache_" + n].view(-1, H, D)[where, h].double() for n in "kv")
            if ring:
                k, v = (torch.cat([x, st[n + "_rows"][start:start + count, h].double()]) for x, n in ((k, "k"), (v, "v")))
            for a in range(0, count, 512):
                b = min(count, a + 512)
                t = torch.arange(first + a, first + b, device="cuda")[:, None]
                hide = kpos > t
                if w:
                    hide = hide | ((kpos <= t - w) & (kpos >= sinks))
                q = st["q"][start + a:start + b, h * G:(h + 1) * G].double()
                scores = torch.einsum("tgd,kd->gtk", q, k) / math.sqrt(D)
                scores = torch.where(hide, -math.inf, scores)
                norm = torch.logsumexp(scores, -1)
                out[start + a:start + b, h * G:(h + 1) * G] = torch.einsum(
                    "gtk,kd->tgd", torch.exp(scores - norm[..., None]), v)
                lse[start + a:start + b, h * G:(h + 1) * G] = norm.T
    return {"out": out, "lse": lse}
