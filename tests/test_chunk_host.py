"""Host side of the chunk operators: refusals without a device, and the page bookkeeping."""
from __future__ import annotations

import ctypes
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

GOOD = (2, 40, 16, 10, 4, 8, 256, 0)


def args(kv, cfg=GOOD, **over):
    a = kv.ChunkArgs()
    for name in ("q", "out", "lse", "cache_k", "cache_v", "page_table", "seq_batch", "first_position", "row_count",
                 "row_start", "raw_q", "raw_k", "raw_v", "q_norm_weight", "k_norm_weight", "cos", "sin", "workspace"):
        setattr(a, name, 4096)
    a.cache_config = kv.make_kv_config(*cfg)
    a.run_count, a.max_row_count, a.rows, a.q_heads = 2, 8, 16, 16
    a.rotary_dim, a.softmax_scale = 256, 1 / 16
    a.workspace_bytes = 1 << 40
    for name, value in over.items():
        setattr(a, name, value)
    return a


def ring(**over):
    return dict(cfg=(2, 40, 16, 10, 4, 8, 256, 160), **over)


COMMON = [dict(run_count=-1), dict(run_count=1025), dict(max_row_count=0), dict(rows=-1), dict(seq_batch=None),
          dict(first_position=None), dict(row_count=None), dict(row_start=None), dict(k_rows=4096), dict(v_rows=4096),
          dict(q=None), dict(q=4100), dict(q_heads=0), dict(q_heads=12)]


@pytest.mark.parametrize("over", COMMON + [
    dict(out=None), dict(out=4104), dict(cache_k=None), dict(cache_v=4098), dict(page_table=None), dict(workspace=None),
    dict(workspace_bytes=0), dict(cache_layer=2), dict(cache_layer=-1), dict(softmax_scale=0.0),
    dict(softmax_scale=float("nan")), dict(window_size=-1), dict(sink_tokens=-1), dict(sink_tokens=4),
    dict(q_heads=8 * 65), dict(cfg=(2, 40, 16, 10, 4, 8, 128, 0)), dict(cfg=(2, 40, 0, 10, 4, 8, 256, 0)),
    dict(cfg=(2, 40, 16, 10, 4, 8, 256, 161)),                       # a ring smaller than its window
    ring(), ring(k_rows=4096, v_rows=4096, window_size=100),         # no room for the run; another window
    ring(k_rows=4096, v_rows=4096, sink_tokens=1)])
def test_attention_refuses(kv, over):
    assert kv.load_library().b200kv_chunk_attention_bf16(ctypes.byref(args(kv, **over)), None) == 1


@pytest.mark.parametrize("over", COMMON + [
    dict(raw_q=None), dict(raw_k=4097), dict(raw_v=4098), dict(q_norm_weight=None), dict(k_norm_weight=None),
    dict(cos=None), dict(sin=None), dict(rotary_dim=128), dict(norm_mode=2), dict(cache_k=None), dict(page_table=None),
    dict(cfg=(2, 40, 16, 10, 4, 8, 512, 0))])
def test_append_refuses(kv, over):
    assert kv.load_library().b200kv_chunk_append_bf16(ctypes.byref(args(kv, **over)), None) == 1


@pytest.mark.parametrize("over", [dict(), dict(k_rows=4096, v_rows=4096, cache_v=None),
                                  dict(k_rows=4096, v_rows=4096, cache_layer=5), dict(k_rows=4096, v_rows=4097)])
def test_write_refuses(kv, over):
    assert kv.load_library().b200kv_chunk_write_bf16(ctypes.byref(args(kv, **over)), None) == 1


@pytest.mark.parametrize("over", [dict(raw_q=None), dict(out=None), ring(), dict(rotary_dim=128), dict(workspace_bytes=0)])
def test_layer_step_refuses_before_it_enqueues(kv, over):
    assert kv.load_library().b200kv_chunk_layer_step_bf16(ctypes.byref(args(kv, **over)), None) == 1


def test_empty_calls_and_null_blocks(kv):
    lib = kv.load_library()
    empty = kv.ChunkArgs()
    for name in ("chunk_append", "chunk_attention", "chunk_write", "chunk_layer_step"):
        fn = getattr(lib, f"b200kv_{name}_bf16")
        assert fn(ctypes.byref(empty), None) == 0
        assert fn(None, None) == 1


def test_give_up_selftest_and_launches_refuse(kv):
    lib = kv.load_library()
    assert lib.b200kv_chunk_attention_launches(None) == 0
    assert lib.b200kv_chunk_attention_give_up_selftest(None, 0, None) == 1
    for over in (dict(), dict(status=4096, run_count=0), dict(status=4096, out=None)):       # no status; nothing to do; no output
        assert lib.b200kv_chunk_attention_give_up_selftest(ctypes.byref(args(kv, **over)), 0, None) == 1
    assert lib.b200kv_chunk_attention_give_up_selftest(ctypes.byref(args(kv, status=4096)), -1, None) == 1
    for over in (dict(run_count=0), dict(rows=0), dict(out=None)):
        assert lib.b200kv_chunk_attention_launches(ctypes.byref(args(kv, **over))) == 0


def test_workspace_bytes(kv):
    w = lambda *a: kv.chunk_workspace_bytes(*a)  # noqa: E731
    small, large = w(16, 8, 256, 1, 1, 148), w(16, 8, 256, 32, 4096, 148)
    assert 0 < small <= large < (256 << 20)
    for bad in ((0, 8, 256, 1, 1, 148), (16, 0, 256, 1, 1, 148), (12, 8, 256, 1, 1, 148), (16, 8, 128, 1, 1, 148),
                (16, 8, 256, 0, 1, 148), (16, 8, 256, 1, 0, 148), (16, 8, 256, 1, 1, 0), (130, 2, 256, 1, 1, 148)):
        assert w(*bad) == 0


@pytest.mark.parametrize("over", [dict(cache_k=None), dict(cache_v=4100), dict(src=None), dict(dst=None),
                                  dict(count=-1), dict(cfg=(2, 40, 3, 10, 4, 1, 4, 0)), dict(cfg=(0, 40, 16, 10, 4, 8, 256, 0))])
def test_copy_pages_refuses(kv, over):
    a = dict(cache_k=4096, cache_v=4096, cfg=GOOD, src=4096, dst=4096, rows=None, count=3)
    a.update(over)
    cfg = kv.make_kv_config(*a["cfg"])
    assert kv.copy_pages(a["cache_k"], a["cache_v"], cfg, a["src"], a["dst"], a["rows"], a["count"], stream=0,
                         check=False) == 1
    assert kv.copy_pages_fp8(a["cache_k"], a["cache_v"], 4096, 4096, cfg, a["src"], a["dst"], a["rows"], a["count"],
                             stream=0, check=False) == 1


def test_copy_pages_fp8_needs_scales_and_blocks_of_eight(kv):
    cfg = kv.make_kv_config(*GOOD)
    assert kv.copy_pages_fp8(4096, 4096, None, 4096, cfg, 4096, 4096, None, 3, stream=0, check=False) == 1
    odd = kv.make_kv_config(2, 40, 12, 10, 4, 8, 256, 0)
    assert kv.copy_pages_fp8(4096, 4096, 4096, 4096, odd, 4096, 4096, None, 3, stream=0, check=False) == 1
    assert kv.copy_pages(4096, 4096, cfg, None, None, None, 0, stream=0) == 0


def test_copy_pages_refuses_rows_that_are_no_multiple_of_eight_elements(kv):
    for heads, dim in ((1, 4), (3, 4), (1, 12)):
        cfg = kv.make_kv_config(2, 40, 16, 10, 4, heads, dim, 0)
        assert kv.copy_pages_fp8(4096, 4096, 4096, 4096, cfg, 4096, 4096, None, 3, stream=0, check=False) == 1
        assert kv.copy_pages(4096, 4096, cfg, 4096, 4096, None, 3, stream=0, check=False) == 1


# --------------------------------------------------------------------------------------------- page bookkeeping
class Pool:
    def __init__(self, kv, pages=12, slots=6, batch=3, ps=4, capacity=8):
        self.kv = kv
        self.cfg = kv.make_kv_config(1, pages, ps, slots, batch, 8, 256, 0)
        self.table = np.full((batch, slots), -1, dtype=np.int32)
        self.refs = np.zeros(pages, dtype=np.int32)
        self.copies = kv.PageCopies(capacity)

    def ensure(self, b, first, count):
        return self.kv.pages_ensure(self.table, self.refs, self.cfg, b, first, count, self.copies)

    def fork(self, src, dst, n):
        return self.kv.pages_fork(self.table, self.refs, self.cfg, src, dst, n)

    def release(self, b, slot, n):
        return self.kv.pages_release(self.table, self.refs, self.cfg, b, slot, n)

    def listed(self):
        n = self.copies.count
        return list(zip(*(x[:n].tolist() for x in (self.copies.src, self.copies.dst, self.copies.rows))))

    def consistent(self):
        counted = np.zeros_like(self.refs)
        for page in self.table[self.table >= 0]:
            counted[page] += 1
        return np.array_equal(counted, self.refs)


def test_ensure_takes_the_lowest_free_pages(kv):
    p = Pool(kv)
    assert p.ensure(1, 0, 9) == 0 and p.table[1].tolist() == [0, 1, 2, -1, -1, -1]
    assert p.ensure(1, 9, 3) == 0 and p.table[1].tolist() == [0, 1, 2, -1, -1, -1]
    assert p.ensure(1, 12, 0) == 0 and p.ensure(0, 4, 1) == 0 and p.table[0].tolist() == [-1, 3, -1, -1, -1, -1]
    assert p.consistent() and p.listed() == []


def test_fork_and_copy_on_write(kv):
    p = Pool(kv)
    p.ensure(0, 0, 10)
    assert p.fork(0, 1, 10) == 0 and p.fork(0, 2, 8) == 0 and p.refs[:3].tolist() == [3, 3, 2]
    assert p.ensure(1, 10, 2) == 0 and p.listed() == [(2, 3, 2)] and p.table[1, 2] == 3
    assert p.ensure(0, 10, 1) == 0 and p.table[0, 2] == 2 and len(p.listed()) == 1      # the last holder writes in place
    assert p.ensure(2, 8, 1) == 0 and p.table[2, 2] == 4 and len(p.listed()) == 1       # starts at a page: no copy
    assert p.consistent()
    p.copies.clear()
    assert p.ensure(2, 4, 1) == 0 and p.table[2, 1] == 5 and p.listed() == []           # rewrites a shared page whole
    assert p.consistent()


def test_recorded_copies_keep_their_pages(kv):
    p = Pool(kv, pages=5)
    p.ensure(0, 0, 6)
    p.fork(0, 1, 6)
    assert p.ensure(1, 6, 1) == 0 and p.listed() == [(1, 2, 2)]
    assert p.fork(1, 2, 7) == 0
    assert p.ensure(2, 7, 1) == -1                    # its source is still to be copied
    p.release(2, 0, 6)
    p.release(1, 0, 6)                                # page 2 is free again, but named by the list
    assert p.ensure(1, 0, 8) == 0 and 2 not in p.table[1] and p.consistent()
    assert p.ensure(1, 8, 1) == -1                    # nothing left but page 2
    p.copies.clear()
    assert p.ensure(1, 8, 1) == 0 and p.table[1, 2] == 2


def test_nothing_changes_when_there_is_no_room(kv):
    p = Pool(kv, pages=4, capacity=0)
    p.ensure(0, 0, 6)
    p.fork(0, 1, 6)
    state = p.table.copy(), p.refs.copy()
    assert p.ensure(1, 6, 1) == -1                    # no room in the list
    assert p.ensure(0, 20, 8) == -1 and p.ensure(2, 0, 12) == -1 and p.ensure(0, 0, 25) == -1
    assert p.fork(0, 1, 3) == -1 and p.fork(0, 0, 3) == -1 and p.fork(0, 2, 100) == -1 and p.fork(0, 3, 1) == -1
    assert p.release(0, 3, 4) == -1 and p.release(3, 0, 1) == -1 and p.ensure(-1, 0, 1) == -1
    assert np.array_equal(state[0], p.table) and np.array_equal(state[1], p.refs)
    ringed = kv.make_kv_config(1, 4, 4, 6, 3, 8, 256, 8)
    assert kv.pages_ensure(p.table, p.refs, ringed, 0, 0, 1, p.copies) == -1
    assert kv.pages_fork(p.table, p.refs, ringed, 0, 2, 1) == -1


def test_release_of_a_page_named_twice(kv):
    """A sequence may map one page in two slots; where the counts say less than the slots, nothing changes."""
    p = Pool(kv)
    p.ensure(0, 0, 12)
    p.table[0, 3], p.refs[1] = 1, 2
    assert p.release(0, 0, 4) == 0 and p.consistent() and p.refs.max() == 0
    p.ensure(0, 0, 12)
    p.table[0, 3] = 1
    state = p.table.copy(), p.refs.copy()
    assert p.release(0, 0, 4) == -1
    assert np.array_equal(state[0], p.table) and np.array_equal(state[1], p.refs)
    p.table[0, 2] = 12                                # not a page of the pool
    assert p.release(0, 0, 3) == -1 and np.array_equal(state[1], p.refs)


def test_release_of_the_middle_for_sinks(kv):
    p = Pool(kv)
    p.ensure(0, 0, 24)
    assert p.release(0, 1, 3) == 0 and p.table[0].tolist() == [0, -1, -1, -1, 4, 5] and p.consistent()
    assert p.fork(0, 1, 24) == 0 and p.table[1].tolist() == p.table[0].tolist() and p.consistent()


@pytest.mark.parametrize("seed", range(6))
def test_compact_fills_the_front(kv, seed):
    rng = np.random.default_rng(seed)
    p = Pool(kv, pages=30, slots=8, batch=5, capacity=30)
    content = {}
    for b in range(3):
        p.ensure(b, 0, int(rng.integers(1, 33)))
    p.fork(0, 3, int(rng.integers(1, 8)))
    p.release(1, 0, 8)
    p.ensure(4, 0, 5)
    p.release(0, 1, 2)
    p.copies.clear()
    content = {page: f"page {page}" for page in range(30)}
    before = [[content[x] if x >= 0 else None for x in row] for row in p.table]
    code, used = kv.pages_compact(p.table, p.refs, p.cfg, p.copies)
    assert code == 0 and p.consistent() and used == int((p.refs > 0).sum())
    assert int(p.table.max()) < used
    srcs, dsts = [c[0] for c in p.listed()], [c[1] for c in p.listed()]
    assert len(set(dsts)) == len(dsts) and not set(srcs) & set(dsts)
    for s, d, rows in p.listed():
        assert rows == 4
        content[d] = content[s]
    assert before == [[content[x] if x >= 0 else None for x in row] for row in p.table]


def test_compact_needs_an_empty_list_and_room(kv):
    p = Pool(kv, capacity=1)
    p.ensure(0, 0, 12)
    p.ensure(1, 0, 8)
    p.release(0, 0, 6)
    state = p.table.copy(), p.refs.copy()
    assert kv.pages_compact(p.table, p.refs, p.cfg, p.copies)[0] == -1          # two moves, room for one
    assert np.array_equal(state[0], p.table) and np.array_equal(state[1], p.refs)
    q = Pool(kv)
    q.ensure(0, 0, 6)
    q.fork(0, 1, 6)
    q.ensure(1, 6, 1)
    assert kv.pages_compact(q.table, q.refs, q.cfg, q.copies)[0] == -1          # a copy is still to be made


OUT_OF_MEMORY = """
import importlib.util, resource, sys
from pathlib import Path
import numpy as np
pkg = Path(sys.argv[1])
spec = importlib.util.spec_from_file_location("gemma_c_b200", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
kv = sys.modules["gemma_c_b200"] = importlib.util.module_from_spec(spec)
spec.loader.exec_module(kv)
kv.load_library()
n = 1 << 24
cfg = kv.make_kv_config(1, n, 1, n, 1, 8, 256, 0)
table, refs, copies = np.full((1, n), -1, dtype=np.int32), np.zeros(n, dtype=np.int32), kv.PageCopies(4)
if sys.argv[2] == "compact":
    table[0, 0], refs[n - 1] = n - 1, 1
state = table.copy(), refs.copy()
size = int(Path("/proc/self/statm").read_text().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (size + (16 << 20), resource.RLIM_INFINITY))
if sys.argv[2] == "compact":
    code = kv.pages_compact(table, refs, cfg, copies)[0]
else:
    code = kv.pages_ensure(table, refs, cfg, 0, 0, n, copies)
resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))
assert code == -1 and copies.count == 0
assert np.array_equal(state[0], table) and np.array_equal(state[1], refs)
"""


@pytest.mark.parametrize("call", ["ensure", "compact"])
def test_a_call_without_memory_fails_and_changes_nothing(kv, call):
    """In a process of its own whose address space has no room for the call's 64 MB: -1, not an exception that ends it."""
    done = subprocess.run([sys.executable, "-c", OUT_OF_MEMORY, str(Path(kv.__file__).parent), call], capture_output=True,
                          text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-500:]


# --------------------------------------------------------------------------------------------- sources
def test_registers_of_tensor_memory_loads_are_tied_to_the_wait(kv):
    """A load from tensor memory is asynchronous: its registers hold nothing before the wait, and nothing but a mention
    of them behind it keeps the compiler from moving what is computed with them ahead of it."""
    sources = sorted((Path(kv.__file__).parent / "csrc").glob("*.cu*"))
    waits = 0
    for path in sources:
        lines = path.read_text().splitlines()
        for at in (i for i, line in enumerate(lines) if "tcgen05.wait::ld" in line):
            waits += 1
            tied = any('asm volatile("" : "+r"(' in line for line in lines[at + 1:at + 4])
            assert tied, f"{path.name}:{at + 1}"
    assert waits >= 3
