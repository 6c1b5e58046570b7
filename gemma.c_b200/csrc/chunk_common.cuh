// Runs of new tokens (include/gemma4_b200kv.h, B200KvChunkArgs): what the append,
// the write and the attention share.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"

namespace b200kv {

// Positions below this leave room for a key tile's arithmetic in 32 bits.
constexpr int32_t kMaxPosition = 2147483647 - 1024;

// Division of 0 .. 2^31 - 1 by a fixed number: the quotient's high part by a 32-bit
// multiplication (Granlund and Montgomery's round-up method).
struct FastDiv {
  uint32_t d, m, shift;
  __device__ __forceinline__ int quotient(int n) const {
    return int((__umulhi(uint32_t(n), m) + uint32_t(n)) >> shift);
  }
  static FastDiv by(uint32_t d) {
    FastDiv f = {d, 0, 0};
    while ((1ull << f.shift) < d) ++f.shift;
    f.m = uint32_t(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
  }
};

// One run as the device sees it; count 0 where the call skips it.
struct ChunkRun {
  int32_t batch = 0;
  int32_t first = 0;
  int32_t count = 0;
  int32_t start = 0;
};

// Run i, or an empty one for an index or values out of range.
__device__ __forceinline__ ChunkRun chunk_run(const ChunkRuns &r, int i, int batch_size) {
  ChunkRun run;
  if (i >= r.run_count) return run;
  const int batch = __ldg(r.seq_batch + i);
  const int first = __ldg(r.first_position + i);
  const int count = __ldg(r.row_count + i);
  const int start = __ldg(r.row_start + i);
  const bool ok = batch >= 0 && batch < batch_size && first >= 0 && count > 0 &&
                  count <= r.max_row_count && start >= 0 &&
                  int64_t(start) + count <= r.rows &&
                  first <= kMaxPosition - count;
  if (!ok) return run;
  run.batch = batch;
  run.first = first;
  run.count = count;
  run.start = start;
  return run;
}

// Physical page of a position, -1 where the sequence has none: past the table of
// a linear cache, unmapped, or not a page of the cache.
__device__ __forceinline__ int chunk_page(const Gemma4KvCacheConfig &c,
                                          const int32_t *page_table, int batch,
                                          int logical_page) {
  if (c.window_size == 0 && logical_page >= c.max_pages_per_seq) return -1;
  const int slot = logical_page % c.max_pages_per_seq;
  const int physical = __ldg(page_table + int64_t(batch) * c.max_pages_per_seq + slot);
  return physical >= 0 && physical < c.num_pages ? physical : -1;
}

// A later row of the run takes the position's place of the ring.
__device__ __forceinline__ bool chunk_overwritten(const Gemma4KvCacheConfig &c,
                                                  const ChunkRun &run, int position) {
  return c.window_size > 0 &&
         position + int64_t(c.max_pages_per_seq) * c.page_size < int64_t(run.first) + run.count;
}

// Element offset (head 0) at which a run's row at `position` is stored, -1 where
// it is not: no page, or a later row of the run takes the same place of the ring.
__device__ __forceinline__ int64_t chunk_store_offset(const Gemma4KvCacheConfig &c,
                                                      const int32_t *page_table, int layer,
                                                      const ChunkRun &run, int position) {
  if (chunk_overwritten(c, run, position)) return -1;
  const int logical_page = position / c.page_size;
  const int physical = chunk_page(c, page_table, run.batch, logical_page);
  if (physical < 0) return -1;
  return cache_offset(c, layer, physical, position - logical_page * c.page_size, 0, 0);
}

inline bool valid_chunk_runs(const ChunkRuns &r) {
  return r.seq_batch != nullptr && r.first_position != nullptr && r.row_count != nullptr &&
         r.row_start != nullptr && r.run_count >= 0 && r.run_count <= B200KV_MAX_RUNS &&
         r.max_row_count > 0 && r.rows >= 0;
}

// The most keys that the rows of `tokens` consecutive tokens of a run can see, whatever
// the lengths: the table's positions and the run's own rows, or the window's and the
// first tokens'. table_end: first position past a linear cache's table.
inline int64_t most_keys(const ChunkAttentionArgs &a, int table_end, int64_t tokens) {
  const int64_t own = a.k_rows != nullptr ? std::min(a.runs.max_row_count, a.runs.rows) : 0;
  const int64_t all = table_end + own;
  return a.window > 0 ? std::min(all, int64_t(a.window) + tokens - 1 + a.sinks) : all;
}

inline bool valid_cache_config(const Gemma4KvCacheConfig &c, int layer) {
  return c.num_layers > 0 && layer >= 0 && layer < c.num_layers && c.num_pages > 0 &&
         c.page_size > 0 && c.max_pages_per_seq > 0 && c.batch_size > 0 && c.num_heads > 0 &&
         c.head_dim > 0 && c.window_size >= 0 &&
         (c.window_size == 0 ||
          int64_t(c.max_pages_per_seq) * c.page_size >= c.window_size);
}

}  // namespace b200kv
