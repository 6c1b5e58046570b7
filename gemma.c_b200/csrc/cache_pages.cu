// Pages as units: copies of whole pages (or their first rows) inside a cache, and
// the host bookkeeping behind sharing them. The reference gives every sequence its
// own pages for good (src/gemma4_kv_cache.cu:108-146) and has neither.
//
// A page of one layer and tensor is page_size * num_heads * head_dim elements in
// one piece, its first r rows the first r * num_heads * head_dim of them (the
// 8-bit K order too, in blocks of eight rows), so a copy is a move of one byte
// range per (pair, layer, tensor). 2 bytes of traffic per byte copied and nothing
// else to do: bound by HBM, few pages by the launch and two loads in a row. A CTA
// moves 16 KB, four 16-byte packs a thread, all asked for before the first is stored.
// Measured: 2000 pages of 64 KB in 4 layers, K and V (1 GB each way) 337 us = 6.2 TB/s;
// 500 pages of an 8-bit cache in 2 layers (131 MB both ways) 25 us; the first rows of
// 16 pages in 4 layers 3.2 us of the GPU.
#include <algorithm>
#include <memory>
#include <new>

#include "chunk_common.cuh"
#include "kernels.cuh"

namespace b200kv {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;                                     // 16-byte packs per thread
constexpr int kPieceBytes = kCopyThreads * kCopyVecs * 16;

struct CopyParams {
  uint8_t *cache[2];
  float *scale[2];
  const int32_t *src_page;
  const int32_t *dst_page;
  const int32_t *row_count;
  int64_t page_bytes;
  int64_t row_bytes;
  int32_t num_pages;
  int32_t page_size;
  int32_t num_heads;
  int32_t row_align;  // rows are copied in multiples of it
};

// grid (piece of the page, layer * 2 + tensor, pair)
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyParams p) {
  const int pair = int(blockIdx.x);
  const int tensor = int(blockIdx.y) & 1;
  const int layer = int(blockIdx.y) >> 1;
  const int src = __ldg(p.src_page + pair);
  const int dst = __ldg(p.dst_page + pair);
  int rows = p.row_count != nullptr ? __ldg(p.row_count + pair) : p.page_size;
  if (src == dst || src < 0 || dst < 0 || src >= p.num_pages || dst >= p.num_pages) return;
  rows = min(rows, p.page_size);
  if (rows <= 0) return;
  rows = div_up(rows, p.row_align) * p.row_align;
  const int64_t bytes = rows * p.row_bytes;
  const int64_t begin = int64_t(blockIdx.z) * kPieceBytes;
  const int64_t first_page = int64_t(layer) * p.num_pages;
  if (begin < bytes) {
    const uint4 *from = reinterpret_cast<const uint4 *>(
        p.cache[tensor] + (first_page + src) * p.page_bytes + begin);
    uint4 *to = reinterpret_cast<uint4 *>(
        p.cache[tensor] + (first_page + dst) * p.page_bytes + begin);
    const int vecs = int(min(int64_t(kPieceBytes), bytes - begin) / 16);
    uint4 v[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i) {
      const int at = int(threadIdx.x) + i * kCopyThreads;
      if (at < vecs) v[i] = from[at];
    }
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i) {
      const int at = int(threadIdx.x) + i * kCopyThreads;
      if (at < vecs) to[at] = v[i];
    }
  }
  if (p.scale[0] != nullptr && blockIdx.z == 0) {
    float *scale = p.scale[tensor];
    for (int h = int(threadIdx.x); h < p.num_heads; h += kCopyThreads) {
      scale[(first_page + dst) * p.num_heads + h] = scale[(first_page + src) * p.num_heads + h];
    }
  }
}

}  // namespace

cudaError_t copy_pages(void *cache_k, void *cache_v, float *scale_k, float *scale_v,
                       Gemma4KvCacheConfig c, int element_bytes, const int32_t *src_page,
                       const int32_t *dst_page, const int32_t *row_count, int32_t count,
                       cudaStream_t stream) {
  if (count == 0) return cudaSuccess;
  const bool fp8 = element_bytes == 1;
  if (count < 0 || cache_k == nullptr || cache_v == nullptr || src_page == nullptr ||
      dst_page == nullptr || c.num_layers <= 0 || c.num_pages <= 0 || c.page_size <= 0 ||
      c.num_heads <= 0 || c.head_dim <= 0 || c.num_layers > 32767 ||
      (fp8 && (scale_k == nullptr || scale_v == nullptr || c.page_size % 8 != 0))) {
    return cudaErrorInvalidValue;
  }
  CopyParams p = {};
  p.row_bytes = int64_t(c.num_heads) * c.head_dim * element_bytes;
  p.page_bytes = p.row_bytes * c.page_size;
  const int64_t pieces = div_up(p.page_bytes, int64_t(kPieceBytes));
  // (16 bytes at a time: an 8-bit row may be an odd number of eights, but eight rows are not)
  if (int64_t(c.num_heads) * c.head_dim % 8 != 0 || pieces > 65535 ||
      ((reinterpret_cast<uintptr_t>(cache_k) | reinterpret_cast<uintptr_t>(cache_v)) & 15u) != 0) {
    return cudaErrorInvalidValue;
  }
  p.cache[0] = static_cast<uint8_t *>(cache_k);
  p.cache[1] = static_cast<uint8_t *>(cache_v);
  p.scale[0] = fp8 ? scale_k : nullptr;
  p.scale[1] = fp8 ? scale_v : nullptr;
  p.src_page = src_page;
  p.dst_page = dst_page;
  p.row_count = row_count;
  p.num_pages = c.num_pages;
  p.page_size = c.page_size;
  p.num_heads = c.num_heads;
  p.row_align = fp8 ? 8 : 1;
  const dim3 grid{unsigned(count), unsigned(c.num_layers * 2), unsigned(pieces)};
  copy_pages_kernel<<<grid, kCopyThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace b200kv

// ===========================================================================
// Host bookkeeping (no device): reference counts on physical pages.
// ===========================================================================
namespace {

// What both the tables' users and the planners take for granted.
bool valid_pool(const int32_t *table, const int32_t *refs, const Gemma4KvCacheConfig *c) {
  return table != nullptr && refs != nullptr && c != nullptr && c->num_pages > 0 &&
         c->page_size > 0 && c->max_pages_per_seq > 0 && c->batch_size > 0;
}

bool valid_copy_list(const int32_t *src, const int32_t *dst, const int32_t *rows,
                     int32_t capacity, const int32_t *count) {
  return count != nullptr && *count >= 0 && capacity >= *count &&
         (capacity == 0 || (src != nullptr && dst != nullptr && rows != nullptr));
}

// n times -1; nullptr where there is no memory for it (no exception leaves a C entry).
std::unique_ptr<int32_t[]> no_pages(int64_t n) {
  std::unique_ptr<int32_t[]> list(new (std::nothrow) int32_t[size_t(n)]);
  if (list != nullptr) std::fill_n(list.get(), n, -1);
  return list;
}

bool holds(const int32_t *list, int32_t count, int32_t page) {
  return count > 0 && std::find(list, list + count, page) != list + count;
}

}  // namespace

extern "C" {

int32_t b200kv_pages_ensure(int32_t *h_page_table, int32_t *h_ref_count,
                            const Gemma4KvCacheConfig *config, int32_t batch,
                            int32_t first, int32_t count, int32_t *h_copy_src,
                            int32_t *h_copy_dst, int32_t *h_copy_rows,
                            int32_t capacity, int32_t *copy_count) {
  if (!valid_pool(h_page_table, h_ref_count, config) || config->window_size != 0 ||
      batch < 0 || batch >= config->batch_size || first < 0 || count < 0 ||
      !valid_copy_list(h_copy_src, h_copy_dst, h_copy_rows, capacity, copy_count)) {
    return -1;
  }
  if (count == 0) return 0;
  const int32_t ps = config->page_size;
  const int64_t last = int64_t(first) + count - 1;
  if (last / ps >= config->max_pages_per_seq) return -1;
  int32_t *table = h_page_table + int64_t(batch) * config->max_pages_per_seq;
  const int32_t lo = first / ps, hi = int32_t(last / ps);
  const int32_t kept_rows = first % ps;  // rows of the first page that stay

  // what every slot needs, before anything changes
  const auto fresh = no_pages(int64_t(hi) - lo + 1);
  if (fresh == nullptr) return -1;
  int32_t cursor = 0, copies = *copy_count;
  for (int32_t slot = lo; slot <= hi; ++slot) {
    const int32_t page = table[slot];
    if (page >= config->num_pages || (page >= 0 && h_ref_count[page] <= 0)) return -1;
    if (page >= 0 && h_ref_count[page] == 1) continue;
    // the lowest free page that no recorded copy still reads or writes
    while (cursor < config->num_pages &&
           (h_ref_count[cursor] != 0 || holds(h_copy_src, *copy_count, cursor) ||
            holds(h_copy_dst, *copy_count, cursor))) {
      ++cursor;
    }
    if (cursor == config->num_pages) return -1;
    fresh[size_t(slot - lo)] = cursor++;
    if (page >= 0 && slot == lo && kept_rows > 0) {
      // its content must be there already, not only recorded to be copied there
      if (copies == capacity || holds(h_copy_dst, *copy_count, page)) return -1;
      ++copies;
    }
  }
  for (int32_t slot = lo; slot <= hi; ++slot) {
    const int32_t to = fresh[size_t(slot - lo)];
    if (to < 0) continue;
    const int32_t page = table[slot];
    if (page >= 0) {
      if (slot == lo && kept_rows > 0) {
        h_copy_src[*copy_count] = page;
        h_copy_dst[*copy_count] = to;
        h_copy_rows[*copy_count] = kept_rows;
        ++*copy_count;
      }
      --h_ref_count[page];
    }
    h_ref_count[to] = 1;
    table[slot] = to;
  }
  return 0;
}

int32_t b200kv_pages_fork(int32_t *h_page_table, int32_t *h_ref_count,
                          const Gemma4KvCacheConfig *config, int32_t src,
                          int32_t dst, int32_t length) {
  if (!valid_pool(h_page_table, h_ref_count, config) || config->window_size != 0 ||
      src < 0 || src >= config->batch_size || dst < 0 || dst >= config->batch_size ||
      src == dst || length < 0) {
    return -1;
  }
  const int32_t slots = config->max_pages_per_seq;
  const int32_t pages = b200kv::div_up(int64_t(length), int64_t(config->page_size));
  if (pages > slots) return -1;
  const int32_t *from = h_page_table + int64_t(src) * slots;
  int32_t *to = h_page_table + int64_t(dst) * slots;
  for (int32_t s = 0; s < slots; ++s) {
    if (to[s] >= 0) return -1;
    if (s < pages && from[s] >= 0 &&
        (from[s] >= config->num_pages || h_ref_count[from[s]] <= 0)) {
      return -1;
    }
  }
  for (int32_t s = 0; s < pages; ++s) {
    to[s] = from[s];
    if (from[s] >= 0) ++h_ref_count[from[s]];
  }
  return 0;
}

int32_t b200kv_pages_release(int32_t *h_page_table, int32_t *h_ref_count,
                             const Gemma4KvCacheConfig *config, int32_t batch,
                             int32_t first_slot, int32_t slot_count) {
  if (!valid_pool(h_page_table, h_ref_count, config) || batch < 0 ||
      batch >= config->batch_size || first_slot < 0 || slot_count < 0 ||
      int64_t(first_slot) + slot_count > config->max_pages_per_seq) {
    return -1;
  }
  int32_t *table = h_page_table + int64_t(batch) * config->max_pages_per_seq + first_slot;
  for (int32_t s = 0; s < slot_count; ++s) {
    if (table[s] < 0) continue;
    // (a page may be named by several of the slots: its count has to last for all)
    if (table[s] < config->num_pages && h_ref_count[table[s]] > 0) {
      --h_ref_count[table[s]];
      continue;
    }
    while (--s >= 0) {
      if (table[s] >= 0) ++h_ref_count[table[s]];
    }
    return -1;
  }
  std::fill_n(table, slot_count, -1);
  return 0;
}

int32_t b200kv_pages_compact(int32_t *h_page_table, int32_t *h_ref_count,
                             const Gemma4KvCacheConfig *config,
                             int32_t *h_copy_src, int32_t *h_copy_dst,
                             int32_t *h_copy_rows, int32_t capacity,
                             int32_t *copy_count, int32_t *used) {
  if (!valid_pool(h_page_table, h_ref_count, config) ||
      !valid_copy_list(h_copy_src, h_copy_dst, h_copy_rows, capacity, copy_count) ||
      *copy_count != 0) {  // every recorded copy must have been made
    return -1;
  }
  const int64_t entries = int64_t(config->batch_size) * config->max_pages_per_seq;
  for (int64_t i = 0; i < entries; ++i) {
    const int32_t page = h_page_table[i];
    if (page >= 0 && (page >= config->num_pages || h_ref_count[page] <= 0)) return -1;
  }
  int32_t live = 0;
  for (int32_t p = 0; p < config->num_pages; ++p) live += h_ref_count[p] > 0 ? 1 : 0;
  int32_t moves = 0;
  for (int32_t p = live; p < config->num_pages; ++p) moves += h_ref_count[p] > 0 ? 1 : 0;
  if (moves > capacity) return -1;
  const auto now = no_pages(config->num_pages);
  if (now == nullptr) return -1;
  int32_t hole = 0;
  for (int32_t p = live; p < config->num_pages; ++p) {
    if (h_ref_count[p] <= 0) continue;
    while (h_ref_count[hole] > 0) ++hole;  // there are as many holes below `live` as moves
    h_copy_src[*copy_count] = p;
    h_copy_dst[*copy_count] = hole;
    h_copy_rows[*copy_count] = config->page_size;
    ++*copy_count;
    now[size_t(p)] = hole;
    h_ref_count[hole] = h_ref_count[p];
    h_ref_count[p] = 0;
  }
  for (int64_t i = 0; i < entries; ++i) {
    const int32_t page = h_page_table[i];
    if (page >= 0 && now[size_t(page)] >= 0) h_page_table[i] = now[size_t(page)];
  }
  if (used != nullptr) *used = live;
  return 0;
}

}  // extern "C"
