// Attention of runs of new tokens over the paged cache (B200KvChunkArgs).
//   out[t, h] = sum_p softmax_p(scale q[t, h] . K[p, h / G]) V[p, h / G]
// over the keys p <= t that have a page, with a window only p > t - window or
// p < sinks. One warp per (row, query head): 16-byte packs of the head dims per
// lane, one pass over the keys with a running maximum and sum in fp32.
#include <algorithm>

#include "chunk_common.cuh"
#include "kernels.cuh"

namespace b200kv {

namespace {

constexpr int kWarps = 4;

template <int D>
__global__ __launch_bounds__(kWarps * 32) void chunk_attention_simple_kernel(ChunkAttentionArgs a) {
  constexpr int kPacks = D / 256;
  const Gemma4KvCacheConfig &c = a.cfg;
  const ChunkRun run = chunk_run(a.runs, int(blockIdx.y), c.batch_size);
  const int r = int(blockIdx.x);
  const int head = int(blockIdx.z) * kWarps + (int(threadIdx.x) >> 5);
  const int lane = int(threadIdx.x) & 31;
  if (r >= run.count || head >= a.q_heads) return;
  const int kv_head = head / (a.q_heads / c.num_heads);
  const int t = run.first + r;
  const int64_t row = (int64_t(run.start) + r) * a.q_heads + head;
  float q[kPacks * 8], acc[kPacks * 8];
  auto unpack = [](uint4 w, float *x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(u[i]);
      x[2 * i + 1] = bf16_hi(u[i]);
    }
  };
#pragma unroll
  for (int v = 0; v < kPacks; ++v) {
    unpack(__ldg(reinterpret_cast<const uint4 *>(a.q + row * D) + lane + 32 * v), q + 8 * v);
  }
#pragma unroll
  for (int i = 0; i < kPacks * 8; ++i) acc[i] = 0.0f;
  const float scale = a.softmax_scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.0f;
  const int lo = a.window > 0 ? max(0, t - a.window + 1) : 0;
  for (int p = 0; p <= t; ++p) {
    if (p < lo && p >= a.sinks) {
      p = lo - 1;
      continue;
    }
    const __nv_bfloat16 *k, *v;
    if (a.k_rows != nullptr && p >= run.first) {
      const int64_t at = ((int64_t(run.start) + p - run.first) * c.num_heads + kv_head) * D;
      k = a.k_rows + at;
      v = a.v_rows + at;
    } else {
      const int page = chunk_page(c, a.page_table, run.batch, p / c.page_size);
      if (page < 0) continue;
      const int64_t at = cache_offset(c, a.layer, page, p % c.page_size, kv_head, 0);
      k = a.cache_k + at;
      v = a.cache_v + at;
    }
    float s = 0.0f;
    float x[8];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      unpack(__ldg(reinterpret_cast<const uint4 *>(k) + lane + 32 * i), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(q[8 * i + j], x[j], s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= scale;
    const float new_m = fmaxf(m, s);
    const float corr = m == -INFINITY ? 0.0f : ex2_approx(m - new_m);
    const float w = ex2_approx(s - new_m);
    l = l * corr + w;
    m = new_m;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      unpack(__ldg(reinterpret_cast<const uint4 *>(v) + lane + 32 * i), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[8 * i + j] = fmaf(w, x[j], acc[8 * i + j] * corr);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int v = 0; v < kPacks; ++v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(acc[8 * v + 2 * i] * inv, acc[8 * v + 2 * i + 1] * inv);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    reinterpret_cast<uint4 *>(a.out + row * D)[lane + 32 * v] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (a.lse != nullptr && lane == 0) {
    a.lse[row] = l > 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  }
}

}  // namespace

size_t chunk_workspace_bytes(int q_heads, int kv_heads, int head_dim, int run_count,
                             int max_row_count, int sm_count) {
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > 64 ||
      (head_dim != 256 && head_dim != 512) || run_count <= 0 || max_row_count <= 0 ||
      sm_count <= 0) {
    return 0;
  }
  return 16;
}

cudaError_t validate_chunk_attention(const ChunkAttentionArgs &a) {
  const Gemma4KvCacheConfig &c = a.cfg;
  if (!valid_chunk_runs(a.runs) || !valid_cache_config(c, a.layer) || a.out == nullptr ||
      a.q == nullptr || a.cache_k == nullptr || a.cache_v == nullptr || a.page_table == nullptr ||
      (a.k_rows == nullptr) != (a.v_rows == nullptr) || a.workspace == nullptr ||
      a.workspace_bytes < 16 || a.q_heads <= 0 || a.q_heads % c.num_heads != 0 || a.q_heads / c.num_heads > 64 ||
      (c.head_dim != 256 && c.head_dim != 512) || a.window < 0 || a.sinks < 0 ||
      (a.sinks > 0 && a.window == 0) || !(a.softmax_scale > 0.0f)) {
    return cudaErrorInvalidValue;
  }
  // a ring has its own window and keeps no first tokens; without the runs' rows
  // beside it, it has to hold every key that the first row sees and the last writes
  if (c.window_size > 0 &&
      (a.window != c.window_size || a.sinks > 0 ||
       (a.k_rows == nullptr && int64_t(c.max_pages_per_seq) * c.page_size <
                                   int64_t(c.window_size) + a.runs.max_row_count - 1))) {
    return cudaErrorInvalidValue;
  }
  const uintptr_t align =
      reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.q) |
      reinterpret_cast<uintptr_t>(a.cache_k) | reinterpret_cast<uintptr_t>(a.cache_v) |
      reinterpret_cast<uintptr_t>(a.k_rows) | reinterpret_cast<uintptr_t>(a.v_rows) |
      reinterpret_cast<uintptr_t>(a.workspace);
  return (align & 15u) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t chunk_attention_bf16(const ChunkAttentionArgs &a, cudaStream_t stream) {
  const cudaError_t valid = validate_chunk_attention(a);
  if (valid != cudaSuccess) return valid;
  if (a.runs.run_count == 0 || a.runs.rows == 0) return cudaSuccess;
  const dim3 grid(unsigned(a.runs.max_row_count), unsigned(a.runs.run_count),
                  unsigned(div_up(a.q_heads, kWarps)));
  if (a.cfg.head_dim == 256) {
    chunk_attention_simple_kernel<256><<<grid, kWarps * 32, 0, stream>>>(a);
  } else {
    chunk_attention_simple_kernel<512><<<grid, kWarps * 32, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace b200kv
