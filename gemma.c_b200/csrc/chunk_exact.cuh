// A row of the attention of runs again, key by key.
//
// The products of a tile multiply the weight 0 of a key that a row does not see with that
// key's V, so a NaN or an infinity there (a token that a later row of the run drafted, a
// key that the first row's window still has) would reach rows that do not see it. Where a
// finished row is not finite, a warp computes it here from the keys that it sees, and what
// was not finite takes those values. (So do sums of finite values that overflowed.) Calls without such values pay for the look at their
// results only. The same formula in fp32, weights included; the walk over the keys is
// bounded by their load latency and as long as the row's history.
#pragma once

#include "chunk_common.cuh"

namespace b200kv {

// Either of the pair is a NaN or an infinity (exponent bits all ones).
__device__ __forceinline__ bool pair_not_finite(uint32_t x) {
  return (((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
}
__device__ __forceinline__ bool pack_not_finite(uint4 v) {
  return pair_not_finite(v.x) || pair_not_finite(v.y) || pair_not_finite(v.z) || pair_not_finite(v.w);
}

// For a whole warp. row: packed row of the token. A lane has 8 output dims, from dim0 on;
// `mine`: it may write them (what they hold is read back).
template <int D>
__device__ __noinline__ void chunk_exact_row(const ChunkAttentionArgs &a, int table_end, int64_t row, int q_head,
                                             int dim0, bool mine) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kPacks = D / 256;  // of 8 dims of K per lane
  constexpr int kAtOnce = 4;       // keys
  const int lane = int(threadIdx.x) & 31;
  const Gemma4KvCacheConfig &c = a.cfg;
  const int head = q_head / (a.q_heads / c.num_heads);
  uint4 *out = reinterpret_cast<uint4 *>(a.out + (row * a.q_heads + q_head) * D + dim0);
  const uint4 was = *out;
  uint32_t now[4] = {was.x, was.y, was.z, was.w};
  uint32_t open = 0;  // dims of this lane that are to be explained
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (mine && ((now[i / 2] >> (16 * (i & 1))) & 0x7f80u) == 0x7f80u) open |= 1u << i;
  }
  const uint32_t bad = open;
  if (!__any_sync(kAll, bad != 0)) return;
  ChunkRun run;  // that names the row
  for (int base = 0; run.count == 0; base += 32) {
    if (base >= a.runs.run_count) return;
    const ChunkRun of = chunk_run(a.runs, base + lane, c.batch_size);
    const uint32_t hit = __ballot_sync(kAll, row >= of.start && row - of.start < of.count);
    if (hit == 0) continue;
    const int from = __ffs(int(hit)) - 1;
    run.count = __shfl_sync(kAll, of.count, from);
    run.first = __shfl_sync(kAll, of.first, from);
    run.start = __shfl_sync(kAll, of.start, from);
    run.batch = __shfl_sync(kAll, of.batch, from);
  }
  const int t = run.first + int(row - run.start);
  const int lo = a.window > 0 ? max(0, t - a.window + 1) : 0;
  const int sink_end = min(a.sinks, lo);
  // The row's keys, newest first, up to four at a time: use(n, offsets of the keys' rows
  // (at the KV head), which of them are in k_rows / v_rows); false ends the walk.
  auto walk = [&](auto use) {
    for (int part = 0; part < 2; ++part) {  // the window, the first tokens
      const int begin = part == 0 ? lo : 0;
      int end = part == 0 ? t + 1 : sink_end;
      while (end > begin) {
        const int from = max(begin, end - 32);
        const int position = from + lane;
        const bool own = a.k_rows != nullptr && position >= run.first;
        int64_t offset = -1;
        if (position < end) {
          if (own) {
            offset = ((int64_t(run.start) + (position - run.first)) * c.num_heads + head) * D;
          } else if (position < table_end) {
            const int page = chunk_page(c, a.page_table, run.batch, position / c.page_size);
            if (page >= 0) offset = cache_offset(c, a.layer, page, position % c.page_size, head, 0);
          }
        }
        uint32_t found = __ballot_sync(kAll, offset >= 0);
        const uint32_t owns = __ballot_sync(kAll, own);
        while (found != 0) {
          int64_t at[kAtOnce];
          bool of_rows[kAtOnce];
          int n = 0;
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            if (found == 0) {  // once more the last one; not used
              at[i] = at[i > 0 ? i - 1 : 0];
              of_rows[i] = of_rows[i > 0 ? i - 1 : 0];
              continue;
            }
            const int key = 31 - __clz(int(found));
            found ^= 1u << key;
            at[i] = __shfl_sync(kAll, offset, key);
            of_rows[i] = ((owns >> key) & 1u) != 0;
            ++n;
          }
          if (!use(n, at, of_rows)) return;
        }
        end = from;
      }
    }
  };
  // A NaN in the dim of a key that the row sees, or an infinity where the result is one:
  // then it is the row's own. (Rows behind a bad one end here, at that one.)
  walk([&](int, const int64_t (&at)[kAtOnce], const bool (&of_rows)[kAtOnce]) {
    uint4 v[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      v[k] = __ldg(reinterpret_cast<const uint4 *>((of_rows[k] ? a.v_rows : a.cache_v) + at[k] + dim0));
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const uint32_t words[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x = (words[i / 2] >> (16 * (i & 1))) & 0x7fffu;
        const uint32_t y = (now[i / 2] >> (16 * (i & 1))) & 0x7fffu;
        if (x > 0x7f80u || (x == 0x7f80u && y == 0x7f80u)) open &= ~(1u << i);
      }
    }
    return __any_sync(kAll, open != 0);
  });
  if (!__any_sync(kAll, open != 0)) return;
  // the row, with a running maximum
  const float scale = a.softmax_scale * 1.4426950408889634f;
  const __nv_bfloat16 *q_row = a.q + (row * a.q_heads + q_head) * D;
  float q[kPacks][8];
#pragma unroll
  for (int n = 0; n < kPacks; ++n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[n][i] = __bfloat162float(q_row[256 * n + lane * 8 + i]);
  }
  float m = -INFINITY, l = 0.0f, acc[8] = {};
  walk([&](int n, const int64_t (&at)[kAtOnce], const bool (&of_rows)[kAtOnce]) {
    float s[kAtOnce];
    uint4 v[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      v[k] = __ldg(reinterpret_cast<const uint4 *>((of_rows[k] ? a.v_rows : a.cache_v) + at[k] + dim0));
      const __nv_bfloat16 *key = (of_rows[k] ? a.k_rows : a.cache_k) + at[k];
      s[k] = 0.0f;
#pragma unroll
      for (int p = 0; p < kPacks; ++p) {
        const uint4 kk = __ldg(reinterpret_cast<const uint4 *>(key + 256 * p) + lane);
        const uint32_t words[4] = {kk.x, kk.y, kk.z, kk.w};
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          s[k] = fmaf(q[p][i], __uint_as_float(words[i / 2] << 16), s[k]);
          s[k] = fmaf(q[p][i + 1], __uint_as_float(words[i / 2] & 0xffff0000u), s[k]);
        }
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) s[k] += __shfl_xor_sync(kAll, s[k], d);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (k >= n) break;
      const float x = s[k] * scale;
      const float top = fmaxf(m, x);
      const float keep = m == -INFINITY ? 0.0f : ex2_approx(m - top);
      const float w = x == -INFINITY ? 0.0f : ex2_approx(x - top);
      m = top;
      // an average all along: large values do not overflow on the way
      const float sum = fmaf(l, keep, w);
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      const float old = l * keep * inv, add = w * inv;
      l = sum;
      const uint32_t words[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        acc[i] = fmaf(add, __uint_as_float(words[i / 2] << 16), acc[i] * old);
        acc[i + 1] = fmaf(add, __uint_as_float(words[i / 2] & 0xffff0000u), acc[i + 1] * old);
      }
    }
    return l == l;  // (a NaN of the scores: so is the row)
  });
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (((bad >> i) & 1u) == 0) continue;
    const uint32_t x = __bfloat16_as_ushort(__float2bfloat16_rn(acc[i]));
    now[i / 2] = (i & 1) != 0 ? (now[i / 2] & 0xffffu) | (x << 16) : (now[i / 2] & 0xffff0000u) | x;
  }
  if (bad != 0) *out = make_uint4(now[0], now[1], now[2], now[3]);
}

}  // namespace b200kv
