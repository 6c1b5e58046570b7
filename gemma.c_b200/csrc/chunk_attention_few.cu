// Attention of small calls (a token, the drafted tokens of a speculative step, a short
// chunk over a short cache): the same definition as chunk_attention.cu, for calls whose
// way is what they cost.
//
// A query tile is 16 rows, tokens x the G query heads of a KV head: the rows of the
// warp-level products (mma.sync m16n8k16). tcgen05 would spend 128 rows, its tensor
// memory and its barriers on them. A cluster of CTAs takes one (query tile,
// KV head) and each of its CTAs an even share of the keys in units of 16, a tile of 64
// (head_dim 512: 32) at a time, brought by TMA a tile ahead: each of the eight warps asks
// for one unit of K or V (head_dim 512: half of one), in a box or two that lie in a page;
// where pages are no whole groups of eight tokens by copies of 16 bytes. (A bulk copy per
// row costs its warp 86 clocks each, 16 of them more than the tile's arithmetic.) Per tile:
//   S = Q K^T     16 keys and 128 dims each, joined through shared memory
//   softmax       16 threads to a row: running maximum and sum in fp32, the weights
//                 rounded to bf16 for P V (by at most 2^-8 of each), summed unrounded
//   O = a O + P V an eighth of the output dims each, fp32 in registers
// At the end every CTA stores in each other one's shared memory what that joins: its
// share of the output dims, with maxima and sums. A CTA joins and writes its share when
// those have come, and waits for nobody to end. One launch, no partial results in memory.
//
// Latency bounds it. Measured, four tokens of 16 + 8 heads of 256 over a ring of 1024
// (8.4 MB of K and V, 1.3 us of HBM): 7.6 us of the GPU in a row of calls, 15.2 by the
// other kernel and its join; one token over 100 keys 6.0; over pages of five 8.0 instead
// of 21.7. Of the way (80 CTAs, 2 tiles each) in clocks: the runs 800, what follows from
// them 1100, page and first tile 1800, a tile 1500 (of which the first is fetching code),
// sending and joining 2000. Earlier forms: 64 CTAs with tiles of 32 keys 10.1 us, a bulk
// copy per row 8.1, all of the rows' copies from one warp 14.2, a softmax in every warp
// for itself 10.7 (twice the code). The code is kept small: a call runs most of it once.
#include <algorithm>
#include <atomic>

#include "chunk_common.cuh"
#include "chunk_exact.cuh"
#include "chunk_maps.cuh"
#include "kernels.cuh"

namespace b200kv {

namespace {

constexpr int kFewRows = 16;
constexpr int kFewUnit = 16;     // keys: a step of P V, and what the CTAs' shares are counted in
constexpr int kFewWarps = 8;
constexpr int kFewStages = 2;
constexpr uint32_t kFewPolls = 1u << 20;  // of a wait; tens of milliseconds at least
constexpr int kFewMaxCluster = 16;

template <int D>
struct FewTraits {
  static constexpr int kKeys = D == 256 ? 64 : 32;        // of a tile
  static constexpr int kUnits = kKeys / kFewUnit;
  static constexpr int kDimParts = kFewWarps / kUnits;    // warps that share 16 keys, 128 dims each
  static constexpr int kUnitBytes = kFewUnit * D * 2;     // D / 256 boxes of 16 keys x 256 dims
  static constexpr int kTileBytes = kUnits * kUnitBytes;  // of K or V
  static constexpr int kPartPitch = kKeys + 8;            // floats of a row of scores
  static constexpr int kOut = D / kFewWarps;              // dims of a warp's part of P V
  static constexpr int kGroups = D / 16;                  // of 16 output dims
};

template <int D>
struct FewShared {
  using T = FewTraits<D>;
  uint8_t tile[kFewStages][2][T::kTileBytes];             // K and V
  float part[T::kDimParts][kFewRows][T::kPartPitch];      // scores
  uint8_t weights[kFewRows][T::kKeys * 2 + 16];           // bf16
  float alpha[kFewRows];                                  // what O is rescaled by
  uint16_t alive[kFewStages][4];  // keys of the tile's units that some row sees
  uint64_t full[kFewStages];      // the tile has landed
  uint64_t joined;                // what the cluster's warps send has landed
  float factor[kFewRows][kFewMaxCluster];  // what a CTA's O counts for in the row
  // What the cluster's CTAs send here: maximum and sum of [rank][row], and [rank][n][row]
  // 16 dims of this CTA's n-th group.
  alignas(16) float2 row[kFewMaxCluster][kFewRows];
  alignas(16) float sent[(T::kGroups + kFewMaxCluster) * kFewRows * 16];
};

struct FewDivs {
  FastDiv page;   // by page_size (tokens)
  FastDiv slots;  // by max_pages_per_seq
  FastDiv group;  // by the query heads of a KV head
  FastDiv ctas;   // by the cluster's size
  FastDiv tiles;  // by the query tiles of the longest run
};

// The units of 16 keys of a query tile, in this order: of the cache [0, ca) (sinks) and
// [cb0, cb1), of the run's own rows [0, oa) (sinks) and [ob0, ob1). Positions ascend.
struct FewKeys {
  int ca, cb0, cb1, oa, ob0, ob1;
  int lo, cache_end, first;
  __device__ __forceinline__ int count() const { return ca + (cb1 - cb0) + oa + (ob1 - ob0); }
  // position of the first key of unit j
  __device__ __forceinline__ int base(int j, bool &own) const {
    own = false;
    if (j < ca) return j * kFewUnit;
    j -= ca;
    if (j < cb1 - cb0) return (cb0 + j) * kFewUnit;
    j -= cb1 - cb0;
    own = true;
    return first + (j < oa ? j : ob0 + j - oa) * kFewUnit;
  }
};

// Of the rows at positions t0 .. t1.
__device__ __forceinline__ FewKeys few_keys(const ChunkAttentionArgs &a, int first, int t0, int t1, int table_end) {
  FewKeys k = {};
  k.first = first;
  k.lo = a.window > 0 ? max(0, t0 - a.window + 1) : 0;
  k.cache_end = min(a.k_rows != nullptr ? first : t1 + 1, table_end);
  const int sink_end = min(a.sinks, k.lo);
  k.ca = div_up(min(sink_end, k.cache_end), kFewUnit);
  if (k.cache_end > k.lo) {
    k.cb0 = k.lo / kFewUnit;
    k.cb1 = div_up(k.cache_end, kFewUnit);
    k.ca = min(k.ca, k.cb0);
  }
  if (a.k_rows != nullptr) {
    k.ob0 = max(k.lo - first, 0) / kFewUnit;
    k.ob1 = (t1 - first) / kFewUnit + 1;
    k.oa = sink_end > first ? min(div_up(sink_end - first, kFewUnit), k.ob0) : 0;
  }
  return k;
}

// bits [0, n) of 16, n clamped
__device__ __forceinline__ uint32_t low16(int n) {
  return n <= 0 ? 0u : (n >= 16 ? 0xffffu : (1u << n) - 1u);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same place in the shared memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t peer_address(uint32_t at, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_peer(uint32_t at, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void arrive_at_peer(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool try_wait_for_peers(uint32_t bar) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void copy_async16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// This lane's copies so far count as one arrival when they have landed.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool few_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t left = kFewPolls; !mbar_try_wait(bar, parity); --left) {
    if (left == 0) return false;
  }
  return true;
}
// Gives the copies of tiles j .. end - 1 time to land (out of line: calls never come here).
__device__ __noinline__ void few_drain(uint32_t bar_full, int j, int end) {
  for (; j < end; ++j) {
    mbar_wait_bounded(bar_full + 8u * uint32_t(j % kFewStages), uint32_t(j / kFewStages) & 1u, 1ll << 26);
  }
}
// This warp's two rows where the lanes of `odd` have a value that is not finite, in the dims
// that the CTA joins (out of line, too). row0: packed row of the tile's first token.
template <int D>
__device__ __noinline__ void few_not_finite(const ChunkAttentionArgs &a, int table_end, int64_t row0, uint32_t odd) {
  const int group = a.q_heads / a.cfg.num_heads, lane = int(threadIdx.x) & 31;
  for (int i = 0; i < 2 * (D / 256); ++i) {  // 256 dims at a time
    if (((odd >> (16 * (i & 1))) & 0xffffu) == 0) continue;
    const int r = int(threadIdx.x) / 32 * 2 + (i & 1), dims = i / 2 * 256 + lane * 8;
    chunk_exact_row<D>(a, table_end, row0 + r / group, int(blockIdx.y) * group + r % group, dims,
                       dims / 16 % int(gridDim.x) == int(blockIdx.x));
  }
}

// grid (CTAs of a cluster, KV heads, query tiles of the runs). give_up_at: the wait for
// this key tile counts as run out (-1 but in the self-test).
template <int D>
__global__ __launch_bounds__(kFewWarps * 32, 1) void chunk_attention_few_kernel(
    const __grid_constant__ ChunkAttentionArgs a, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k_rows,
    const __grid_constant__ CUtensorMap map_v_rows, int table_end, int box, FewDivs div, int give_up_at) {
  using T = FewTraits<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  FewShared<D> &s = *reinterpret_cast<FewShared<D> *>(smem_raw);
  const int tid = int(threadIdx.x);
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const Gemma4KvCacheConfig &c = a.cfg;
  const int heads = c.num_heads;
  const int group = int(div.group.d);
  const int ctas = int(gridDim.x);
  const int rank = int(blockIdx.x);
  const int head = int(blockIdx.y);
  const uint32_t bar_full = smem_u32(&s.full[0]);
  const uint32_t bar_joined = smem_u32(&s.joined);
  // groups of 16 output dims that this CTA joins: number n of the dims is CTA n % ctas's
  const int slots = div.ctas.quotient(T::kGroups + ctas - 1 - rank);
  if (tid == 0) {
    // a warp's word, and without boxes each lane's copies
    for (int i = 0; i < kFewStages; ++i) mbar_init(bar_full + 8u * i, box > 0 ? kFewWarps : 33 * kFewWarps);
    mbar_init(bar_joined, uint32_t(ctas * kFewWarps));
    mbar_fence_init();
    if (box > 0) {
      prefetch_map(&map_k);
      prefetch_map(&map_v);
      if (a.k_rows != nullptr) {
        prefetch_map(&map_k_rows);
        prefetch_map(&map_v_rows);
      }
    }
  }
  __syncthreads();
  cluster_arrive();  // (its CTAs must have started before they are written to)
  pdl_wait_for_predecessor();
  pdl_release_successor();
  const int of_run = div.tiles.quotient(int(blockIdx.z));
  const ChunkRun run = chunk_run(a.runs, of_run, c.batch_size);
  const int token0 = (int(blockIdx.z) - of_run * int(div.tiles.d)) * div.group.quotient(kFewRows);
  if (token0 >= run.count) {  // the whole cluster
    cluster_wait();
    return;
  }
  const int tokens = min(div.group.quotient(kFewRows), run.count - token0);
  const int rows = tokens * group;
  const int t0 = run.first + token0, t1 = t0 + tokens - 1;
  const int64_t row0 = int64_t(run.start) + token0;  // packed row of the first token
  const FewKeys keys = few_keys(a, run.first, t0, t1, table_end);
  const int total = keys.count();
  const int even = div.ctas.quotient(total);
  const int rest = total - even * ctas;  // the first CTAs have one more
  const int unit0 = even * rank + min(rank, rest);
  const int units = even + (rank < rest ? 1 : 0);
  const int tiles = div_up(units, T::kUnits);

  // ---- K and V: this warp's unit of a tile. Lanes 2 i and 2 i + 1 look up the first and
  // the last eight keys of the unit of tile i, 16 tiles at a time.
  const bool is_v = (warp & 1) != 0;
  const int my_unit = (warp >> 1) % T::kUnits;
  const int block0 = (warp >> 1) / T::kUnits * (kBoxDims / 64);  // head_dim 512: dims from 256 on
  const int page_groups = c.page_size / 8;
  int token_group = -1;  // cache: group of eight tokens; -1: none
  auto look_up = [&](int j) {
    token_group = -1;
    if (box == 0) return;
    const int ask = j * T::kUnits + my_unit + (lane >> 1) * T::kUnits;
    bool own;
    const int at = keys.base(unit0 + ask, own) + 8 * (lane & 1);
    if (ask < units && !own && at < keys.cache_end) {
      const int logical = div.page.quotient(at);
      const int slot = c.window_size > 0 ? logical - div.slots.quotient(logical) * c.max_pages_per_seq : logical;
      const int page = __ldg(a.page_table + int64_t(run.batch) * c.max_pages_per_seq + slot);
      if (page >= 0 && page < c.num_pages) {
        token_group = (a.layer * c.num_pages + page) * page_groups + ((at - logical * c.page_size) >> 3);
      }
    }
  };
  look_up(0);
  auto issue = [&](int j) {
    if (j >= tiles) return;
    const int unit = j * T::kUnits + my_unit;
    if (j > 0 && (j & 15) == 0) look_up(j);
    // the keys of the unit that some row sees
    bool own;
    const int base = keys.base(unit0 + unit, own);
    uint32_t alive = unit >= units ? 0u
                                   : low16((own ? t1 + 1 : keys.cache_end) - base) &
                                         (~low16(keys.lo - base) | low16(a.sinks - base));
    const int stage = j % kFewStages;
    const uint32_t bar = bar_full + 8u * uint32_t(stage);
    const uint32_t to = smem_u32(&s.tile[stage][is_v][my_unit * T::kUnitBytes]) + uint32_t(block0 * 2048);
    if (box == 0) {  // pages of no whole groups of eight: row by row
      int64_t offset = -1;  // of row `lane` of the unit
      if (((alive >> lane) & 1u) != 0) {
        const int at = base + lane;
        if (own) {
          offset = ((int64_t(run.start) + (at - run.first)) * heads + head) * D;
        } else {
          const int logical = div.page.quotient(at);
          const int slot = c.window_size > 0 ? logical - div.slots.quotient(logical) * c.max_pages_per_seq : logical;
          const int page = __ldg(a.page_table + int64_t(run.batch) * c.max_pages_per_seq + slot);
          if (page >= 0 && page < c.num_pages) {
            offset = cache_offset(c, a.layer, page, at - logical * c.page_size, head, 0);
          }
        }
      }
      alive = __ballot_sync(0xffffffffu, offset >= 0);
      const __nv_bfloat16 *rows_of = own ? (is_v ? a.v_rows : a.k_rows) : (is_v ? a.cache_v : a.cache_k);
      // eight lanes to 128 bytes of a row
#pragma unroll
      for (int r4 = 0; r4 < kFewUnit; r4 += 4) {
        const int r = r4 + (lane >> 3);
        const int64_t at = __shfl_sync(0xffffffffu, offset, r);
        if (at >= 0) {
          const __nv_bfloat16 *from = rows_of + at + block0 * 64 + (lane & 7) * 8;
          const uint32_t dst = to + uint32_t((r >> 3) * 4096 + (r & 7) * 128 + (((lane & 7) ^ (r & 7)) << 4));
#pragma unroll
          for (int b = 0; b < kBoxDims / 64; ++b) copy_async16(dst + uint32_t(1024 * b), from + 64 * b);
        }
      }
      copies_arrive(bar);
      if (lane == 0) {
        if (!is_v && block0 == 0) s.alive[stage][my_unit] = uint16_t(alive);
        mbar_arrive(bar);
      }
      __syncwarp();
      return;
    }
    const int group0 = __shfl_sync(0xffffffffu, token_group, 2 * (j & 15));
    const int group1 = __shfl_sync(0xffffffffu, token_group, 2 * (j & 15) + 1);
    if (!own) alive &= (group0 >= 0 ? 0xffu : 0u) | (group1 >= 0 ? 0xff00u : 0u);
    const bool both = !own && box == 16;  // one box for both groups of eight
    const bool half0 = (alive & 0xffu) != 0 || (both && alive != 0), half1 = (alive >> 8) != 0 && !both;
    if (lane == 0) {
      if (!is_v && block0 == 0) s.alive[stage][my_unit] = uint16_t(alive);
      mbar_arrive_expect_tx(bar, uint32_t((half0 ? (both ? 2 : 1) : 0) + (half1 ? 1 : 0)) * 4096u);
      const CUtensorMap *map = own ? (is_v ? &map_v_rows : &map_k_rows) : (is_v ? &map_v : &map_k);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (!(h == 0 ? half0 : half1)) continue;
        if (own) {
          tma_load_rows_box(to + uint32_t(4096 * h), map, block0, run.start + base - run.first + 8 * h, head, bar);
        } else {
          tma_load_page_box(to + uint32_t(4096 * h), map, block0, h == 0 ? group0 : group1, head, bar);
        }
      }
    }
    __syncwarp();
  };
  // ---- Q: the A operand for this warp's 128 dims (rows behind the last: zeros)
  const int key16 = (warp % T::kUnits) * 16, dim_part = warp / T::kUnits;
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  uint32_t q[8][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = g + 8 * h;
    const int token = div.group.quotient(row);
    const __nv_bfloat16 *from =
        a.q + ((row0 + token) * a.q_heads + head * group + (row - token * group)) * D + dim_part * 128 + t2;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      q[k][h] = row < rows ? __ldg(reinterpret_cast<const uint32_t *>(from + 16 * k)) : 0u;
      q[k][h + 2] = row < rows ? __ldg(reinterpret_cast<const uint32_t *>(from + 16 * k + 8)) : 0u;
    }
  }

  issue(0);

  // ---- this thread's row and keys of the softmax
  constexpr int kMine = T::kKeys / 16;
  const int row = tid >> 4, place = tid & 15;
  const int t = t0 + div.group.quotient(row);
  const float scale = a.softmax_scale * 1.4426950408889634f;
  const int in8 = (lane & 7) + ((lane >> 3) & 1) * 8;  // row that the lane names to ldmatrix
  const uint32_t tile_at = smem_u32(&s.tile[0][0][0]);
  float m = -INFINITY, l = 0.0f;  // l: of this thread's keys
  float o[T::kOut / 8][4] = {};
  bool ok = true;

#pragma unroll 1
  for (int j = 0; j < tiles; ++j) {
    const int stage = j % kFewStages;
    issue(j + 1);  // (its place was read before the barrier among the scores of tile j - 1)
    ok = j != give_up_at && few_wait(bar_full + 8u * uint32_t(stage), uint32_t(j / kFewStages) & 1u);
    const uint32_t k_at = tile_at + uint32_t(2 * stage * T::kTileBytes);
    const uint32_t v_at = k_at + uint32_t(T::kTileBytes);
    {  // a part of the scores
      float sc[2][2][4] = {};
      // (unit, group of eight keys, block of 64 dims, key, its 16-byte chunks swizzled)
      const uint32_t from = k_at + uint32_t(key16 / 16 * T::kUnitBytes + (dim_part >> 1) * 8192 + (lane >> 4) * 4096 +
                                            (dim_part & 1) * 2048 + (lane & 7) * 128);
      const uint32_t chunk = uint32_t(((lane >> 3) & 1) ^ (lane & 7)) << 4;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t b[4];
        ldmatrix_x4(b, from + uint32_t(k >> 2) * 1024u + (chunk ^ (uint32_t(k & 3) << 5)));
        mma_bf16(sc[k & 1][0], q[k], b[0], b[1]);
        mma_bf16(sc[k & 1][1], q[k], b[2], b[3]);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float *to = &s.part[dim_part][g][key16 + 8 * n + t2];
        *reinterpret_cast<float2 *>(to) = make_float2(sc[0][n][0] + sc[1][n][0], sc[0][n][1] + sc[1][n][1]);
        *reinterpret_cast<float2 *>(to + 8 * T::kPartPitch) =
            make_float2(sc[0][n][2] + sc[1][n][2], sc[0][n][3] + sc[1][n][3]);
      }
    }
    // what does not wait for the scores: which of the thread's keys its row sees, and V
    uint32_t sees;
    {
      bool own;
      const int first = kMine * place;
      const int at = keys.base(unit0 + j * T::kUnits + first / kFewUnit, own) + first % kFewUnit;
      sees = uint32_t(s.alive[stage][first / kFewUnit] >> (first % kFewUnit)) & low16(t + 1 - at);
      if (a.window > 0) sees &= ~low16(t - a.window + 1 - at) | low16(a.sinks - at);
    }
    uint32_t v[T::kUnits][T::kOut / 16][4];
    const int v_block = warp * T::kOut / 64;  // of 64 dims
#pragma unroll
    for (int u = 0; u < T::kUnits; ++u) {
      const uint32_t from = v_at + uint32_t(u * T::kUnitBytes + (v_block >> 2) * 8192 + (in8 >> 3) * 4096 +
                                            (v_block & 3) * 1024 + (in8 & 7) * 128);
      const uint32_t chunk = uint32_t((((warp * T::kOut) & 63) / 8 + (lane >> 4)) ^ (in8 & 7)) << 4;
#pragma unroll
      for (int n = 0; n < T::kOut / 16; ++n) ldmatrix_x4_trans(v[u][n], from + (chunk ^ uint32_t(32 * n)));
      // keys that nobody sees may hold anything (0 * NaN): this lane has keys 2 (lane % 4),
      // + 1, + 8 and + 9
      const uint32_t alive = s.alive[stage][u];
      if (alive != 0xffffu) {
        const uint32_t mine = alive >> t2;
        const uint32_t keep0 = ((mine & 1u) != 0 ? 0xffffu : 0u) | ((mine & 2u) != 0 ? 0xffff0000u : 0u);
        const uint32_t keep1 = ((mine & 0x100u) != 0 ? 0xffffu : 0u) | ((mine & 0x200u) != 0 ? 0xffff0000u : 0u);
#pragma unroll
        for (int n = 0; n < T::kOut / 16; ++n) {
          v[u][n][0] &= keep0;
          v[u][n][1] &= keep1;
          v[u][n][2] &= keep0;
          v[u][n][3] &= keep1;
        }
      }
    }
    ok = __syncthreads_and(ok);
    if (!ok) {
      // A tile did not come: its copies and those of the next one, asked for above, get the
      // time to land before the CTA gives its shared memory back. A NaN in the sums makes
      // the rows and their log-sum-exp NaN, whichever CTA joins them.
      few_drain(bar_full, j, min(j + 2, tiles));
      set_status(a.status, B200KV_STATUS_WAIT_TIMEOUT);
      l = __int_as_float(0x7fffffff);
      break;
    }
    {
      float x[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) x[i] = 0.0f;
#pragma unroll
      for (int d = 0; d < T::kDimParts; ++d) {
        float part[kMine];
        if constexpr (kMine == 4) {
          *reinterpret_cast<float4 *>(part) = *reinterpret_cast<const float4 *>(&s.part[d][row][4 * place]);
        } else {
          *reinterpret_cast<float2 *>(part) = *reinterpret_cast<const float2 *>(&s.part[d][row][2 * place]);
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) x[i] += part[i];
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        x[i] = ((sees >> i) & 1u) != 0 ? x[i] * scale : -INFINITY;
        top = fmaxf(top, x[i]);
      }
#pragma unroll
      for (int d = 8; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float now = fmaxf(m, top);
      const float alpha = m == -INFINITY ? 0.0f : ex2_approx(m - now);
      const float neg = now == -INFINITY ? 0.0f : -now;
      l *= alpha;
      m = now;
      uint32_t w[kMine / 2];
#pragma unroll
      for (int i = 0; i < kMine; i += 2) {
        const float e0 = ex2_approx(x[i] + neg), e1 = ex2_approx(x[i + 1] + neg);
        l += e0 + e1;
        const __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
        w[i / 2] = *reinterpret_cast<const uint32_t *>(&b2);
      }
      if constexpr (kMine == 4) {
        *reinterpret_cast<uint2 *>(&s.weights[row][8 * place]) = make_uint2(w[0], w[1]);
      } else {
        *reinterpret_cast<uint32_t *>(&s.weights[row][4 * place]) = w[0];
      }
      if (place == 0) s.alpha[row] = alpha;
    }
    __syncthreads();
    const float alpha0 = s.alpha[g], alpha1 = s.alpha[g + 8];
#pragma unroll
    for (int n = 0; n < T::kOut / 8; ++n) {
      o[n][0] *= alpha0;
      o[n][1] *= alpha0;
      o[n][2] *= alpha1;
      o[n][3] *= alpha1;
    }
#pragma unroll
    for (int u = 0; u < T::kUnits; ++u) {
      uint32_t w[4];
      ldmatrix_x4(w, smem_u32(&s.weights[in8][0]) + uint32_t(32 * u + (lane >> 4) * 16));
#pragma unroll
      for (int n = 0; n < T::kOut / 16; ++n) {
        mma_bf16(o[2 * n], w, v[u][n][0], v[u][n][1]);
        mma_bf16(o[2 * n + 1], w, v[u][n][2], v[u][n][3]);
      }
    }
  }
  // ---- to the CTAs that join the dims: a group is 16 rows x 16 dims
#pragma unroll
  for (int d = 8; d > 0; d /= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
  cluster_wait();
  if (place < ctas) store_peer(peer_address(smem_u32(&s.row[rank][row]), uint32_t(place)), m, l);
#pragma unroll
  for (int n = 0; n < T::kOut / 16; ++n) {
    const int of_dims = warp * (T::kOut / 16) + n;
    const int slot = div.ctas.quotient(of_dims);
    const int owner = of_dims - slot * ctas;
    const int theirs = div.ctas.quotient(T::kGroups + ctas - 1 - owner);
    const uint32_t at = peer_address(smem_u32(&s.sent[(rank * theirs + slot) * 256 + g * 16 + t2]), uint32_t(owner));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      store_peer(at + 32u * uint32_t(h), o[2 * n + h][0], o[2 * n + h][1]);
      store_peer(at + 32u * uint32_t(h) + 512u, o[2 * n + h][2], o[2 * n + h][3]);
    }
  }
  __syncwarp();
  if (lane < ctas) arrive_at_peer(peer_address(bar_joined, uint32_t(lane)));
  // (longer than any wait of a CTA that is to arrive)
  ok = true;
  for (uint32_t left = 32 * kFewPolls; ok && !try_wait_for_peers(bar_joined); --left) ok = left > 0;
  ok = __all_sync(0xffffffffu, ok);
  // ---- joined: out = sum 2^(m_k - M) O_k / sum 2^(m_k - M) l_k
  bool odd = false;  // a value is not finite, and not because the scores are not
  if (row < rows) {
    float2 ml = make_float2(-INFINITY, 0.0f);  // of CTA `place`
    if (place < ctas) ml = s.row[place][row];
    const uint32_t lanes = 0xffffu << (lane & 16);
    float top = ml.x;
#pragma unroll
    for (int d = 8; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(lanes, top, d));
    // (a CTA without a visible key has zeros; one that saw only NaN has a NaN sum)
    const float f = ml.y == 0.0f ? 0.0f : ex2_approx(ml.x == -INFINITY ? 0.0f : ml.x - top);
    float sum = f * ml.y;
#pragma unroll
    for (int d = 8; d > 0; d /= 2) sum += __shfl_xor_sync(lanes, sum, d);
    if (!ok) sum = __int_as_float(0x7fffffff);  // some CTA has not sent its share
    s.factor[row][place] = f * (sum != 0.0f ? 1.0f / sum : 0.0f);
    __syncwarp(lanes);
    const int token = div.group.quotient(row);
    const int64_t out = (row0 + token) * a.q_heads + head * group + (row - token * group);
#pragma unroll 1
    for (int slot = 0; slot < slots; ++slot) {
      float acc = 0.0f;
#pragma unroll 4
      for (int k = 0; k < ctas; ++k) {
        acc = fmaf(s.factor[row][k], s.sent[((k * slots + slot) * kFewRows + row) * 16 + place], acc);
      }
      a.out[out * D + (slot * ctas + rank) * 16 + place] = __float2bfloat16_rn(acc);
      odd |= !(fabsf(acc) < INFINITY);
    }
    odd = odd && sum == sum;
    if (a.lse != nullptr && rank == 0 && place == 0) {
      a.lse[out] = sum != 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
  }
  const uint32_t odd_lanes = __ballot_sync(0xffffffffu, odd);
  if (odd_lanes != 0) few_not_finite<D>(a, table_end, row0, odd_lanes);
  if (!ok) set_status(a.status, B200KV_STATUS_WAIT_TIMEOUT);
}

struct FewLaunch {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[2];
  FewLaunch(int cluster, int heads, int tiles, int smem, cudaStream_t stream) {
    config.gridDim = dim3(unsigned(cluster), unsigned(heads), unsigned(tiles));
    config.blockDim = dim3(kFewWarps * 32);
    config.dynamicSmemBytes = size_t(smem);
    config.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 2;
  }
};

// Clusters of this size that the device runs at once: they lie within a group of SMs,
// and the groups differ (148 SMs: 7 of 16 or 11, 11 of 10, 15 of 8, 33 of 4).
template <int D>
int clusters_at_once(int device, int cluster) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kFewMaxCluster + 1];  // 0: not asked yet
  if (device < kDevices) {
    const int n = known[device][cluster].load(std::memory_order_relaxed);
    if (n > 0) return n - 1;
  }
  FewLaunch launch(cluster, 1, 1, int(sizeof(FewShared<D>)), nullptr);
  launch.config.numAttrs = 1;
  int count = 0;
  if (cudaOccupancyMaxActiveClusters(&count, chunk_attention_few_kernel<D>, &launch.config) != cudaSuccess) {
    cudaGetLastError();
    count = 0;  // not a size for this device
  }
  if (device < kDevices) known[device][cluster].store(count + 1, std::memory_order_relaxed);
  return count;
}

// Query tiles of the longest run.
int64_t few_tiles(const ChunkAttentionArgs &a) {
  return div_up(int64_t(std::min(a.runs.max_row_count, a.runs.rows)), kFewRows / (a.q_heads / a.cfg.num_heads));
}

// The clusters' size for the call; *cluster 0: it is not a small one.
template <int D>
cudaError_t few_cluster(const ChunkAttentionArgs &a, int device, int table_end, int *cluster) {
  *cluster = 0;
  const int64_t items = a.runs.run_count * a.cfg.num_heads * few_tiles(a);
  constexpr int kSmem = int(sizeof(FewShared<D>));
  static_assert(kSmem <= 227 * 1024, "the tiles must fit one SM");
  const auto kernel = chunk_attention_few_kernel<D>;
  cudaError_t st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (st == cudaSuccess) st = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (st != cudaSuccess) return st;
  int size = kFewMaxCluster;  // the largest of which all run at once
  while (size >= 1 && items > clusters_at_once<D>(device, size)) --size;
  if (size < 1) return cudaSuccess;
  // A tile of 64 keys is 1.2 us here behind some 5.6 of start and end; the other kernel and
  // its join take 12 to 17 and hardly more for more keys, so up to 640 keys of 256 dims to a
  // CTA belong here. Of the lengths the host knows the most that a row can see. GPU
  // time here / there, eight heads of 256: four tokens of one sequence over 500, 4000, 8000
  // keys 6.4 / 14.1, 13.4 / 17.0, 20.7 / 19.9 us; of four over 2000 14.5 / 18.9, of eight
  // over 500 9.6 / 21.8; 40 tokens over 500, 2000 8.6 / 16.9, 18.2 / 18.3; 100 over 50, 500
  // 8.4 / 16.0, 16.8 / 18.5; 16 tokens of 16 heads of 512 on one KV head over 500, 2000 10.0
  // / 18.9, 18.8 / 20.3. Where the lengths differ the longest counts here: four tokens of
  // four sequences over 100 .. 4000 keys 24.0 / 19.1.
  if (most_keys(a, table_end, 1) * D <= 640 * 256 * int64_t(size)) *cluster = size;
  return cudaSuccess;
}

template <int D>
cudaError_t try_few(const ChunkAttentionArgs &a, int device, int table_end, cudaStream_t stream, bool *taken,
                    int give_up_at) {
  int cluster = 0;
  const cudaError_t st = few_cluster<D>(a, device, table_end, &cluster);
  if (st != cudaSuccess || cluster == 0) return st;
  *taken = true;
  const int box = box_tokens(a.cfg.page_size, kFewUnit);
  const int tiles = int(few_tiles(a));  // (no more than clusters that run at once)
  CUtensorMap map_k = {}, map_v = {}, map_k_rows = {}, map_v_rows = {};
  if (box > 0 &&
      (!make_cache_map(&map_k, a.cache_k, a.cfg, box) || !make_cache_map(&map_v, a.cache_v, a.cfg, box) ||
       (a.k_rows != nullptr &&
        (!make_rows_map(&map_k_rows, a.k_rows, a.runs.rows, a.cfg.num_heads, D) ||
         !make_rows_map(&map_v_rows, a.v_rows, a.runs.rows, a.cfg.num_heads, D))))) {
    return cudaErrorInvalidValue;
  }
  const FewLaunch launch(cluster, a.cfg.num_heads, a.runs.run_count * tiles, int(sizeof(FewShared<D>)), stream);
  const FewDivs div = {FastDiv::by(uint32_t(a.cfg.page_size)), FastDiv::by(uint32_t(a.cfg.max_pages_per_seq)),
                       FastDiv::by(uint32_t(a.q_heads / a.cfg.num_heads)), FastDiv::by(uint32_t(cluster)),
                       FastDiv::by(uint32_t(tiles))};
  return cudaLaunchKernelEx(&launch.config, chunk_attention_few_kernel<D>, a, map_k, map_v, map_k_rows, map_v_rows,
                            table_end, box, div, give_up_at);
}

}  // namespace

bool chunk_attention_few_takes(const ChunkAttentionArgs &a, int device, int table_end) {
  if (a.q_heads / a.cfg.num_heads > kFewRows) return false;
  int cluster = 0;
  const cudaError_t st = a.cfg.head_dim == 256 ? few_cluster<256>(a, device, table_end, &cluster)
                                               : few_cluster<512>(a, device, table_end, &cluster);
  return st == cudaSuccess && cluster > 0;
}

cudaError_t chunk_attention_few_bf16(const ChunkAttentionArgs &a, int device, int table_end,
                                     cudaStream_t stream, bool *taken, int give_up_at) {
  *taken = false;
  if (a.q_heads / a.cfg.num_heads > kFewRows) return cudaSuccess;
  return a.cfg.head_dim == 256 ? try_few<256>(a, device, table_end, stream, taken, give_up_at)
                               : try_few<512>(a, device, table_end, stream, taken, give_up_at);
}

}  // namespace b200kv
