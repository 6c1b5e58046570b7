// Attention of runs with few query rows (a token, the drafted tokens of a
// speculative step) over few sequences: the same definition as chunk_attention.cu,
// for calls so small that the way through a call is what it costs.
//
// All rows of a run (tokens x the G query heads of a KV head, at most 16) are the 16
// rows of the warp-level products (mma.sync m16n8k16): tcgen05 would spend its 128
// rows, its tensor memory and its barriers on them. A cluster of CTAs takes one (run,
// KV head) and each of its CTAs an even share of the keys, in tiles of 32. K and V rows
// come by 16-byte asynchronous copies, several tiles ahead, whatever the page size;
// rows that nobody sees arrive as zeros. Per tile, eight warps:
//   S = Q K^T     two halves of the keys x four quarters of the dims, joined through
//                 shared memory
//   softmax       16 threads to a row, two keys each; running maximum and sum in fp32,
//                 the weights rounded to bf16 for P V (by at most 2^-8 of each), summed
//                 unrounded
//   O = a O + P V an eighth of the output dims each, fp32 in registers
// At the end every CTA sends each other one its share of the output dims, with maxima
// and sums, over distributed shared memory; after one cluster barrier a CTA joins and
// writes its share. One launch, no partial results in memory.
#include <algorithm>

#include "chunk_common.cuh"
#include "kernels.cuh"

namespace b200kv {

namespace {

constexpr int kFewRows = 16;
constexpr int kFewKeys = 32;
constexpr int kFewThreads = 256;
constexpr int kFewMaxCluster = 16;

template <int D>
struct FewTraits {
  static constexpr int kStages = D == 256 ? 4 : 2;
  static constexpr int kPitch = D * 2 + 16;               // bytes of a row: no bank twice
  static constexpr int kTileBytes = kFewKeys * kPitch;    // of K or V
  static constexpr int kQuarter = D / 4;                  // dims of a warp's part of Q K^T
  static constexpr int kOut = D / 8;                      // dims of a warp's part of P V
};

template <int D>
struct FewShared {
  uint8_t tile[FewTraits<D>::kStages][2][FewTraits<D>::kTileBytes];
  float part[4][kFewRows][kFewKeys];            // scores of a quarter of the dims
  uint8_t weights[kFewRows][kFewKeys * 2 + 16];  // bf16
  float alpha[kFewRows];                        // what O is rescaled by
  uint8_t alive[FewTraits<D>::kStages][kFewKeys];
  // what the cluster's CTAs send here: [rank][row][dim of this CTA's share] and per
  // [rank][row] maximum and sum
  float2 row[kFewMaxCluster][kFewRows];
  float sent[kFewRows * D];
};

// The key tiles of a run, in this order: of the cache [0, ca) (sinks) and [cb0, cb1), of
// the run's own rows [0, oa) (sinks) and [ob0, ob1).
struct FewTiles {
  int ca, cb0, cb1, oa, ob0, ob1;
  int lo, cache_end, first;
  __device__ __forceinline__ int count() const { return ca + (cb1 - cb0) + oa + (ob1 - ob0); }
  // position of the first key of tile j
  __device__ __forceinline__ int base(int j, bool &own) const {
    own = false;
    if (j < ca) return j * kFewKeys;
    j -= ca;
    if (j < cb1 - cb0) return (cb0 + j) * kFewKeys;
    j -= cb1 - cb0;
    own = true;
    return first + (j < oa ? j : ob0 + j - oa) * kFewKeys;
  }
};

__device__ __forceinline__ FewTiles few_tiles(const ChunkAttentionArgs &a, const ChunkRun &run, int table_end) {
  FewTiles k = {};
  const int t1 = run.first + run.count - 1;
  k.first = run.first;
  k.lo = a.window > 0 ? max(0, run.first - a.window + 1) : 0;
  k.cache_end = min(a.k_rows != nullptr ? run.first : t1 + 1, table_end);
  const int sink_end = min(a.sinks, k.lo);
  k.ca = div_up(min(sink_end, k.cache_end), kFewKeys);
  if (k.cache_end > k.lo) {
    k.cb0 = k.lo / kFewKeys;
    k.cb1 = div_up(k.cache_end, kFewKeys);
    k.ca = min(k.ca, k.cb0);
  }
  if (a.k_rows != nullptr) {
    // (no key of a run comes before its window: lo <= first)
    k.ob1 = (t1 - run.first) / kFewKeys + 1;
  }
  return k;
}

__device__ __forceinline__ void copy16_or_zeros(uint32_t to, const void *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from),
               "r"(there ? 16u : 0u)
               : "memory");
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
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
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

template <int D>
__global__ __launch_bounds__(kFewThreads, 1) void chunk_attention_few_kernel(
    const __grid_constant__ ChunkAttentionArgs a, int table_end) {
  using T = FewTraits<D>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  FewShared<D> &s = *reinterpret_cast<FewShared<D> *>(smem_raw);
  const int tid = int(threadIdx.x);
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const Gemma4KvCacheConfig &c = a.cfg;
  const int heads = c.num_heads;
  const int group = a.q_heads / heads;
  const int ctas = int(cluster_size());
  const int rank = int(cluster_rank());
  const int item = int(blockIdx.x) / ctas;
  const int head = item % heads;

  pdl_wait_for_predecessor();
  pdl_release_successor();
  const ChunkRun run = chunk_run(a.runs, item / heads, c.batch_size);
  if (run.count == 0) return;  // the whole cluster
  cluster_arrive();            // (its CTAs must have started before they are sent to)
  const int rows = run.count * group;
  const FewTiles keys = few_tiles(a, run, table_end);
  const int total = keys.count();
  const int tile0 = int(int64_t(total) * rank / ctas);
  const int tiles = int(int64_t(total) * (rank + 1) / ctas) - tile0;

  // ---- where the rows of the tiles lie. A warp copies rows 4 w .. 4 w + 3 of every tile;
  // lane l knows row l % 4 of tile l / 4 of a batch of eight tiles.
  constexpr int64_t kOwn = int64_t(1) << 62;
  auto look_up = [&](int batch) -> int64_t {  // element offset (kOwn: of the run's rows), -1: nobody sees it
    const int j = 8 * batch + (lane >> 2);
    if (j >= tiles) return -1;
    bool own;
    const int base = keys.base(tile0 + j, own);
    const int at = base + 4 * warp + (lane & 3);
    if (own) {
      return at - run.first < run.count
                 ? kOwn + ((int64_t(run.start) + (at - run.first)) * heads + head) * D
                 : -1;
    }
    if (at >= keys.cache_end || (at < keys.lo && at >= a.sinks)) return -1;
    const int logical = at / c.page_size;
    const int page = chunk_page(c, a.page_table, run.batch, logical);
    return page < 0 ? -1 : cache_offset(c, a.layer, page, at - logical * c.page_size, head, 0);
  };
  int64_t here = look_up(0), next = look_up(1);
  const uint32_t tile_at = smem_u32(&s.tile[0][0][0]);
  auto issue = [&](int j) {
    if (j < tiles) {
      const int stage = j % T::kStages;
      if (j > 0 && (j & 7) == 0) {
        here = next;
        next = look_up((j >> 3) + 1);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t at = __shfl_sync(0xffffffffu, here, (j & 7) * 4 + r);
        const bool there = at >= 0;
        const bool own = there && (at & kOwn) != 0;
        const int64_t offset = there ? at & ~kOwn : 0;
        const int row = 4 * warp + r;
        if (lane == 0) s.alive[stage][row] = there ? 1 : 0;
#pragma unroll
        for (int v = 0; v < D / 256; ++v) {
          const uint32_t to = tile_at + uint32_t(2 * stage * T::kTileBytes + row * T::kPitch + (lane + 32 * v) * 16);
          const int64_t from = offset + (lane + 32 * v) * 8;
          copy16_or_zeros(to, (own ? a.k_rows : a.cache_k) + from, there);
          copy16_or_zeros(to + uint32_t(T::kTileBytes), (own ? a.v_rows : a.cache_v) + from, there);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < T::kStages - 1; ++i) issue(i);

  // ---- Q: the A operand of this warp's quarter of the dims (rows behind the last: zeros)
  const int key_half = warp & 1, quarter = warp >> 1;
  const int g = lane >> 2, t2 = (lane & 3) * 2;
  uint32_t q[T::kQuarter / 16][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = g + 8 * h;
    const int token = row / group;
    const __nv_bfloat16 *from = a.q + ((int64_t(run.start) + token) * a.q_heads + head * group + (row - token * group)) * D +
                                quarter * T::kQuarter + t2;
#pragma unroll
    for (int k = 0; k < T::kQuarter / 16; ++k) {
      q[k][h] = row < rows ? __ldg(reinterpret_cast<const uint32_t *>(from + 16 * k)) : 0u;
      q[k][h + 2] = row < rows ? __ldg(reinterpret_cast<const uint32_t *>(from + 16 * k + 8)) : 0u;
    }
  }

  // ---- softmax: this thread's row and keys
  const int row = tid >> 4, pair = tid & 15;
  const int t = run.first + row / group;
  const float scale = a.softmax_scale * 1.4426950408889634f;
  float m = -INFINITY, l = 0.0f;  // l: of this thread's keys
  float o[T::kOut / 8][4] = {};

  for (int j = 0; j < tiles; ++j) {
    const int stage = j % T::kStages;
    asm volatile("cp.async.wait_group %0;" ::"n"(T::kStages - 2) : "memory");
    __syncthreads();
    issue(j + T::kStages - 1);
    const uint32_t k_at = tile_at + uint32_t(2 * stage * T::kTileBytes);
    const uint32_t v_at = k_at + uint32_t(T::kTileBytes);
    {  // a part of the scores: 16 keys, a quarter of the dims
      float sc[2][4] = {};
      const uint32_t from = k_at + uint32_t((16 * key_half + (lane & 7) + ((lane >> 4) & 1) * 8) * T::kPitch +
                                            quarter * T::kQuarter * 2 + ((lane >> 3) & 1) * 16);
#pragma unroll
      for (int k = 0; k < T::kQuarter / 16; ++k) {
        uint32_t b[4];
        ldmatrix_x4(b, from + 32u * uint32_t(k));
        mma_bf16(sc[0], q[k], b[0], b[1]);
        mma_bf16(sc[1], q[k], b[2], b[3]);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float *to = &s.part[quarter][g][16 * key_half + 8 * n + t2];
        *reinterpret_cast<float2 *>(to) = make_float2(sc[n][0], sc[n][1]);
        *reinterpret_cast<float2 *>(to + 8 * kFewKeys) = make_float2(sc[n][2], sc[n][3]);
      }
    }
    __syncthreads();
    {
      bool own;
      const int at = keys.base(tile0 + j, own) + 2 * pair;
      float x[2];
      const float2 p0 = *reinterpret_cast<const float2 *>(&s.part[0][row][2 * pair]);
      const float2 p1 = *reinterpret_cast<const float2 *>(&s.part[1][row][2 * pair]);
      const float2 p2 = *reinterpret_cast<const float2 *>(&s.part[2][row][2 * pair]);
      const float2 p3 = *reinterpret_cast<const float2 *>(&s.part[3][row][2 * pair]);
      x[0] = ((p0.x + p1.x) + (p2.x + p3.x)) * scale;
      x[1] = ((p0.y + p1.y) + (p2.y + p3.y)) * scale;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool sees = s.alive[stage][2 * pair + i] != 0 && at + i <= t &&
                          (a.window == 0 || at + i > t - a.window || at + i < a.sinks);
        if (!sees) x[i] = -INFINITY;
      }
      float top = fmaxf(x[0], x[1]);
#pragma unroll
      for (int d = 8; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float now = fmaxf(m, top);
      const float alpha = m == -INFINITY ? 0.0f : ex2_approx(m - now);
      const float neg = now == -INFINITY ? 0.0f : -now;
      const float e0 = ex2_approx(x[0] + neg), e1 = ex2_approx(x[1] + neg);
      l = fmaf(l, alpha, e0 + e1);
      m = now;
      const __nv_bfloat162 w = __floats2bfloat162_rn(e0, e1);
      *reinterpret_cast<__nv_bfloat162 *>(&s.weights[row][4 * pair]) = w;
      if (pair == 0) s.alpha[row] = alpha;
    }
    __syncthreads();
    {
      const float alpha0 = s.alpha[g], alpha1 = s.alpha[g + 8];
#pragma unroll
      for (int n = 0; n < T::kOut / 8; ++n) {
        o[n][0] *= alpha0;
        o[n][1] *= alpha0;
        o[n][2] *= alpha1;
        o[n][3] *= alpha1;
      }
      const int in8 = (lane & 7) + ((lane >> 3) & 1) * 8;
      const uint32_t w_from = smem_u32(&s.weights[in8][0]) + uint32_t(lane >> 4) * 16u;
      const uint32_t v_from =
          v_at + uint32_t(in8 * T::kPitch + warp * T::kOut * 2 + (lane >> 4) * 16);
#pragma unroll
      for (int k = 0; k < kFewKeys / 16; ++k) {
        uint32_t w[4];
        ldmatrix_x4(w, w_from + 32u * uint32_t(k));
#pragma unroll
        for (int n = 0; n < T::kOut / 16; ++n) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, v_from + uint32_t(16 * k * T::kPitch + 32 * n));
          mma_bf16(o[2 * n], w, b[0], b[1]);
          mma_bf16(o[2 * n + 1], w, b[2], b[3]);
        }
      }
    }
  }

  // ---- to the CTAs that own the dims: columns [rank * D / ctas, ...) each
#pragma unroll
  for (int d = 8; d > 0; d /= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
  const int share = D / ctas;  // 16 dims at least
  cluster_wait();
  if (pair < ctas) store_peer(peer_address(smem_u32(&s.row[rank][row]), uint32_t(pair)), m, l);
  const uint32_t sent_at = smem_u32(&s.sent[rank * kFewRows * share]);
#pragma unroll
  for (int n = 0; n < T::kOut / 8; ++n) {
    const int column = warp * T::kOut + 8 * n + t2;
    const int owner = column / share;
    const uint32_t at = peer_address(sent_at + uint32_t((g * share + column - owner * share) * 4), uint32_t(owner));
    store_peer(at, o[n][0], o[n][1]);
    store_peer(at + uint32_t(8 * share * 4), o[n][2], o[n][3]);
  }
  cluster_arrive();
  cluster_wait();
  // ---- joined: out = sum 2^(m_r - M) O_r / sum 2^(m_r - M) l_r
  const int pairs = share / 2;
  for (int i = tid; i < rows * pairs; i += kFewThreads) {
    const int r = i / pairs;
    const int column = 2 * (i - r * pairs);
    float top = -INFINITY;
    for (int k = 0; k < ctas; ++k) top = fmaxf(top, s.row[k][r].x);
    float sum = 0.0f, x = 0.0f, y = 0.0f;
    for (int k = 0; k < ctas; ++k) {
      const float2 ml = s.row[k][r];
      const float2 v = *reinterpret_cast<const float2 *>(&s.sent[(k * kFewRows + r) * share + column]);
      // (a CTA without a visible key has zeros; one that saw only NaN has a NaN sum)
      const float f = ml.y == 0.0f ? 0.0f : ex2_approx(ml.x == -INFINITY ? 0.0f : ml.x - top);
      sum = fmaf(f, ml.y, sum);
      x = fmaf(f, v.x, x);
      y = fmaf(f, v.y, y);
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    const int token = r / group;
    const int64_t at = (int64_t(run.start) + token) * a.q_heads + head * group + (r - token * group);
    *reinterpret_cast<__nv_bfloat162 *>(a.out + at * D + rank * share + column) =
        __floats2bfloat162_rn(x * inv, y * inv);
    if (a.lse != nullptr && rank == 0 && column == 0) {
      a.lse[at] = sum != 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
  }
}

template <int D>
cudaError_t launch_few(const ChunkAttentionArgs &a, int cluster, int table_end, cudaStream_t stream) {
  constexpr int kSmem = int(sizeof(FewShared<D>));
  static_assert(kSmem <= 227 * 1024, "the tiles must fit one SM");
  const auto kernel = chunk_attention_few_kernel<D>;
  cudaError_t st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (st == cudaSuccess && cluster > 8) {
    st = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }
  if (st != cudaSuccess) return st;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(a.runs.run_count * a.cfg.num_heads * cluster));
  config.blockDim = dim3(kFewThreads);
  config.dynamicSmemBytes = kSmem;
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, kernel, a, table_end);
}

}  // namespace

int chunk_few_cluster(const ChunkAttentionArgs &a, int sm_count, int table_end) {
  const int group = a.q_heads / a.cfg.num_heads;
  if (int64_t(std::min(a.runs.max_row_count, a.runs.rows)) * group > kFewRows) return 0;
  const int64_t items = int64_t(a.runs.run_count) * a.cfg.num_heads;
  // Clusters lie within a group of SMs, and not all of its SMs fill up: 7 clusters of 16,
  // 15 of 8, 33 of 4 run at once on 148 SMs. One more than that costs a second round.
  int cluster = kFewMaxCluster;
  while (cluster > 1 && items * cluster * 4 > int64_t(sm_count) * 3) cluster /= 2;
  if (cluster < 4) return 0;
  const int64_t most = a.window > 0 ? int64_t(a.window) + a.sinks : table_end;  // keys of a row
  return most <= 512 * int64_t(cluster) ? cluster : 0;
}

cudaError_t chunk_attention_few_bf16(const ChunkAttentionArgs &a, int cluster, int table_end,
                                     cudaStream_t stream) {
  return a.cfg.head_dim == 256 ? launch_few<256>(a, cluster, table_end, stream)
                               : launch_few<512>(a, cluster, table_end, stream);
}

}  // namespace b200kv
