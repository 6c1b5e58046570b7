// Attention of runs of new tokens over the paged cache (B200KvChunkArgs):
//   out[t, h] = sum_p softmax_p(scale q[t, h] . K[p, h / G]) V[p, h / G]
// over the keys p <= t that have a page, with a window only p > t - window or
// p < sinks; G query heads share a KV head.
//
// Work. A tile of queries is 128 rows: 128 / G tokens of a run times the G query
// heads of one KV head (row = token * G + head), so that K and V are read once for
// the whole group and one token of 16 heads fills as many rows as eight tokens of
// two. Keys come in tiles of 64: of the cache at positions that are multiples of 64,
// of the runs' own rows counted from the run's first. An item is a (query tile, KV
// head, part of the output dims); its keys are laid end to end with those of all
// other items, in units of one key tile, and cut evenly: every CTA of the grid (one
// per SM) takes one contiguous piece, whatever the lengths. A CTA that has all of an
// item's keys writes the item's rows; a piece of an item leaves its rows' maximum,
// sum and accumulator in the workspace, and chunk_combine_kernel joins them.
//
// One CTA: eleven warps.
//   warps 0-7  softmax: two groups of four warps, a thread per query row; group g
//              takes the key tiles with number n % 2 == g
//   warps 8, 9 load K and V tiles (TMA boxes that lie inside one page, or 16-byte
//              copies where pages are no multiple of eight tokens); a box costs its
//              warp about 130 clocks and a page-table entry a round trip, so the
//              tensors have a warp each, which looks up 32 boxes at a time and those
//              a batch ahead. The K warp also tells the others what a segment (this
//              CTA's piece of an item) and a key tile are.
//   warp 10    issues the MMAs
// Tensor memory (512 columns): O (128 x 256 fp32), Q (128 x 256 bf16: the A operand
// of Q K^T), and two score buffers of 64 columns. K and V tiles go through two rings
// of 32 KB shared-memory slots (64 keys x 256 dims, 128-byte swizzle); a segment's Q
// comes through two slots of the K ring, ahead of its keys, and is copied to tensor
// memory from there (tcgen05.cp), so the softmax warps never touch it.
// head_dim 256: 3 + 3 slots, and two buffers (16 KB) for the bf16 weights, the A
// operand of P V. A score buffer is free as soon as it has been read, so Q K^T runs
// two tiles ahead of P V: the tensor pipe always has work queued, and a group of
// softmax warps has two tiles' time for one.
// head_dim 512: a tile takes two K slots and one V slot, the upper half of Q lies in
// shared memory, 3 + 2 slots remain; the weights go back into tensor memory over the
// scores they come from (in two halves: P V starts on the first under the second), so
// Q K^T runs one tile ahead. The output dims are two parts computed by different
// items, each with all of Q K^T.
//
// Softmax: the maximum that a row's weights are scaled by is passed from tile to
// tile (through shared memory, from one group to the other) and raised only when a
// tile exceeds it by 2^8, so rescaling O is rare; scores, maxima, sums and O are
// fp32, the weights are rounded to bf16 for P V (by at most 2^-8 of each, which the
// average over keys does not add up), the sum takes them unrounded.
//
// Keys that no row of the tile sees (before the window, behind the last row, pages
// that are not mapped) may hold anything: their scores are replaced, and their V
// rows cleared in shared memory before P V (0 * NaN). A NaN or an infinity in V that some
// rows of the tile see and others do not is left to the results: a row that is not finite,
// although its scores are, is computed again from the keys that it sees (chunk_exact.cuh),
// by the combine. The look at what is written costs about 1 % (in a row of calls the ragged
// runs below 139.8 -> 141.6 us, head_dim 512 295 -> 298).
//
// Every wait is bounded; one that runs out writes B200KV_STATUS_WAIT_TIMEOUT and
// makes the CTA fall through to its exit, which frees the tensor memory.
//
// What bounds it. Long runs: the tensor pipe, then the way of K and V from L2 (64 KB per
// tile and CTA: 45 bytes a clock and SM at the rates below). A tile of head_dim 256 is
// 1024 clocks of MMAs (Q K^T from tensor memory 32 a step, P V 128 a step) and takes 1350
// to 1450; of head_dim 512 1792 (the upper half of Q is read from shared memory, 48 a
// step) and 2500. An item's start and end cost some 10k clocks in which the tensor pipe
// has little to do: draining P V (1.1k), reading O back and writing it (4k; 7k the first
// time, when the code has to be fetched), the first tile's softmax, the masked tiles. Few
// rows: HBM. Measured (16 + 8 heads of 256 unless said), in the first fraction of a second
// and in a row of calls under the power cap: 4096 tokens behind 12288 0.82 and 1.00 ms (1160
// and 960 TFLOP/s); 32 runs of 1 .. 8 tokens over 512 .. 12000 keys 262 and 283 us (6.5 TB/s
// at best); runs of 239 .. 1211 tokens over rings of 1024 116 and 141 us; 64 tokens with a
// window of 2048 and 4 sinks 171 and 188 us; three runs of 406 .. 695 tokens of 16 heads of
// 512 on one KV head 250 and 298 us. Pages of five tokens (a copy of 16 bytes per lane by
// one warp, a tile of 64 keys some 5000 clocks), at best: 453, 204, 212 (725 .. 896 tokens,
// window 2048), 530.
//
// The roles share one instruction cache and much of what was tried is about that: waits
// out of line and rolled MMA and epilogue loops (6000 to 4500 instructions) made the tile
// a quarter faster; four more warps for the epilogue, an epilogue put off until the next
// item's first tile (more registers and code), and for head_dim 512 both groups on every
// tile (448k clocks instead of 430k) did not pay. Nor did, for head_dim 512, two CTAs with
// half of the dims each that send one another their part of the scores: 1024 clocks of
// MMAs a tile instead of 1792 and a third less from L2, but 32 KB of scores a tile and
// CTA between shared memories took 4400 (390 us instead of 250).
#include <algorithm>

#include "chunk_common.cuh"
#include "chunk_exact.cuh"
#include "chunk_maps.cuh"
#include "kernels.cuh"
#include "umma_common.cuh"

namespace b200kv {

namespace {

constexpr int kRows = 128;                    // query rows per tile
constexpr int kKeys = 64;                     // keys per tile
constexpr int kPartDims = 256;                // output dims per item
constexpr int kSlotBytes = kKeys * kPartDims * 2;
// A slot is laid down in groups of eight keys: [key / 8][block of 64 dims][key % 8]
// [64 dims], 128-byte swizzle. The 8 x 64 atoms of the MMA operands then have one
// stride between key groups whatever the page size, and one TMA box brings all the
// groups and blocks that lie in a page.
constexpr int kGroupBytes = 8 * kPartDims * 2;
constexpr int kBlockBytes = 8 * 128;
constexpr int kQBlockBytes = kRows * 128;     // 128 rows x 64 dims
constexpr int kPTileBytes = kRows * kKeys * 2;  // weights of a tile
constexpr int kMaxSlots = 3;                  // of a ring
constexpr int kSoftmaxWarps = 8;
constexpr int kThreads = (kSoftmaxWarps + 3) * 32;
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kTmemQ = 256;
constexpr uint32_t kTmemS = 384;              // + 64 * buffer
constexpr float kRescaleSlack = 8.0f;         // log2 units
// Key tiles and segments whose description is kept. The K warp describes tile n when K
// of tile n - 1 has a slot, which takes Q K^T of tile n - 4 (n - 3 for head_dim 512) to
// be complete and so the softmax of tile n - 6 (n - 5) to have begun.
constexpr int kInfos = 8;
constexpr int kSegments = 8;
constexpr long long kTileWaitClocks = 1ll << 26;
constexpr uint32_t kWaitPolls = 1u << 20;     // tens of milliseconds at least; a tile takes microseconds
// What starting an item costs next to a key tile (loading Q, reading O back: some 10k
// of a tile's 1.4k cycles), and the least a CTA is given, both in key tiles: they
// shape the cut only. Item cost 3, 5, 8 on ragged runs over a ring: 117.2, 116.1,
// 115.9 us; least share 2, 4, 8 for four tokens over a ring of 1024: 15.9, 16.1, 20.1.
constexpr int kItemCost = 8;
constexpr int kMinShare = 4;
constexpr int kNotFinite = 4;  // in a meta word's w

template <int kHeadDim_>
struct ChunkTraits {
  static constexpr int kHeadDim = kHeadDim_;
  static constexpr int kKSlots = kHeadDim / 256;      // slots of one K tile
  static constexpr int kParts = kHeadDim / kPartDims;
  static constexpr int kQHiBytes = (kHeadDim - 256) * kRows * 2;
  static constexpr bool kPShared = kHeadDim == 256;   // the weights in shared memory
  static constexpr int kPBytes = kPShared ? 2 * kPTileBytes : 0;
  static constexpr int kKRing = 3;
  static constexpr int kVRing = kHeadDim == 256 ? 3 : 2;
  static constexpr int kLag = kPShared ? 2 : 1;       // tiles that Q K^T is ahead of P V
  // shared memory: upper half of Q, weights, K ring, V ring
  static constexpr int kPAt = kQHiBytes;
  static constexpr int kKAt = kPAt + kPBytes;
  static constexpr int kVAt = kKAt + kKRing * kSlotBytes;
  static constexpr int kTileBytes = kVAt + kVRing * kSlotBytes;
};

struct ChunkParams {
  __nv_bfloat16 *out;
  float *lse;
  const __nv_bfloat16 *q;
  const __nv_bfloat16 *cache_k;
  const __nv_bfloat16 *cache_v;
  const __nv_bfloat16 *k_rows;
  const __nv_bfloat16 *v_rows;
  Gemma4KvCacheConfig cfg;
  const int32_t *page_table;
  ChunkRuns runs;
  int32_t layer;
  int32_t q_heads;
  int32_t group;
  int32_t tile_tokens;   // 128 / group
  int32_t tiles_per_run; // query tiles of the longest run
  int32_t q_box;         // tokens of a query box
  int32_t q_slots;       // K slots that a segment's Q takes
  int32_t window;
  int32_t sinks;
  int32_t table_end;     // first position past a linear cache's table
  int32_t box;           // tokens per TMA box; 0: rows are copied one by one
  FastDiv page_div;      // by page_size
  FastDiv slot_div;      // by max_pages_per_seq
  FastDiv run_div;       // by tiles_per_run
  FastDiv group_div;     // by group
  float scale_log2;
  int4 *meta;            // per CTA: see PartialMeta
  float *partials;       // [cta][2] x (acc [rows_cap][256], m [rows_cap], l [rows_cap])
  int32_t rows_cap;
  int32_t *status;
};

// The key tiles of a query tile, in this order: of the cache [0, ca) (sinks) and
// [cb0, cb1), of the run's own rows [0, oa) (sinks) and [ob0, ob1).
struct KeyTiles {
  int ca, cb0, cb1, oa, ob0, ob1;
  __device__ __forceinline__ int count() const { return ca + (cb1 - cb0) + oa + (ob1 - ob0); }
};

__device__ __forceinline__ KeyTiles key_tiles(const ChunkParams &p, int first, int t0, int t1) {
  KeyTiles k = {};
  const int lo = p.window > 0 ? max(0, t0 - p.window + 1) : 0;
  const int sink_end = min(p.sinks, lo);
  const int c_lim = min(p.k_rows != nullptr ? min(first, t1 + 1) : t1 + 1, p.table_end);
  k.ca = div_up(min(sink_end, c_lim), kKeys);
  if (c_lim > lo) {
    k.cb0 = lo / kKeys;
    k.cb1 = div_up(c_lim, kKeys);
    k.ca = min(k.ca, k.cb0);
  }
  if (p.k_rows != nullptr) {
    k.ob0 = (max(lo, first) - first) / kKeys;
    k.ob1 = (t1 - first) / kKeys + 1;
    k.oa = sink_end > first ? min(div_up(sink_end - first, kKeys), k.ob0) : 0;
  } else if (k.ca == 0 && k.cb1 == 0) {
    k.cb1 = 1;  // no key at all: a tile that nobody sees gives the rows their zeros
  }
  return k;
}

// A piece of an item's key tiles: what one CTA does between loading Q and writing rows.
struct Segment {
  ChunkRun run;
  KeyTiles keys;
  int hp;            // part * KV heads + KV head
  int token0;        // first token of the tile within the run
  int rows;          // query rows
  int t0, t1;        // positions of the first and last row
  int begin, end;    // key tiles [begin, end) of the item
  int total;
};

// Walks the items of a CTA's share (the two loader warps do, each by itself). The
// lanes hold 32 runs at a time.
struct Walk {
  int left;
  int hp, run, tile, offset;

  __device__ __forceinline__ bool next(const ChunkParams &p, Segment &s, ChunkRun &mine, int &first_run) {
    while (left > 0) {
      if (run < first_run || run >= first_run + 32) {
        first_run = run & ~31;
        mine = chunk_run(p.runs, first_run + (int(threadIdx.x) & 31), p.cfg.batch_size);
      }
      const int from = run - first_run;
      s.run.count = __shfl_sync(0xffffffffu, mine.count, from);
      s.run.first = __shfl_sync(0xffffffffu, mine.first, from);
      s.run.start = __shfl_sync(0xffffffffu, mine.start, from);
      s.run.batch = __shfl_sync(0xffffffffu, mine.batch, from);
      s.token0 = tile * p.tile_tokens;
      if (s.token0 >= s.run.count) {  // the run has no such tile
        tile = 0;
        offset = 0;
        if (++run == p.runs.run_count) {
          run = 0;
          ++hp;
        }
        continue;
      }
      const int tokens = min(p.tile_tokens, s.run.count - s.token0);
      s.t0 = s.run.first + s.token0;
      s.t1 = s.t0 + tokens - 1;
      s.rows = tokens * p.group;
      s.keys = key_tiles(p, s.run.first, s.t0, s.t1);
      s.total = s.keys.count();
      s.hp = hp;
      const int cost = s.total + kItemCost;
      const int take = min(cost - offset, left);
      s.begin = max(0, offset - kItemCost);
      s.end = max(0, offset + take - kItemCost);
      left -= take;
      offset += take;
      if (offset == cost) {
        offset = 0;
        ++tile;
      }
      if (s.begin < s.end) return true;
    }
    return false;
  }
};

// What the softmax needs to know about a key tile, left by the loader.
struct TileInfo {
  unsigned long long live;  // keys that some row of the query tile sees
  int base;                 // position of the tile's first key
  int edge;                 // some row does not see all 64
};

// What the softmax and the MMA warp need to know about a segment.
struct SegmentInfo {
  int tiles;   // key tiles; 0: there is no further segment
  int rows;    // query rows
  int t0;      // position of the first
  int row0;    // its token's row in the packed tensors
  int hp;      // part * KV heads + KV head
  int piece;   // 0, 1: which of the CTA's partial results; -1: the item is whole
  int pad[2];
};

struct SmallState {
  uint64_t k_full[kMaxSlots]; // the slot's tile (or half of Q) has landed
  uint64_t k_done[kMaxSlots]; // the MMAs (or copies) that read the slot are complete
  uint64_t v_full[kMaxSlots];
  uint64_t v_done[kMaxSlots];
  uint64_t s_full[2];         // scores of the tile in S[b] complete
  uint64_t p_full[2][2];      // half of its weights written (and O rescaled where needed)
  uint64_t m_full[2][4];      // row_ref[b] of 32 rows written
  uint64_t l_full[2][4];      // row_sum of 32 rows written by the group
  uint64_t v_raw;             // a V tile that still has rows to be cleared has landed
  uint64_t s_free[2];         // kPShared: the scores in S[b] have been read
  uint64_t q_hi_full;         // head_dim 512: the upper half of the segment's Q has landed
  uint64_t q_free;            // the segment's last Q K^T is complete
  uint64_t o_full;            // its last P V is complete
  uint64_t o_free;            // its O has been read back
  uint64_t drained;           // giving up: the MMAs issued so far are complete
  uint64_t seg_full[kSegments];
  TileInfo info[kInfos];
  SegmentInfo segment[kSegments];
  float row_ref[2][kRows];
  float row_sum[2][kRows];
  int scan[kThreads / 32];
  Walk start;
  int4 meta;                  // of this CTA, for the combine
  uint32_t tmem_base;
  int abort;
  int not_finite;             // a row that this CTA has written is not
};

template <class T>
constexpr int kChunkSmemBytes = T::kTileBytes + int(sizeof(SmallState));

// 64 fp32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&r)[64]) {
  uint32_t u[64];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t *v = u + 32 * h;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
          "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
          "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
          "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
          "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr + 32u * uint32_t(h))
        : "memory");
  }
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    asm volatile("" : "+r"(u[i]));  // not used before the wait
    r[i] = __uint_as_float(u[i]);
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  return fmaxf(a, fmaxf(b, c));
}
using f32x2 = unsigned long long;  // two fp32, each operation with the scalar one's rounding
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2_rn(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2_rn(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// bits [0, n) of a 64-bit word, n clamped to 0 .. 64
__device__ __forceinline__ unsigned long long low_bits(int n) {
  return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1ull);
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// 128 rows x 32 bytes of a swizzled block to eight columns of tensor memory.
__device__ __forceinline__ void tmem_copy_warp(uint32_t d_tmem, uint32_t lo, uint32_t hi, bool leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b64 d;\n\tsetp.ne.b32 q, %3, 0;\n\tmov.b64 d, {%1, %2};\n\t"
      "@q tcgen05.cp.cta_group::1.128x256b [%0], d;\n\t}\n" ::"r"(d_tmem),
      "r"(lo), "r"(hi), "r"(uint32_t(leader))
      : "memory");
}
// One box of query rows x 64 dims: box tokens x the query heads of one KV head.
__device__ __forceinline__ void tma_load_block(uint32_t dst, const CUtensorMap *map, int x, int head,
                                               int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(bar)
      : "memory");
}

__device__ __noinline__ bool wait_slowly(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  for (uint32_t left = kWaitPolls; !mbar_try_wait(bar, parity); --left) {
    if (left == 0 || ((left & 31u) == 0 && *abort_flag != 0)) return false;
  }
  return true;
}

template <class T>
__global__ __launch_bounds__(kThreads, 1) void chunk_attention_kernel(
    const __grid_constant__ ChunkParams p, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k_rows,
    const __grid_constant__ CUtensorMap map_v_rows, const __grid_constant__ CUtensorMap map_q) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  SmallState &small = *reinterpret_cast<SmallState *>(smem_raw + T::kTileBytes);
  const uint32_t s_q_hi = smem_u32(smem_raw);
  const uint32_t s_p = s_q_hi + T::kPAt;
  const int tid = int(threadIdx.x);
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int heads = p.cfg.num_heads;
  if ((s_q_hi & 1023u) != 0) {  // the swizzle's atoms; the window starts on such a boundary
    if (tid == 0) {
      set_status(p.status, B200KV_STATUS_WAIT_TIMEOUT);
      pdl_wait_for_predecessor();
      p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    return;
  }

  const uint32_t bar_k_full = smem_u32(&small.k_full[0]);  // + 8 slot
  const uint32_t bar_k_done = smem_u32(&small.k_done[0]);  // + 8 slot
  const uint32_t bar_v_full = smem_u32(&small.v_full[0]);  // + 8 slot
  const uint32_t bar_v_done = smem_u32(&small.v_done[0]);  // + 8 slot
  const uint32_t bar_s_full = smem_u32(&small.s_full[0]);  // + 8 b
  const uint32_t bar_p_full = smem_u32(&small.p_full[0][0]);  // + 16 b + 8 half
  const uint32_t bar_m_full = smem_u32(&small.m_full[0][0]);  // + 32 b + 8 warp quarter
  const uint32_t bar_l_full = smem_u32(&small.l_full[0][0]);  // + 32 group + 8 warp quarter
  const uint32_t bar_s_free = smem_u32(&small.s_free[0]);  // + 8 b
  const uint32_t bar_q_hi_full = smem_u32(&small.q_hi_full);
  const uint32_t bar_v_raw = smem_u32(&small.v_raw);
  const uint32_t bar_q_free = smem_u32(&small.q_free);
  const uint32_t bar_o_full = smem_u32(&small.o_full);
  const uint32_t bar_o_free = smem_u32(&small.o_free);
  const uint32_t bar_drained = smem_u32(&small.drained);
  const uint32_t bar_seg_full = smem_u32(&small.seg_full[0]);  // + 8 (segment % kSegments)
  if (tid == 0) {
    for (int i = 0; i < kMaxSlots; ++i) {
      mbar_init(bar_k_full + 8u * i, 1);
      mbar_init(bar_k_done + 8u * i, 1);
      mbar_init(bar_v_full + 8u * i, 1);
      mbar_init(bar_v_done + 8u * i, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_s_full + 8u * b, 1);
      mbar_init(bar_p_full + 16u * b, 4);
      mbar_init(bar_p_full + 16u * b + 8u, 4);
      for (int w = 0; w < 4; ++w) {
        mbar_init(bar_m_full + 32u * b + 8u * w, 1);
        mbar_init(bar_l_full + 32u * b + 8u * w, 1);
      }
    }
    mbar_init(bar_s_free, 4);
    mbar_init(bar_s_free + 8u, 4);
    mbar_init(bar_q_hi_full, 1);
    mbar_init(bar_v_raw, 1);
    mbar_init(bar_q_free, 1);
    mbar_init(bar_o_full, 1);
    mbar_init(bar_o_free, kSoftmaxWarps);
    mbar_init(bar_drained, 1);
    for (int i = 0; i < kSegments; ++i) mbar_init(bar_seg_full + 8u * i, 1);
    small.abort = 0;
    small.not_finite = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&small.tmem_base)),
                 "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // everything up to here is this kernel's own; the runs, the rows and the cache
  // may be what the kernel before it writes
  pdl_wait_for_predecessor();
  // the combine's blocks may take their places; they wait for this kernel's end
  pdl_release_successor();

  // ---- this CTA's share: the costs of all (run, query tile) pairs, summed
  const int pairs = p.runs.run_count * p.tiles_per_run;
  const int per_thread = div_up(pairs, kThreads);
  auto pair_cost = [&](int pair) -> int {
    const int of_run = p.run_div.quotient(pair);
    const ChunkRun run = chunk_run(p.runs, of_run, p.cfg.batch_size);
    const int token0 = (pair - of_run * p.tiles_per_run) * p.tile_tokens;
    if (token0 >= run.count) return 0;
    const int t0 = run.first + token0;
    const int t1 = t0 + min(p.tile_tokens, run.count - token0) - 1;
    return key_tiles(p, run.first, t0, t1).count() + kItemCost;
  };
  int mine = 0;
  for (int i = 0; i < per_thread; ++i) {
    const int pair = tid * per_thread + i;
    if (pair < pairs) mine += pair_cost(pair);
  }
  int before = mine;  // inclusive scan over the warp
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += up;
  }
  if (lane == 31) small.scan[warp] = before;
  __syncthreads();
  int warps_before = 0, per_head = 0;
#pragma unroll 1
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) warps_before += small.scan[w];
    per_head += small.scan[w];
  }
  before += warps_before - mine;  // costs before this thread's first pair
  // an even cut (the host has seen to it that all of this fits 32 bits)
  const uint32_t total = uint32_t(per_head) * uint32_t(heads * T::kParts);
  const uint32_t ctas = max(1u, min(gridDim.x, total / kMinShare));
  const uint32_t share = total / ctas;
  const uint32_t extra = total - share * ctas;  // the first CTAs have one more
  const uint32_t cta = blockIdx.x;
  const int c0 = cta < ctas ? int(share * cta + min(cta, extra)) : 0;
  const int c1 = cta < ctas ? c0 + int(share + (cta < extra ? 1 : 0)) : 0;
  if (tid == 0) {
    small.start.left = 0;
    small.start.hp = small.start.run = small.start.tile = small.start.offset = 0;
  }
  __syncthreads();
  if (c1 > c0) {
    const int hp = int(uint32_t(c0) / uint32_t(per_head));
    int rem = c0 - hp * per_head;
    if (rem >= before && rem < before + mine) {
      rem -= before;
      int pair = tid * per_thread;
      for (int cost; rem >= (cost = pair_cost(pair)); ++pair) rem -= cost;
      small.start.left = c1 - c0;
      small.start.hp = hp;
      small.start.run = p.run_div.quotient(pair);
      small.start.tile = pair - small.start.run * p.tiles_per_run;
      small.start.offset = rem;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = small.tmem_base;
  volatile int *abort_flag = &small.abort;
  Walk walk = small.start;

  // Bounded wait that also gives up when another role has; false = give up (the role
  // says so at the end). What is not ready at once is waited for out of line: there are
  // dozens of waits, and the roles share one instruction cache.
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    return mbar_try_wait(bar, parity) || wait_slowly(bar, parity, &small.abort);
  };
  // The same in line, for where a call would have to save a tile's scores.
  auto wait_here = [&](uint32_t bar, uint32_t parity) -> bool {
    for (uint32_t left = kWaitPolls; !mbar_try_wait(bar, parity); --left) {
      if (left == 0) return false;
    }
    return true;
  };
  bool failed = false;
  // A ring's slots are filled and freed in order: a role keeps the slot of its next
  // fill and the parity of that slot's use. V of key tile n is fill n of its ring.
  struct Cursor {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void advance(uint32_t slots) {
      if (++slot == slots) {
        slot = 0;
        phase ^= 1u;
      }
    }
  };
  auto v_slot = [](int tile) { return uint32_t(tile % T::kVRing); };
  auto v_parity = [](int tile) { return uint32_t(tile / T::kVRing) & 1u; };

  if (warp == kSoftmaxWarps || warp == kSoftmaxWarps + 1) {
    // ------------------------------------------------------------ loaders of K and V
    const bool is_v = warp == kSoftmaxWarps + 1;
    const __nv_bfloat16 *cache = is_v ? p.cache_v : p.cache_k;
    const __nv_bfloat16 *rows = is_v ? p.v_rows : p.k_rows;
    const CUtensorMap *map = is_v ? &map_v : &map_k;
    const CUtensorMap *map_rows = is_v ? &map_v_rows : &map_k_rows;
    const int box_shift = p.box > 0 ? 31 - __clz(p.box) : 0;
    const int tile_boxes = p.box > 0 ? kKeys >> box_shift : 0;  // boxes of a key tile
    const int batch_tiles = p.box > 0 ? 32 / tile_boxes : 1;    // key tiles of a look-up
    const int page_groups = p.cfg.page_size / 8;
    const int layer_group = p.layer * p.cfg.num_pages * page_groups;
    const uint32_t ring = s_q_hi + (is_v ? T::kVAt : T::kKAt);
    const uint32_t ring_slots = is_v ? T::kVRing : T::kKRing;
    const uint32_t bar_full = is_v ? bar_v_full : bar_k_full;
    const uint32_t bar_done = is_v ? bar_v_done : bar_k_done;
    Cursor at;
    uint32_t raw_phase = 0;  // of v_raw
    int n = 0, segments = 0;
    int4 meta = make_int4(-1, 0, 0, 0);
    ChunkRun mine;
    int first_run = -32;
    Segment s;
    bool ok = true;
    auto tell_segment = [&](int tiles) {
      if (is_v) return;
      if (lane == 0) {
        SegmentInfo &info = small.segment[segments % kSegments];
        info.tiles = tiles;
        info.rows = s.rows;
        info.t0 = s.t0;
        info.row0 = s.run.start + s.token0;
        info.hp = s.hp;
        info.piece = s.begin > 0 ? 0 : (s.end < s.total ? 1 : -1);
        mbar_arrive(bar_seg_full + 8u * uint32_t(segments % kSegments));
      }
      ++segments;
    };
    // box == 0: the slot whose copies are on their way. It is said to be full when the next
    // slot's have been asked for, or at the segment's end.
    uint32_t copied = 0;
    auto copies_landed = [&](bool all) {
      if (copied == 0) return;
      if (all) {
        asm volatile("cp.async.wait_all;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(copied);
      copied = 0;
    };
    while (ok && walk.next(p, s, mine, first_run)) {
      const int head = s.hp % heads;
      const int part = s.hp / heads;
      tell_segment(s.end - s.begin);
      if (!is_v) {
        if (s.begin > 0) meta.w = s.end == s.total ? 1 : 2;
        if (s.begin == 0 && s.end < s.total) {
          meta.x = s.hp;
          meta.y = s.run.start + s.token0;
          meta.z = s.rows;
        }
        // Q: 64-dim blocks, two to a slot, or all four where the box has at most 64 rows
        // (rows behind the segment's are other runs', or zeros, or for a box of more than 64 what
        // the slot held: nobody looks at what comes of them)
        const int token = s.run.start + s.token0;
        const uint32_t block_bytes = uint32_t(p.q_box * p.group) * 128u;
        for (int h = 0; h < p.q_slots && ok; ++h) {
          ok = __all_sync(0xffffffffu, wait(bar_k_done + 8u * at.slot, at.phase ^ 1u));
          if (!ok) break;
          const uint32_t blocks = 4u / uint32_t(p.q_slots);
          if (p.q_slots == 1) {
            // Rows behind the box: zeros. The products' time is that of 128 rows however few
            // are queries, but zeros cost them little power, and power is what sets the clock
            // in a row of calls: with these and zero weights 1 .. 8 tokens of 32 runs run at
            // 1225 MHz instead of 1000, 289 -> 279 us, one token of 64 runs 193 -> 184.
            uint8_t *behind = smem_raw + T::kKAt + at.slot * kSlotBytes + lane * 16;
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
#pragma unroll 1
              for (int c = p.q_box * p.group * 128; c < kSlotBytes / 4 - lane * 16; c += 512) {
                *reinterpret_cast<uint4 *>(behind + b * (kSlotBytes / 4) + c) = make_uint4(0u, 0u, 0u, 0u);
              }
            }
            fence_proxy_async_shared();
          }
          if (lane == 0) mbar_arrive_expect_tx(bar_k_full + 8u * at.slot, blocks * block_bytes);
          __syncwarp();
          if (uint32_t(lane) < blocks) {
            tma_load_block(ring + at.slot * kSlotBytes + uint32_t(lane) * (kSlotBytes / blocks), &map_q,
                           (int(blocks) * h + lane) * 64, head * p.group, token,
                           bar_k_full + 8u * at.slot);
          }
          at.advance(ring_slots);
        }
        if constexpr (T::kKSlots == 2) {
          // its place is free when the last segment's rows are out (they go through it)
          if (ok && segments > 1) {
            ok = __all_sync(0xffffffffu, wait(bar_o_free, uint32_t(segments - 2) & 1u));
          }
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(bar_q_hi_full, 4u * block_bytes);
            for (int b = 0; b < 4; ++b) {
              tma_load_block(s_q_hi + uint32_t(b) * kQBlockBytes, &map_q, 256 + b * 64,
                             head * p.group, token, bar_q_hi_full);
            }
          }
          __syncwarp();
        }
      }
      int j = s.begin;
      while (j < s.end && ok) {
        // the contiguous key tiles from j on
        int k = j, stop;
        bool own = false;
        if (k < s.keys.ca) {
          stop = s.keys.ca;
        } else if ((k -= s.keys.ca) < s.keys.cb1 - s.keys.cb0) {
          k += s.keys.cb0;
          stop = s.keys.cb1;
        } else {
          k -= s.keys.cb1 - s.keys.cb0;
          own = true;
          stop = s.keys.oa;
          if (k >= s.keys.oa) {
            k += s.keys.ob0 - s.keys.oa;
            stop = s.keys.ob1;
          }
        }
        const int count = min(stop - k, s.end - j);
        j += count;
        const int origin = own ? s.run.first : 0;
        const int limit = own ? s.t1 + 1
                              : min(p.k_rows != nullptr ? min(s.run.first, s.t1 + 1) : s.t1 + 1, p.table_end);
        // keys of the tile that some row sees, pages aside
        auto seen = [&](int base) -> unsigned long long {
          unsigned long long live = low_bits(limit - base);
          if (p.window > 0) {
            live &= ~low_bits(s.t0 - p.window + 1 - base) | low_bits(p.sinks - base);
          }
          return live;
        };
        // box > 0: token group of box `lane` of the 32 from position `at` on, -1
        // without a page; asked for raw, checked when it is used
        int raw = -1, raw_offset = 0;
        auto ask = [&](uint32_t at) {  // (32 boxes on, this may be past 2^31)
          raw = -1;
          const int position = int(min(at + (uint32_t(lane) << box_shift), uint32_t(limit)));
          if (position >= limit) return;
          int logical = p.page_div.quotient(position);
          raw_offset = (position - logical * p.cfg.page_size) >> 3;
          const int slots = p.cfg.max_pages_per_seq;
          if (p.cfg.window_size > 0) logical -= p.slot_div.quotient(logical) * slots;
          raw = __ldg(p.page_table + int64_t(s.run.batch) * slots + logical);
        };
        int group_of_box = -1;
        int in_batch = batch_tiles;  // the current batch is used up
        if (!own && p.box > 0) ask(uint32_t(k * kKeys));
        for (int i = 0; i < count; ++i, ++n) {
          const int base = origin + (k + i) * kKeys;
          unsigned long long live = ~0ull;
          if (base + kKeys > limit || (p.window > 0 && base <= s.t0 - p.window)) live = seen(base);
          int group = -1;  // of this lane's box of the tile
          if (!own && p.box > 0) {
            if (in_batch == batch_tiles) {
              group_of_box = raw >= 0 && raw < p.cfg.num_pages
                                 ? layer_group + raw * page_groups + raw_offset
                                 : -1;
              in_batch = 0;
              ask(uint32_t(base) + 32u * uint32_t(p.box));
            }
            group = __shfl_sync(0xffffffffu, group_of_box, (in_batch * tile_boxes + lane) & 31);
            ++in_batch;
            if (lane >= tile_boxes ||
                ((live >> (lane << box_shift)) & (p.box == 64 ? ~0ull : (1ull << p.box) - 1ull)) == 0) {
              group = -1;
            }
            const uint32_t boxes = __ballot_sync(0xffffffffu, group >= 0);
            if (boxes != (tile_boxes == 32 ? ~0u : (1u << tile_boxes) - 1u)) {
              unsigned long long mapped = 0;
              for (int b = 0; b < tile_boxes; ++b) {
                if ((boxes >> b) & 1u) mapped |= low_bits(p.box) << (b << box_shift);
              }
              live &= mapped;
            }
          }
          int page[2], offset[2];  // box == 0: of rows lane and lane + 32
          if (p.box == 0 && !own) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              page[r] = -1;
              const int at = lane + 32 * r;
              if (((live >> at) & 1ull) != 0) {
                int logical = p.page_div.quotient(base + at);
                offset[r] = base + at - logical * p.cfg.page_size;
                const int slots = p.cfg.max_pages_per_seq;
                if (p.cfg.window_size > 0) logical -= p.slot_div.quotient(logical) * slots;
                page[r] = __ldg(p.page_table + int64_t(s.run.batch) * slots + logical);
                if (page[r] >= p.cfg.num_pages) page[r] = -1;
              }
            }
            const uint32_t lo = __ballot_sync(0xffffffffu, page[0] >= 0);
            const uint32_t hi = __ballot_sync(0xffffffffu, page[1] >= 0);
            live &= (uint64_t(hi) << 32) | lo;
          }
#pragma unroll
          for (int f = 0; f < T::kKSlots; ++f) {
            if (is_v && f > 0) break;
            const int block0 = is_v ? part * 4 : f * 4;
            // the slot's last reader is done (a slot's first use waits for nothing)
            ok = __all_sync(0xffffffffu, wait(bar_done + 8u * at.slot, at.phase ^ 1u));
            if (!ok) break;
            if (!is_v && f == 0 && lane == 0) {
              const bool edge = live != ~0ull || base + kKeys - 1 > s.t0 ||
                                (p.window > 0 && base <= s.t1 - p.window && base + kKeys > p.sinks);
              small.info[n % kInfos] = {live, base, edge ? 1 : 0};
            }
            const bool clear = is_v && live != ~0ull;
            const uint32_t bar = clear && p.box > 0 ? bar_v_raw : bar_full + 8u * at.slot;
            const uint32_t dst = ring + at.slot * kSlotBytes;
            if (p.box == 0) {
              int64_t row_at[2];  // element offset of rows lane, lane + 32
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                row_at[r] = -1;
                const int at = lane + 32 * r;
                if (((live >> at) & 1ull) == 0) continue;
                row_at[r] = own ? ((int64_t(s.run.start) + (k + i) * kKeys + at) * heads + head) * T::kHeadDim
                                : cache_offset(p.cfg, p.layer, page[r], offset[r], head, 0);
              }
              const __nv_bfloat16 *from = own ? rows : cache;
              // eight lanes to 128 bytes of a row, four rows at a time, block by block
#pragma unroll 4
              for (int r4 = 0; r4 < kKeys; r4 += 4) {
                const int r = r4 + (lane >> 3);
                const int64_t at = __shfl_sync(0xffffffffu, row_at[r4 >> 5], r & 31);
                if (at >= 0) {
                  const __nv_bfloat16 *src = from + at + block0 * 64 + (lane & 7) * 8;
                  const uint32_t to = dst + uint32_t(r >> 3) * kGroupBytes + uint32_t(r & 7) * 128u +
                                      ((uint32_t(lane & 7) ^ uint32_t(r & 7)) << 4);
#pragma unroll
                  for (int b = 0; b < kPartDims / 64; ++b) cp_async16(to + uint32_t(b) * kBlockBytes, src + b * 64);
                }
              }
              asm volatile("cp.async.commit_group;" ::: "memory");
            } else if (own) {
              if (lane == 0) mbar_arrive_expect_tx(bar, kSlotBytes);
              __syncwarp();
              if (lane < kKeys / 8) {
                tma_load_rows_box(dst + uint32_t(lane) * kGroupBytes, map_rows, block0,
                                  s.run.start + (k + i) * kKeys + lane * 8, head, bar);
              }
            } else {
              const uint32_t boxes = __ballot_sync(0xffffffffu, group >= 0);
              if (lane == 0) {
                mbar_arrive_expect_tx(bar, uint32_t(__popc(boxes) << box_shift) * (kPartDims * 2));
              }
              __syncwarp();
              if (group >= 0) {
                tma_load_page_box(dst + (uint32_t(lane << box_shift) >> 3) * kGroupBytes, map, block0, group,
                                  head, bar);
              }
            }
            if (clear) {
              if (p.box > 0) {
                ok = __all_sync(0xffffffffu, wait(bar_v_raw, raw_phase));
                if (!ok) {
                  mbar_wait_bounded(bar_v_raw, raw_phase, kTileWaitClocks);
                  break;
                }
                raw_phase ^= 1u;
              }
              uint8_t *row0 = smem_raw + T::kVAt + at.slot * kSlotBytes + (lane >> 3) * kBlockBytes +
                              (lane & 7) * 16;
#pragma unroll 1
              for (int g = 0; g < 8; ++g) {  // groups of eight rows
                const uint32_t alive = uint32_t(live >> (8 * g));
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                  if (((alive >> r) & 1u) == 0) {
                    *reinterpret_cast<uint4 *>(row0 + g * kGroupBytes + r * 128) = make_uint4(0, 0, 0, 0);
                  }
                }
              }
              if (p.box > 0) {
                fence_proxy_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_v_full + 8u * at.slot);
              }
            }
            if (p.box == 0) {
              copies_landed(false);
              copied = bar_full + 8u * at.slot;
            }
            at.advance(ring_slots);
          }
          if (!ok) break;
        }
      }
      copies_landed(true);
    }
    if (ok) tell_segment(0);
    failed = !ok;
    if (!is_v && lane == 0) small.meta = meta;
    if (!ok || *abort_flag != 0) {
      // nobody may be waiting for the last loads any more: see them land before the
      // CTA gives its shared memory back. The slots before the cursor were filled in
      // its phase, those behind it in the phase before (a slot that never was passes:
      // parity 1 of a fresh barrier counts as complete).
      for (uint32_t i = 0; i < ring_slots; ++i) {
        mbar_wait_bounded(bar_full + 8u * i, i < at.slot ? at.phase : at.phase ^ 1u, kTileWaitClocks);
      }
      if (T::kKSlots == 2 && !is_v && segments > 0) {
        mbar_wait_bounded(bar_q_hi_full, uint32_t(segments - 1) & 1u, kTileWaitClocks);
      }
    }
  } else if (warp == kSoftmaxWarps + 2) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t kIdescQK = umma_idesc(kKeys, false);
    constexpr uint32_t kIdescPV = umma_idesc(kPartDims, true);
    // descriptor words of a slot's tile: K (K-major; the leading stride is not used)
    // and V (MN-major), and of the upper half of Q
    constexpr uint32_t kLoK = 1u << 16;
    constexpr uint32_t kLoV = uint32_t(kBlockBytes >> 4) << 16;
    constexpr uint32_t kHiSlot = uint32_t(kGroupBytes >> 4) | (1u << 14) | (2u << 29);
    constexpr uint32_t kHiQ = 64u | (1u << 14) | (2u << 29);
    const bool leader = elect_one();
    auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, wait(bar, parity));
    };
    Cursor k_at, v_at;  // K of the next tile to score, V of the next to add
    uint32_t v_last_slot = 0, v_last_phase = 0;  // V of the last tile added
    int n = 0;          // tiles whose Q K^T has been issued
    int added = 0;      // tiles whose P V has been issued
    int segments = 0;
    bool ok = true;
    auto s_free_parity = [&]() { return uint32_t((n - 2) >> 1) & 1u; };
    auto p_bar = [&](int half) { return bar_p_full + 16u * (uint32_t(added) & 1u) + 8u * uint32_t(half); };
    auto p_parity = [&]() { return uint32_t(added >> 1) & 1u; };
    // S[n & 1] = Q K^T of tile n: 16 steps of 16 dims per K slot, four to a block
    auto issue_qk = [&](bool waited, bool last) -> bool {
      const uint32_t d = tmem + kTmemS + uint32_t(n & 1) * kKeys;
#pragma unroll
      for (int f = 0; f < T::kKSlots; ++f) {
        if (!(waited && f == 0) && !warp_wait(bar_k_full + 8u * k_at.slot, k_at.phase)) return false;
        // S[n & 1] held the weights of tile n - 2: asked for behind K, whose wait runs
        // under that product
        if (!T::kPShared && f == 0 && n >= 2 && !warp_wait(bar_v_done + 8u * v_last_slot, v_last_phase)) {
          return false;
        }
        tc_fence_after();
        const uint32_t k = ((s_q_hi + T::kKAt + k_at.slot * kSlotBytes) >> 4) | kLoK;
        const uint32_t q_hi = (s_q_hi >> 4) | kLoK;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const uint32_t at = uint32_t(i >> 2) * (kBlockBytes >> 4) + uint32_t(i & 3) * 2u;
          if (f == 0) {
            umma_bf16_a_tmem_warp(d, tmem + kTmemQ + 8u * uint32_t(i), k + at, kHiSlot, kIdescQK,
                                  i > 0, leader);
          } else {
            umma_bf16_warp(d, q_hi + uint32_t(i >> 2) * (kQBlockBytes >> 4) + uint32_t(i & 3) * 2u,
                           kHiQ, k + at, kHiSlot, kIdescQK, true, leader);
          }
        }
        umma_commit_warp(bar_k_done + 8u * k_at.slot, leader);
        k_at.advance(T::kKRing);
      }
      umma_commit_warp(bar_s_full + 8u * uint32_t(n & 1), leader);
      if (last) umma_commit_warp(bar_q_free, leader);
      ++n;
      return true;
    };
    // O (+)= P V of tile `added`: four steps of 16 keys
    auto issue_pv = [&](bool waited, bool accumulate) -> bool {
      const uint32_t b = uint32_t(added) & 1u;
      if (!waited && !warp_wait(bar_v_full + 8u * v_at.slot, v_at.phase)) return false;
      const uint32_t v = ((s_q_hi + T::kVAt + v_at.slot * kSlotBytes) >> 4) | kLoV;
#pragma unroll
      for (int i = 0; i < kKeys / 16; ++i) {
        if (i == 0 || (i == 2 && !T::kPShared)) {
          if (!waited && !warp_wait(p_bar(i / 2), p_parity())) return false;
          tc_fence_after();
        }
        const uint32_t vi = v + uint32_t(i) * (2u * kGroupBytes >> 4);
        if constexpr (T::kPShared) {
          umma_bf16_warp(tmem, ((s_p + b * kPTileBytes) >> 4 | kLoK) + uint32_t(i) * 2u, kHiQ, vi,
                         kHiSlot, kIdescPV, accumulate || i > 0, leader);
        } else {
          umma_bf16_a_tmem_warp(tmem, tmem + kTmemS + b * kKeys + 8u * uint32_t(i), vi, kHiSlot,
                                kIdescPV, accumulate || i > 0, leader);
        }
      }
      umma_commit_warp(bar_v_done + 8u * v_at.slot, leader);
      v_last_slot = v_at.slot;
      v_last_phase = v_at.phase;
      v_at.advance(T::kVRing);
      ++added;
      return true;
    };
    for (; ok; ++segments) {
      ok = warp_wait(bar_seg_full + 8u * uint32_t(segments % kSegments),
                     uint32_t(segments / kSegments) & 1u);
      if (!ok) break;
      const int tiles = small.segment[segments % kSegments].tiles;
      if (tiles == 0) break;
      const int first = n;
      // Q into tensor memory, when the last segment's Q K^T no longer reads what is there
      if (segments > 0) ok = warp_wait(bar_q_free, uint32_t(segments - 1) & 1u);
      for (int h = 0; h < p.q_slots && ok; ++h) {
        ok = warp_wait(bar_k_full + 8u * k_at.slot, k_at.phase);
        if (!ok) break;
        tc_fence_after();
        // (with one slot a copy's 128 rows reach into what lies behind the block's 64:
        // rows without a query)
        const int blocks = 4 / p.q_slots;
        const uint32_t q = ((s_q_hi + T::kKAt + k_at.slot * kSlotBytes) >> 4) | kLoK;
        for (int i = 0; i < 4 * blocks; ++i) {
          tmem_copy_warp(tmem + kTmemQ + 8u * uint32_t(4 * blocks * h + i),
                         q + uint32_t(i >> 2) * uint32_t((kSlotBytes >> 4) / blocks) + uint32_t(i & 3) * 2u,
                         kHiQ, leader);
        }
        umma_commit_warp(bar_k_done + 8u * k_at.slot, leader);
        k_at.advance(T::kKRing);
      }
      if (T::kKSlots == 2) ok = ok && warp_wait(bar_q_hi_full, uint32_t(segments & 1));
      // one step beyond the segment's tiles per tile that P V lags behind
      for (int j = 0; j < tiles + T::kLag && ok; ++j) {
        bool ready = false;
        if (T::kPShared && j < tiles && j >= T::kLag) {
          // What both products wait for, asked for at once: a wait costs its latency
          // even where nothing is waited for, and the tensor pipe has only what is
          // queued to run under it.
          ready = mbar_try_wait(bar_s_free + 8u * uint32_t(n & 1), s_free_parity()) &
                  mbar_try_wait(bar_k_full + 8u * k_at.slot, k_at.phase) &
                  mbar_try_wait(bar_v_full + 8u * v_at.slot, v_at.phase) &
                  mbar_try_wait(p_bar(0), p_parity());
          ready = __all_sync(0xffffffffu, ready);
        }
        if (j < tiles) {
          // S[n & 1] held the scores of tile n - 2
          if (T::kPShared && n >= 2 && !ready) {
            ok = warp_wait(bar_s_free + 8u * uint32_t(n & 1), s_free_parity());
          }
          ok = ok && issue_qk(ready, j + 1 == tiles);
          if (!ok) break;
        }
        if (j >= T::kLag) {
          if (!T::kPShared) {  // with P in two halves, each with its barrier
            ready = mbar_try_wait(bar_v_full + 8u * v_at.slot, v_at.phase) &
                    mbar_try_wait(p_bar(0), p_parity()) & mbar_try_wait(p_bar(1), p_parity());
            ready = __all_sync(0xffffffffu, ready);
          }
          // the segment's first P V writes O anew: the last segment's rows must be out
          if (added == first && segments > 0) {
            ok = warp_wait(bar_o_free, uint32_t(segments - 1) & 1u);
            if (!ok) break;
          }
          ok = issue_pv(ready, added > first);
        }
      }
      if (ok) umma_commit_warp(bar_o_full, leader);
    }
    failed = !ok;
    if (failed) {  // nothing reads shared memory or writes tensor memory when the CTA ends
      umma_commit_warp(bar_drained, leader);
      mbar_wait_bounded(bar_drained, 0, kTileWaitClocks);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int group = warp >> 2;
    const int quarter = warp & 3;
    const int row = tid & (kRows - 1);
    const uint32_t lanes = uint32_t(32 * quarter) << 16;
    const float scale = p.scale_log2;
    int n0 = 0;        // key tiles before this segment
    int segments = 0;
    bool ok = true;
    // every lane waits; the warp goes on or gives up as one
    auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, wait(bar, parity));
    };
    const int token = p.group_div.quotient(row);  // of the query tile
    const int head_of_group = row - token * p.group;
    // What is kept of a segment while its tiles go by.
    struct Rows {
      int64_t at;    // output row of this thread's query
      int rows;      // of the tile
      int t;         // this row's position (rows behind the last: not used)
      int tiles;
      int part;
      int piece;     // 0, 1: which of the CTA's partial results; -1: the item is whole
    };
    int asked = 0;  // segments so far
    auto next_segment = [&](Rows &kept) -> bool {
      if (!warp_wait(bar_seg_full + 8u * uint32_t(asked % kSegments),
                     uint32_t(asked / kSegments) & 1u)) {
        ok = false;
        return false;
      }
      const SegmentInfo s = small.segment[asked % kSegments];
      ++asked;
      if (s.tiles == 0) return false;
      kept.rows = s.rows;
      kept.t = s.t0 + token;
      kept.tiles = s.tiles;
      kept.part = s.hp / heads;
      kept.piece = s.piece;
      kept.at = (int64_t(s.row0) + token) * p.q_heads + (s.hp - kept.part * heads) * p.group + head_of_group;
      return true;
    };
    if constexpr (T::kPShared) {  // weights of rows that never are queries
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        *reinterpret_cast<uint4 *>(smem_raw + T::kPAt + group * kPTileBytes + row * 128 + 16 * c) =
            make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_shared();
    }
    Rows now_rows;
    bool more = next_segment(now_rows);
    while (more && ok) {
      const bool active = 32 * quarter < now_rows.rows;  // some row of the warp is a query
      const int t = now_rows.t;
      const int n1 = n0 + now_rows.tiles;
      float l_run = 0.0f;
      float ref = -INFINITY;  // what l_run's weights are scaled by
      if (!active) {
        // no row of this warp is a query: it keeps the barriers' phases, which go by the
        // tile's number
        for (int n = n0 + ((n0 ^ group) & 1); n < n1; n += 2) {
          ok = warp_wait(bar_s_full + 8u * uint32_t(group), uint32_t(n >> 1) & 1u);
          if (!ok) break;
          if (T::kPShared && n >= 2) {  // not a phase ahead of the other warps' weights
            ok = warp_wait(bar_v_done + 8u * v_slot(n - 2), v_parity(n - 2));
            if (!ok) break;
          }
          __syncwarp();
          if (lane == 0) {
            if constexpr (T::kPShared) mbar_arrive(bar_s_free + 8u * uint32_t(group));
            mbar_arrive(bar_m_full + 32u * uint32_t(group) + 8u * uint32_t(quarter));
            mbar_arrive(bar_p_full + 16u * uint32_t(group));
            if constexpr (!T::kPShared) mbar_arrive(bar_p_full + 16u * uint32_t(group) + 8u);
          }
        }
      } else {
        for (int n = n0 + ((n0 ^ group) & 1); n < n1; n += 2) {
          ok = warp_wait(bar_s_full + 8u * uint32_t(group), uint32_t(n >> 1) & 1u);
          if (!ok) break;
          tc_fence_after();
          const TileInfo info = small.info[n % kInfos];
          float sc[64];
          const uint32_t s_at = tmem + lanes + kTmemS + uint32_t(group) * kKeys;
          tmem_ld64(s_at, sc);
          if constexpr (T::kPShared) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_s_free + 8u * uint32_t(group));
          }
          if (info.edge) {
            asm volatile("" ::: "memory");  // a branch, not 64 selects on every tile
            unsigned long long sees = info.live & low_bits(t + 1 - info.base);
            if (p.window > 0) {
              sees &= ~low_bits(t - p.window + 1 - info.base) | low_bits(p.sinks - info.base);
            }
            const uint32_t lo = uint32_t(sees), hi = uint32_t(sees >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (((lo >> c) & 1u) == 0) sc[c] = -INFINITY;
              if (((hi >> c) & 1u) == 0) sc[c + 32] = -INFINITY;
            }
          }
          float mx[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
          for (int c = 4; c < 60; c += 8) {
#pragma unroll
            for (int u = 0; u < 4; ++u) mx[u] = max3(mx[u], sc[c + u], sc[c + 4 + u]);
          }
          float m_tile = fmaxf(max3(mx[0], mx[1], max3(mx[2], mx[3], sc[60])),
                               max3(sc[61], sc[62], sc[63])) * scale;
          // rows behind the last hold anything: they must not make the warp rescale, and
          // their weights are zeros
          if (row >= now_rows.rows) m_tile = 3.0e38f;
          // the reference so far: the other group's tile before this one
          float last = -INFINITY;
          if (n > n0) {
            ok = __all_sync(0xffffffffu, wait_here(bar_m_full + 32u * uint32_t(group ^ 1) +
                                                       8u * uint32_t(quarter),
                                                   uint32_t((n - 1) >> 1) & 1u));
            if (!ok) break;
            last = small.row_ref[group ^ 1][row];
          }
          const float now = m_tile > last + kRescaleSlack || last == -INFINITY ? m_tile : last;
          small.row_ref[group][row] = now;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_m_full + 32u * uint32_t(group) + 8u * uint32_t(quarter));
          // Raising is rare. Tensor-memory accesses are warp-wide: the warp rescales its
          // rows of O if any of them must, once P V of the tile before no longer adds to
          // them.
          if (__any_sync(0xffffffffu, ref != now)) {
            l_run = ref == -INFINITY ? 0.0f : l_run * ex2_approx(ref - now);
            ref = now;
            const bool raised = last != -INFINITY && now != last;
            if (__any_sync(0xffffffffu, raised)) {
              ok = __all_sync(0xffffffffu, wait_here(bar_v_done + 8u * v_slot(n - 1), v_parity(n - 1)));
              if (!ok) break;
              tc_fence_after();
              const float factor = raised ? ex2_approx(last - now) : 1.0f;
#pragma unroll 1
              for (int c = 0; c < kPartDims; c += 16) {
                float o[16];
                uint32_t x[16];
                tmem_ld<16>(tmem + lanes + uint32_t(c), o);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(o[i] * factor);
                tmem_st16(tmem + lanes + uint32_t(c), x);
              }
            }
          }
          if (T::kPShared && n >= 2) {  // the buffer's last weights have been used
            ok = __all_sync(0xffffffffu, wait_here(bar_v_done + 8u * v_slot(n - 2), v_parity(n - 2)));
            if (!ok) break;
          }
          // the weights, in packed pairs; rounded to bf16 for P V, summed unrounded
          const float neg = now == -INFINITY ? 0.0f : -now;
          const f32x2 neg2 = pack2(neg, neg), scale2 = pack2(scale, scale);
          f32x2 sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float e0, e1;
              unpack2(fma2_rn(pack2(sc[32 * h + 2 * i], sc[32 * h + 2 * i + 1]), scale2, neg2), e0, e1);
              e0 = ex2_approx(e0);
              e1 = ex2_approx(e1);
              sum[i & 1] = add2_rn(sum[i & 1], pack2(e0, e1));
              const __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
              w[i] = *reinterpret_cast<const uint32_t *>(&b2);
            }
            if constexpr (T::kPShared) {  // row of 128 bytes, its 16-byte chunks swizzled
              uint8_t *to = smem_raw + T::kPAt + group * kPTileBytes + row * 128;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                *reinterpret_cast<uint4 *>(to + (((4 * h + c) ^ (row & 7)) << 4)) =
                    make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
              }
              if (h == 1) fence_proxy_async_shared();
            } else {
              tmem_st16(s_at + 16u * uint32_t(h), w);
            }
            if (!T::kPShared || h == 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(bar_p_full + 16u * uint32_t(group) + (T::kPShared ? 0u : 8u * uint32_t(h)));
              }
            }
          }
          float a0, a1;
          unpack2(add2_rn(sum[0], sum[1]), a0, a1);
          l_run += a0 + a1;
        }
      }
      if (!ok) break;

      // ---- the segment's end
      const int last = n1 - 1;
      const bool owner = (last & 1) == group;
      if (active) {
        if (!owner) {
          ok = warp_wait(bar_m_full + 32u * uint32_t(group ^ 1) + 8u * uint32_t(quarter),
                         uint32_t(last >> 1) & 1u);
          if (!ok) break;
          const float now = small.row_ref[group ^ 1][row];
          if (ref != now) {
            l_run = ref == -INFINITY ? 0.0f : l_run * ex2_approx(ref - now);
            ref = now;
          }
        }
      }
      ok = warp_wait(bar_o_full, uint32_t(segments & 1));
      if (!ok) break;
      tc_fence_after();
      if (active) small.row_sum[group][row] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_l_full + 32u * uint32_t(group) + 8u * uint32_t(quarter));
      ok = warp_wait(bar_l_full + 32u * uint32_t(group ^ 1) + 8u * uint32_t(quarter),
                     uint32_t(segments & 1));
      if (!ok) break;
      const bool whole = now_rows.piece < 0;
      const bool writes = active && row < now_rows.rows;
      const float l_row = active ? small.row_sum[0][row] + small.row_sum[1][row] : 0.0f;
      // (a sum of zero: no key; of NaN: the row is NaN)
      const float inv = whole ? (l_row != 0.0f ? 1.0f / l_row : 0.0f) : 1.0f;
      float *piece = p.partials + (int64_t(blockIdx.x) * 2 + (whole ? 0 : now_rows.piece)) *
                                      (int64_t(p.rows_cap) * (kPartDims + 2));
      // This group's 128 columns of O, 32 lines of 128 bytes per warp at a time: 64
      // columns as bf16, or 32 as fp32, through 4 KB of shared memory per warp so that a
      // store covers whole lines, not 32 rows of 16 bytes: the weights' buffers (P V is
      // complete), or for head_dim 512 the upper half of Q (so is Q K^T). Rolled loops:
      // this code runs once per segment and costs what it takes to fetch it.
      const int steps = whole ? 2 : 4;
      const int step_columns = whole ? 64 : 32;
      static_assert(T::kPShared || T::kQHiBytes >= kSoftmaxWarps * 4096, "place for the rows");
      uint8_t *stage = smem_raw + (T::kPShared ? T::kPAt : 0) + (4 * group + quarter) * 4096;
      const int valid = now_rows.rows - 32 * quarter;  // rows of the warp
      const __nv_bfloat162 none = __floats2bfloat162_rn(0.0f, 0.0f);
      __nv_bfloat162 odd = none;  // 0 times what is written: NaN if any of it is not finite
#pragma unroll 1
      for (int h = 0; h < steps; ++h) {
        const int column = 128 * group + step_columns * h;
        uint8_t *line;  // this row's 128 bytes
        if (whole) {
          line = reinterpret_cast<uint8_t *>(p.out + now_rows.at * T::kHeadDim +
                                             now_rows.part * kPartDims + column);
        } else {
          line = reinterpret_cast<uint8_t *>(piece + row * kPartDims + column);
        }
        if (active) {
#pragma unroll 1
          for (int c = 0; c < 8; c += 4) {  // four 16-byte chunks of the line
            uint4 w[4];
            if (whole) {
              float o[32];
              tmem_ld<32>(tmem + lanes + uint32_t(column + 8 * c), o);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                w[i] = make_uint4(bf16_pair(o[8 * i] * inv, o[8 * i + 1] * inv),
                                  bf16_pair(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                  bf16_pair(o[8 * i + 4] * inv, o[8 * i + 5] * inv),
                                  bf16_pair(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  odd = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&words[j]), none, odd);
                }
              }
            } else {
              float o[16];
              tmem_ld<16>(tmem + lanes + uint32_t(column + 4 * c), o);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                w[i] = make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]),
                                  __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3]));
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              *reinterpret_cast<uint4 *>(stage + lane * 128 + (((c + i) ^ (lane & 7)) << 4)) = w[i];
            }
          }
        }
        if (T::kPShared && h + 1 == steps) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_o_free);
        }
        if (active) {
          __syncwarp();
#pragma unroll 2
          for (int i = 0; i < 8; ++i) {  // eight lanes store a row's line
            const int r = 4 * i + (lane >> 3);
            const int c = lane & 7;
            const uint4 v = *reinterpret_cast<const uint4 *>(stage + r * 128 + ((c ^ (r & 7)) << 4));
            uint8_t *to = reinterpret_cast<uint8_t *>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(line), r));
            if (r < valid) reinterpret_cast<uint4 *>(to)[c] = v;
          }
          __syncwarp();
        }
      }
      if constexpr (!T::kPShared) {  // the next upper half of Q comes where the rows went through
        fence_proxy_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_o_free);
      }
      // (a NaN of the sum comes of the scores: the row's own)
      if (writes && l_row == l_row && pair_not_finite(*reinterpret_cast<const uint32_t *>(&odd))) small.not_finite = 1;
      if (writes && group == 0) {
        if (!whole) {
          piece[p.rows_cap * kPartDims + row] = ref;
          piece[p.rows_cap * (kPartDims + 1) + row] = l_row;
        } else if (p.lse != nullptr && now_rows.part == 0) {
          p.lse[now_rows.at] = l_row != 0.0f ? (ref + log2f(l_row)) * 0.6931471805599453f : -INFINITY;
        }
      }
      n0 = n1;
      more = next_segment(now_rows);
      ++segments;
    }
    failed = !ok;
  }
  if (failed) {
    set_status(p.status, B200KV_STATUS_WAIT_TIMEOUT);
    *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) {
    int4 meta = small.meta;
    if (small.not_finite != 0) meta.w |= kNotFinite;
    p.meta[blockIdx.x] = meta;
  }
  if (warp == 0) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemColumns)
                 : "memory");
  }
}

// Rows that one CTA has written whole, where some are not finite. The combine's blocks of the
// CTAs that say so look through all rows between them, but for those of items that are
// joined (their joins look by themselves).
template <int D>
__device__ __noinline__ void combine_not_finite(const ChunkParams &p, const ChunkAttentionArgs &a) {
  const int lane = int(threadIdx.x) & 31;
  const int parts = D / kPartDims;
  int ctas = 0, before = 0;  // CTAs that say so, those before this one
  for (int c = 0; c < int(gridDim.x); c += 32) {
    const bool says = c + lane < int(gridDim.x) && (p.meta[c + lane].w & kNotFinite) != 0;
    ctas += __popc(__ballot_sync(0xffffffffu, says));
    before += __popc(__ballot_sync(0xffffffffu, says && c + lane < int(blockIdx.x)));
  }
  const int block_warps = int(blockDim.x) / 32;
  const int64_t warps = int64_t(ctas) * gridDim.y * block_warps;
  const int64_t rows = int64_t(a.runs.rows) * a.q_heads * parts;
  for (int64_t i = (int64_t(before) * gridDim.y + blockIdx.y) * block_warps + threadIdx.x / 32; i < rows; i += warps) {
    const int part = int(i % parts);
    const int q_head = int(i / parts % a.q_heads);
    const int64_t row = i / parts / a.q_heads;
    const int dims = part * kPartDims + lane * 8;
    const uint4 v = *reinterpret_cast<const uint4 *>(a.out + (row * a.q_heads + q_head) * D + dims);
    if (!__any_sync(0xffffffffu, pack_not_finite(v))) continue;
    bool joined = false;
    for (int c = lane; c < int(gridDim.x); c += 32) {
      const int4 meta = p.meta[c];
      joined |= meta.x == part * p.cfg.num_heads + q_head / p.group && row >= meta.y &&
                (row - meta.y) * p.group < meta.z;
    }
    if (__any_sync(0xffffffffu, joined)) continue;
    chunk_exact_row<D>(a, p.table_end, row, q_head, dims, true);
  }
}

// Joins the partial rows of items that several CTAs share. Block (i, y): the item
// whose first key tiles CTA i has (meta.x >= 0: KV head and part; meta.y: packed row of
// its first token; meta.z: query rows); the pieces behind it are the first of CTA i + 1,
// i + 2, ... up to the one that has the item's end (meta.w 1; 2: goes on). A warp per
// row, 8 columns per lane:
//   M = max m, out = sum 2^(m - M) acc / sum 2^(m - M) l, lse = (M + log2 sum) ln 2
// Bound by the latency of its few dependent loads: the pieces' rows are asked for four
// at a time, together with what weighs them.
constexpr int kCombineWarps = 4;
template <int D>
__global__ __launch_bounds__(kCombineWarps * 32, 8) void chunk_combine_kernel(
    const __grid_constant__ ChunkParams p, const __grid_constant__ ChunkAttentionArgs a) {
  pdl_wait_for_predecessor();
  const int lane = int(threadIdx.x) & 31;
  const int row = int(blockIdx.y) * kCombineWarps + (int(threadIdx.x) >> 5);
  const int ctas = int(gridDim.x);
  const int cta = int(blockIdx.x);
  const int4 meta = p.meta[cta];
  int state = cta + 1 + lane < ctas ? p.meta[cta + 1 + lane].w : 1;
  if ((meta.w & kNotFinite) != 0) combine_not_finite<D>(p, a);
  if (meta.x < 0 || row >= meta.z) return;
  int pieces = 1;  // the first and those behind it
  for (int base = cta + 1;;) {
    const uint32_t end = __ballot_sync(0xffffffffu, (state & ~kNotFinite) != 2);
    if (end != 0) {
      pieces += __ffs(int(end));
      break;
    }
    pieces += 32;
    base += 32;
    state = base + lane < ctas ? p.meta[base + lane].w : 1;
  }
  pieces = min(pieces, ctas - cta);
  const int64_t slot_floats = int64_t(p.rows_cap) * (kPartDims + 2);
  // piece 0: the second partial result of CTA i; piece k: the first of CTA i + k
  const float *base = p.partials + int64_t(cta) * 2 * slot_floats;
  auto piece = [&](int i) { return base + (i == 0 ? slot_floats : int64_t(i) * 2 * slot_floats); };
  float m = -INFINITY, l = 0.0f;
  float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < pieces; i0 += 4) {
    float mi[4], li[4];
    float4 a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mi[k] = -INFINITY;
      li[k] = 0.0f;
      a[k] = b[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i0 + k >= pieces) continue;
      const float *from = piece(i0 + k);
      mi[k] = __ldg(from + p.rows_cap * kPartDims + row);
      li[k] = __ldg(from + p.rows_cap * (kPartDims + 1) + row);
      a[k] = __ldg(reinterpret_cast<const float4 *>(from + row * kPartDims + lane * 8));
      b[k] = __ldg(reinterpret_cast<const float4 *>(from + row * kPartDims + lane * 8) + 1);
    }
    const float now = fmaxf(fmaxf(fmaxf(mi[0], mi[1]), fmaxf(mi[2], mi[3])), m);
    const float keep = m == -INFINITY ? 0.0f : ex2_approx(m - now);
    l *= keep;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= keep;
    m = now;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // (a piece without a visible key has accumulated zeros)
      const float f = mi[k] == -INFINITY ? 0.0f : ex2_approx(mi[k] - now);
      l = fmaf(f, li[k], l);
      acc[0] = fmaf(f, a[k].x, acc[0]);
      acc[1] = fmaf(f, a[k].y, acc[1]);
      acc[2] = fmaf(f, a[k].z, acc[2]);
      acc[3] = fmaf(f, a[k].w, acc[3]);
      acc[4] = fmaf(f, b[k].x, acc[4]);
      acc[5] = fmaf(f, b[k].y, acc[5]);
      acc[6] = fmaf(f, b[k].z, acc[6]);
      acc[7] = fmaf(f, b[k].w, acc[7]);
    }
  }
  const int part = meta.x / p.cfg.num_heads;
  const int head = meta.x - part * p.cfg.num_heads;
  const int token = p.group_div.quotient(row);
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const int64_t at = (int64_t(meta.y) + token) * p.q_heads + head * p.group + (row - token * p.group);
  const uint4 packed = make_uint4(bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv),
                                  bf16_pair(acc[4] * inv, acc[5] * inv), bf16_pair(acc[6] * inv, acc[7] * inv));
  reinterpret_cast<uint4 *>(p.out + at * D + part * kPartDims)[lane] = packed;
  if (p.lse != nullptr && part == 0 && lane == 0) {
    p.lse[at] = l != 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  }
  if (l == l && __any_sync(0xffffffffu, pack_not_finite(packed))) {
    chunk_exact_row<D>(a, p.table_end, int64_t(meta.y) + token, head * p.group + (row - token * p.group),
                       part * kPartDims + lane * 8, true);
  }
}

int table_end(const Gemma4KvCacheConfig &c) {
  if (c.window_size > 0) return kMaxPosition;  // a ring has a place for every position
  return int(std::min<int64_t>(kMaxPosition, int64_t(c.max_pages_per_seq) * c.page_size));
}

bool make_q_map(CUtensorMap *map, const __nv_bfloat16 *q, int rows, int q_heads, int head_dim,
                int group, int box_tokens) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return false;
  const cuuint64_t row = cuuint64_t(q_heads) * head_dim * 2;
  const cuuint64_t dims[3] = {cuuint64_t(head_dim), cuuint64_t(q_heads), cuuint64_t(rows)};
  const cuuint64_t strides[2] = {cuuint64_t(head_dim) * 2, row};
  const cuuint32_t box[3] = {64, cuuint32_t(group), cuuint32_t(box_tokens)};
  const cuuint32_t steps[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16 *>(q), dims,
                strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query rows a partial result can have, and the workspace of one CTA: its meta word
// and two partial results.
int partial_rows(int group, int max_row_count) {
  const int tokens = std::min(kRows / group, max_row_count);
  return div_up(tokens * group, 8) * 8;
}
int64_t workspace_per_cta(int group, int max_row_count) {
  return 16 + int64_t(partial_rows(group, max_row_count)) * (kPartDims + 2) * 4 * 2;
}

template <class T>
cudaError_t launch_chunk(const ChunkAttentionArgs &a, int ctas, cudaStream_t stream) {
  static_assert(kChunkSmemBytes<T> <= 227 * 1024, "the ring and the small state must fit one SM");
  const Gemma4KvCacheConfig &c = a.cfg;
  ChunkParams p = {};
  p.out = a.out;
  p.lse = a.lse;
  p.q = a.q;
  p.cache_k = a.cache_k;
  p.cache_v = a.cache_v;
  p.k_rows = a.k_rows;
  p.v_rows = a.v_rows;
  p.cfg = c;
  p.page_table = a.page_table;
  p.runs = a.runs;
  p.layer = a.layer;
  p.q_heads = a.q_heads;
  p.group = a.q_heads / c.num_heads;
  p.tile_tokens = kRows / p.group;
  p.tiles_per_run = div_up(std::min(a.runs.max_row_count, a.runs.rows), p.tile_tokens);
  p.window = a.window;
  p.sinks = a.sinks;
  p.table_end = table_end(c);
  p.box = box_tokens(c.page_size, kKeys);
  p.page_div = FastDiv::by(uint32_t(c.page_size));
  p.slot_div = FastDiv::by(uint32_t(c.max_pages_per_seq));
  p.group_div = FastDiv::by(uint32_t(p.group));
  p.run_div = FastDiv::by(uint32_t(p.tiles_per_run));
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  p.rows_cap = partial_rows(p.group, a.runs.max_row_count);
  p.meta = static_cast<int4 *>(a.workspace);
  p.partials = reinterpret_cast<float *>(p.meta + ctas);
  p.status = a.status;
  p.q_box = std::min(p.tile_tokens, a.runs.max_row_count);
  p.q_slots = p.q_box * p.group <= kRows / 2 ? 1 : 2;
  CUtensorMap map_q = {}, map_k = {}, map_v = {}, map_k_rows = {}, map_v_rows = {};
  if (!make_q_map(&map_q, a.q, a.runs.rows, a.q_heads, c.head_dim, p.group, p.q_box)) {
    return cudaErrorInvalidValue;
  }
  if (p.box > 0 && (!make_cache_map(&map_k, a.cache_k, c, p.box) ||
                    !make_cache_map(&map_v, a.cache_v, c, p.box))) {
    return cudaErrorInvalidValue;
  }
  if (p.box > 0 && a.k_rows != nullptr &&
      (!make_rows_map(&map_k_rows, a.k_rows, a.runs.rows, c.num_heads, c.head_dim) ||
       !make_rows_map(&map_v_rows, a.v_rows, a.runs.rows, c.num_heads, c.head_dim))) {
    return cudaErrorInvalidValue;
  }
  cudaError_t st = cudaFuncSetAttribute(chunk_attention_kernel<T>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, kChunkSmemBytes<T>);
  if (st != cudaSuccess) return st;
  st = launch_pdl(chunk_attention_kernel<T>, dim3(unsigned(ctas)), dim3(kThreads),
                  size_t(kChunkSmemBytes<T>), stream, p, map_k, map_v, map_k_rows, map_v_rows,
                  map_q);
  if (st != cudaSuccess) return st;
  const unsigned row_blocks = unsigned(div_up(p.rows_cap, kCombineWarps));
  return launch_pdl(chunk_combine_kernel<T::kHeadDim>, dim3(unsigned(ctas), row_blocks), dim3(kCombineWarps * 32), 0,
                    stream, p, a);
}

}  // namespace

size_t chunk_workspace_bytes(int q_heads, int kv_heads, int head_dim, int run_count,
                             int max_row_count, int sm_count) {
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > 64 ||
      (head_dim != 256 && head_dim != 512) || run_count <= 0 || max_row_count <= 0 ||
      sm_count <= 0) {
    return 0;
  }
  return size_t(workspace_per_cta(q_heads / kv_heads, max_row_count)) * size_t(sm_count);
}

cudaError_t validate_chunk_attention(const ChunkAttentionArgs &a) {
  const Gemma4KvCacheConfig &c = a.cfg;
  if (!valid_chunk_runs(a.runs) || !valid_cache_config(c, a.layer) || a.out == nullptr ||
      a.q == nullptr || a.cache_k == nullptr || a.cache_v == nullptr || a.page_table == nullptr ||
      (a.k_rows == nullptr) != (a.v_rows == nullptr) || a.workspace == nullptr ||
      a.q_heads <= 0 || a.q_heads % c.num_heads != 0 || a.q_heads / c.num_heads > 64 ||
      (c.head_dim != 256 && c.head_dim != 512) || a.window < 0 || a.sinks < 0 ||
      (a.sinks > 0 && a.window == 0) || !(a.softmax_scale > 0.0f)) {
    return cudaErrorInvalidValue;
  }
  // (run, query tile) pairs that every CTA adds up, and the most key tiles they can have
  const int64_t tokens = kRows / (a.q_heads / c.num_heads);
  const int64_t pairs = a.runs.run_count * div_up(int64_t(std::min(a.runs.max_row_count, a.runs.rows)), tokens);
  const int64_t keys = most_keys(a, table_end(c), tokens);
  // (each of the four stretches of keys may begin and end inside a tile)
  const double cost = double(keys / kKeys + 8 + kItemCost) * double(pairs) * c.num_heads * (c.head_dim / kPartDims);
  if (pairs > (1 << 24) || cost >= 2147483648.0) return cudaErrorInvalidValue;
  if (int64_t(a.workspace_bytes) < workspace_per_cta(a.q_heads / c.num_heads, a.runs.max_row_count)) {
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

// A window of all the positions hides nothing; cut to those, the distance of its start
// from a key tile behind the row (t - window + 1 - base) fits 32 bits in both kernels.
static ChunkAttentionArgs with_window_cut(ChunkAttentionArgs a) {
  a.window = std::min(a.window, kMaxPosition);
  return a;
}

cudaError_t chunk_attention_bf16(const ChunkAttentionArgs &given, cudaStream_t stream) {
  const cudaError_t valid = validate_chunk_attention(given);
  if (valid != cudaSuccess) return valid;
  const ChunkAttentionArgs a = with_window_cut(given);
  if (a.runs.run_count == 0 || a.runs.rows == 0) return cudaSuccess;
  int device = 0, sms = 0;
  cudaError_t st = cudaGetDevice(&device);
  if (st != cudaSuccess) return st;
  st = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (st != cudaSuccess) return st;
  bool taken = false;
  st = chunk_attention_few_bf16(a, device, table_end(a.cfg), stream, &taken);
  if (st != cudaSuccess || taken) return st;
  // one CTA per SM, or as many as the workspace has room for
  const int64_t room = int64_t(a.workspace_bytes) /
                       workspace_per_cta(a.q_heads / a.cfg.num_heads, a.runs.max_row_count);
  const int ctas = int(std::min<int64_t>(sms, room));
  return a.cfg.head_dim == 256 ? launch_chunk<ChunkTraits<256>>(a, ctas, stream)
                               : launch_chunk<ChunkTraits<512>>(a, ctas, stream);
}

int chunk_attention_launches(const ChunkAttentionArgs &a) {
  int device = 0;
  if (validate_chunk_attention(a) != cudaSuccess || a.runs.run_count == 0 || a.runs.rows == 0 ||
      cudaGetDevice(&device) != cudaSuccess) {
    return 0;
  }
  return chunk_attention_few_takes(a, device, table_end(a.cfg)) ? 1 : 2;  // the other one's join
}

cudaError_t chunk_attention_give_up_selftest(const ChunkAttentionArgs &a, int32_t tile,
                                             cudaStream_t stream) {
  const cudaError_t valid = validate_chunk_attention(a);
  if (valid != cudaSuccess) return valid;
  if (a.status == nullptr || tile < 0 || a.runs.run_count == 0 || a.runs.rows == 0) return cudaErrorInvalidValue;
  int device = 0;
  cudaError_t st = cudaGetDevice(&device);
  if (st != cudaSuccess) return st;
  bool taken = false;
  st = chunk_attention_few_bf16(with_window_cut(a), device, table_end(a.cfg), stream, &taken, tile);
  return st != cudaSuccess || taken ? st : cudaErrorInvalidValue;
}

}  // namespace b200kv
