// Product of two microscaled FP4 operands, many rows on both sides: persistent kernel on pairs of CTAs.
//
//   out[i, j] = T( ga gb sum_k a[i, k] b[j, k] )
//
// Bound by the tensor pipe (a pair's MMA of 256 x 256 x 64 takes 128 cycles at the FP4 rate), by the shared memory that
// the copies write and the MMAs and scale copies read (36-39 KB and about as much per stage of 512 MMA cycles), and on
// long runs by the power cap: 6.0 PFLOP/s on 4096 x 9472 x 16384, 5.2 on 8192 x 24576 x 4096 in short runs and 4.7 at the
// cap.  A cluster of two CTAs owns a tile: each loads its 128 rows of a and its half of the 256 rows of b,
// tcgen05.mma.cta_group::2 reads both halves of b, and each CTA accumulates its 128 rows x 256 columns.
//
//   warp 0      copies of both operands' codes and scale tiles by TMA; every CTA needs the scales of all 256 rows of
//               b.  Both CTAs' copies complete on the first CTA's barrier (the cta_group::2 form of the copy)
//   warp 1      first CTA: scales to tensor memory (both CTAs') and MMAs
//   warps 2-9   epilogue
//
// Tensor memory holds two accumulators of 256 columns that overlap, [0, 256) and [208, 464), beside the 48 columns
// of scales.  The epilogue reads the shared columns of a tile first and gives them back at once; the next
// tile's MMAs start then and run beside the rest of the epilogue.
//
// kSplit: fewer tiles than half the pairs of SMs.  A tile on its own needs 700 cycles per stage of K; two pairs of a
// cluster share it then, each with half of K, push the FP32 sums of the columns they do not own to the pair that does
// (distributed shared memory, over the ring that has been read), and both pairs add and store their columns, always in
// the same order.  (256 x 6144 x 4096 in two halves 11.5 us, 13.4 without.  Four pairs, clusters of eight CTAs
// with 200 KB each, took 20 us: too few of them fit on the chip at once.)
#include "fp4_tc.cuh"

namespace lbl {
namespace {

constexpr int kRowsCta = 128;   // rows of a, and of b, that one CTA loads
constexpr int kRowsPair = 256;
constexpr int kEpilogueWarps = 8;  // two per quarter of the lanes, a chunk of columns each in turn
constexpr int kThreads = 32 * (2 + kEpilogueWarps);
constexpr int kMaxStages = 6;
constexpr int kStatusPairWait = 620;
constexpr int kTmemColumns = 512;
constexpr int kScaleColumn = 512 - 48;
constexpr int kSecondAccumulator = kScaleColumn - kRowsPair;  // 208
constexpr int kChunk = 64;  // columns an epilogue warp handles at a time
constexpr int kStagingBytes = 32 * kChunk * 2;  // per epilogue warp
constexpr int kSmemLimit = 227 * 1024;
constexpr int kGroupRows = 16;  // row tiles walked together, for reuse in the L2 (8192 x 24576 x 4096 at the power cap: 4, 8, 16, 32 rows 380, 362, 352, 350 us)

struct PairParams {
  const float* factor_a;
  const float* factor_b;
  void* out;
  int64_t out_pitch;
  int rows_a, rows_b;
  int cols_padded;
  int tiles_a, tiles_b;
  int out_bytes;  // rows of out start on 16 or 8 bytes, or anywhere (2)
  int* status;
};

struct PairBarriers {
  uint64_t full[kMaxStages];   // first CTA's: both CTAs' copies have landed
  uint64_t empty[kMaxStages];  // the MMAs have read the stage (cluster-wide commit)
  uint64_t acc_full;           // a tile's accumulators are complete (cluster-wide commit)
  uint64_t acc_free;           // first CTA's: both CTAs have read the shared columns
  uint32_t tmem_base;
  int abort_flag;
};

template <int kFormat>
struct PairTile {
  static constexpr int kTiles = kStageCols / fp4::Format<kFormat>::kTileCols;
  static constexpr int kBytesCodes = kRowsCta * kRowBytes;      // of one operand
  static constexpr int kBytesScaleA = kTiles * 512;
  static constexpr int kBytesScaleB = 2 * kTiles * 512;
  static constexpr int kStageBytes = 2 * kBytesCodes + kBytesScaleA + kBytesScaleB;
  static constexpr int kStages = (kSmemLimit - 1280 - kEpilogueWarps * kStagingBytes) / kStageBytes < kMaxStages
                                     ? (kSmemLimit - 1280 - kEpilogueWarps * kStagingBytes) / kStageBytes
                                     : kMaxStages;
  static constexpr int kSmemBytes = kStages * kStageBytes + kEpilogueWarps * kStagingBytes + 1024;
  static_assert(kTiles * 4 * 3 <= 48, "scale columns");
};

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_result, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_result)),
               "r"(cols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// Arrives on the barrier at this shared-memory offset in both CTAs of the pair (cluster ranks `leader` and
// leader + 1) once every MMA issued so far has finished.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"(static_cast<uint16_t>(3u << leader))
      : "memory");
}
// Tiled load into this CTA's shared memory that completes on a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, int c0, int c1,
                                                 uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(smem_dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(cluster_bar)
      : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Tile t: groups of kGroupRows row tiles, walked column by column.
__device__ __forceinline__ void tile_of(const PairParams& p, int t, int* tile_a, int* tile_b) {
  const int per_group = kGroupRows * p.tiles_b;
  const int group = t / per_group;
  const int first = group * kGroupRows;
  const int rows = min(kGroupRows, p.tiles_a - first);
  const int rest = t - group * per_group;
  *tile_a = first + rest % rows;
  *tile_b = rest / rows;
}

// One warp's 32 rows x 64 columns of sums, a row per lane, to out through the warp's staging memory, so that rows leave
// as whole 128-byte runs: in 16- or 8-byte pieces where rows of out start on those, and otherwise a row per store, in
// 4-byte words that start on a word (one column later on rows that do not).
template <typename T>
__device__ __forceinline__ void store_chunk(const PairParams& p, const uint32_t (&v)[2][32], float alpha,
                                            uint8_t* staging, int row0, int col0, int lane) {
  // Row `lane`: eight pieces of 16 bytes, swizzled over the banks.
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t* f = &v[i >> 2][(i & 3) * 8];
    uint4 q;
    q.x = two_rounded<T>(__uint_as_float(f[0]) * alpha, __uint_as_float(f[1]) * alpha);
    q.y = two_rounded<T>(__uint_as_float(f[2]) * alpha, __uint_as_float(f[3]) * alpha);
    q.z = two_rounded<T>(__uint_as_float(f[4]) * alpha, __uint_as_float(f[5]) * alpha);
    q.w = two_rounded<T>(__uint_as_float(f[6]) * alpha, __uint_as_float(f[7]) * alpha);
    *reinterpret_cast<uint4*>(staging + lane * 128 + ((i ^ (lane & 7)) << 4)) = q;
  }
  __syncwarp();
  T* out = static_cast<T*>(p.out);
  if (p.out_bytes == 16) {  // rows_b is a multiple of eight then
    const int piece = lane & 7;
    const int col = col0 + piece * 8;
#pragma unroll
    for (int r = lane >> 3; r < 32; r += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(staging + r * 128 + ((piece ^ (r & 7)) << 4));
      if (row0 + r < p.rows_a && col < p.rows_b) *reinterpret_cast<uint4*>(out + (row0 + r) * p.out_pitch + col) = q;
    }
  } else if (p.out_bytes == 8) {  // of four
    const int piece = lane & 15;
    const int col = col0 + piece * 4;
#pragma unroll
    for (int r = lane >> 4; r < 32; r += 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(staging + r * 128 + (((piece >> 1) ^ (r & 7)) << 4) + (piece & 1) * 8);
      if (row0 + r < p.rows_a && col < p.rows_b) *reinterpret_cast<uint2*>(out + (row0 + r) * p.out_pitch + col) = q;
    }
  } else {
    // Four rows at a time, without a branch: which lanes store what depends on whether the row starts on a word.
    // (4096 x 16386 x 128: one row after the other, with branches for its ends, 103 us, so 75; eight at a time 73, but the
    // registers cost the other paths 3 %.)
    const int columns = p.rows_b - col0;
    const int rows = p.rows_a - row0;
    unsigned short* line = reinterpret_cast<unsigned short*>(out + row0 * p.out_pitch + col0);
    const uint32_t late_first = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(line) >> 1) & 1;
    const uint32_t alternate = static_cast<uint32_t>(p.out_pitch) & 1;
    const bool pair_at[2] = {2 * lane + 1 < columns, 2 * lane + 2 < columns && lane < 31};
    const bool last_at[2] = {2 * lane + 1 == columns, 2 * lane + 1 < columns && !pair_at[1]};
    const bool first_at = lane == 0 && columns > 0;
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 4) {
      uint32_t words[4], next[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        words[i] = *reinterpret_cast<const uint32_t*>(staging + (r0 + i) * 128 + (((lane >> 2) ^ ((r0 + i) & 7)) << 4) + (lane & 3) * 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = __shfl_down_sync(0xffffffffu, words[i], 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool late = (late_first ^ (alternate & i)) != 0;
        const bool here = r0 + i < rows;
        // The word of columns 2 lane and 2 lane + 1; one column later the upper half joins the next lane's lower one.
        const uint32_t word = late ? __funnelshift_r(words[i], next[i], 16) : words[i];
        unsigned short* dst = line + 2 * lane + late;
        if (here && (late ? pair_at[1] : pair_at[0])) *reinterpret_cast<uint32_t*>(dst) = word;
        if (here && (late ? last_at[1] : last_at[0])) *dst = static_cast<unsigned short>(word);
        if (here && late && first_at) *line = static_cast<unsigned short>(words[i]);
        line += p.out_pitch;
      }
    }
  }
  __syncwarp();
}

template <int kFormat, bool kSplit, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                    const PairParams p) {
  using Tile = PairTile<kFormat>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem_a + Tile::kStages * Tile::kBytesCodes;
  uint8_t* smem_sa = smem_b + Tile::kStages * Tile::kBytesCodes;
  uint8_t* smem_sb = smem_sa + Tile::kStages * Tile::kBytesScaleA;
  uint8_t* staging = smem_sb + Tile::kStages * Tile::kBytesScaleB;
  __shared__ PairBarriers bars;
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t in_cluster = cluster_rank();
  const uint32_t rank = in_cluster & 1;        // in the pair; 0 issues the MMAs
  const uint32_t leader = in_cluster & ~1u;    // cluster rank of the pair's first CTA
  const int slice = kSplit ? static_cast<int>(in_cluster >> 1) : 0;
  const int first_tile = kSplit ? blockIdx.x >> 2 : blockIdx.x >> 1;
  const int tiles = p.tiles_a * p.tiles_b;
  const int tile_step = kSplit ? tiles : gridDim.x >> 1;  // kSplit: one tile per cluster
  const int k_stages = (p.cols_padded + kStageCols - 1) / kStageCols;
  const int kb_begin = kSplit ? k_stages * slice / 2 : 0;
  const int kb_end = kSplit ? k_stages * (slice + 1) / 2 : k_stages;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Tile::kStages; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    mbar_init(&bars.acc_full, 1);
    mbar_init(&bars.acc_free, 2 * kEpilogueWarps);
    bars.abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 0 && elect_one()) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    prefetch_map(&map_sa);
    prefetch_map(&map_sb);
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars.tmem_base, kTmemColumns);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  // Both CTAs' barriers exist and both allocations are done before anybody signals across.
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_base);
  pdl_wait_for_previous_kernel();
  pdl_allow_next_kernel();

  if (warp == 0) {
    const uint32_t full = map_to_cta(smem_addr(&bars.full[0]), leader);
    RingPosition at;
    at.parity = 1;  // the first round finds every stage free
    for (int t = first_tile; t < tiles; t += tile_step) {
      int tile_a, tile_b;
      tile_of(p, t, &tile_a, &tile_b);
      // Rows and scale tiles past the end of an operand read as zeros.
      const int row_a = tile_a * kRowsPair + static_cast<int>(rank) * kRowsCta;
      const int row_b = tile_b * kRowsPair + static_cast<int>(rank) * kRowsCta;
      bool ok = true;
      for (int kb = kb_begin; kb < kb_end; ++kb, at.next(Tile::kStages)) {
        const int s = at.slot;
        ok = warp_wait(&bars.empty[s], at.parity, abort_flag, p.status, kStatusPairWait + 1);
        if (!ok) break;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&bars.full[s], 2 * Tile::kStageBytes);
          const uint32_t bar = full + 8u * static_cast<uint32_t>(s);
          tma_load_2d_pair(smem_a + s * Tile::kBytesCodes, &map_a, kb * kRowBytes, row_a, bar);
          tma_load_2d_pair(smem_b + s * Tile::kBytesCodes, &map_b, kb * kRowBytes, row_b, bar);
          tma_load_2d_pair(smem_sa + s * Tile::kBytesScaleA, &map_sa, kb * Tile::kBytesScaleA / 8, row_a / 128, bar);
          tma_load_2d_pair(smem_sb + s * Tile::kBytesScaleB, &map_sb, kb * Tile::kBytesScaleA / 8, tile_b * 2, bar);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t a_addr = smem_addr(smem_a), b_addr = smem_addr(smem_b);
      const uint32_t sa_addr = smem_addr(smem_sa), sb_addr = smem_addr(smem_sb);
      RingPosition at;
      int n = 0;
      for (int t = first_tile; t < tiles; t += tile_step, ++n) {
        // Tile n may use its accumulator once the epilogue has read the shared columns of tile n - 1 (and with
        // them, in program order, all of tile n - 2).
        bool ok = n == 0 || warp_wait_pair(&bars.acc_free, (n - 1) & 1, abort_flag, p.status, kStatusPairWait + 2);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t acc = tmem + (n & 1) * kSecondAccumulator;
        for (int kb = kb_begin; kb < kb_end; ++kb, at.next(Tile::kStages)) {
          const int s = at.slot;
          ok = warp_wait(&bars.full[s], at.parity, abort_flag, p.status, kStatusPairWait + 3);
          if (!ok) break;
          tc_fence_after_sync();
          if (elect_one()) {
            issue_stage<kFormat, 2, kRowsPair, kRowsPair>(
                acc, tmem + kScaleColumn, a_addr + s * Tile::kBytesCodes, b_addr + s * Tile::kBytesCodes,
                sa_addr + s * Tile::kBytesScaleA, sb_addr + s * Tile::kBytesScaleB, p.cols_padded - kb * kStageCols,
                kb != kb_begin);
            mma_commit_pair(&bars.empty[s], leader);
            if (kb == kb_end - 1) mma_commit_pair(&bars.acc_full, leader);
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
  } else if constexpr (!kSplit) {
    const float alpha = product_factor(p.factor_a, p.factor_b);
    const uint32_t acc_free = map_to_cta(smem_addr(&bars.acc_free), leader);
    const int quarter = warp & 3;
    const int group = (warp - 2) >> 2;
    uint8_t* mine = staging + (warp - 2) * kStagingBytes;
    int n = 0;
    for (int t = first_tile; t < tiles; t += tile_step, ++n) {
      int tile_a, tile_b;
      tile_of(p, t, &tile_a, &tile_b);
      const int row0 = tile_a * kRowsPair + static_cast<int>(rank) * kRowsCta + quarter * 32;
      const int col0 = tile_b * kRowsPair;
      if (!warp_wait(&bars.acc_full, n & 1, abort_flag, p.status, kStatusPairWait + 4)) break;
      tc_fence_after_sync();
      const uint32_t acc = tmem + (n & 1) * kSecondAccumulator + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c = group; c < kRowsPair / kChunk; c += kEpilogueWarps / 4) {
        // The columns shared with the other accumulator come first: the last ones of [0, 256), the first of [208, 464).
        const int first_col = ((n & 1) ? c : kRowsPair / kChunk - 1 - c) * kChunk;
        uint32_t v[2][32];
        tmem_load_32cols(acc + first_col, v[0]);
        tmem_load_32cols(acc + first_col + 32, v[1]);
        tmem_load_wait();
        if (c == group) {  // the shared columns have been read, or this warp has no part in them: tile n - 1 is done
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) arrive_remote(acc_free);
        }
        store_chunk<T>(p, v, alpha, mine, row0, col0 + first_col, lane);
      }
    }
  }

  if constexpr (kSplit) {
    constexpr int kOwnChunks = kRowsPair / kChunk / 2;  // a pair stores half of the columns
    const int quarter = warp & 3;
    const int group = (warp - 2) >> 2;
    const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    bool ok = false;
    if (warp >= 2) {
      ok = warp_wait(&bars.acc_full, 0, abort_flag, p.status, kStatusPairWait + 4);
      tc_fence_after_sync();
    }
    // Every CTA of the cluster has read its ring to the end: the other pair's sums may land there,
    // [own chunks][64 columns][128 rows] FP32.
    __syncwarp();
    cluster_sync_all();
    const uint32_t place = smem_addr(smem) + static_cast<uint32_t>(quarter * 32 + lane) * 4;
    if (ok) {
#pragma unroll 1
      for (int c = group; c < kOwnChunks; c += kEpilogueWarps / 4) {
        const int column = ((1 - slice) * kOwnChunks + c) * kChunk;
        const uint32_t to = map_to_cta(place + static_cast<uint32_t>(c) * (kChunk * kRowsCta * 4), in_cluster ^ 2u);
        uint32_t v[2][32];
        tmem_load_32cols(acc + column, v[0]);
        tmem_load_32cols(acc + column + 32, v[1]);
        tmem_load_wait();
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + j * kRowsCta * 4), "r"(v[j >> 5][j & 31]) : "memory");
        }
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (ok) {
      const float alpha = product_factor(p.factor_a, p.factor_b);
      int tile_a, tile_b;
      tile_of(p, first_tile, &tile_a, &tile_b);
      const int row0 = tile_a * kRowsPair + static_cast<int>(rank) * kRowsCta + quarter * 32;
#pragma unroll 1
      for (int c = group; c < kOwnChunks; c += kEpilogueWarps / 4) {
        const int column = (slice * kOwnChunks + c) * kChunk;
        uint32_t v[2][32];
        tmem_load_32cols(acc + column, v[0]);
        tmem_load_32cols(acc + column + 32, v[1]);
        tmem_load_wait();
        const float* part = reinterpret_cast<const float*>(smem) + c * (kChunk * kRowsCta) + quarter * 32 + lane;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          v[j >> 5][j & 31] = __float_as_uint(__uint_as_float(v[j >> 5][j & 31]) + part[j * kRowsCta]);
        }
        store_chunk<T>(p, v, alpha, staging + (warp - 2) * kStagingBytes, row0, tile_b * kRowsPair + column, lane);
      }
    }
  }

  if (*abort_flag) {
    // Give copies that are still in flight time to land before the shared memory is released.
    const long long start = clock64();
    while (clock64() - start < 200000) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  // Neither CTA may leave (or free tensor memory) while the other could still signal it.
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, kTmemColumns);
  }
}

// Scale tiles as rows of 8-byte elements, one row per 128 rows of the operand.
template <int kFormat>
bool encode_scales(CUtensorMap* map, const uint8_t* scales, int64_t rows, int64_t K, int box_rows) {
  const int64_t pitch = fp4::scale_tiles(K, kFormat) * 512;
  const uint64_t dims[2] = {static_cast<uint64_t>(pitch / 8), static_cast<uint64_t>((rows + 127) / 128)};
  const uint64_t strides[1] = {static_cast<uint64_t>(pitch)};
  const uint32_t box[2] = {PairTile<kFormat>::kBytesScaleA / 8, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, scales, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int kFormat, bool kSplit, typename T>
cudaError_t launch(const Fp4Operand& a, const Fp4Operand& b, void* out, int64_t K, int sm_count, int* status,
                   cudaStream_t stream) {
  using Tile = PairTile<kFormat>;
  const int64_t pitch = fp4::code_pitch(K);
  CUtensorMap map_a, map_b, map_sa, map_sb;
  if (!encode_codes(&map_a, a.codes, a.rows, pitch, kRowsCta) || !encode_codes(&map_b, b.codes, b.rows, pitch, kRowsCta) ||
      !encode_scales<kFormat>(&map_sa, a.scales, a.rows, K, 1) || !encode_scales<kFormat>(&map_sb, b.scales, b.rows, K, 2)) {
    return cudaErrorInvalidValue;
  }
  PairParams params;
  params.factor_a = a.factor;
  params.factor_b = b.factor;
  params.out = out;
  params.out_pitch = b.rows;
  params.rows_a = static_cast<int>(a.rows);
  params.rows_b = static_cast<int>(b.rows);
  params.cols_padded = static_cast<int>(fp4::padded_cols(K));
  const int64_t tiles_a = (a.rows + kRowsPair - 1) / kRowsPair;
  const int64_t tiles_b = (b.rows + kRowsPair - 1) / kRowsPair;
  if (tiles_a * tiles_b > 0x3fffffffLL) return cudaErrorInvalidConfiguration;
  params.tiles_a = static_cast<int>(tiles_a);
  params.tiles_b = static_cast<int>(tiles_b);
  const uintptr_t out_bits = reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(b.rows * sizeof(T));
  params.out_bytes = out_bits % 16 == 0 ? 16 : out_bits % 8 == 0 ? 8 : 2;
  params.status = status;

  auto kernel = fp4_pair_kernel<kFormat, kSplit, T>;
  static bool configured[64] = {};
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device < 0 || device >= 64 || !configured[device]) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile::kSmemBytes);
    if (err != cudaSuccess) return err;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  const int64_t slots = sm_count >= 2 ? sm_count / 2 : 1;
  int64_t pairs = tiles_a * tiles_b < slots ? tiles_a * tiles_b : slots;
  if (kSplit) pairs = 2 * tiles_a * tiles_b;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Tile::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kSplit ? 4 : 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1] = fp4::programmatic_launch();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_sa, map_sb, params);
}

template <int kFormat, typename T>
cudaError_t pair_product(const Fp4Operand& a, const Fp4Operand& b, void* out, int64_t K, int sm_count, int* status,
                         cudaStream_t stream) {
  const int64_t tiles = ((a.rows + kRowsPair - 1) / kRowsPair) * ((b.rows + kRowsPair - 1) / kRowsPair);
  const bool split = 2 * tiles <= sm_count / 2 && fp4::padded_cols(K) > 3 * kStageCols;
  return split ? launch<kFormat, true, T>(a, b, out, K, sm_count, status, stream)
               : launch<kFormat, false, T>(a, b, out, K, sm_count, status, stream);
}

}  // namespace

cudaError_t launch_fp4_pair(const Fp4Operand& a, const Fp4Operand& b, int format, void* out, int out_type, int64_t K,
                            int sm_count, int* status_word, cudaStream_t stream) {
  if (format == fp4::kNv) {
    return out_type == kTypeBf16 ? pair_product<fp4::kNv, __nv_bfloat16>(a, b, out, K, sm_count, status_word, stream)
                                 : pair_product<fp4::kNv, __half>(a, b, out, K, sm_count, status_word, stream);
  }
  return out_type == kTypeBf16 ? pair_product<fp4::kMx, __nv_bfloat16>(a, b, out, K, sm_count, status_word, stream)
                               : pair_product<fp4::kMx, __half>(a, b, out, K, sm_count, status_word, stream);
}

}  // namespace lbl
