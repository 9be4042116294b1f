// Product of a microscaled FP4 weight with few rows of activations: y[q, p] = sum_k x[q, k] w[p, k].
//
// Bound by the weight's bytes, so the weight takes the M side of the MMA (128 rows per CTA, streamed once
// through a ring of TMA stages) and the activations its N side (kQ = 16 .. 256 of them).  K is cut into
// as many slices as fill the SMs; the CTAs of one row block's slices form a cluster, leave their FP32
// partial tiles in shared memory and add them in slice order through distributed shared memory: no
// scratch, no atomics, the same bits every time.
//
//   kFused (kQ <= 32): the activations come in 16 bits and every CTA quantises its slice of them into shared
//   memory while its first weight stages are on their way (the rounding of fp4_common.cuh), one launch
//   for the whole linear layer.  Otherwise both operands are codes and tiled scales.
//
//   warp 0      copies: codes by TMA (rows of 128 bytes, 128-byte swizzle), scale tiles by bulk copies
//   warp 1      scales to tensor memory, MMAs
//   the others  quantisation (kFused), epilogue
#include "fp4_tc.cuh"

namespace lbl {
namespace {

constexpr int kP = 128;
constexpr int kMaxStages = 8;
constexpr int kMaxSplit = 8;
constexpr int kStatusStreamWait = 600;

struct StreamParams {
  const uint8_t* sf_p;
  const uint8_t* sf_q;
  const float* factor_p;
  const float* factor_q;
  const void* x;  // kFused: 16-bit activations
  int64_t x_stride;
  void* out;
  int64_t out_pitch;
  int rows_p, rows_q;
  int cols;         // K
  int cols_padded;  // to 32
  int scale_tiles;  // along K
  int out_words;    // rows of out start on eight bytes
  int stages;
  int split;        // CTAs of a cluster, a power of two
  int split_shift;  // its logarithm
  int x_access;     // how rows of x may be read
  int early_weight;  // fetch the weight before the kernel in front is complete
  int receive_offset;  // where partial sums arrive in shared memory; 0: over the ring
  int* status;
};

struct StreamBarriers {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
};

template <int kFormat, int kQ, bool kFused>
struct StreamTile {
  static constexpr int kTiles = kStageCols / fp4::Format<kFormat>::kTileCols;
  static constexpr int kQBlocks = (kQ + 127) / 128;
  static constexpr int kBytesP = kP * kRowBytes;
  static constexpr int kBytesQ = kQ * kRowBytes;
  static constexpr int kBytesScaleP = kTiles * 512;
  static constexpr int kBytesScaleQ = kTiles * 512 * kQBlocks;
  static constexpr int kStageBytes = kBytesP + kBytesScaleP + (kFused ? 0 : kBytesQ + kBytesScaleQ);
  static constexpr int kPartialBytes = kP * kQ * 4;
  static constexpr int kColumns = kQ + kTiles * 4 * (1 + kQBlocks);
  static constexpr int kTmemColumns = kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
  static constexpr int kWorkers = 8;  // warps
  static constexpr int kThreads = 32 * (2 + kWorkers);
};

// Rounds this CTA's slice of the activations: sixteen columns of a row per thread and step, stage by
// stage, into the swizzled code tiles and the scale tiles the MMAs read.  Rows past rows_q are left as
// they are: they only reach columns of the accumulator that nobody reads.
template <int kFormat, int kQ, typename T>
__device__ __forceinline__ void quantise_slice(const StreamParams& p, int k_begin, int stages_here, uint8_t* codes,
                                               uint8_t* scales, int worker, int workers) {
  using Tile = StreamTile<kFormat, kQ, true>;
  const fp4::TensorFactor factor = fp4::tensor_factor(kFormat == fp4::kNv ? p.factor_q : nullptr);
  const int per_stage = p.rows_q * 16;  // even: both halves of an MXFP4 block are in one warp
  const int total = stages_here * per_stage;
  const int rounds = (total + workers - 1) / workers;
  for (int i = 0; i < rounds; ++i) {
    const int item = i * workers + worker;
    const bool have = item < total;
    const int stage = have ? item / per_stage : 0;
    const int rest = item - stage * per_stage;
    const int row = have ? rest >> 4 : 0;
    const int unit = rest & 15;
    const int col = (k_begin + stage) * kStageCols + unit * 16;
    const int valid = have ? min(16, max(0, p.cols - col)) : 0;
    const T* src = static_cast<const T*>(p.x) + row * p.x_stride + col;
    fp4::Sixteen<T> v;
    if (valid == 16 && p.x_access != fp4::kRowsAny) {
      v.load_vector(src, p.x_access);
    } else {
      v.load_masked(src, valid);
    }
    uint32_t amax = v.amax_bits();
    fp4::BlockStep step;
    if constexpr (kFormat == fp4::kMx) {
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      step = fp4::mx_step(amax);
    } else {
      step = fp4::nv_step(amax, factor);
    }
    const uint2 out = fp4::round_sixteen<kFormat>(v, step);
    if (have) {
      const uint32_t chunk = unit >> 1;
      uint8_t* dst = codes + stage * Tile::kBytesQ + (row >> 3) * 1024 + (row & 7) * 128 +
                     ((chunk ^ (row & 7)) << 4) + (unit & 1) * 8;
      *reinterpret_cast<uint2*>(dst) = out;
      const int block = kFormat == fp4::kMx ? unit >> 1 : unit;
      scales[stage * Tile::kBytesScaleQ + (block >> 2) * 512 + row * 16 + (block & 3)] = static_cast<uint8_t>(step.byte);
    }
  }
}

template <int kFormat, int kQ, bool kFused, typename T>
__global__ void __launch_bounds__(StreamTile<kFormat, kQ, kFused>::kThreads, 2)
    fp4_stream_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                      const StreamParams p) {
  using Tile = StreamTile<kFormat, kQ, kFused>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ StreamBarriers bars;
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = p.split > 1 ? cluster_rank() : 0;
  const int p0 = (blockIdx.x >> p.split_shift) * kP;
  const int q0 = blockIdx.y * kQ;
  const int used = min(kQ, p.rows_q - q0);  // activation rows of this tile
  const int k_stages = (p.cols_padded + kStageCols - 1) / kStageCols;
  const int k_begin = static_cast<int>(static_cast<int64_t>(k_stages) * rank >> p.split_shift);
  const int k_end = static_cast<int>(static_cast<int64_t>(k_stages) * (rank + 1) >> p.split_shift);
  const int stages_here = k_end - k_begin;

  // Code tiles first (swizzled tiles start on 1024 bytes).  kFused: Q holds the whole slice.
  const int q_slots = kFused ? stages_here : p.stages;
  uint8_t* smem_p = smem;
  uint8_t* smem_q = smem_p + p.stages * Tile::kBytesP;
  uint8_t* smem_sp = smem_q + q_slots * Tile::kBytesQ;
  uint8_t* smem_sq = smem_sp + p.stages * Tile::kBytesScaleP;

  const int tile_step = Tile::kTiles;
  auto load_p = [&](int i, int s) {
    const int kb = k_begin + i;
    const uint32_t bytes = min(tile_step, p.scale_tiles - kb * tile_step) * 512;
    int blocks_q = 0;
    if (!kFused) {
      for (int b = 0; b < Tile::kQBlocks; ++b) blocks_q += b * 128 < used ? 1 : 0;
    }
    mbar_arrive_expect_tx(&bars.full[s], Tile::kBytesP + bytes + (kFused ? 0 : Tile::kBytesQ + bytes * blocks_q));
    tma_load_2d(smem_p + s * Tile::kBytesP, &map_p, kb * kRowBytes, p0, &bars.full[s]);
    bulk_load(smem_sp + s * Tile::kBytesScaleP,
              p.sf_p + (static_cast<int64_t>(p0 / 128) * p.scale_tiles + kb * tile_step) * 512, bytes, &bars.full[s]);
  };
  auto load_q = [&](int i, int s) {
    const int kb = k_begin + i;
    const uint32_t bytes = min(tile_step, p.scale_tiles - kb * tile_step) * 512;
    tma_load_2d(smem_q + s * Tile::kBytesQ, &map_q, kb * kRowBytes, q0, &bars.full[s]);
    for (int b = 0; b < Tile::kQBlocks && b * 128 < used; ++b) {
      bulk_load(smem_sq + s * Tile::kBytesScaleQ + b * tile_step * 512,
                p.sf_q + (static_cast<int64_t>(q0 / 128 + b) * p.scale_tiles + kb * tile_step) * 512, bytes, &bars.full[s]);
    }
  };
  const int ahead = min(p.stages, stages_here);

  // The weight's first stages are on their way before anything else is set up.  The activations may come from the
  // kernel in front of this one; the weight does not when that is the call's own quantiser or the caller says so.
  if (warp == 0) {
    if (elect_one()) {
      for (int s = 0; s < p.stages; ++s) {
        mbar_init(&bars.full[s], 1);
        mbar_init(&bars.empty[s], 1);
      }
      mbar_init(&bars.done, 1);
      bars.abort_flag = 0;
      mbar_init_fence();
      if (!p.early_weight) pdl_wait_for_previous_kernel();
      for (int i = 0; i < ahead; ++i) load_p(i, i);
      if constexpr (!kFused) {
        pdl_wait_for_previous_kernel();
        for (int i = 0; i < ahead; ++i) load_q(i, i);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(&bars.tmem_base, Tile::kTmemColumns);
    tmem_relinquish();
  } else {
    pdl_wait_for_previous_kernel();
    if constexpr (kFused) {
      quantise_slice<kFormat, kQ, T>(p, k_begin, stages_here, smem_q, smem_sq, threadIdx.x - 64, Tile::kWorkers * 32);
      fence_async_proxy();
    }
  }
  // A partial sum may go to a neighbour once it has started (its receiving memory is its own) or, where that
  // memory is the ring's, once its MMAs are complete.
  if (p.split > 1 && p.receive_offset != 0) cluster_arrive();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_base);
  pdl_allow_next_kernel();

  if (warp == 0) {
    RingPosition at;
    for (int i = ahead; i < stages_here; ++i, at.next(p.stages)) {
      if (!warp_wait(&bars.empty[at.slot], at.parity, abort_flag, p.status, kStatusStreamWait + 1)) break;
      if (elect_one()) {
        load_p(i, at.slot);
        if constexpr (!kFused) load_q(i, at.slot);
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    const uint32_t p_addr = smem_addr(smem_p), q_addr = smem_addr(smem_q);
    const uint32_t sp_addr = smem_addr(smem_sp), sq_addr = smem_addr(smem_sq);
    RingPosition at;
    for (int i = 0; i < stages_here; ++i, at.next(p.stages)) {
      const int s = at.slot;
      if (!warp_wait(&bars.full[s], at.parity, abort_flag, p.status, kStatusStreamWait + 2)) break;
      tc_fence_after_sync();
      const int sq = kFused ? i : s;
      if (elect_one()) {
        issue_stage<kFormat, 1, kP, kQ>(tmem, tmem + kQ, p_addr + s * Tile::kBytesP, q_addr + sq * Tile::kBytesQ,
                                        sp_addr + s * Tile::kBytesScaleP, sq_addr + sq * Tile::kBytesScaleQ,
                                        p.cols_padded - (k_begin + i) * kStageCols, i != 0);
        mma_commit(&bars.empty[s]);
        if (i == stages_here - 1) mma_commit(&bars.done);
      }
      __syncwarp();
    }
  }
  // When this barrier has passed every MMA of the CTA is complete and every copy has been read.
  warp_wait(&bars.done, 0, abort_flag, p.status, kStatusStreamWait + 3);
  tc_fence_after_sync();
  if (*abort_flag) {
    // Give copies that are still in flight time to land before the shared memory is used otherwise.
    const long long start = clock64();
    while (clock64() - start < 200000) {
    }
  }
  __syncthreads();
  if (p.split > 1) {
    if (p.receive_offset == 0) cluster_arrive();
    cluster_wait();
  }

  // Row q of the tile is summed by CTA q % split, which receives [slice][q / split][128] FP32.
  const int slots = kQ >> p.split_shift;
  uint8_t* received = smem + p.receive_offset;
  if (warp >= 2) {
    // Two warps per quarter of the lanes, 32 columns in turn.
    const int quarter = warp & 3;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t mine = smem_addr(received) + (rank * slots * kP + quarter * 32 + lane) * 4;
    for (int c0 = ((warp - 2) >> 2) * 32; c0 < used; c0 += 64) {
      uint32_t v[32];
      tmem_load_32cols(taddr + c0, v);
      tmem_load_wait();
      if (p.split == 1) {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          if (c0 + c >= used) break;
          asm volatile("st.shared::cta.b32 [%0], %1;" ::"r"(mine + (c0 + c) * kP * 4), "r"(v[c]) : "memory");
        }
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int q = c0 + c;
          if (q >= used) break;
          const uint32_t to = map_to_cta(mine + (q >> p.split_shift) * kP * 4, q & (p.split - 1));
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(v[c]) : "memory");
        }
      }
    }
  }
  tc_fence_before_sync();
  if (p.split > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, Tile::kTmemColumns);
  }

  // Four neighbouring rows of the weight and one activation row per thread and step; slices in their order.
  const float alpha = product_factor(p.factor_p, p.factor_q);
  T* out = static_cast<T*>(p.out);
  const int my_rows = used > static_cast<int>(rank) ? (used - static_cast<int>(rank) + p.split - 1) >> p.split_shift : 0;
  const int stride = slots * (kP / 4);
#pragma unroll 4
  for (int item = threadIdx.x; item < my_rows * (kP / 4); item += Tile::kThreads) {
    const int slot = item / (kP / 4);
    const int row = (item % (kP / 4)) * 4;
    const float4* part = reinterpret_cast<const float4*>(received) + item;
    float4 sum = part[0];
    for (int r = 1; r < p.split; ++r) {
      const float4 v = part[r * stride];
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    const int left = p.rows_p - (p0 + row);
    T* dst = out + (q0 + (slot << p.split_shift) + rank) * p.out_pitch + p0 + row;
    const uint32_t y[2] = {two_rounded<T>(sum.x * alpha, sum.y * alpha), two_rounded<T>(sum.z * alpha, sum.w * alpha)};
    if (p.out_words && left >= 4) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < left) reinterpret_cast<unsigned short*>(dst)[i] = static_cast<unsigned short>(y[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

constexpr int kSmemLimit = 226 * 1024;     // dynamic shared memory of a CTA
constexpr int kSmemPerSm = 228 * 1024;
constexpr int kStaticSmem = (sizeof(StreamBarriers) + 127) / 128 * 128;
constexpr int kFusedRows = 16;
constexpr int kRingStages = 6;

// Slices of K, each on a CTA of its own: doubled while the CTAs still fit the SMs once and a slice keeps two stages
// (four with more than 32 activation rows, whose sums cost more to join), and once more, to two CTAs on some SMs, while
// it keeps six (eight).  Measured, us, 1 / 2 / 4 / 8 slices: 1 row, 32 row blocks of 16 stages 6.2 / 5.5 / 4.3 / 4.4,
// of 48 stages 13.8 / 9.3 / 6.7 / 6.5; 32 rows, 48 blocks of 16 stages 7.5 / 6.5 / 9.8 / 9.5; 64 rows, 32 blocks of 16
// stages 7.3 / 6.8 / 5.6 / 6.6; 77 rows, 40 blocks of 4 stages 5.1 / 5.6 / 6.3 / 6.3; 100 rows, 64 blocks of 32 stages
// 17.3 / 13.8 / 12.4 / 20.7; 16 rows, 192 blocks of 16 stages 13.7 / 17.2 / 20.6 / 29.9.
int choose_split(int64_t tiles, int k_stages, int tile_rows, int sm_count) {
  const int least = tile_rows <= 32 ? 2 : 4;  // stages of a slice
  const int least_beyond = tile_rows <= 32 ? 6 : 8;
  int split = 1;
  while (split < kMaxSplit && ((k_stages >= 2 * split * least && 2 * tiles * split <= sm_count) ||
                               (k_stages >= 2 * split * least_beyond && tiles * split < sm_count))) {
    split *= 2;
  }
  return split;
}

int stages_of(int64_t K) { return static_cast<int>((fp4::padded_cols(K) + kStageCols - 1) / kStageCols); }

template <int kFormat, int kQ, bool kFused, typename T>
cudaError_t launch(const Fp4Operand& w, const Fp4Operand& x, const void* raw, int64_t raw_stride, void* out, int64_t K,
                   int sm_count, int* status, bool early_weight, cudaStream_t stream) {
  using Tile = StreamTile<kFormat, kQ, kFused>;
  const int64_t pitch = fp4::code_pitch(K);
  CUtensorMap map_p, map_q;
  if (!encode_codes(&map_p, w.codes, w.rows, pitch, kP)) return cudaErrorInvalidValue;
  if constexpr (kFused) {
    map_q = map_p;  // not used
  } else {
    if (!encode_codes(&map_q, x.codes, x.rows, pitch, kQ)) return cudaErrorInvalidValue;
  }
  const int64_t blocks_p = (w.rows + kP - 1) / kP;
  const int64_t blocks_q = (x.rows + kQ - 1) / kQ;
  const int k_stages = stages_of(K);
  const int split = choose_split(blocks_p * blocks_q, k_stages, kQ, sm_count);
  const int slice = (k_stages + split - 1) / split;

  StreamParams params;
  params.sf_p = w.scales;
  params.sf_q = x.scales;
  params.factor_p = w.factor;
  params.factor_q = x.factor;
  params.x = raw;
  params.x_stride = raw_stride;
  params.out = out;
  params.out_pitch = w.rows;
  params.rows_p = static_cast<int>(w.rows);
  params.rows_q = static_cast<int>(x.rows);
  params.cols = static_cast<int>(K);
  params.cols_padded = static_cast<int>(fp4::padded_cols(K));
  params.scale_tiles = static_cast<int>(fp4::scale_tiles(K, kFormat));
  params.out_words = w.rows % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
  params.split = split;
  params.split_shift = 0;
  while ((1 << params.split_shift) < split) ++params.split_shift;
  params.x_access = fp4::row_access(raw, raw_stride * 2);
  params.status = status;
  // Received partial sums have memory of their own while they are small, and lie over the ring otherwise.
  const bool own_memory = split > 1 && kQ <= 32;
  const int fixed = 1024 + (kFused ? slice * (Tile::kBytesQ + Tile::kBytesScaleQ) : 0) + (own_memory ? Tile::kPartialBytes : 0);
  // All CTAs on the SMs at once where that leaves two stages: a CTA that has to wait for another one's end starts
  // its pipeline cold.  At least two on an SM in any case, for the next kernel of the stream.
  const int64_t ctas = blocks_p * blocks_q * split;
  const int64_t per_sm = ctas <= 2 * sm_count ? 2 : ctas <= 3 * sm_count ? 3 : 4;
  const int budget = static_cast<int>(kSmemPerSm / per_sm) - 1024 - kStaticSmem;  // the driver takes 1 KB of each CTA's share
  int stages = slice < kRingStages ? slice : kRingStages;
  while (stages > 2 && fixed + stages * Tile::kStageBytes > budget) --stages;
  params.stages = stages;
  int smem = fixed + stages * Tile::kStageBytes;
  params.receive_offset = own_memory ? smem - 1024 - Tile::kPartialBytes : 0;
  if (smem < Tile::kPartialBytes + 1024) smem = Tile::kPartialBytes + 1024;
  if (smem > kSmemLimit) return cudaErrorInvalidValue;

  auto kernel = fp4_stream_kernel<kFormat, kQ, kFused, T>;
  static bool configured[64] = {};
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device < 0 || device >= 64 || !configured[device]) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (err != cudaSuccess) return err;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  if (blocks_q > 65535 || blocks_p * split > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks_p * split), static_cast<unsigned>(blocks_q));
  cfg.blockDim = dim3(Tile::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int attrs = 0;
  if (split > 1) {
    attr[attrs].id = cudaLaunchAttributeClusterDimension;
    attr[attrs].val.clusterDim.x = split;
    attr[attrs].val.clusterDim.y = 1;
    attr[attrs].val.clusterDim.z = 1;
    ++attrs;
  }
  attr[attrs++] = fp4::programmatic_launch();
  cfg.attrs = attr;
  cfg.numAttrs = attrs;
  return cudaLaunchKernelEx(&cfg, kernel, map_p, map_q, params);
}

}  // namespace

template <int kFormat, typename T>
static cudaError_t stream_product(const Fp4Operand& a, const Fp4Operand& b, void* out, int64_t K, int sm_count,
                                  int* status, bool early_weight, cudaStream_t stream) {
  if (a.rows <= 16) return launch<kFormat, 16, false, T>(b, a, nullptr, 0, out, K, sm_count, status, early_weight, stream);
  if (a.rows <= 32) return launch<kFormat, 32, false, T>(b, a, nullptr, 0, out, K, sm_count, status, early_weight, stream);
  if (a.rows <= 64) return launch<kFormat, 64, false, T>(b, a, nullptr, 0, out, K, sm_count, status, early_weight, stream);
  return launch<kFormat, 128, false, T>(b, a, nullptr, 0, out, K, sm_count, status, early_weight, stream);
}

cudaError_t launch_fp4_stream(const Fp4Operand& a, const Fp4Operand& b, int format, void* out, int out_type, int64_t K,
                              int sm_count, int* status_word, bool early_weight, cudaStream_t stream) {
  if (format == fp4::kNv) {
    return out_type == kTypeBf16 ? stream_product<fp4::kNv, __nv_bfloat16>(a, b, out, K, sm_count, status_word, early_weight, stream)
                                 : stream_product<fp4::kNv, __half>(a, b, out, K, sm_count, status_word, early_weight, stream);
  }
  return out_type == kTypeBf16 ? stream_product<fp4::kMx, __nv_bfloat16>(a, b, out, K, sm_count, status_word, early_weight, stream)
                               : stream_product<fp4::kMx, __half>(a, b, out, K, sm_count, status_word, early_weight, stream);
}

// Every CTA rounds its slice of the activations itself: worth a launch while that is four rounds of the quantising warps
// (three where CTAs share an SM) and the slice leaves three stages to the ring.  Measured, us, one launch / two, NVFP4:
// 4096 x 4096 (slices of 4 stages, 128 CTAs) 1 row 4.5 / 6.9, 8 rows 5.6 / 6.9, 16 rows 6.9 / 7.0; 6144 x 4096 (8, 96
// CTAs) 8 rows 7.8 / 7.6, 12 rows 8.8 / 7.7; 8192 x 8192 (8, 256 CTAs) 1 row 9.4 / 12.5, 6 rows 11.2 / 12.5, 12 rows 13.5
// / 12.5; 5120 x 12288 (12, 160 CTAs) 1 row 9.7 / 12.2, 6 rows 12.8 / 12.2; 24576 x 4096 (16, 192 CTAs; two stages left)
// 1 row 14.7 / 13.9, in MXFP4 (smaller scale tiles, three stages) 11.7 / 13.2.
bool fp4_fused_supports(int64_t M, int64_t N, int64_t K, int format, int sm_count) {
  if (M > kFusedRows) return false;
  const int64_t k_stages = stages_of(K);
  const int64_t blocks = (N + kP - 1) / kP;
  const int split = choose_split(blocks, static_cast<int>(k_stages), kFusedRows, sm_count);
  const int64_t slice = (k_stages + split - 1) / split;
  if (blocks * split <= sm_count) return slice <= 16 && M * slice <= 64;
  return slice <= (format == fp4::kNv ? 12 : 16) && M * slice <= 48;
}

cudaError_t launch_fp4_fused_linear(const void* x, int x_type, int64_t x_stride, int64_t M, const float* x_factor,
                                    const Fp4Operand& w, int format, void* out, int64_t K, int sm_count,
                                    int* status_word, bool early_weight, cudaStream_t stream) {
  const Fp4Operand a = {nullptr, nullptr, x_factor, M};
  if (format == fp4::kNv) {
    return x_type == kTypeBf16
               ? launch<fp4::kNv, kFusedRows, true, __nv_bfloat16>(w, a, x, x_stride, out, K, sm_count, status_word, early_weight, stream)
               : launch<fp4::kNv, kFusedRows, true, __half>(w, a, x, x_stride, out, K, sm_count, status_word, early_weight, stream);
  }
  return x_type == kTypeBf16
             ? launch<fp4::kMx, kFusedRows, true, __nv_bfloat16>(w, a, x, x_stride, out, K, sm_count, status_word, early_weight, stream)
             : launch<fp4::kMx, kFusedRows, true, __half>(w, a, x, x_stride, out, K, sm_count, status_word, early_weight, stream);
}

}  // namespace lbl
