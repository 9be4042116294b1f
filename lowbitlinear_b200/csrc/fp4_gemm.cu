// Product of two microscaled FP4 operands on the block-scaled tensor cores of sm_100a.
//
//   out[i, j] = T( ga gb sum_k a[i, k] b[j, k] ),   a and b as codes and tiled scales (fp4_common.cuh)
//
// tcgen05.mma reads E2M1 codes from shared memory and the block scales from tensor memory: the
// products and their scaling by powers of two (MXFP4) or E4M3 numbers (NVFP4) are exact, sums are FP32.
// One CTA computes a tile of 128 rows of operand P by kQ rows of operand Q; P is `a` when there are many
// rows of it and `b` (the weights) when there are few, the epilogue transposing the tile then.
//
//   warp 0      TMA: per 256 columns of K the codes of both operands (rows of 128 bytes, 128-byte swizzle) and
//               their scale tiles (plain bulk copies: the tiles of a row block follow each other along K)
//   warp 1      tcgen05.cp of the scale tiles into tensor memory, then the MMAs (64 columns each); both run in
//               issue order, so the scales need no buffering
//   warps 2-5   epilogue
//
// Columns past K are zero codes (row padding) or outside the tensor (the copy engine fills zeros); the
// last stage issues only the MMAs that have columns, so no scale byte is used that was not loaded.
#include "fp4_common.cuh"
#include "kernels.h"
#include "tc_common.cuh"
#include "tensor_map.h"

namespace lbl {
namespace {

constexpr int kP = 128;           // rows of operand P per tile: the lanes of the accumulator
constexpr int kStageCols = 256;   // columns of K per stage
constexpr int kRowBytes = kStageCols / 2;
constexpr int kThreads = 192;
constexpr int kStatusFp4Wait = 600;
constexpr int kMaxStages = 8;

struct Fp4Params {
  const uint8_t* sf_p;  // tiled scales
  const uint8_t* sf_q;
  const float* factor_p;  // FP32 tensor factors, null = 1
  const float* factor_q;
  void* out;
  int64_t out_pitch;  // elements between rows of out
  int rows_p, rows_q;
  int cols;         // padded K
  int scale_tiles;  // along K
  int stages;
  int* status;
};

struct Fp4Barriers {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
};

// Untiled bulk copy of `bytes` (a multiple of 16) from global to shared memory.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// 512 bytes of scales (32 rows of 16 bytes, four 128-byte groups of eight rows) into four columns of
// tensor memory, the same in each quarter of the lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem_byte_addr) {
  const uint32_t lo = (smem_byte_addr >> 4) & 0x3FFFu;
  const uint32_t hi = (128u >> 4) | (1u << 14);  // stride between the groups, descriptor version; no swizzle
  const uint64_t desc = (static_cast<uint64_t>(hi) << 32) | lo;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Instruction descriptor of the block-scaled kinds: A = B = E2M1 (1 at bits 7 and 10), both K-major, N / 8
// at bits 17-22, scale type at bit 23 (1: E8M0), M / 128 at bits 27-28, which bytes of the scale
// columns to use at bits 4-5 (B) and 29-30 (A).
template <int kFormat>
__host__ __device__ constexpr uint32_t fp4_instr_desc(uint32_t m, uint32_t n, uint32_t scale_id) {
  return (scale_id << 4) | (1u << 7) | (1u << 10) | ((n / 8) << 17) | ((kFormat == fp4::kMx ? 1u : 0u) << 23) |
         ((m / 128) << 27) | (scale_id << 29);
}

template <int kFormat>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t sf_a, uint32_t sf_b, uint32_t accumulate) {
  if constexpr (kFormat == fp4::kMx) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sf_a), "r"(sf_b), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sf_a), "r"(sf_b), "r"(accumulate)
        : "memory");
  }
}

template <typename T>
__device__ __forceinline__ T rounded(float v);
template <>
__device__ __forceinline__ __half rounded<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <int kFormat, int kQ>
struct Fp4Tile {
  static constexpr int kTilesPerStage = kStageCols / fp4::Format<kFormat>::kTileCols;  // scale tiles: 2 or 4
  static constexpr int kQBlocks = (kQ + 127) / 128;
  static constexpr int kBytesP = kP * kRowBytes;
  static constexpr int kBytesQ = (kQ < 8 ? 8 : kQ) * kRowBytes;
  static constexpr int kBytesScales = kTilesPerStage * 512 * (1 + kQBlocks);
  static constexpr int kStageBytes = kBytesP + kBytesQ + kBytesScales;
  static constexpr int kScaleColumns = kTilesPerStage * 4 * (1 + kQBlocks);
  static constexpr int kTmemColumns = kQ + kScaleColumns <= 64    ? 64
                                      : kQ + kScaleColumns <= 128 ? 128
                                      : kQ + kScaleColumns <= 256 ? 256
                                                                  : 512;
};

template <int kFormat, int kQ, bool kTransposed, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                    const Fp4Params p) {
  using Tile = Fp4Tile<kFormat, kQ>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // Ring of codes first (swizzled tiles start on 1024 bytes), then the scales.
  uint8_t* smem_p = smem;
  uint8_t* smem_q = smem_p + p.stages * Tile::kBytesP;
  uint8_t* smem_s = smem_q + p.stages * Tile::kBytesQ;
  __shared__ Fp4Barriers bars;
  volatile int* abort_flag = &bars.abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int p0 = blockIdx.x * kP;
  const int q0 = blockIdx.y * kQ;
  const int k_stages = (p.cols + kStageCols - 1) / kStageCols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&bars.full[s], 1);
      mbar_init(&bars.empty[s], 1);
    }
    mbar_init(&bars.done, 1);
    bars.abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    tmem_alloc(&bars.tmem_base, Tile::kTmemColumns);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_base);

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = 0; kb < k_stages; ++kb) {
        const int s = kb % p.stages;
        const int round = kb / p.stages;
        if (round > 0) mbar_wait_bounded(&bars.empty[s], (round - 1) & 1, abort_flag, p.status, kStatusFp4Wait + 1);
        if (*abort_flag) break;
        const int tile0 = kb * Tile::kTilesPerStage;
        const int tiles = min(Tile::kTilesPerStage, p.scale_tiles - tile0);
        const uint32_t bytes = tiles * 512;
        int blocks_q = 0;
        for (int b = 0; b < Tile::kQBlocks; ++b) blocks_q += q0 + b * 128 < p.rows_q ? 1 : 0;
        mbar_arrive_expect_tx(&bars.full[s], Tile::kBytesP + Tile::kBytesQ + bytes * (1 + blocks_q));
        tma_load_2d(smem_p + s * Tile::kBytesP, &map_p, kb * kRowBytes, p0, &bars.full[s]);
        tma_load_2d(smem_q + s * Tile::kBytesQ, &map_q, kb * kRowBytes, q0, &bars.full[s]);
        uint8_t* sf = smem_s + s * Tile::kBytesScales;
        bulk_load(sf, p.sf_p + (static_cast<int64_t>(p0 / 128) * p.scale_tiles + tile0) * 512, bytes, &bars.full[s]);
        for (int b = 0; b < blocks_q; ++b) {
          bulk_load(sf + (1 + b) * Tile::kTilesPerStage * 512,
                    p.sf_q + (static_cast<int64_t>(q0 / 128 + b) * p.scale_tiles + tile0) * 512, bytes, &bars.full[s]);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t sf_p = tmem + kQ;
      const uint32_t sf_q = sf_p + Tile::kTilesPerStage * 4;
      for (int kb = 0; kb < k_stages; ++kb) {
        const int s = kb % p.stages;
        mbar_wait_bounded(&bars.full[s], (kb / p.stages) & 1, abort_flag, p.status, kStatusFp4Wait + 2);
        if (*abort_flag) break;
        tc_fence_after_sync();
        const int tiles = min(Tile::kTilesPerStage, p.scale_tiles - kb * Tile::kTilesPerStage);
        const uint32_t sf = smem_addr(smem_s + s * Tile::kBytesScales);
        for (int t = 0; t < tiles; ++t) {
          scales_to_tmem(sf_p + t * 4, sf + t * 512);
          for (int b = 0; b < Tile::kQBlocks; ++b) {
            scales_to_tmem(sf_q + t * 4 * Tile::kQBlocks + b * 4, sf + ((1 + b) * Tile::kTilesPerStage + t) * 512);
          }
        }
        const uint32_t a_addr = smem_addr(smem_p + s * Tile::kBytesP);
        const uint32_t b_addr = smem_addr(smem_q + s * Tile::kBytesQ);
        const int steps = min(kStageCols / 64, (p.cols - kb * kStageCols + 63) / 64);
        for (int j = 0; j < steps; ++j) {
          // MXFP4: a scale tile serves two MMAs, bytes 0-1 and 2-3; NVFP4: one.
          const int t = kFormat == fp4::kMx ? j / 2 : j;
          const uint32_t id = kFormat == fp4::kMx ? (j & 1) * 2u : 0u;
          mma_fp4<kFormat>(tmem, smem_desc_k_major_sw128(a_addr + j * 32), smem_desc_k_major_sw128(b_addr + j * 32),
                           fp4_instr_desc<kFormat>(kP, kQ, id), sf_p + t * 4, sf_q + t * 4 * Tile::kQBlocks,
                           (kb | j) != 0 ? 1u : 0u);
        }
        mma_commit(&bars.empty[s]);
      }
      if (!*abort_flag) mma_commit(&bars.done);
    }
  } else {
    float alpha = 1.0f;
    if (p.factor_p != nullptr) alpha *= __ldg(p.factor_p);
    if (p.factor_q != nullptr) alpha *= __ldg(p.factor_q);
    const bool ok = mbar_wait_bounded(&bars.done, 0, abort_flag, p.status, kStatusFp4Wait + 3);
    tc_fence_after_sync();
    if (ok) {
      const int quarter = warp & 3;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
      const int row_p = p0 + quarter * 32 + lane;
      T* out = static_cast<T*>(p.out);
      constexpr int kChunk = 32;
      for (int c0 = 0; c0 < kQ; c0 += kChunk) {
        uint32_t v[kChunk];
        tmem_load_32cols(taddr + c0, v);
        tmem_load_wait();
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          const int row_q = q0 + c0 + i;
          if (row_p < p.rows_p && row_q < p.rows_q && c0 + i < kQ) {
            const T y = rounded<T>(__uint_as_float(v[i]) * alpha);
            if (kTransposed) {
              out[row_q * p.out_pitch + row_p] = y;
            } else {
              out[row_p * p.out_pitch + row_q] = y;
            }
          }
        }
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
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, Tile::kTmemColumns);
  }
}

bool encode_codes(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t pitch, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(pitch), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(pitch)};
  const uint32_t box[2] = {kRowBytes, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kFormat, int kQ, bool kTransposed, typename T>
cudaError_t launch(const Fp4Operand& P, const Fp4Operand& Q, void* out, int64_t out_pitch, int64_t K, int* status,
                   cudaStream_t stream) {
  using Tile = Fp4Tile<kFormat, kQ>;
  const int64_t pitch = fp4::code_pitch(K);
  CUtensorMap map_p, map_q;
  if (!encode_codes(&map_p, P.codes, P.rows, pitch, kP) || !encode_codes(&map_q, Q.codes, Q.rows, pitch, kQ)) {
    return cudaErrorInvalidValue;
  }
  Fp4Params params;
  params.sf_p = P.scales;
  params.sf_q = Q.scales;
  params.factor_p = P.factor;
  params.factor_q = Q.factor;
  params.out = out;
  params.out_pitch = out_pitch;
  params.rows_p = static_cast<int>(P.rows);
  params.rows_q = static_cast<int>(Q.rows);
  params.cols = static_cast<int>(fp4::padded_cols(K));
  params.scale_tiles = static_cast<int>(fp4::scale_tiles(K, kFormat));
  params.stages = 4;
  params.status = status;
  const int smem = params.stages * Tile::kStageBytes + 1024;
  auto kernel = fp4_gemm_kernel<kFormat, kQ, kTransposed, T>;
  static bool configured[64] = {};
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device < 0 || device >= 64 || !configured[device]) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
    if (device >= 0 && device < 64) configured[device] = true;
  }
  const int64_t blocks_p = (P.rows + kP - 1) / kP;
  const int64_t blocks_q = (Q.rows + kQ - 1) / kQ;
  if (blocks_q > 65535 || blocks_p > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks_p), static_cast<unsigned>(blocks_q));
  kernel<<<grid, kThreads, smem, stream>>>(map_p, map_q, params);
  return cudaGetLastError();
}

template <int kFormat, typename T>
cudaError_t dispatch(const Fp4Operand& a, const Fp4Operand& b, void* out, int64_t K, int* status,
                     cudaStream_t stream) {
  const int64_t N = b.rows;
  if (a.rows <= 32) return launch<kFormat, 32, true, T>(b, a, out, N, K, status, stream);
  if (a.rows <= 64) return launch<kFormat, 64, true, T>(b, a, out, N, K, status, stream);
  return launch<kFormat, 128, false, T>(a, b, out, N, K, status, stream);
}

}  // namespace

cudaError_t launch_fp4_gemm(const Fp4Operand& a, const Fp4Operand& b, int format, void* out, int out_type, int64_t K,
                            int* status_word, cudaStream_t stream) {
  if (format == fp4::kNv) {
    return out_type == kTypeBf16 ? dispatch<fp4::kNv, __nv_bfloat16>(a, b, out, K, status_word, stream)
                                 : dispatch<fp4::kNv, __half>(a, b, out, K, status_word, stream);
  }
  return out_type == kTypeBf16 ? dispatch<fp4::kMx, __nv_bfloat16>(a, b, out, K, status_word, stream)
                               : dispatch<fp4::kMx, __half>(a, b, out, K, status_word, stream);
}

}  // namespace lbl
