// tcgen05 wrappers of the block-scaled FP4 kernels, on one CTA (kCtas = 1) or a pair of them (2).
//
// tcgen05.mma reads E2M1 codes from shared memory and block scales from tensor memory.  The products and
// their scaling by powers of two (MXFP4) or E4M3 numbers (NVFP4) are exact; sums are FP32.  Scale tiles
// reach tensor memory by tcgen05.cp, which the issuing thread's later MMAs follow in order, so one
// set of scale columns serves every stage.
#pragma once

#include "fp4_common.cuh"
#include "kernels.h"
#include "tc_common.cuh"
#include "tensor_map.h"

namespace lbl {
namespace {

constexpr int kStageCols = 256;  // columns of K per pipeline stage
constexpr int kRowBytes = kStageCols / 2;  // 128: one swizzle row
constexpr int kMmaCols = 64;     // columns of K per MMA

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Untiled bulk copy of `bytes` (a multiple of 16) from global to shared memory.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// 512 bytes of scales (32 rows of 16 bytes, four 128-byte groups of eight rows, no swizzle) into four
// columns of tensor memory, the same in each quarter of the lanes; for a pair in both CTAs, each from its
// own shared memory.
template <int kCtas>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem_byte_addr) {
  const uint32_t lo = (smem_byte_addr >> 4) & 0x3FFFu;
  const uint32_t hi = (128u >> 4) | (1u << 14);  // stride between the groups, descriptor version
  const uint64_t desc = (static_cast<uint64_t>(hi) << 32) | lo;
  if constexpr (kCtas == 1) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  } else {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  }
}

// Instruction descriptor of the block-scaled kinds: A = B = E2M1 (1 at bits 7 and 10), both K-major, N / 8
// at bits 17-22, scale type at bit 23 (1: E8M0), M / 128 at bits 27-28, which bytes of the scale
// columns to use at bits 4-5 (B) and 29-30 (A).
template <int kFormat>
__host__ __device__ constexpr uint32_t fp4_instr_desc(uint32_t m, uint32_t n, uint32_t scale_id) {
  return (scale_id << 4) | (1u << 7) | (1u << 10) | ((n / 8) << 17) | ((kFormat == fp4::kMx ? 1u : 0u) << 23) |
         ((m / 128) << 27) | (scale_id << 29);
}

#define LBL_FP4_MMA(instruction)                                                                              \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t" instruction                                  \
               " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),                                        \
               "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sf_a), "r"(sf_b), "r"(accumulate)                    \
               : "memory")
template <int kFormat, int kCtas>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t sf_a, uint32_t sf_b, uint32_t accumulate) {
  if constexpr (kFormat == fp4::kMx && kCtas == 1) {
    LBL_FP4_MMA("tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X");
  } else if constexpr (kFormat == fp4::kMx) {
    LBL_FP4_MMA("tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X");
  } else if constexpr (kCtas == 1) {
    LBL_FP4_MMA("tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X");
  } else {
    LBL_FP4_MMA("tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X");
  }
}
#undef LBL_FP4_MMA

// Copies the scale tiles of one stage and issues its MMAs.  kRowsP / kRowsQ: rows of the instruction;
// scales of P: one 128-row tile per CTA, of Q: kQBlocks tiles.  The last stage of K (not kWhole) issues only the MMAs
// that have columns, so no scale byte is used that was not loaded.
template <int kFormat, int kCtas, int kRowsP, int kRowsQ, bool kWhole>
__device__ __forceinline__ void issue_stage(uint32_t d_tmem, uint32_t sf_tmem, uint32_t p_addr, uint32_t q_addr,
                                            uint32_t sf_p_addr, uint32_t sf_q_addr, int cols_left, uint32_t accumulate) {
  constexpr int kTileCols = fp4::Format<kFormat>::kTileCols;
  constexpr int kTiles = kStageCols / kTileCols;
  constexpr int kQBlocks = (kRowsQ + 127) / 128;
  const uint32_t sf_p = sf_tmem;
  const uint32_t sf_q = sf_tmem + kTiles * 4;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    if (kWhole || t * kTileCols < cols_left) {
      scales_to_tmem<kCtas>(sf_p + t * 4, sf_p_addr + t * 512);
#pragma unroll
      for (int b = 0; b < kQBlocks; ++b) {
        scales_to_tmem<kCtas>(sf_q + (t * kQBlocks + b) * 4, sf_q_addr + (b * kTiles + t) * 512);
      }
    }
  }
  const uint64_t p_desc = smem_desc_k_major_sw128(p_addr);
  const uint64_t q_desc = smem_desc_k_major_sw128(q_addr);
#pragma unroll
  for (int j = 0; j < kStageCols / kMmaCols; ++j) {
    if (kWhole || j * kMmaCols < cols_left) {
      // MXFP4: a scale tile serves two MMAs, bytes 0-1 and 2-3; NVFP4: one.  64 columns are 32 bytes: two units of the
      // descriptors' addresses.
      const int t = kFormat == fp4::kMx ? j / 2 : j;
      const uint32_t id = kFormat == fp4::kMx ? (j & 1) * 2u : 0u;
      mma_fp4<kFormat, kCtas>(d_tmem, p_desc + 2 * j, q_desc + 2 * j, fp4_instr_desc<kFormat>(kRowsP, kRowsQ, id),
                              sf_p + t * 4, sf_q + t * 4 * kQBlocks, j == 0 ? accumulate : 1u);
    }
  }
}
template <int kFormat, int kCtas, int kRowsP, int kRowsQ>
__device__ __forceinline__ void issue_stage(uint32_t d_tmem, uint32_t sf_tmem, uint32_t p_addr, uint32_t q_addr,
                                            uint32_t sf_p_addr, uint32_t sf_q_addr, int cols_left, uint32_t accumulate) {
  if (cols_left >= kStageCols) {
    issue_stage<kFormat, kCtas, kRowsP, kRowsQ, true>(d_tmem, sf_tmem, p_addr, q_addr, sf_p_addr, sf_q_addr, cols_left, accumulate);
  } else {
    issue_stage<kFormat, kCtas, kRowsP, kRowsQ, false>(d_tmem, sf_tmem, p_addr, q_addr, sf_p_addr, sf_q_addr, cols_left, accumulate);
  }
}

// Bounded wait that keeps polling: a warp parked with a time hint is not always woken early by an arrival
// that comes from the tensor core or another CTA, and these kernels hand a stage on every 500 cycles.
__device__ __forceinline__ bool mbar_spin_bounded(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                                  int* status_word, int status_code) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
    }
    if (*abort_flag) return false;
    if (clock64() - start > kWaitLimitCycles) {
      *abort_flag = 1;
      atomicCAS(status_word, 0, status_code);
      return false;
    }
  }
}

// The same for all lanes of a warp, with one verdict: false when anybody has given up.  A phase that is already
// complete costs one poll and one vote: the loops that issue copies and MMAs have 500 cycles per stage, and every
// instruction in front of them counts.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status_word,
                                          int status_code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  mbar_spin_bounded(bar, parity, abort_flag, status_word, status_code);
  return __any_sync(0xffffffffu, *abort_flag) == 0;
}

// Position in a ring of `stages` slots.
struct RingPosition {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++slot == stages) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

// warp_wait for a barrier on which both CTAs of a pair arrive: what the other CTA did before its arrival is
// ordered before what follows here.
__device__ __forceinline__ bool warp_wait_pair(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                               int* status_word, int status_code) {
  const long long start = clock64();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done != 0)) return true;
    const bool late = clock64() - start > kWaitLimitCycles;
    if (late) {
      *abort_flag = 1;
      atomicCAS(status_word, 0, status_code);
    }
    if (__any_sync(0xffffffffu, late || *abort_flag != 0)) return false;
  }
}

// One lane of a converged warp.  The warps that issue copies and MMAs run their loops with all lanes and
// choose one only around the instructions: addresses and descriptors are then the same for the warp as the
// compiler sees it and stay in uniform registers.  In a branch on the lane number each tcgen05
// instruction took 52-64 cycles to issue (a stage of four MMAs and six scale copies 629 cycles, NVFP4 with twelve
// 932), with the elected lane the MMAs' own 512.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// ---- clusters --------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// shared::cluster address of `addr` (a shared::cta address of this CTA) in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- output ----------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t two_rounded(float a, float b);
template <>
__device__ __forceinline__ uint32_t two_rounded<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t two_rounded<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float product_factor(const float* factor_p, const float* factor_q) {
  float alpha = 1.0f;
  if (factor_p != nullptr) alpha *= __ldg(factor_p);
  if (factor_q != nullptr) alpha *= __ldg(factor_q);
  return alpha;
}

// ---- host --------------------------------------------------------------------------------------
inline bool encode_codes(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t pitch, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(pitch), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(pitch)};
  const uint32_t box[2] = {kRowBytes, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace
}  // namespace lbl
