// Microscaled FP4 quantiser and its inverse.
//
//   quantise    step = f(largest magnitude of the block), code = nearest E2M1 number to x / step, ties
//               to even (fp4_common.cuh has the two rules and why every decision is exact)
//   dequantise  x = code * step, one rounding to the output type
//
// Both are bound by HBM: a value is read (or written) once in 2 or 4 bytes, and 0.53 (MXFP4) or 0.56
// (NVFP4) bytes per value go the other way.  A thread owns sixteen neighbouring columns: one NVFP4
// block, or half of an MXFP4 block whose other half sits in the neighbouring lane, so the largest
// magnitude takes at most one shuffle; four scale bytes meet by shuffles and leave as one word.  Rows are read and
// written in 32-byte pieces per lane; rows that do not start on 16 bytes go through shared memory, where a warp
// turns its 512 neighbouring columns from "a lane, one column after the other" to sixteen per lane.
#include "fp4_common.cuh"
#include "kernels.h"

namespace lbl {
namespace {

constexpr int kThreads = 256;
constexpr int kWarpCols = 512;  // columns of a row that one warp handles

// One thread per (row, sixteen columns); rows are padded to whole scale tiles, so that every byte of
// the scale buffer is written (zero where there is no value).
template <typename T, int kFormat>
__global__ void __launch_bounds__(kThreads)
    fp4_quantize_kernel(const T* __restrict__ x, int64_t row_stride, const float* __restrict__ factor,
                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int rows, int cols, int pitch,
                        int tiles, int access, bool early_successor) {
  pdl_wait_for_previous_kernel();
  if (early_successor) pdl_allow_next_kernel();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * blockDim.y + threadIdx.y;  // of this launch: fewer than 65536
  const int unit = blockIdx.x * blockDim.x + threadIdx.x;  // blockDim.x is a multiple of 32: a warp has one row
  if (row >= ((rows + 127) & ~127)) return;
  const int first = unit * 16;
  const int valid = row < rows ? min(16, cols - first) : 0;  // columns to read; below zero past the last one

  fp4::Sixteen<T> v;
  const T* src = x + (row * row_stride + first);
  if (access == fp4::kRowsAny) {
    extern __shared__ __align__(32) uint8_t turned[];
    T* mine = reinterpret_cast<T*>(turned) + (threadIdx.y * blockDim.x + threadIdx.x) / 32 * kWarpCols;
    const T* line = src - lane * 16;
    const int end = row < rows ? cols - first + lane * 16 : 0;
#pragma unroll
    for (int i = 0; i < kWarpCols / 32; ++i) {
      const int c = i * 32 + lane;
      mine[c] = c < end ? line[c] : static_cast<T>(0.0f);
    }
    __syncwarp();
    v.load_vector(mine + lane * 16, fp4::kRows16);
  } else if (valid == 16) {
    v.load_vector(src, access);
  } else {
    v.load_masked(src, valid);
  }
  uint32_t amax = v.amax_bits();
  fp4::BlockStep step;
  if constexpr (kFormat == fp4::kMx) {
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    step = fp4::mx_step(amax);
  } else {
    step = fp4::nv_step(amax, fp4::tensor_factor(factor));
  }
  const uint2 out = fp4::round_sixteen<kFormat>(v, step);
  const bool stored = row < rows && unit * 8 < pitch;
  if (stored) *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(row) * pitch + unit * 8) = out;

  // Blocks with no column (padding of the last tile, padding rows) have scale zero.
  uint32_t byte = stored ? step.byte : 0u;
  constexpr int kSpan = kFormat == fp4::kMx ? 2 : 1;  // lanes per block
  const int place = (lane / kSpan) & 3;
  uint32_t word = byte << (8 * place);
  word |= __shfl_xor_sync(0xffffffffu, word, kSpan);
  word |= __shfl_xor_sync(0xffffffffu, word, 2 * kSpan);
  const int tile = unit / (4 * kSpan);
  if (lane % (4 * kSpan) == 0 && tile < tiles) {
    *reinterpret_cast<uint32_t*>(scales + fp4::scale_word_offset(row, tile, tiles)) = word;
  }
}

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

// One thread per (row, sixteen columns).
template <typename T, int kFormat>
__global__ void __launch_bounds__(kThreads)
    fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                          const float* __restrict__ factor, T* __restrict__ out, int rows, int cols, int pitch,
                          int tiles, int access) {
  pdl_wait_for_previous_kernel();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * blockDim.y + threadIdx.y;  // of this launch: fewer than 65536
  const int unit = blockIdx.x * blockDim.x + threadIdx.x;  // blockDim.x is a multiple of 32: a warp has one row
  const int first = unit * 16;
  if (row >= rows) return;
  float v[16];
  if (first < cols) {
    const uint2 raw = __ldg(reinterpret_cast<const uint2*>(codes + static_cast<int64_t>(row) * pitch + unit * 8));
    constexpr int kSpan = kFormat == fp4::kMx ? 2 : 1;
    const int block = unit / kSpan;
    const uint32_t byte = __ldg(scales + fp4::scale_word_offset(row, block >> 2, tiles) + (block & 3));
    float g = 1.0f;
    if constexpr (kFormat == fp4::kNv) g = factor == nullptr ? 1.0f : __ldg(factor);
    const float step = fp4::step_of<kFormat>(byte, g);
    uint32_t pairs[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fp4::eight_values(h == 0 ? raw.x : raw.y, pairs);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = fp4::pair_to_float<__half>(pairs[i]);
        v[h * 8 + 2 * i] = f.x * step;
        v[h * 8 + 2 * i + 1] = f.y * step;
      }
    }
  }
  T* dst = out + (static_cast<int64_t>(row) * cols + first);
  if (access == fp4::kRowsAny) {
    extern __shared__ __align__(32) uint8_t turned[];
    T* mine = reinterpret_cast<T*>(turned) + (threadIdx.y * blockDim.x + threadIdx.x) / 32 * kWarpCols;
    if (first < cols) {
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[lane * 16 + i] = static_cast<T>(v[i]);
    }
    __syncwarp();
    T* line = dst - lane * 16;
    const int end = cols - first + lane * 16;
#pragma unroll
    for (int i = 0; i < kWarpCols / 32; ++i) {
      const int c = i * 32 + lane;
      if (c < end) line[c] = mine[c];
    }
  } else if (first + 16 <= cols) {
    uint32_t w[8];
#pragma unroll
    for (int piece = 0; piece < static_cast<int>(sizeof(T)) / 2; ++piece) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) {
          w[i] = __float_as_uint(v[piece * 8 + i]);
        } else {
          w[i] = two_rounded<T>(v[2 * i], v[2 * i + 1]);
        }
      }
      if (access == fp4::kRows32) {
        fp4::store_32_bytes(dst + piece * 8, w);
      } else {
        uint4* to = reinterpret_cast<uint4*>(dst + piece * 8);
        to[0] = make_uint4(w[0], w[1], w[2], w[3]);
        to[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  } else if (first < cols) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (first + i < cols) dst[i] = static_cast<T>(v[i]);
    }
  }
}

// blockDim = (32 * columns of warps, rows): short rows share a CTA.
dim3 block_for(int64_t units) {
  const int64_t warps = (units + 31) / 32;
  int x = 1;
  while (x < 8 && x < warps) x *= 2;
  return dim3(32 * x, kThreads / (32 * x));
}

constexpr int64_t kRowsPerLaunch = 65535 / 128 * 128;  // limit of the grid's y extent, in whole scale tiles

template <typename... Parameters, typename... Arguments>
cudaError_t launch(void (*kernel)(Parameters...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                   Arguments... arguments) {
  cudaLaunchAttribute attr = fp4::programmatic_launch();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Parameters(arguments)...);
}

template <typename T, int kFormat>
cudaError_t quantize(const void* x, int64_t row_stride, const float* factor, uint8_t* codes, uint8_t* scales,
                     int64_t rows, int64_t cols, bool early_successor, cudaStream_t stream) {
  const int64_t tiles = fp4::scale_tiles(cols, kFormat);
  const int64_t units = tiles * fp4::Format<kFormat>::kTileCols / 16;
  const dim3 block = block_for(units);
  const int64_t blocks_x = (units + block.x - 1) / block.x;
  const int64_t padded = (rows + 127) / 128 * 128;
  if (blocks_x > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const int access = fp4::row_access(x, row_stride * static_cast<int64_t>(sizeof(T)));
  const size_t smem = access == fp4::kRowsAny ? kThreads / 32 * kWarpCols * sizeof(T) : 0;
  for (int64_t r0 = 0; r0 < padded; r0 += kRowsPerLaunch) {
    const int64_t here = rows - r0 < kRowsPerLaunch ? rows - r0 : kRowsPerLaunch;
    const int64_t here_padded = (here + 127) / 128 * 128;
    const dim3 grid(static_cast<unsigned>(blocks_x), static_cast<unsigned>((here_padded + block.y - 1) / block.y));
    const cudaError_t err = launch(
        fp4_quantize_kernel<T, kFormat>, grid, block, smem, stream, static_cast<const T*>(x) + r0 * row_stride, row_stride, factor, codes + r0 * fp4::code_pitch(cols),
        scales + r0 / 128 * tiles * 512, static_cast<int>(here), static_cast<int>(cols),
        static_cast<int>(fp4::code_pitch(cols)), static_cast<int>(tiles), access, early_successor);
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

template <typename T, int kFormat>
cudaError_t dequantize(const uint8_t* codes, const uint8_t* scales, const float* factor, void* out, int64_t rows,
                       int64_t cols, cudaStream_t stream) {
  const int64_t tiles = fp4::scale_tiles(cols, kFormat);
  const int64_t units = (cols + 15) / 16;
  const dim3 block = block_for(units);
  const int64_t blocks_x = (units + block.x - 1) / block.x;
  if (blocks_x > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const int access = fp4::row_access(out, cols * static_cast<int64_t>(sizeof(T)));
  const size_t smem = access == fp4::kRowsAny ? kThreads / 32 * kWarpCols * sizeof(T) : 0;
  for (int64_t r0 = 0; r0 < rows; r0 += kRowsPerLaunch) {
    const int64_t here = rows - r0 < kRowsPerLaunch ? rows - r0 : kRowsPerLaunch;
    const dim3 grid(static_cast<unsigned>(blocks_x), static_cast<unsigned>((here + block.y - 1) / block.y));
    const cudaError_t err = launch(
        fp4_dequantize_kernel<T, kFormat>, grid, block, smem, stream, codes + r0 * fp4::code_pitch(cols), scales + r0 / 128 * tiles * 512, factor, static_cast<T*>(out) + r0 * cols,
        static_cast<int>(here), static_cast<int>(cols), static_cast<int>(fp4::code_pitch(cols)), static_cast<int>(tiles),
        access);
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_fp4_quantize(const void* x, int x_type, int64_t row_stride, int format, const float* factor,
                                uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, bool early_successor,
                                cudaStream_t stream) {
  const bool nv = format == fp4::kNv;
  switch (x_type) {
    case kTypeF16:
      return nv ? quantize<__half, fp4::kNv>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream)
                : quantize<__half, fp4::kMx>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream);
    case kTypeBf16:
      return nv ? quantize<__nv_bfloat16, fp4::kNv>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream)
                : quantize<__nv_bfloat16, fp4::kMx>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream);
    case kTypeF32:
      return nv ? quantize<float, fp4::kNv>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream)
                : quantize<float, fp4::kMx>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_fp4_dequantize(const uint8_t* codes, const uint8_t* scales, int format, const float* factor,
                                  void* out, int out_type, int64_t rows, int64_t cols, cudaStream_t stream) {
  const bool nv = format == fp4::kNv;
  switch (out_type) {
    case kTypeF16:
      return nv ? dequantize<__half, fp4::kNv>(codes, scales, factor, out, rows, cols, stream)
                : dequantize<__half, fp4::kMx>(codes, scales, factor, out, rows, cols, stream);
    case kTypeBf16:
      return nv ? dequantize<__nv_bfloat16, fp4::kNv>(codes, scales, factor, out, rows, cols, stream)
                : dequantize<__nv_bfloat16, fp4::kMx>(codes, scales, factor, out, rows, cols, stream);
    case kTypeF32:
      return nv ? dequantize<float, fp4::kNv>(codes, scales, factor, out, rows, cols, stream)
                : dequantize<float, fp4::kMx>(codes, scales, factor, out, rows, cols, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace lbl
