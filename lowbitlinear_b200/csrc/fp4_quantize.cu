// Microscaled FP4 quantiser and its inverse.
//
//   quantise    step = f(largest magnitude of the block), code = nearest E2M1 number to x / step, ties
//               to even (fp4_common.cuh has the two rules and why every decision is exact)
//   dequantise  x = code * step, one rounding to the output type
//
// Both are bound by HBM: a value is read (or written) once in 2 or 4 bytes, and 0.53 (MXFP4) or 0.56
// (NVFP4) bytes per value go the other way.  A thread owns sixteen neighbouring columns; the quantiser of a large
// matrix of a 16-bit type 32, so that what a thread does besides its values (addresses, steps, scale words)
// weighs less: at two bytes per value the instructions are as scarce as the bandwidth (24576 x 4096 FP16 to NVFP4
// 49.4 us with sixteen, 42.7 with 32; 333 x 1003 2.0 and 2.8).  The largest magnitude of a block takes at most one
// shuffle; four scale bytes meet by shuffles and leave as one word.  Rows are read and written in 32-byte pieces
// per lane; rows that do not start on 16 bytes go through shared memory, where a warp turns its columns from a word per
// lane to sixteen columns per lane (24576 x 4095 BF16 to NVFP4 68 us and back 59; a value at a time 69 and 63).
#include "fp4_common.cuh"
#include "kernels.h"

namespace lbl {
namespace {

constexpr int kThreads = 256;
constexpr int kWarpUnits = 32 * 16;  // columns of a row that one warp handles, per sixteen of a thread
constexpr int kWarpWords = kWarpUnits / 2;         // of two 16-bit columns
constexpr int kTurnedBytes = kWarpWords * 4 + 16;  // shared memory in which a warp turns them: one word more, on 16 bytes

// Columns [0, end) of a row of 16-bit values that starts on any address, as eight words of two columns per lane: lane l
// gets columns 16 l to 16 l + 15, zero past the end.  Read a word per lane, from the last word boundary at or before the
// row's start; the value that shares a word with something else is read alone.
__device__ __forceinline__ void load_any_row(const unsigned short* line, int end, uint8_t* turned, int lane, uint32_t (&w)[8]) {
  uint32_t* words = reinterpret_cast<uint32_t*>(turned);
  const int late = static_cast<int>(reinterpret_cast<uintptr_t>(line) >> 1) & 1;  // word k: columns 2 k - late, 2 k - late + 1
  const int last = min(end, kWarpUnits) - 1;
  uint32_t raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = 2 * (i * 32 + lane) - late;
    raw[i] = c >= 0 && c + 1 < end ? *reinterpret_cast<const uint32_t*>(line + c) : 0u;
  }
  const bool single = lane == 0 ? late && end > 0 : lane == 1 && last >= 0 && ((last + late) & 1) == 0;
  const int at = lane == 0 ? 0 : last;
  const unsigned short value = single ? line[at] : static_cast<unsigned short>(0);
#pragma unroll
  for (int i = 0; i < 8; ++i) words[i * 32 + lane] = raw[i];
  if (lane == 0) words[kWarpWords] = 0;
  __syncwarp();
  if (single) reinterpret_cast<unsigned short*>(turned)[at + late] = value;
  __syncwarp();
  const uint4 a = *reinterpret_cast<const uint4*>(words + lane * 8);
  const uint4 b = *reinterpret_cast<const uint4*>(words + lane * 8 + 4);
  w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  if (late) {
    const uint32_t next = words[lane * 8 + 8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __funnelshift_r(w[i], i < 7 ? w[i + 1] : next, 16);
  }
}

// The inverse: words of columns 16 l to 16 l + 15 of lane l to columns [0, end) of such a row.
__device__ __forceinline__ void store_any_row(unsigned short* line, int end, uint8_t* turned, int lane, const uint32_t (&w)[8]) {
  uint32_t* words = reinterpret_cast<uint32_t*>(turned);
  const int late = static_cast<int>(reinterpret_cast<uintptr_t>(line) >> 1) & 1;  // words start one column later
  const int last = min(end, kWarpUnits) - 1;
  *reinterpret_cast<uint4*>(words + lane * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(words + lane * 8 + 4) = make_uint4(w[4], w[5], w[6], w[7]);
  __syncwarp();
  uint32_t raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = i * 32 + lane;
    raw[i] = late ? __funnelshift_r(words[k], words[k + 1], 16) : words[k];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = 2 * (i * 32 + lane) + late;
    if (c + 1 <= last) *reinterpret_cast<uint32_t*>(line + c) = raw[i];
  }
  const bool single = lane == 0 ? late && end > 0 : lane == 1 && last >= late && ((last - late) & 1) == 0;
  const int at = lane == 0 ? 0 : last;
  if (single) line[at] = reinterpret_cast<const unsigned short*>(turned)[at];
}

// One thread per (row, 16 kUnits columns); rows are padded to whole scale tiles, so that every byte of
// the scale buffer is written (zero where there is no value).
template <typename T, int kFormat, int kUnits>
__global__ void __launch_bounds__(kThreads)
    fp4_quantize_kernel(const T* __restrict__ x, int64_t row_stride, const float* __restrict__ factor,
                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int rows, int cols, int pitch,
                        int tiles, int access, bool early_successor) {
  pdl_wait_for_previous_kernel();
  if (early_successor) pdl_allow_next_kernel();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * blockDim.y + threadIdx.y;  // of this launch: fewer than 65536
  const int thread = blockIdx.x * blockDim.x + threadIdx.x;  // blockDim.x is a multiple of 32: a warp has one row
  if (row >= ((rows + 127) & ~127)) return;
  const int first = thread * (16 * kUnits);
  const int left = row < rows ? cols - first : 0;  // columns to read; below zero past the last one

  fp4::Sixteen<T> v[kUnits];
  const T* src = x + (row * row_stride + first);
  if (kUnits == 1 && access == fp4::kRowsAny) {
    extern __shared__ __align__(32) uint8_t turned[];
    const int warp = (threadIdx.y * blockDim.x + threadIdx.x) / 32;
    const T* line = src - lane * 16;
    const int end = row < rows ? cols - first + lane * 16 : 0;
    if constexpr (sizeof(T) == 2) {
      load_any_row(reinterpret_cast<const unsigned short*>(line), end, turned + warp * kTurnedBytes, lane, v[0].w);
    } else {
      T* mine = reinterpret_cast<T*>(turned) + warp * kWarpUnits;
#pragma unroll
      for (int i = 0; i < kWarpUnits / 32; ++i) {
        const int c = i * 32 + lane;
        mine[c] = c < end ? line[c] : static_cast<T>(0.0f);
      }
      __syncwarp();
      v[0].load_vector(mine + lane * 16, fp4::kRows16);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (left >= 16 * (u + 1)) {
        v[u].load_vector(src + 16 * u, access);
      } else {
        v[u].load_masked(src + 16 * u, left - 16 * u);
      }
    }
  }

  // Bytes of this thread's blocks, at their place in the word of four; blocks with no column (padding of the last tile,
  // padding rows) have scale zero.
  constexpr int kLanesPerWord = 8 / kUnits / (kFormat == fp4::kNv ? 2 : 1);
  const bool stored = row < rows && first < 2 * pitch;
  uint32_t word = 0;
  uint2 out[kUnits];
  if constexpr (kFormat == fp4::kMx) {
    uint32_t amax = v[0].amax_bits();
    if constexpr (kUnits == 2) {
      amax = max(amax, v[1].amax_bits());
    } else {
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    }
    const fp4::BlockStep step = fp4::mx_step(amax);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) out[u] = fp4::round_sixteen<kFormat>(v[u], step);
    if (stored) word = step.byte << (8 * (lane * kUnits / 2 & 3));
  } else {
    const fp4::TensorFactor g = fp4::tensor_factor(factor);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const fp4::BlockStep step = fp4::nv_step(v[u].amax_bits(), g);
      out[u] = fp4::round_sixteen<kFormat>(v[u], step);
      if (stored) word |= step.byte << (8 * (lane * kUnits + u & 3));
    }
  }
  if (stored) {
    uint8_t* dst = codes + (static_cast<int64_t>(row) * pitch + first / 2);
    if constexpr (kUnits == 2) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(out[0].x, out[0].y, out[1].x, out[1].y);
    } else {
      *reinterpret_cast<uint2*>(dst) = out[0];
    }
  }
#pragma unroll
  for (int offset = kLanesPerWord / 2; offset > 0; offset >>= 1) word |= __shfl_xor_sync(0xffffffffu, word, offset);
  const int tile = thread / kLanesPerWord;
  if (lane % kLanesPerWord == 0 && tile < tiles) {
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
  float v[16] = {};
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
    const int warp = (threadIdx.y * blockDim.x + threadIdx.x) / 32;
    T* line = dst - lane * 16;
    const int end = cols - first + lane * 16;
    if constexpr (sizeof(T) == 2) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = two_rounded<T>(v[2 * i], v[2 * i + 1]);
      store_any_row(reinterpret_cast<unsigned short*>(line), end, turned + warp * kTurnedBytes, lane, w);
    } else {
      T* mine = reinterpret_cast<T*>(turned) + warp * kWarpUnits;
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[lane * 16 + i] = v[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kWarpUnits / 32; ++i) {
        const int c = i * 32 + lane;
        if (c < end) line[c] = mine[c];
      }
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

// blockDim = (32 * warps along a row, rows): eight warps, of which as many work along a row as leave the fewest idle
// in its last CTA.
dim3 block_for(int64_t threads) {
  const int64_t warps = (threads + 31) / 32;
  int best = 1;
  for (int x = 2; x <= 8 && x <= warps; x *= 2) {
    if ((warps + x - 1) / x * x <= (warps + best - 1) / best * best) best = x;
  }
  return dim3(32 * best, kThreads / (32 * best));
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

template <typename T>
constexpr size_t turned_bytes() {
  return kThreads / 32 * (sizeof(T) == 2 ? kTurnedBytes : kWarpUnits * sizeof(T));
}

template <typename T, int kFormat, int kUnits>
cudaError_t quantize_units(const void* x, int64_t row_stride, const float* factor, uint8_t* codes, uint8_t* scales,
                           int64_t rows, int64_t cols, bool early_successor, cudaStream_t stream) {
  const int64_t tiles = fp4::scale_tiles(cols, kFormat);
  const int64_t pitch = fp4::code_pitch(cols);
  const int64_t threads = tiles * fp4::Format<kFormat>::kTileCols / (16 * kUnits);
  const dim3 block = block_for(threads);
  const int64_t blocks_x = (threads + block.x - 1) / block.x;
  const int64_t padded = (rows + 127) / 128 * 128;
  if (blocks_x > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const int access = fp4::row_access(x, row_stride * static_cast<int64_t>(sizeof(T)));
  const size_t smem = access == fp4::kRowsAny ? turned_bytes<T>() : 0;
  for (int64_t r0 = 0; r0 < padded; r0 += kRowsPerLaunch) {
    const int64_t here = rows - r0 < kRowsPerLaunch ? rows - r0 : kRowsPerLaunch;
    const int64_t here_padded = (here + 127) / 128 * 128;
    const dim3 grid(static_cast<unsigned>(blocks_x), static_cast<unsigned>((here_padded + block.y - 1) / block.y));
    const cudaError_t err = launch(
        fp4_quantize_kernel<T, kFormat, kUnits>, grid, block, smem, stream, static_cast<const T*>(x) + r0 * row_stride,
        row_stride, factor, codes + r0 * pitch, scales + r0 / 128 * tiles * 512, here, cols, pitch, tiles, access,
        early_successor);
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

template <typename T, int kFormat>
cudaError_t quantize(const void* x, int64_t row_stride, const float* factor, uint8_t* codes, uint8_t* scales,
                     int64_t rows, int64_t cols, bool early_successor, cudaStream_t stream) {
  // 32 columns per thread once that still fills a B200 twice with threads; rows that go through shared memory keep
  // sixteen (20000 x 1003 to MXFP4 13.0 us, in values rather than words 13.4, with 32 of them 15.6).
  if constexpr (sizeof(T) == 2) {
    if (rows * cols >= 2LL * 148 * 2048 * 32 && fp4::row_access(x, row_stride * 2) != fp4::kRowsAny) {
      return quantize_units<T, kFormat, 2>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream);
    }
  }
  return quantize_units<T, kFormat, 1>(x, row_stride, factor, codes, scales, rows, cols, early_successor, stream);
}

template <typename T, int kFormat>
cudaError_t dequantize(const uint8_t* codes, const uint8_t* scales, const float* factor, void* out, int64_t rows,
                       int64_t cols, cudaStream_t stream) {
  const int64_t tiles = fp4::scale_tiles(cols, kFormat);
  const int64_t pitch = fp4::code_pitch(cols);
  const int64_t units = (cols + 15) / 16;
  const dim3 block = block_for(units);
  const int64_t blocks_x = (units + block.x - 1) / block.x;
  if (blocks_x > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const int access = fp4::row_access(out, cols * static_cast<int64_t>(sizeof(T)));
  const size_t smem = access == fp4::kRowsAny ? turned_bytes<T>() : 0;
  for (int64_t r0 = 0; r0 < rows; r0 += kRowsPerLaunch) {
    const int64_t here = rows - r0 < kRowsPerLaunch ? rows - r0 : kRowsPerLaunch;
    const dim3 grid(static_cast<unsigned>(blocks_x), static_cast<unsigned>((here + block.y - 1) / block.y));
    const cudaError_t err = launch(
        fp4_dequantize_kernel<T, kFormat>, grid, block, smem, stream, codes + r0 * pitch, scales + r0 / 128 * tiles * 512,
        factor, static_cast<T*>(out) + r0 * cols, here, cols, pitch, tiles, access);
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
