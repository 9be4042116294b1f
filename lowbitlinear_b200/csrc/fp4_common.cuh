// Microscaled FP4 on the device: the two storage formats, the rounding of a block, and the place of
// a scale byte in its tile.
//
//   MXFP4  blocks of 32 columns, E8M0 scale byte b (2^(b - 127))
//   NVFP4  blocks of 16 columns, E4M3 scale byte, one FP32 factor g for the whole tensor
//
// E2M1 codes lie two to a byte, low nibble first; a row of K columns takes 16 * ceil(K / 32) bytes, so
// every row starts on a 16-byte boundary.  Scales lie in tiles of 512 bytes, 128 rows by 4 blocks,
// in the order in which tcgen05.cp moves them to tensor memory.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

namespace lbl {
namespace fp4 {

constexpr int kMx = 0;  // LBL_FP4_MX
constexpr int kNv = 1;  // LBL_FP4_NV

template <int kFormat>
struct Format {
  static constexpr int kBlock = kFormat == kNv ? 16 : 32;
  static constexpr int kTileCols = 4 * kBlock;  // columns covered by one scale tile
  static constexpr uint32_t kNanScale = kFormat == kNv ? 0x7Fu : 0xFFu;
};

__host__ __device__ constexpr int64_t code_pitch(int64_t K) { return (K + 31) / 32 * 16; }
__host__ __device__ constexpr int64_t padded_cols(int64_t K) { return (K + 31) / 32 * 32; }
// Scale tiles along K.
__host__ __device__ constexpr int64_t scale_tiles(int64_t K, int format) {
  const int tile_cols = format == kNv ? 64 : 128;
  return (padded_cols(K) + tile_cols - 1) / tile_cols;
}
// Byte offset of the four scales of row r that belong to tile t along K.
__device__ __forceinline__ int64_t scale_word_offset(int r, int t, int tiles) {
  return (static_cast<int64_t>(r >> 7) * tiles + t) * 512 + ((r & 31) * 16 + ((r >> 5) & 3) * 4);
}

// Tensor factors outside this range would let a step or its reciprocal leave the normal FP32
// numbers; a tensor quantised with one gets the NaN scale everywhere instead of silent garbage.
__device__ __forceinline__ bool factor_ok(float g) { return g >= 0x1p-64f && g <= 0x1p64f; }

__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
  __nv_fp8_e4m3 v;
  v.__x = static_cast<__nv_fp8_storage_t>(byte);
  return static_cast<float>(v);
}

// What one block needs to round its values.  mul + mul_low is the reciprocal of the step to more than 40 bits, mul a
// little below it (MXFP4: mul alone, exact).
struct BlockStep {
  uint32_t byte;  // scale as stored
  float step, mul, mul_low;
  bool short_step;  // NVFP4: the step has the four bits of an E4M3 number (g is a power of two)
};

// A number rounded to 17 significant bits.  Every border between two codes (or two E4M3 numbers) is
// on this grid, so a quotient that was computed with an error of a few units in the last place of
// FP32 lands exactly on a border whenever the true quotient is that near to it.
__device__ __forceinline__ float round_to_17_bits(float v) {
  return __uint_as_float((__float_as_uint(v) + 0x20u) & ~0x3Fu);
}
// x / d (x >= 0) on the right side of every border: t is the quotient on the 17-bit grid, the sign of
// the remainder x - t d is exact (one rounding), and one unit in the last place moves t off a border
// the way the true quotient lies.
__device__ __forceinline__ float sided_quotient(float x, float d, float mul) {
  const float t = round_to_17_bits(x * mul);
  const int remainder = __float_as_int(fmaf(-t, d, x));
  const int up = static_cast<int>(min(static_cast<uint32_t>(remainder), 1u));  // 0 when there is none
  return __int_as_float(__float_as_int(t) + up + 2 * (remainder >> 31));
}

// MXFP4: 2^(floor(log2 amax) - 2), at least 2^-127; everything is exact.
__device__ __forceinline__ BlockStep mx_step(uint32_t amax_bits) {
  BlockStep b;
  const uint32_t exponent = amax_bits >> 23;
  const uint32_t byte = exponent >= 2 ? exponent - 2 : 0u;
  const bool bad = exponent == 255u;
  b.byte = bad ? 0xFFu : byte;
  b.mul = bad ? 0.0f : __uint_as_float((254u - byte) << 23);
  b.step = 0.0f, b.mul_low = 0.0f, b.short_step = false;  // not used
  return b;
}

// NVFP4: s = nearest E4M3 to amax / (6 g), step = s g in FP32.
struct TensorFactor {
  float g, six_g, mul;
  bool ok, power_of_two;
};
__device__ __forceinline__ TensorFactor tensor_factor(const float* factor) {
  TensorFactor f;
  f.g = factor == nullptr ? 1.0f : __ldg(factor);
  f.ok = factor_ok(f.g);
  f.six_g = f.ok ? 6.0f * f.g : 1.0f;
  f.mul = __fdividef(1.0f, f.six_g);
  f.power_of_two = (__float_as_uint(f.g) & 0x7FFFFFu) == 0;
  return f;
}
__device__ __forceinline__ BlockStep nv_step(uint32_t amax_bits, const TensorFactor& f) {
  BlockStep b;
  const float amax = fminf(__uint_as_float(amax_bits), 1024.0f * f.six_g);  // far above saturation
  const float quotient = sided_quotient(amax, f.six_g, f.mul);
  const uint32_t byte = __nv_cvt_float_to_fp8(quotient, __NV_SATFINITE, __NV_E4M3);
  const bool bad = amax_bits >= 0x7F800000u || !f.ok;
  b.byte = bad ? 0x7Fu : byte;
  b.step = e4m3_to_float(byte) * f.g;
  const bool none = bad || byte == 0;  // a step of zero: every code is zero
  // The quotient is off by two units in the last place at most; 2^-21 below it lies under the reciprocal for certain.
  b.mul = none ? 0.0f : __fdividef(1.0f - 0x1p-21f, b.step);
  b.mul_low = none ? 0.0f : fmaf(-b.mul, b.step, 1.0f) * b.mul;
  b.short_step = f.power_of_two;
  return b;
}

// The two-operand conversion puts its first operand in the upper nibble.
__device__ __forceinline__ uint32_t eight_codes(const float (&q)[8]) {
  uint32_t out;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(out)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return out;
}

// NVFP4 quotients of eight values, to 40 bits and rounded once; both products have the sign of x, zeros included.
// kSettled: a number of at most eleven bits over a step of four is either on a border (at most seven bits: three
// of the border, four of the step), and then comes out as the border itself, or at least 2^-11 of it away.
// Otherwise the rounding may have put a quotient on a border that it only comes near to.  Borders have three bits;
// when one of the quotients has no more (a zero, or one in 2^20), the sign of its exact remainder decides, and one
// unit in the last place moves it to its side.
template <bool kSettled>
__device__ __forceinline__ void nv_quotients(const float (&x)[8], const BlockStep& b, float (&q)[8]) {
  uint32_t lowest = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = fmaf(x[i], b.mul, x[i] * b.mul_low);
    if (!kSettled) lowest = min(lowest, __float_as_uint(q[i]) << 11);
  }
  if (!kSettled && lowest == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float size = fabsf(q[i]);
      const float remainder = fmaf(-size, b.step, fabsf(x[i]));
      const int move = (remainder > 0.0f ? 1 : 0) - (remainder < 0.0f ? 1 : 0);
      const bool border = (__float_as_uint(size) << 11) == 0 && size < 8.0f;  // beyond, everything becomes 6
      if (border) q[i] = copysignf(__int_as_float(__float_as_int(size) + move), x[i]);
    }
  }
}

// Codes of sixteen neighbouring values (Sixteen<T> below).
template <int kFormat, typename Values>
__device__ __forceinline__ uint2 round_sixteen(const Values& v, const BlockStep& b) {
  uint32_t codes[2];
  float x[8], q[8];
  if constexpr (kFormat == kMx) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v.eight(h, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = x[i] * b.mul;  // exact
      codes[h] = eight_codes(q);
    }
  } else if (Values::kHalf && b.short_step) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v.eight(h, x);
      nv_quotients<true>(x, b, q);
      codes[h] = eight_codes(q);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v.eight(h, x);
      nv_quotients<false>(x, b, q);
      codes[h] = eight_codes(q);
    }
  }
  const bool bad = b.byte == Format<kFormat>::kNanScale;
  return make_uint2(bad ? 0u : codes[0], bad ? 0u : codes[1]);
}

// Eight codes as four pairs of FP16 numbers in column order (exact).
__device__ __forceinline__ void eight_values(uint32_t codes, uint32_t (&pairs)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(pairs[0]), "=r"(pairs[1]), "=r"(pairs[2]), "=r"(pairs[3])
      : "r"(codes));
}

// Scale byte -> step in FP32.
template <int kFormat>
__device__ __forceinline__ float step_of(uint32_t byte, float g) {
  if constexpr (kFormat == kMx) {
    if (byte == 255u) return __uint_as_float(0x7FC00000u);
    return byte == 0u ? 0x1p-127f : __uint_as_float(byte << 23);
  } else {
    return e4m3_to_float(byte) * g;
  }
}

// ---- sixteen neighbouring activations or weights as they lie in memory -------------------------
// Every FP4 kernel is launched with programmatic dependent launch: its set-up overlaps the end of the kernel in front,
// and it reads and writes global memory only after griddepcontrol.wait, when that kernel is complete
// (LBL_FLAG_PDL: the weight is fetched before).  Every CTA waits, so a kernel ends after its predecessor, and it lets
// its successor start only after the wait, so whatever ran two kernels earlier is complete by then.  The
// quantiser of weights and the dequantiser never let a successor start early.
inline cudaLaunchAttribute programmatic_launch() {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  return attr;
}

// How the rows of a matrix may be read or written, by the alignment of its base and pitch.
constexpr int kRows32 = 2;  // 32-byte accesses
constexpr int kRows16 = 1;  // 16-byte accesses
constexpr int kRowsAny = 0;
inline int row_access(const void* base, int64_t pitch_bytes) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(pitch_bytes);
  return bits % 32 == 0 ? kRows32 : bits % 16 == 0 ? kRows16 : kRowsAny;
}

// 32 bytes in one access (the address a multiple of 32).  With two 16-byte accesses per lane each
// touches half of every 32-byte sector it reaches.
__device__ __forceinline__ void load_32_bytes(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
      : "l"(p));
}
__device__ __forceinline__ void store_32_bytes(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

template <typename T>
struct Sixteen;
template <>
struct Sixteen<float> {
  static constexpr bool kHalf = false;
  float v[16];
  __device__ __forceinline__ void load_vector(const float* p, int access) {
    if (access == kRows32) {
      uint32_t w[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_32_bytes(p + 8 * h, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * h + i] = __uint_as_float(w[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 q = reinterpret_cast<const float4*>(p)[i];
        v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
      }
    }
  }
  __device__ __forceinline__ void load_masked(const float* p, int valid) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < valid ? p[i] : 0.0f;
  }
  // Bits of the largest magnitude as FP32; integer order, so that NaN beats infinity beats all.
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
  }
  __device__ __forceinline__ void eight(int half, float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = v[half * 8 + i];
  }
};

template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t bits);
template <>
__device__ __forceinline__ float2 pair_to_float<__half>(uint32_t bits) {
  return __half22float2(*reinterpret_cast<const __half2*>(&bits));
}
template <>
__device__ __forceinline__ float2 pair_to_float<__nv_bfloat16>(uint32_t bits) {
  return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xFFFF0000u));
}

template <typename T>
__device__ __forceinline__ uint32_t max_magnitude(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t max_magnitude<__half>(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
template <>
__device__ __forceinline__ uint32_t max_magnitude<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}

template <typename T>
struct SixteenHalves {
  static constexpr bool kHalf = true;
  uint32_t w[8];
  __device__ __forceinline__ void load_vector(const T* p, int access) {
    if (access == kRows32) {
      load_32_bytes(p, w);
    } else {
      const uint4 a = reinterpret_cast<const uint4*>(p)[0];
      const uint4 b = reinterpret_cast<const uint4*>(p)[1];
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
  }
  __device__ __forceinline__ void load_masked(const T* p, int valid) {
    const unsigned short* raw = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = 2 * i < valid ? raw[2 * i] : 0u;
      const uint32_t hi = 2 * i + 1 < valid ? raw[2 * i + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
  }
  // Magnitudes two at a time; the sign of the running maximum is noise until the end, NaN stays.
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = w[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_magnitude<T>(m, w[i]);
    m &= 0x7FFF7FFFu;
    const uint32_t top = max(m & 0xFFFFu, m >> 16);
    return __float_as_uint(pair_to_float<T>(top).x);
  }
  __device__ __forceinline__ void eight(int half, float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pair_to_float<T>(w[half * 4 + i]);
      out[2 * i] = f.x, out[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Sixteen<__half> : SixteenHalves<__half> {};
template <>
struct Sixteen<__nv_bfloat16> : SixteenHalves<__nv_bfloat16> {};

}  // namespace fp4
}  // namespace lbl
