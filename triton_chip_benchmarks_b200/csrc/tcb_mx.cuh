// Pieces shared by the MX FP4 kernels: E2M1 conversion, E8M0 scales, 16-bit
// pairs and the sizes of the packed layout.
#pragma once

#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tcb {
namespace mx_detail {

// Values of a row of codes: whole groups of 32.
__host__ __device__ inline long long mx_padded(long long n) { return (n + 31) / 32 * 32; }
// 128-wide tiles of an axis whose packed scales are padded to 256 values.
__host__ __device__ inline long long mx_tiles(long long n) { return (n + 255) / 256 * 2; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Rounds to nearest even.
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (sizeof(T) == 4) {
    return v;
  } else if constexpr (std::is_same_v<T, __half>) {
    return __float2half_rn(v);
  } else {
    return __float2bfloat16_rn(v);
  }
}

// The two 16-bit values of a word (low half first) as fp32, exactly.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x, hi = f.y;
  } else {
    lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xFFFF0000u);
  }
}

// Two fp32 values rounded to nearest even into one word (low half first).
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t w;
  if constexpr (std::is_same_v<T, __half>) {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  }
  return w;
}

// E8M0 code of a group whose largest |v| has the fp32 bits `top`: the biased
// exponent less 2 (E2M1's largest exponent), one more where rounding up needs
// it (mantissa above 1.5 = 6 / 4), at least 0; 127 for a group of zeros and 255
// (NaN) where a value is infinite or not a number.
__device__ __forceinline__ uint32_t scale_code(uint32_t top, int up) {
  int e = static_cast<int>(top >> 23) - 2;
  if (up && (top & 0x7FFFFFu) > 0x400000u) ++e;
  e = max(e, 0);
  if (top == 0) e = 127;
  if (top >= 0x7F800000u) e = 255;
  return static_cast<uint32_t>(e);
}

// 2^(127 - code) for a code of scale_code (at most 253, or 255: any number).
__device__ __forceinline__ float inverse_scale(uint32_t e8) {
  return __uint_as_float((254u - min(e8, 253u)) << 23);
}

// 2^(code - 127); code 0 is the subnormal 2^-127, code 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t e8) {
  return __uint_as_float(e8 == 0 ? 0x00400000u : e8 == 255 ? 0x7FC00000u : e8 << 23);
}

// Eight values as E2M1 codes, the first in the low nibble (nearest even, saturating).
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}

// The two 16-bit values of a word times powers of two, in fp32.  bf16: one
// instruction a value (adding -0 keeps the sign of zeros).
template <typename T>
__device__ __forceinline__ void scale2(uint32_t w, float inv_lo, float inv_hi, float& lo, float& hi) {
  if constexpr (std::is_same_v<T, __half>) {
    unpack2<T>(w, lo, hi);
    lo *= inv_lo;
    hi *= inv_hi;
  } else {
    const uint16_t a = static_cast<uint16_t>(__float_as_uint(inv_lo) >> 16);
    const uint16_t b = static_cast<uint16_t>(__float_as_uint(inv_hi) >> 16);
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "fma.rn.f32.bf16 %0, l, %3, 0f80000000;\n\tfma.rn.f32.bf16 %1, h, %4, 0f80000000;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(w), "h"(a), "h"(b));
  }
}

// One E2M1 code (0..15) as fp32: |code| 0 and 1 are 0 and 1/2, the others
// (2 + c % 2) * 2^(c / 2 - 2).
__device__ __forceinline__ float decode1(uint32_t code) {
  const uint32_t c = code & 7u;
  const uint32_t bits = c < 2 ? c * 0x3F000000u : (c << 22) + (126u << 23);
  return __uint_as_float(bits | (code & 8u) << 28);
}

// Eight E2M1 codes as four fp16 pairs (exact).  A byte at a time: where the word
// stayed in use, taking it apart with one vector mov decoded bytes as zeros
// (nvcc 12.9).
__device__ __forceinline__ void decode8(uint32_t w, uint32_t (&h)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
        : "=r"(h[i])
        : "r"(w >> (8 * i)));
}

}  // namespace mx_detail
}  // namespace tcb
