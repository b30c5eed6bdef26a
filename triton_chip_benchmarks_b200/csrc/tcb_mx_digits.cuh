// 16-bit rows as MX FP4 digits: what the few-row kernel and the CTA-pair GEMM
// share.
//
// A group of 32 values with the largest in [2^(e+1), 2^(e+2)) is split exactly
// into E2M1 digits,
//   u_0 = x * 2^-e (|u_0| < 4),  d_i = RNE_E2M1(u_i),  u_{i+1} = 8 (u_i - d_i),
//   x = sum_i d_i 2^(e - 3i):  |u_i| <= 4 keeps the rounding below 1/2, so each
// digit gives three bits more.  Eight digits hold a value to 2^-23 of its
// group's largest (half of 8^-7 in units of 2^e, the largest being at least two
// of them): bf16 values down to 2^-15 of it (fp16: 2^-12) without any error,
// smaller ones as a fixed-point number of about the precision that an fp32 sum
// holding the largest has.  The digits are eight rows of an MX tensor
// whose scales differ by 2^3: a block-scaled MMA multiplies them as it does any
// rows, and the epilogue adds a token's eight results, smallest first.
// Infinities and NaN have no digits: they count as zero there, and the NaN scale
// on their group's last digit tells the epilogue (odd_products).
#pragma once

#include "tcb_mx.cuh"

namespace tcb {
namespace mx_detail {

constexpr int kDigits = 8;
constexpr int kDigitBits = 3;

__device__ __forceinline__ float value16(uint16_t bits, bool bf16) {
  return bf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16)
              : __half2float(__ushort_as_half(bits));
}

__device__ __forceinline__ bool is_odd(float v) {
  return (__float_as_uint(v) & 0x7FFFFFFFu) >= 0x7F800000u;
}

// Packed E8M0 code of (row, group).
__device__ __forceinline__ uint32_t packed_scale(const uint8_t* scales, int kblocks, long long row, int group) {
  return scales[((row >> 7) * kblocks + (group >> 3)) * 1024 + ((group >> 2) & 1) * 512 + (row & 31) * 16 +
                ((row & 127) >> 5) * 4 + (group & 3)];
}

// The products of a row's infinities and NaN in [k0, k1) with weight row n: what
// its result is when it has any, whatever the rest sums to.
static __device__ __noinline__ float odd_products(const uint16_t* x, bool bf16, const uint8_t* w,
                                                  long long pitch, const uint8_t* sw, int kblocks,
                                                  long long n, int k0, int k1) {
  float sum = 0.0f;
  for (int k = k0; k < k1; ++k) {
    const float v = value16(x[k], bf16);
    if (!is_odd(v)) continue;
    const uint32_t code = w[n * pitch + k / 2] >> (4 * (k & 1)) & 15u;
    sum += v * (decode1(code) * scale_value(packed_scale(sw, kblocks, n, k / 32)));
  }
  return sum;
}

// A token's result from its eight columns r[0..7]; `*odd` where odd_products has
// to be added (the last digit is not a number).
__device__ __forceinline__ float sum_digits(const float* r, bool* odd) {
  *odd = isnan(r[kDigits - 1]);
  float sum = *odd ? 0.0f : r[kDigits - 1];
#pragma unroll
  for (int d = kDigits - 2; d >= 0; --d) sum += r[d];
  return sum;
}

}  // namespace mx_detail
}  // namespace tcb
