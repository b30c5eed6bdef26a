// 16-bit rows as MX FP4 digits: what the few-row kernel and the CTA-pair GEMM
// share.
//
// A group of 32 values with the largest in [2^(e+1), 2^(e+2)) is split into E2M1
// digits,
//   u_0 = x * 2^-e (|u_0| < 4),  d_i = RNE_E2M1(u_i),  u_{i+1} = 8 (u_i - d_i),
//   x = sum_{i<D} d_i 2^(e - 3i) + u_D 2^(e - 3D):  |u_i| <= 4 keeps the rounding below
// 1/2, so each digit gives three bits more.  The digits are D rows of an MX tensor
// whose scales differ by 2^3: a block-scaled MMA multiplies them as it does any
// rows, and the epilogue adds a token's D results, smallest first.
//
// What is left.  Eight digits hold a value to 2^-23 of its group's largest: bf16
// values down to 2^-15 of it (fp16: 2^-12) without any error.  Smaller ones may leave
// something, and the largest value's weight may be zero (E2M1 has that code), so it
// counts.  All of the following take part as fp32 products beside the MMA, so that x is
// not rounded at all:
//   * u_D 2^(e - 3D), exact in fp32 (a multiple of the value's last bit);
//   * digits whose scale would be below 2^-127 (groups below about 2^-105): the digit is
//     zero, and u goes on without it;
//   * values from 2^126 on, infinities and NaN, which count as zero in the digits (the
//     first digit may be a seventh larger than its value, which must not overflow).
// Few values leave anything: of 8192 normal ones whose channels have log-normal sizes,
// with eight digits 0.8 in bf16 and 5.6 in fp16, with nine a thirteenth of that.  They are
// listed by token and place, a list for a few tokens and 256 values of K; a list that is
// too short only counts, and its readers split the rows again (right for any rows, fast
// for those that leave little: 16 x 4096 x 4096 bf16 takes 9.0 us for normal rows, 10.8 with
// six channels and 12.3 with 24 a thousand times larger; 16 x 8192 x 8192 with a value
// 2^20 times larger in every group 1.9 ms).
// The few-row kernel takes its lists along with a stage and finds the weights in shared
// memory.  The CTA-pair GEMM's spare warps gather them from L2, 32 bytes for half of
// one (1024 x 8192 x 8192 with eight digits: 194 us became 258 in bf16, 755 in fp16), so
// rows for it have nine digits (227, 238).
#pragma once

#include "tcb_mx.cuh"

namespace tcb {
namespace mx_detail {

constexpr int kDigitBits = 3;

// How tokens lie in an MX tensor of digits: digit d of token j of list i is row
// i * kRows + j * kDigits + d.  A list covers kTokens tokens and 256 values of K;
// kPerTile lists (of neighbouring tokens) lie side by side.
template <int DIGITS, int TOKENS, int ROWS, int PER_TILE>
struct DigitLayout {
  static constexpr int kDigits = DIGITS, kTokens = TOKENS, kRows = ROWS, kPerTile = PER_TILE;
  static_assert(DIGITS * TOKENS <= ROWS, "rows of a list");
  static __host__ __device__ long long lists(long long m) { return (m + TOKENS - 1) / TOKENS; }
  static __host__ __device__ long long rows(long long m) { return lists(m) * ROWS; }
  static __host__ __device__ long long index(long long list, int kb, int kblocks) {
    return (list / PER_TILE * kblocks + kb) * PER_TILE + list % PER_TILE;
  }
  static constexpr int kTileTokens = PER_TILE * TOKENS;
  // First column of token t of a tile; columns of m tokens, in eights.
  static __host__ __device__ int column(int t) { return t / TOKENS * ROWS + t % TOKENS * DIGITS; }
  static __host__ __device__ int columns(int m) { return (column(m - 1) + DIGITS + 7) / 8 * 8; }
};
// Few-row kernel, a tile of 128 columns: 16 bf16 or 14 fp16 tokens.  fp16 values have three
// bits more, and with a ninth digit leave as little as bf16 values do with eight (33 x 5000
// x 4136: 16.0 us with eight, 13.9 with nine; 16 x 16384 x 8192, two tiles, 24.5 and 26.4).
using Bf16Tile = DigitLayout<8, 4, 32, 4>;
using Fp16Tile = DigitLayout<9, 7, 64, 2>;
// CTA-pair GEMM: seven tokens a slice of 64 columns.
using SliceDigits = DigitLayout<9, 7, 64, 1>;

__device__ __forceinline__ float value16(uint16_t bits, bool bf16) {
  return bf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16)
              : __half2float(__ushort_as_half(bits));
}

// No digits: at least 2^126, infinite or not a number.
__device__ __forceinline__ bool is_large(float v) {
  return (__float_as_uint(v) & 0x7FFFFFFFu) >= 0x7E800000u;
}

// 16-bit rows [m][k], pitch ld elements; vec: every row starts on a 16-byte boundary.
struct ValueRows {
  const uint16_t* x;
  long long ld;
  int m, k;
  int bf16, vec;
};

// MX rows [n], of pitch code bytes, with packed scales.
struct MxRows {
  const uint8_t* codes;
  long long pitch;
  const uint8_t* scales;
  int kblocks;
  long long n;
};

// The lane's eight of 256 values from k on, zeros past the end.
__device__ __forceinline__ uint4 load_values(const ValueRows& rows, long long token, int k) {
  const uint16_t* row = rows.x + token * rows.ld;
  if (rows.vec && k + 8 <= rows.k) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < rows.k) w[i / 2] |= static_cast<uint32_t>(row[k + i]) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Value i of a lane's eight.
__device__ __forceinline__ float lane_value(uint4 raw, bool bf16, int i) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return value16(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1))), bf16);
}

// A lane's eight values (four lanes a group) as digits: put(d, code, words) for digit
// d, with the E8M0 code of its scale.  Returns whether the lane's values leave
// anything; u[] (u_DIGITS) and e8 are for left_of.
template <int DIGITS, typename Put>
__device__ __forceinline__ bool split_digits(uint4 raw, bool bf16, float (&u)[8], int& e8, Put put) {
  uint32_t top = 0, any = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    u[i] = lane_value(raw, bf16, i);
    if (is_large(u[i])) {
      u[i] = 0.0f;
      any = 1;
    }
    top = max(top, __float_as_uint(u[i]) & 0x7FFFFFFFu);
  }
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  // The first digit's code; a group of zeros has one that makes all of them valid.
  e8 = top == 0 ? 127 + (DIGITS - 1) * kDigitBits : max(static_cast<int>(top >> 23) - 1, 0);
  const float inv = inverse_scale(static_cast<uint32_t>(e8));
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] *= inv;
#pragma unroll
  for (int d = 0; d < DIGITS; ++d) {
    const int code = e8 - kDigitBits * d;
    const uint32_t codes = code >= 0 ? encode8(u) : 0u;
    uint32_t h[4];
    decode8(codes, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      unpack2<__half>(h[i], lo, hi);
      u[2 * i] = (u[2 * i] - lo) * static_cast<float>(1 << kDigitBits);
      u[2 * i + 1] = (u[2 * i + 1] - hi) * static_cast<float>(1 << kDigitBits);
    }
    put(d, static_cast<uint8_t>(max(code, 0)), codes);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) any |= __float_as_uint(u[i]) << 1;  // but for signs of zeros
  return any != 0;
}

// What split_digits leaves of the lane's values: u becomes that.
template <int DIGITS>
__device__ __forceinline__ void left_of(uint4 raw, bool bf16, float (&u)[8], int e8) {
  // Two exact products: the last digit's scale over eight alone may be too small a number.
  constexpr float kPast = 1.0f / (1 << DIGITS * kDigitBits);
  const float unit = scale_value(static_cast<uint32_t>(e8));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = lane_value(raw, bf16, i);
    u[i] = is_large(v) ? v : u[i] * kPast * unit;
  }
}

// How many of the lane's values leave something.
__device__ __forceinline__ int count_left(const float (&left)[8]) {
  int n = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) n += left[i] != 0.0f;  // NaN too
  return n;
}

// The sum of left . a weight row (a row a lane) over a block of 256 values of K, `left`
// being spread over the warp's `lanes`: codes(from) are the eight codes at lane from's
// values, scale(group) their group's.
template <typename Codes, typename Scale>
__device__ __forceinline__ float left_block(const float (&left)[8], uint32_t lanes, Codes codes, Scale scale) {
  float sum = 0.0f;
  for (; lanes != 0; lanes &= lanes - 1) {
    const int from = __ffs(lanes) - 1;
    const uint32_t word = codes(from);
    const float s = scale(from / 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = __shfl_sync(0xFFFFFFFFu, left[i], from);
      if (v != 0.0f) sum += v * (decode1(word >> (4 * i) & 15u) * s);
    }
  }
  return sum;
}

// What the digits of a list's tokens leave in 256 values of K, in order.  More than
// kLeftEntries are counted, not listed.
constexpr int kLeftEntries = 15;
struct __align__(16) LeftList {
  uint32_t count;
  uint32_t unused;
  uint2 entries[kLeftEntries];  // a LeftEntry; the fp32 value
};
// A place in a block of 256 values of K and a token, as its reader wants them: the byte
// and nibble of the code, and where the scale lies in the row's 1 KB of packed scales.
struct LeftEntry {
  uint32_t bits;
  static __device__ __forceinline__ uint32_t token(uint32_t t) { return t << 24; }
  static __device__ __forceinline__ LeftEntry of(uint32_t t, uint32_t place) {
    return {token(t) | ((place >> 7) * 512 + (place >> 5 & 3u)) << 11 | (place & 1u) << 10 | place >> 1};
  }
  __device__ __forceinline__ uint32_t byte() const { return bits & 127u; }
  __device__ __forceinline__ uint32_t shift() const { return bits >> 8 & 4u; }
  __device__ __forceinline__ uint32_t scale() const { return bits >> 11 & 1023u; }
  __device__ __forceinline__ uint32_t token() const { return bits >> 24; }
};
static_assert(sizeof(LeftList) == 128, "eight lanes read 16 bytes each");

// Appends a warp's values to a list whose first `at` entries are other tokens'; a lane
// has `mine`.
__device__ __forceinline__ void append_left(LeftList* list, uint32_t at, uint32_t mine, uint32_t token,
                                            const float (&left)[8]) {
  const int lane = threadIdx.x & 31;
  uint32_t end = mine;
#pragma unroll
  for (int step = 1; step < 32; step *= 2) {
    const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, end, step);
    if (lane >= step) end += before;
  }
  at += end - mine;
  if (mine == 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (left[i] != 0.0f && at < kLeftEntries)
      list->entries[at++] = make_uint2(LeftEntry::of(token, lane * 8 + i).bits, __float_as_uint(left[i]));
}

// What the digits of a token leave in K block kb, split again, times a weight row (a row
// a lane; codes and scale as in left_block).
template <int DIGITS, typename Codes, typename Scale>
__device__ __forceinline__ float left_again(const ValueRows& rows, long long token, int kb, Codes codes, Scale scale) {
  const uint4 raw = load_values(rows, token, kb * 256 + (threadIdx.x & 31) * 8);
  float left[8];
  int e8;
  const bool any = split_digits<DIGITS>(raw, rows.bf16, left, e8, [](int, uint8_t, uint32_t) {});
  left_of<DIGITS>(raw, rows.bf16, left, e8);
  return left_block(left, __ballot_sync(0xFFFFFFFFu, any), codes, scale);
}

// acc[t] = the products of weight row n (a row a lane) with what the digits of token
// first + t, t < Layout::kTokens, leave; `lists` are that list's, a K block each.
// Returns whether there is anything (acc is not written otherwise).  One entry at a time:
// there are few, and the code, which runs now and then, costs what fetching it takes
// (64 x 16384 x 4096 bf16: 30.6 us so, 34.1 with eight weights in flight).
template <typename Layout>
__device__ __noinline__ bool left_products(const LeftList* lists, const ValueRows& rows, long long first,
                                           const MxRows& w, long long n, float* acc) {
  const int lane = threadIdx.x & 31;
  const long long m = min(n, w.n - 1);  // rows past the end: any row
  const uint8_t* row = w.codes + m * w.pitch;
  const uint8_t* scales = w.scales + (m >> 7) * w.kblocks * 1024 + (m & 31) * 16 + ((m & 127) >> 5) * 4;
  bool any = false;
  for (int base = 0; base < w.kblocks; base += 32) {
    // A list a lane: its count and first entry.
    uint4 head = make_uint4(0, 0, 0, 0);
    if (base + lane < w.kblocks) head = *reinterpret_cast<const uint4*>(lists + base + lane);
    uint32_t some = __ballot_sync(0xFFFFFFFFu, head.x != 0);
    if (some == 0) continue;
    if (!any)
      for (int t = 0; t < Layout::kTokens; ++t) acc[t] = 0.0f;
    any = true;
#pragma unroll 1
    for (; some != 0; some &= some - 1) {
      const int from = __ffs(some) - 1, kb = base + from;
      const int count = static_cast<int>(__shfl_sync(0xFFFFFFFFu, head.x, from));
      const uint8_t* codes = row + kb * 128ll;
      const uint8_t* scale = scales + kb * 1024ll;
      if (count > kLeftEntries) {
        for (int t = 0; t < Layout::kTokens && first + t < rows.m; ++t)
          acc[t] += left_again<Layout::kDigits>(
              rows, first + t, kb, [&](int at) { return *reinterpret_cast<const uint32_t*>(codes + at * 4); },
              [&](int group) { return scale_value(scale[(group >> 2) * 512 + (group & 3)]); });
        continue;
      }
      uint2 entry = make_uint2(__shfl_sync(0xFFFFFFFFu, head.z, from), __shfl_sync(0xFFFFFFFFu, head.w, from));
#pragma unroll 1
      for (int e = 0;;) {
        const LeftEntry at{entry.x};
        acc[at.token()] += __uint_as_float(entry.y) *
                           (decode1(codes[at.byte()] >> at.shift() & 15u) * scale_value(scale[at.scale()]));
        if (++e >= count) break;
        entry = lists[kb].entries[e];
      }
    }
  }
  return any;
}

// A token's result from its columns r[0..DIGITS - 1], smallest first.
template <int DIGITS>
__device__ __forceinline__ float sum_digits(const float* r) {
  float sum = r[DIGITS - 1];
#pragma unroll
  for (int d = DIGITS - 2; d >= 0; --d) sum += r[d];
  return sum;
}

}  // namespace mx_detail
}  // namespace tcb
