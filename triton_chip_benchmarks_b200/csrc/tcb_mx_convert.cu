// MX FP4 quantisation and dequantisation (sm_100a).
//
// A group of 32 neighbours v_i shares the scale 2^e and keeps the E2M1 codes
//   c_i = RNE_E2M1(v_i * 2^-e), saturating at +-6,
//   e   = floor(log2 max|v|) - 2        (TCB_MX_FLOOR, the OCP MX rule), or
//         the least e with 6 * 2^e >= max|v|   (TCB_MX_UP, nothing saturates),
// with e >= -127.  A power of two scales exactly, so the only rounding is the
// one to E2M1.  e comes from the exponent (and, rounding up, the mantissa) bits
// of the largest |v|, held as the integer maximum of the fp32 bit patterns: it
// orders NaN above infinity above every number, so one compare finds both.
//
// Tiles.  128 x 128 values a CTA of 256 threads: along either axis they hold
// 128 rows x 4 groups, which is exactly one 512-byte half of the packed scale
// layout that the GEMM reads, so the scales leave as one contiguous piece for
// the row-wise and for the column-wise tensor, padding included (values past
// the edge count as zero, and an all-zero group has the unit scale 127).  A
// thread takes 16 values (half a group) of four rows; inside the matrix its
// loads are straight-line code, all issued before the first is used (with a
// bounds test around each they went out one by one: 74 us instead of 26.5 for
// 8192 x 8192 bf16).  16-bit values stay packed for the search of the largest:
// two a word, one instruction a word, and bf16 is scaled by a mixed-precision FMA
// without being taken apart first (26.5 to 24.4 us; 170 MB, 6.9 TB/s: HBM).
//
// Both axes in one read.  The tile goes to shared memory with cp.async (zeros
// past the edge), 16-byte chunks swizzled so that neither the row-wise nor the
// column-wise loads conflict; a thread takes four times 16 values of a row, then
// 32 rows of one word (two 16-bit columns, or one fp32), and the column codes
// are turned round through shared memory into 64-byte runs.  8192 x 4096 bf16:
// 20.5 us, 103 MB, 5.0 TB/s; the integer pipe is 64 % busy and the issue slots
// 72 %, so instructions bound it (46 us with the loads one by one, 23.5 before the
// mixed-precision scaling).  Rows that do not start on 16-byte boundaries come through
// the same tile: inside the matrix a thread reads the two aligned chunks that its
// 16 bytes lie in and shifts them together (element by element 70 us instead of
// 41 for 8191 x 8191 bf16 along the rows, 97 instead of 62 along both axes).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcb_device.cuh"
#include "tcb_host.h"
#include "tcb_mx.cuh"

namespace tcb {
namespace {

using namespace mx_detail;

constexpr int kTile = 128;       // rows and columns of a CTA's tile
constexpr int kThreads = 256;
constexpr int kVec = 16;         // consecutive values of one thread in one row
constexpr int kLanesPerRow = kTile / kVec;
constexpr int kRowsPerPass = kThreads / kLanesPerRow;
constexpr int kPasses = kTile / kRowsPerPass;
constexpr int kCodesPitch = 80;  // bytes of a column's 64 code bytes in shared memory
constexpr int kHalfBytes = 512;  // scales of 128 rows x 4 groups

struct QuantArgs {
  const void* x;
  uint8_t* codes;     // [rows][cols_p / 2]
  uint8_t* scales;    // packed, of [rows][cols_p / 32]
  uint8_t* codes_t;   // [cols][rows_p / 2]
  uint8_t* scales_t;  // packed, of [cols][rows_p / 32]
  long long rows, cols, ld;
  long long tiles_x;  // column tiles (an even number)
  int up;
};

// The values' words: 8 of two 16-bit values, or 16 of one fp32 value.
template <typename T>
constexpr int kWords = kVec * static_cast<int>(sizeof(T)) / 4;

// 16 bytes of a row, zero past its end; `valid` values are in the matrix.
template <typename T>
__device__ __forceinline__ uint4 load_edge(const T* p, int valid) {
  constexpr int kPer = 16 / sizeof(T);
  if (valid >= kPer) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (i >= valid) continue;
    if constexpr (sizeof(T) == 4)
      w[i] = __float_as_uint(p[i]);
    else
      w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The 16 bytes that start `m` bytes into lo (0..15; hi follows it).
__device__ __forceinline__ uint4 shift_together(uint4 lo, uint4 hi, uint32_t m) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = m & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = m & 4 ? w[i + 1] : w[i];
  const uint32_t bits = (m & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// 16 bytes global -> shared, of which the first `bytes` are read and the rest
// are zeros.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes)
               : "memory");
}

// Byte offset of 16-byte chunk c of a row of the tile in shared memory: the
// eight lanes of a row read chunks 2l + j (fp32: 4l + j), which the swizzle
// spreads over all banks.
template <typename T>
__device__ __forceinline__ int tile_chunk(int row, int c) {
  constexpr int kMask = sizeof(T) == 4 ? 3 : 1;
  return row * kTile * static_cast<int>(sizeof(T)) + ((c ^ ((c >> 3) & kMask)) << 4);
}

// Running maximum of magnitudes, a word at a time: one fp32 pattern, or the two
// halves of a 16-bit pair with a NaN winning (the hardware's magnitude maximum
// leaves some sign in `top`).
template <typename T>
__device__ __forceinline__ uint32_t top_of(uint32_t top, uint32_t w) {
  if constexpr (sizeof(T) == 4)
    return max(top, w & 0x7FFFFFFFu);
  else if constexpr (std::is_same_v<T, __half>)
    asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(top) : "r"(w));
  else
    asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(w));
  return top;
}

// fp32 bits of the larger (which = -1) or of one of the magnitudes in `top`.
template <typename T>
__device__ __forceinline__ uint32_t magnitude(uint32_t top, int which) {
  if constexpr (sizeof(T) == 4) {
    return top;
  } else {
    top &= 0x7FFF7FFFu;
    return which < 0 ? max(top & 0xFFFFu, top >> 16) : which ? top >> 16 : top & 0xFFFFu;
  }
}

// Eight consecutive values (their words) times 2^-e as E2M1 codes; zeros where
// the scale is NaN.
template <typename T>
__device__ __forceinline__ uint32_t encode_words(const uint32_t* w, uint32_t e8) {
  const float inv = inverse_scale(e8);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]) * inv;
    } else if (i % 2 == 0) {
      scale2<T>(w[i / 2], inv, inv, v[i], v[i + 1]);
    }
  }
  return e8 == 255 ? 0u : encode8(v);
}

// fp32 bits of a magnitude given by T's bits.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t magnitude) {
  if constexpr (sizeof(T) == 4) {
    return magnitude;
  } else if constexpr (std::is_same_v<T, __half>) {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(magnitude))));
  } else {
    return magnitude << 16;
  }
}

template <typename T, bool VEC, bool ROWS, bool COLS>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? (COLS ? 3 : 2) : COLS && !std::is_same_v<T, __half> ? 5 : 4)
    quantize_kernel(const __grid_constant__ QuantArgs args) {
  constexpr bool kTiled = COLS || !VEC;
  constexpr int kChunks = kWords<T> / 4;  // 16-byte chunks of a thread's values
  extern __shared__ __align__(16) uint8_t smem[];
  // [tile][row scales][column scales][column codes]
  uint8_t* s_scales = smem + (kTiled ? kTile * kTile * sizeof(T) : 0);
  uint8_t* s_scales_t = s_scales + (ROWS ? kHalfBytes : 0);
  uint8_t* s_codes_t = s_scales_t + kHalfBytes;

  const int tid = threadIdx.x;
  const long long tx = static_cast<long long>(blockIdx.x) % args.tiles_x;
  const long long ty = static_cast<long long>(blockIdx.x) / args.tiles_x;
  const long long r0 = ty * kTile, c0 = tx * kTile;
  const int lane_col = tid % kLanesPerRow;
  const int col = lane_col * kVec;
  const int row = tid / kLanesPerRow;
  const T* x = static_cast<const T*>(args.x);
  let_next_kernel_start();
  wait_for_previous_kernels();

  // Rows alone: a thread's values straight into registers.
  [[maybe_unused]] uint4 raw[kTiled ? 1 : kPasses][kChunks];
  if constexpr (!kTiled) {
    if (r0 + kTile <= args.rows && c0 + kTile <= args.cols) {
      const T* p = x + (r0 + row) * args.ld + c0 + col;
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
#pragma unroll
        for (int q = 0; q < kChunks; ++q)
          raw[i][q] = reinterpret_cast<const uint4*>(p + i * kRowsPerPass * args.ld)[q];
    } else {
      const long long left = args.cols - c0 - col;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const long long r = r0 + row + i * kRowsPerPass;
#pragma unroll
        for (int q = 0; q < kChunks; ++q) {
          constexpr int kPer = 16 / sizeof(T);
          const int valid = r < args.rows ? static_cast<int>(min(max(left - q * kPer, 0ll), 16ll)) : 0;
          raw[i][q] = valid ? load_edge(x + r * args.ld + c0 + col + q * kPer, valid)
                            : make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else if constexpr (VEC) {
    constexpr int kRowChunks = kTile * static_cast<int>(sizeof(T)) / 16;
    constexpr int kStep = kThreads / kRowChunks;  // rows a round of loads covers
    const int c = tid % kRowChunks;
    const long long at = c0 + c * (16 / static_cast<int>(sizeof(T)));
    const long long left = (args.cols - at) * static_cast<long long>(sizeof(T));
    const int bytes = left <= 0 ? 0 : left >= 16 ? 16 : static_cast<int>(left);
#pragma unroll
    for (int i = 0; i < kTile / kStep; ++i) {
      const int lr = tid / kRowChunks + i * kStep;
      const bool in = bytes > 0 && r0 + lr < args.rows;
      cp_async16(smem + tile_chunk<T>(lr, c), in ? x + (r0 + lr) * args.ld + at : x, in ? bytes : 0);
    }
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  } else {
    constexpr int kPer = 16 / sizeof(T);
    constexpr int kRowChunks = kTile / kPer;
    constexpr int kStep = kThreads / kRowChunks;  // rows a round of loads covers
    const int c = tid % kRowChunks, lr0 = tid / kRowChunks;
    const long long at = c0 + c * kPer;
    // A tile inside the matrix, and not at either end of X: the aligned chunks
    // around its values are X's too (the next or the last row's, or the gap's).
    const bool inside = r0 + kTile <= args.rows && c0 + kTile <= args.cols && (r0 > 0 || c0 > 0) &&
                        (r0 + kTile < args.rows || c0 + kTile + 16 <= args.cols);
    if (inside) {
      constexpr int kBatch = 4;
#pragma unroll 1
      for (int i = 0; i < kTile / kStep; i += kBatch) {
        uint4 lo[kBatch], hi[kBatch];
        uint32_t m[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const char* p = reinterpret_cast<const char*>(x + (r0 + lr0 + (i + j) * kStep) * args.ld + at);
          m[j] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
          const uint4* q = reinterpret_cast<const uint4*>(p - m[j]);
          lo[j] = q[0];
          hi[j] = q[1];
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          *reinterpret_cast<uint4*>(smem + tile_chunk<T>(lr0 + (i + j) * kStep, c)) =
              shift_together(lo[j], hi[j], m[j]);
      }
    } else {
#pragma unroll 8
      for (int i = tid; i < kTile * kTile; i += kThreads) {
        const int r = i / kTile, col_in = i % kTile;
        const bool in = r0 + r < args.rows && c0 + col_in < args.cols;
        T v = from_float<T>(0.0f);
        if (in) v = x[(r0 + r) * args.ld + c0 + col_in];
        *reinterpret_cast<T*>(smem + tile_chunk<T>(r, col_in / kPer) + col_in % kPer * sizeof(T)) = v;
      }
    }
    __syncthreads();
  }
  if constexpr (ROWS) {
    const long long pitch = mx_padded(args.cols) / 2;
    const bool in_cols = c0 + col < 2 * pitch;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int lr = row + i * kRowsPerPass;
      uint32_t w[kWords<T>];
      uint32_t top = 0;
#pragma unroll
      for (int q = 0; q < kChunks; ++q) {
        uint4 v;
        if constexpr (kTiled)
          v = *reinterpret_cast<const uint4*>(smem + tile_chunk<T>(lr, lane_col * kChunks + q));
        else
          v = raw[i][q];
        w[4 * q] = v.x, w[4 * q + 1] = v.y, w[4 * q + 2] = v.z, w[4 * q + 3] = v.w;
      }
#pragma unroll
      for (int q = 0; q < kWords<T>; ++q) top = top_of<T>(top, w[q]);
      top = top_of<T>(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      const uint32_t e8 = scale_code(top_bits<T>(magnitude<T>(top, -1)), args.up);
      uint32_t codes[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) codes[h] = encode_words<T>(w + h * (kWords<T> / 2), e8);
      if (in_cols && r0 + lr < args.rows)
        *reinterpret_cast<uint2*>(args.codes + (r0 + lr) * pitch + (c0 + col) / 2) =
            make_uint2(codes[0], codes[1]);
      if ((tid & 1) == 0)
        s_scales[(lr & 31) * 16 + (lr >> 5) * 4 + (col >> 5)] = static_cast<uint8_t>(e8);
    }
  }
  __syncthreads();
  if constexpr (ROWS) {
    if (tid < kHalfBytes / 16) {
      // Column tile tx is half tx % 2 of group block tx / 2 of row block ty.
      uint8_t* dst = args.scales + (ty * args.tiles_x + tx) * kHalfBytes;
      reinterpret_cast<uint4*>(dst)[tid] = reinterpret_cast<const uint4*>(s_scales)[tid];
    }
  }
  if constexpr (COLS) {
    constexpr int kColsPerWord = 4 / sizeof(T);
    constexpr int kLanes = kTile / kColsPerWord;  // threads across the tile's columns
#pragma unroll 1
    for (int task = tid; task < 4 * kLanes; task += kThreads) {
      const int word = task % kLanes, group = task / kLanes;
      const uint8_t* src = smem + tile_chunk<T>(group * 32, word / 4) + word % 4 * 4;
      uint32_t w[32];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        w[i] = *reinterpret_cast<const uint32_t*>(src + i * kTile * sizeof(T));
        top = top_of<T>(top, w[i]);
      }
      uint32_t e8[kColsPerWord], codes[kColsPerWord][4];
#pragma unroll
      for (int k = 0; k < kColsPerWord; ++k) e8[k] = scale_code(top_bits<T>(magnitude<T>(top, k)), args.up);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (sizeof(T) == 4) {
          codes[0][q] = encode_words<T>(w + 8 * q, e8[0]);
        } else {
          float lo[8], hi[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            scale2<T>(w[8 * q + i], inverse_scale(e8[0]), inverse_scale(e8[1]), lo[i], hi[i]);
          codes[0][q] = e8[0] == 255 ? 0u : encode8(lo);
          codes[1][q] = e8[1] == 255 ? 0u : encode8(hi);
        }
      }
#pragma unroll
      for (int k = 0; k < kColsPerWord; ++k) {
        const int c = word * kColsPerWord + k;
        *reinterpret_cast<uint4*>(s_codes_t + c * kCodesPitch + group * 16) =
            make_uint4(codes[k][0], codes[k][1], codes[k][2], codes[k][3]);
        s_scales_t[(c & 31) * 16 + (c >> 5) * 4 + group] = static_cast<uint8_t>(e8[k]);
      }
    }
    __syncthreads();
    const long long pitch_t = mx_padded(args.rows) / 2;
    const long long tiles_y = mx_tiles(args.rows);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int c = (tid >> 2) + 64 * p, part = tid & 3;
      const long long at = r0 / 2 + part * 16;
      if (c0 + c < args.cols && at < pitch_t)
        *reinterpret_cast<uint4*>(args.codes_t + (c0 + c) * pitch_t + at) =
            *reinterpret_cast<const uint4*>(s_codes_t + c * kCodesPitch + part * 16);
    }
    if (tid < kHalfBytes / 16) {
      uint8_t* out = args.scales_t + (tx * tiles_y + ty) * kHalfBytes;
      reinterpret_cast<uint4*>(out)[tid] = reinterpret_cast<const uint4*>(s_scales_t)[tid];
    }
  }
}

template <typename T, bool VEC, bool ROWS, bool COLS>
int launch_quantize(const QuantArgs& args, long long tiles, const DeviceFacts& facts,
                    cudaStream_t stream) {
  const int smem = (COLS || !VEC ? kTile * kTile * static_cast<int>(sizeof(T)) : 0) +
                   (ROWS ? kHalfBytes : 0) + (COLS ? kHalfBytes + kTile * kCodesPitch : 0);
  auto fn = quantize_kernel<T, VEC, ROWS, COLS>;
  static DeviceIntCache cap_cache;
  const int cap = cap_cache.get(facts.device, [&] {
    return raise_dynamic_smem(reinterpret_cast<const void*>(fn), facts.max_smem_optin);
  });
  if (cap < smem) return TCB_ERR_RESOURCE;
  return launch_overlapping(fn, dim3(static_cast<unsigned>(tiles)), kThreads, static_cast<size_t>(smem), 1,
                            stream, args);
}

template <typename T>
int run_quantize(const QuantArgs& args, long long tiles, const DeviceFacts& facts,
                 cudaStream_t stream) {
  // 16-byte loads need a 16-byte base and row pitch.
  const bool vec = aligned(args.x, 16) && args.ld * static_cast<long long>(sizeof(T)) % 16 == 0;
  const bool rows = args.codes != nullptr, cols = args.codes_t != nullptr;
  if (vec) {
    if (rows && cols) return launch_quantize<T, true, true, true>(args, tiles, facts, stream);
    if (rows) return launch_quantize<T, true, true, false>(args, tiles, facts, stream);
    return launch_quantize<T, true, false, true>(args, tiles, facts, stream);
  }
  if (rows && cols) return launch_quantize<T, false, true, true>(args, tiles, facts, stream);
  if (rows) return launch_quantize<T, false, true, false>(args, tiles, facts, stream);
  return launch_quantize<T, false, false, true>(args, tiles, facts, stream);
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  void* y;
  long long rows, cols, ld;
  long long tiles_x;
  int wide;  // fp32 rows start on 32-byte boundaries
};

// The same tiles the other way.  code * 2^e is exact in fp32 and is rounded
// once to T.  VEC: a thread turns 4 code bytes of a row into 8 values, 16-byte
// stores (fp32 rows on 32-byte boundaries: one 32-byte store; as two 16-byte
// stores of half a sector each they took 13.6 us instead of 8.4 for 4099 x 2072).
// Otherwise rows of Y start anywhere, and a warp stores 32 values of a row side
// by side, their codes brought round by a shuffle (8 values a thread, element by
// element, took 42 us instead of 10.7 for 2072 x 4099 fp32).  8192 x 8192 bf16:
// 26.7 us, 170 MB, 6.4 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(const __grid_constant__ DequantArgs args) {
  constexpr int kDeqVec = 8;
  constexpr int kDeqLanes = kTile / kDeqVec, kDeqRows = kThreads / kDeqLanes;
  constexpr int kDeqPasses = kTile / kDeqRows;
  __shared__ __align__(16) uint8_t s_scales[kHalfBytes];
  const int tid = threadIdx.x;
  const long long tiles_x = args.tiles_x;  // tiles that hold values (the last may be half past the edge)
  const long long tx = static_cast<long long>(blockIdx.x) % tiles_x;
  const long long ty = static_cast<long long>(blockIdx.x) / tiles_x;
  const long long r0 = ty * kTile, c0 = tx * kTile;
  const long long pitch = mx_padded(args.cols) / 2;
  const int col = (tid % kDeqLanes) * kDeqVec;
  const int row = tid / kDeqLanes;
  const long long left = args.cols - c0 - col;
  const int valid = left <= 0 ? 0 : left >= kDeqVec ? kDeqVec : static_cast<int>(left);
  uint32_t w[kDeqPasses];
  let_next_kernel_start();
  wait_for_previous_kernels();
  if constexpr (VEC) {
#pragma unroll
    for (int p = 0; p < kDeqPasses; ++p) {
      const long long r = r0 + row + p * kDeqRows;
      w[p] = valid > 0 && r < args.rows
                 ? *reinterpret_cast<const uint32_t*>(args.codes + r * pitch + (c0 + col) / 2)
                 : 0u;
    }
  }
  if (tid < kHalfBytes / 16)
    reinterpret_cast<uint4*>(s_scales)[tid] =
        reinterpret_cast<const uint4*>(args.scales + (ty * mx_tiles(args.cols) + tx) * kHalfBytes)[tid];
  __syncthreads();
  if constexpr (VEC) {
#pragma unroll
    for (int p = 0; p < kDeqPasses; ++p) {
      const int lr = row + p * kDeqRows;
      const long long r = r0 + lr;
      if (valid == 0 || r >= args.rows) continue;
      const float scale = scale_value(s_scales[(lr & 31) * 16 + (lr >> 5) * 4 + (col >> 5)]);
      uint32_t h[4];
      decode8(w[p], h);
      float v[kDeqVec];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unpack2<__half>(h[i], v[2 * i], v[2 * i + 1]);
        v[2 * i] *= scale;
        v[2 * i + 1] *= scale;
      }
      T* dst = static_cast<T*>(args.y) + r * args.ld + c0 + col;
      if (valid == kDeqVec) {
        if constexpr (sizeof(T) == 4) {
          if (args.wide) {
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]),
                         "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                         : "memory");
          } else {
            reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        } else {
          *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                      pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kDeqVec; ++i)
          if (i < valid) dst[i] = from_float<T>(v[i]);
      }
    }
  } else {
    // A lane's word i holds codes 8 (lane % 16).. of row 2 i + lane / 16 of the
    // warp's 16.
    constexpr int kRows = kTile / (kThreads / 32);
    const int warp = tid >> 5, lane = tid & 31;
    uint32_t codes[kRows / 2];
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i) {
      const long long r = r0 + warp * kRows + 2 * i + (lane >> 4);
      const long long at = c0 / 2 + (lane & 15) * 4;
      codes[i] = r < args.rows && at < pitch
                     ? *reinterpret_cast<const uint32_t*>(args.codes + r * pitch + at)
                     : 0u;
    }
    // ... and scale i is that of row (lane + 32 i) / 4, group lane % 4.
    float scales[kRows / 8];
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i) {
      const int lr = warp * kRows + 8 * i + (lane >> 2);
      scales[i] = scale_value(s_scales[(lr & 31) * 16 + (lr >> 5) * 4 + (lane & 3)]);
    }
    const int shift = 4 * (lane & 7);
    const int rows = static_cast<int>(min(static_cast<long long>(kRows), args.rows - r0 - warp * kRows));
    const int cols = static_cast<int>(min(static_cast<long long>(kTile), args.cols - c0));
    T* dst = static_cast<T*>(args.y) + (r0 + warp * kRows) * args.ld + c0 + lane;
#pragma unroll
    for (int i = 0; i < kRows; ++i, dst += args.ld) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t word = __shfl_sync(0xFFFFFFFFu, codes[i / 2], (i & 1) * 16 + 4 * g + (lane >> 3));
        const float scale = __shfl_sync(0xFFFFFFFFu, scales[i / 8], (i & 7) * 4 + g);
        const float v = decode1(word >> shift & 15u) * scale;
        if (i < rows && 32 * g + lane < cols) dst[32 * g] = from_float<T>(v);
      }
    }
  }
}

template <typename T>
int launch_dequantize(DequantArgs args, cudaStream_t stream) {
  args.wide = sizeof(T) == 4 && aligned(args.y, 32) && args.ld % 8 == 0;
  const bool vec = aligned(args.y, 16) && args.ld * static_cast<long long>(sizeof(T)) % 16 == 0;
  const long long tiles = args.tiles_x * ((args.rows + kTile - 1) / kTile);
  if (tiles > INT_MAX) return TCB_ERR_RESOURCE;
  return launch_overlapping(vec ? dequantize_kernel<T, true> : dequantize_kernel<T, false>,
                            dim3(static_cast<unsigned>(tiles)), kThreads, 0, 1, stream, args);
}

}  // namespace
}  // namespace tcb

using namespace tcb;

extern "C" int tcb_mx_quantize(int dtype, const void* X, long long rows, long long cols,
                               long long ld, int rule, void* codes, void* scales, void* codes_t,
                               void* scales_t, tcb_stream_t stream) {
  if (rows < 0 || cols < 0 || rows > INT_MAX || cols > INT_MAX || ld < cols ||
      (rule != TCB_MX_FLOOR && rule != TCB_MX_UP) || (codes == nullptr) != (scales == nullptr) ||
      (codes_t == nullptr) != (scales_t == nullptr) || (codes == nullptr && codes_t == nullptr))
    return TCB_ERR_INVALID_ARGUMENT;
  if (dtype != TCB_T_BF16 && dtype != TCB_T_FP16 && dtype != TCB_T_FP32) return TCB_ERR_UNSUPPORTED;
  if (rows == 0 || cols == 0) return TCB_OK;
  if (X == nullptr) return TCB_ERR_INVALID_ARGUMENT;
  if (!aligned(X, dtype == TCB_T_FP32 ? 4 : 2) || !aligned(codes, 16) || !aligned(scales, 16) ||
      !aligned(codes_t, 16) || !aligned(scales_t, 16))
    return TCB_ERR_ALIGNMENT;
  DeviceFacts facts;
  const int rc = current_device_facts(&facts);
  if (rc != TCB_OK) return rc;
  if (facts.major != 10) return TCB_ERR_UNSUPPORTED;
  QuantArgs args;
  args.x = X;
  args.codes = static_cast<uint8_t*>(codes);
  args.scales = static_cast<uint8_t*>(scales);
  args.codes_t = static_cast<uint8_t*>(codes_t);
  args.scales_t = static_cast<uint8_t*>(scales_t);
  args.rows = rows;
  args.cols = cols;
  args.ld = ld;
  args.tiles_x = mx_detail::mx_tiles(cols);
  args.up = rule == TCB_MX_UP;
  const long long tiles = args.tiles_x * mx_detail::mx_tiles(rows);
  if (tiles > INT_MAX) return TCB_ERR_RESOURCE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TCB_T_BF16) return run_quantize<__nv_bfloat16>(args, tiles, facts, s);
  if (dtype == TCB_T_FP16) return run_quantize<__half>(args, tiles, facts, s);
  return run_quantize<float>(args, tiles, facts, s);
}

extern "C" int tcb_mx_dequantize(int dtype, const void* codes, const void* scales, long long rows,
                                 long long cols, void* Y, long long ld, tcb_stream_t stream) {
  if (rows < 0 || cols < 0 || rows > INT_MAX || cols > INT_MAX || ld < cols)
    return TCB_ERR_INVALID_ARGUMENT;
  if (dtype != TCB_T_BF16 && dtype != TCB_T_FP16 && dtype != TCB_T_FP32) return TCB_ERR_UNSUPPORTED;
  if (rows == 0 || cols == 0) return TCB_OK;
  if (codes == nullptr || scales == nullptr || Y == nullptr) return TCB_ERR_INVALID_ARGUMENT;
  if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(Y, dtype == TCB_T_FP32 ? 4 : 2))
    return TCB_ERR_ALIGNMENT;
  DeviceFacts facts;
  const int rc = current_device_facts(&facts);
  if (rc != TCB_OK) return rc;
  if (facts.major != 10) return TCB_ERR_UNSUPPORTED;
  DequantArgs args;
  args.codes = static_cast<const uint8_t*>(codes);
  args.scales = static_cast<const uint8_t*>(scales);
  args.y = Y;
  args.rows = rows;
  args.cols = cols;
  args.ld = ld;
  args.tiles_x = (cols + kTile - 1) / kTile;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TCB_T_BF16) return launch_dequantize<__nv_bfloat16>(args, s);
  if (dtype == TCB_T_FP16) return launch_dequantize<__half>(args, s);
  return launch_dequantize<float>(args, s);
}
