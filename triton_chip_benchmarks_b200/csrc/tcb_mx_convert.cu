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
// the edge count as zero, and an all-zero group has the unit scale 127).  All
// eight 16-byte loads of a thread are issued before the first is used.
//
// Both axes in one read.  The tile is kept in shared memory on its way through
// the row pass; a thread then takes two neighbouring columns of one 32-row
// group (a warp reads 32 consecutive words per row: no bank conflicts) and the
// codes are turned round through shared memory into 64-byte runs.
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
constexpr int kVec = 8;          // consecutive values of one thread in one row
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

// Eight values of one row as fp32 bit patterns; zero past the matrix.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int valid, float (&v)[kVec]) {
  if (VEC && valid >= kVec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p));
      const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = i < valid ? to_float(p[i]) : 0.0f;
  }
}

template <typename T, bool VEC, bool ROWS, bool COLS>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const __grid_constant__ QuantArgs args) {
  extern __shared__ __align__(16) uint8_t smem[];
  // [tile as fp32 or T][row scales][column scales][column codes]
  T* tile = reinterpret_cast<T*>(smem);
  uint8_t* s_scales = smem + (COLS ? kTile * kTile * sizeof(T) : 0);
  uint8_t* s_scales_t = s_scales + (ROWS ? kHalfBytes : 0);
  uint8_t* s_codes_t = s_scales_t + kHalfBytes;

  const int tid = threadIdx.x;
  const long long tx = static_cast<long long>(blockIdx.x) % args.tiles_x;
  const long long ty = static_cast<long long>(blockIdx.x) / args.tiles_x;
  const long long r0 = ty * kTile, c0 = tx * kTile;
  const int col = (tid % kLanesPerRow) * kVec;
  const int row = tid / kLanesPerRow;
  const long long left = args.cols - c0 - col;
  const int valid = left <= 0 ? 0 : left >= kVec ? kVec : static_cast<int>(left);

  float v[kPasses][kVec];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const long long r = r0 + row + p * kRowsPerPass;
    load8<T, VEC>(static_cast<const T*>(args.x) + (r < args.rows ? r * args.ld + c0 + col : 0),
                  r < args.rows ? valid : 0, v[p]);
  }
  const long long pitch = mx_padded(args.cols) / 2;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int lr = row + p * kRowsPerPass;
    if constexpr (COLS) {
      // The values are T's, so converting back is exact.
      T* dst = tile + lr * kTile + col;
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[p][0], v[p][1], v[p][2], v[p][3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[p][4], v[p][5], v[p][6], v[p][7]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2<T>(v[p][2 * i], v[p][2 * i + 1]);
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if constexpr (ROWS) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) top = max(top, __float_as_uint(v[p][i]) & 0x7FFFFFFFu);
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const uint32_t e8 = scale_code(top, args.up);
      const uint32_t codes = encode8(v[p], inverse_scale(e8), e8);
      const long long r = r0 + lr;
      if (r < args.rows && c0 + col < 2 * pitch)
        *reinterpret_cast<uint32_t*>(args.codes + r * pitch + (c0 + col) / 2) = codes;
      if ((tid & 3) == 0)
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
    const int pair = tid & 63, group = tid >> 6;  // columns 2 pair, 2 pair + 1; rows 32 group..
    float a[32], b[32];
    uint32_t ta = 0, tb = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const T* src = tile + (group * 32 + i) * kTile + 2 * pair;
      if constexpr (sizeof(T) == 4) {
        const float2 f = *reinterpret_cast<const float2*>(src);
        a[i] = f.x, b[i] = f.y;
      } else {
        unpack2<T>(*reinterpret_cast<const uint32_t*>(src), a[i], b[i]);
      }
      ta = max(ta, __float_as_uint(a[i]) & 0x7FFFFFFFu);
      tb = max(tb, __float_as_uint(b[i]) & 0x7FFFFFFFu);
    }
    const uint32_t ea = scale_code(ta, args.up), eb = scale_code(tb, args.up);
    uint32_t ca[4], cb[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f[kVec], g[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] = a[8 * q + i], g[i] = b[8 * q + i];
      ca[q] = encode8(f, inverse_scale(ea), ea);
      cb[q] = encode8(g, inverse_scale(eb), eb);
    }
    uint8_t* dst = s_codes_t + 2 * pair * kCodesPitch + group * 16;
    *reinterpret_cast<uint4*>(dst) = make_uint4(ca[0], ca[1], ca[2], ca[3]);
    *reinterpret_cast<uint4*>(dst + kCodesPitch) = make_uint4(cb[0], cb[1], cb[2], cb[3]);
    const int ca0 = 2 * pair, cb0 = ca0 + 1;
    s_scales_t[(ca0 & 31) * 16 + (ca0 >> 5) * 4 + group] = static_cast<uint8_t>(ea);
    s_scales_t[(cb0 & 31) * 16 + (cb0 >> 5) * 4 + group] = static_cast<uint8_t>(eb);
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
  const int smem = (COLS ? kTile * kTile * static_cast<int>(sizeof(T)) : 0) + (ROWS ? kHalfBytes : 0) +
                   (COLS ? kHalfBytes + kTile * kCodesPitch : 0);
  auto fn = quantize_kernel<T, VEC, ROWS, COLS>;
  static DeviceIntCache cap_cache;
  const int cap = cap_cache.get(facts.device, [&] {
    return raise_dynamic_smem(reinterpret_cast<const void*>(fn), facts.max_smem_optin);
  });
  if (cap < smem) return TCB_ERR_RESOURCE;
  clear_stale_error();
  fn<<<static_cast<unsigned>(tiles), kThreads, smem, stream>>>(args);
  return launch_status();
}

template <typename T>
int run_quantize(const QuantArgs& args, long long tiles, const DeviceFacts& facts,
                 cudaStream_t stream) {
  // 16-byte loads need a 16-byte base and row pitch; anything else is read
  // element by element.
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
  int vec;  // rows of y start on 16-byte boundaries
};

// The same tiles the other way: a thread turns 4 code bytes of a row into 8
// values.  code * 2^e is exact in fp32 and is rounded once to T.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(const __grid_constant__ DequantArgs args) {
  __shared__ __align__(16) uint8_t s_scales[kHalfBytes];
  const int tid = threadIdx.x;
  const long long tiles_x = args.tiles_x;  // tiles that hold values (the last may be half past the edge)
  const long long tx = static_cast<long long>(blockIdx.x) % tiles_x;
  const long long ty = static_cast<long long>(blockIdx.x) / tiles_x;
  const long long r0 = ty * kTile, c0 = tx * kTile;
  const int col = (tid % kLanesPerRow) * kVec;
  const int row = tid / kLanesPerRow;
  const long long pitch = mx_padded(args.cols) / 2;
  const long long left = args.cols - c0 - col;
  const int valid = left <= 0 ? 0 : left >= kVec ? kVec : static_cast<int>(left);
  uint32_t w[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const long long r = r0 + row + p * kRowsPerPass;
    w[p] = valid > 0 && r < args.rows
               ? __ldg(reinterpret_cast<const uint32_t*>(args.codes + r * pitch + (c0 + col) / 2))
               : 0u;
  }
  if (tid < kHalfBytes / 16)
    reinterpret_cast<uint4*>(s_scales)[tid] = __ldg(
        reinterpret_cast<const uint4*>(args.scales + (ty * mx_tiles(args.cols) + tx) * kHalfBytes) + tid);
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int lr = row + p * kRowsPerPass;
    const long long r = r0 + lr;
    if (valid == 0 || r >= args.rows) continue;
    const float scale = scale_value(s_scales[(lr & 31) * 16 + (lr >> 5) * 4 + (col >> 5)]);
    uint32_t h[4];
    decode8(w[p], h);
    float v[kVec];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unpack2<__half>(h[i], v[2 * i], v[2 * i + 1]);
      v[2 * i] *= scale;
      v[2 * i + 1] *= scale;
    }
    T* dst = static_cast<T*>(args.y) + r * args.ld + c0 + col;
    if (args.vec && valid == kVec) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                    pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (i < valid) dst[i] = from_float<T>(v[i]);
    }
  }
}

template <typename T>
int launch_dequantize(DequantArgs args, cudaStream_t stream) {
  args.vec = aligned(args.y, 16) && args.ld * static_cast<long long>(sizeof(T)) % 16 == 0;
  const long long tiles = args.tiles_x * ((args.rows + kTile - 1) / kTile);
  if (tiles > INT_MAX) return TCB_ERR_RESOURCE;
  clear_stale_error();
  dequantize_kernel<T><<<static_cast<unsigned>(tiles), kThreads, 0, stream>>>(args);
  return launch_status();
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
