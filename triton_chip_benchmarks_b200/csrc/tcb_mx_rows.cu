// Products of a few rows with an MX FP4 weight (sm_100a): Y = X . W^T.
//
// X has M rows (tokens) of bf16, fp16 or MX FP4; W [N][K] is MX FP4.  With few
// rows the weight's bytes are all that counts: 17/32 byte a weight, read once.
// The tensor core does the arithmetic as mma.sync m16n8k16 (fp16 x fp16 ->
// fp32) with 16 weight rows as the M side and 8 tokens as the N side: E2M1 is
// exact in fp16, and one cvt decodes two codes.  (tcgen05 would want the
// decoded weights back in shared memory or tensor memory; here they go from
// registers straight into the MMA.)
//
//   y[t][n] = sum_blocks 2^ex(t, block) sum_groups 2^ew(n, group) tmp,
//   tmp = sum over the group's 32 values of x'[t][k] * code(w[n][k]).
//
// tmp is one pair of MMAs from a zero accumulator; the group's weight scale is
// applied to it in fp32, so any E8M0 scale is exact.  bf16 rows are brought
// into fp16's range by a power of two per token and 256 values of K, which
// puts the largest at 2^14..2^15: values down to 2^-31 of the largest stay
// exact and smaller ones are rounded to 2^-39 of it, below what an fp32 sum
// that holds the largest can show.  fp16 rows are taken as they are; MX rows
// are decoded, their scale per group applied with the weight's.
//
// Data flow.  A CTA owns 128 rows of W and a slice of K.  A producer warp
// TMA-loads stages of 256 K values (128 bytes of codes x 128 rows in the
// 128-byte swizzle, 1 KB of packed scales, the X tile) into a ring; four X warps
// turn the X tile into fp16 fragments in place; eight consumer warps take 16
// weight rows each.  A lane's four code bytes of a row (a quarter of a group)
// are k = 8t..8t+7 of the group; the order of k inside an MMA is free as long
// as X follows it, so its X fragment is one 16-byte load.
//
// Split over K.  With fewer row tiles than SMs, up to eight CTAs of a cluster
// share a row tile, each with a part of K, and add their partial sums through
// distributed shared memory in rank order: one launch, no workspace, the same
// result every time.
#include <cudaTypedefs.h>

#include "tcb_device.cuh"
#include "tcb_gemm_common.cuh"
#include "tcb_host.h"
#include "tcb_mx.cuh"
#include "tcb_mx_rows.h"

namespace tcb {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace {

using namespace mx_detail;
using gemm_detail::bulk_load_1d;
using gemm_detail::mbar_arrive;
using gemm_detail::wait_or_abort;

constexpr int kRowTile = 128;
constexpr int kConsumerWarps = kRowTile / 16;
constexpr int kXWarps = 4;
constexpr int kProducerWarp = kConsumerWarps;
constexpr int kRowsThreads = (kConsumerWarps + 1 + kXWarps) * 32;
constexpr int kBlockK = 256;                       // K values of a stage
constexpr int kWBytes = kRowTile * kBlockK / 2;    // 16 KB of codes
constexpr int kScaleBytes = kRowTile * kBlockK / 32;
constexpr int kMaxRingStages = 8;
constexpr int kPartialPitch = kRowTile + 4;        // floats of a token's partial sums
constexpr int kMaxSplit = 8;

// NT token tiles of 8.
template <int XT, int NT>
struct Rows {
  static constexpr int kTokens = 8 * NT;
  static constexpr int kXBytes = kTokens * kBlockK * 2;                       // fp16 fragments
  static constexpr int kXScales = XT == kRowsMx ? 8 * kTokens : kTokens;      // fp32 factors
  static constexpr int kRawBytes = XT == kRowsMx ? kTokens * kBlockK / 2 + kScaleBytes : 0;
  static constexpr int kStageBytes =
      (kWBytes + kScaleBytes + kXBytes + kRawBytes + kXScales * 4 + 1023) / 1024 * 1024;
  static constexpr int kCtas = NT <= 2 ? 2 : 1;    // per SM
  static constexpr int kBudget = (kCtas == 2 ? 112 : 224) * 1024 - 1024;
  static constexpr int kStages =
      kBudget / kStageBytes > kMaxRingStages ? kMaxRingStages : kBudget / kStageBytes;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static_assert(kStages >= 2, "a ring needs two stages");
  static_assert(kTokens * kPartialPitch * 4 <= kStages * kStageBytes, "partial sums reuse the ring");
};

struct RowsArgs {
  const uint8_t* sw;    // packed scales of W
  const uint8_t* sx;    // packed scales of X (MX)
  const void* x;        // X, for rows that TMA cannot read
  const void* bias;
  void* y;
  long long ldx, ldy;
  int* status;
  int m, n, k;
  int kblocks;
  int split;            // CTAs of a cluster
  int x_tma;
  int y_type;           // RowsType of y and the bias
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1, const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
        "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// 16-byte chunk c of a token's 512 bytes of fragments: tokens 2i and 2i + 1,
// which a quarter-warp reads together, use opposite halves of a 128-byte line.
__device__ __forceinline__ int x_chunk(int token, int c) { return token * 32 + (c ^ ((token & 1) << 2)); }

// One lane's 8 values of a token (16-bit words) as fp16 fragments; returns the
// factor that the block's sums are multiplied with.
template <int XT>
__device__ __forceinline__ float x_fragment(const uint32_t (&w)[4], uint32_t (&h)[4]) {
  if constexpr (XT == kRowsFp16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = w[i];
    return 1.0f;
  } else {
    float v[8];
    uint32_t top = 0;  // largest finite |x|
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2<__nv_bfloat16>(w[i], v[2 * i], v[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(v[i]) & 0x7FFFFFFFu;
      top = max(top, u < 0x7F800000u ? u : 0u);
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    // 2^(14 - exponent of the largest), at most 2^127, and its reciprocal.
    const uint32_t fe = min(268u - (top >> 23), 254u);
    const float factor = __uint_as_float(fe << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = pack2<__half>(v[2 * i] * factor, v[2 * i + 1] * factor);
    return __uint_as_float(fe == 254u ? 0x00400000u : (254u - fe) << 23);
  }
}

template <int XT, int NT>
__global__ void __launch_bounds__(kRowsThreads, Rows<XT, NT>::kCtas)
    mx_rows_kernel(const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ RowsArgs args) {
  using R = Rows<XT, NT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t loaded[R::kStages];
  __shared__ __align__(8) uint64_t ready[R::kStages];
  __shared__ __align__(8) uint64_t empty[R::kStages];
  __shared__ volatile int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / args.split, rank = blockIdx.x % args.split;
  const int token0 = blockIdx.y * R::kTokens;
  const int kb0 = static_cast<int>(static_cast<long long>(args.kblocks) * rank / args.split);
  const int kb1 = static_cast<int>(static_cast<long long>(args.kblocks) * (rank + 1) / args.split);

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    if (args.x_tma) prefetch_tensormap(&map_x);
    for (int s = 0; s < R::kStages; ++s) {
      mbar_init(&loaded[s], 1);
      mbar_init(&ready[s], kXWarps);
      mbar_init(&empty[s], kConsumerWarps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  float total[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) total[n][i] = 0.0f;

  if (warp == kProducerWarp) {
    if (lane == 0) {
      const uint32_t bytes = kWBytes + kScaleBytes +
                             (args.x_tma ? (XT == kRowsMx ? R::kTokens * kBlockK / 2 : R::kXBytes) : 0) +
                             (XT == kRowsMx ? kScaleBytes : 0);
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % R::kStages;
        if (!wait_or_abort(&empty[s], (static_cast<uint32_t>(it / R::kStages) & 1u) ^ 1u,
                           &abort_flag, args.status))
          break;
        uint8_t* stage = smem + s * R::kStageBytes;
        mbar_arrive_expect_tx(&loaded[s], bytes);
        tma_load_2d(stage, &map_w, kb * (kBlockK / 2), tile * kRowTile, &loaded[s]);
        bulk_load_1d(stage + kWBytes,
                     args.sw + (static_cast<long long>(tile) * args.kblocks + kb) * kScaleBytes,
                     kScaleBytes, &loaded[s]);
        uint8_t* xs = stage + kWBytes + kScaleBytes;
        if constexpr (XT == kRowsMx) {
          tma_load_2d(xs + R::kXBytes, &map_x, kb * (kBlockK / 2), token0, &loaded[s]);
          bulk_load_1d(xs + R::kXBytes + R::kTokens * kBlockK / 2,
                       args.sx + (static_cast<long long>(token0 / 128) * args.kblocks + kb) * kScaleBytes,
                       kScaleBytes, &loaded[s]);
        } else if (args.x_tma) {
          tma_load_2d(xs, &map_x, kb * kBlockK, token0, &loaded[s]);
        }
      }
      // After an abort too, no load is left in flight (each of the last round's
      // barriers is still in the phase it was armed for).
      for (int j = it > R::kStages ? it - R::kStages : 0; j < it; ++j)
        mbar_wait(&loaded[j % R::kStages], static_cast<uint32_t>(j / R::kStages) & 1u);
    }
    __syncwarp();
  } else if (warp > kProducerWarp) {
    // -------------------------------------------------------------- X warps
    for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
      const int s = it % R::kStages;
      if (!__all_sync(0xFFFFFFFFu, wait_or_abort(&loaded[s], static_cast<uint32_t>(it / R::kStages) & 1u,
                                                 &abort_flag, args.status)))
        break;
      uint8_t* x = smem + s * R::kStageBytes + kWBytes + kScaleBytes;
      uint4* chunks = reinterpret_cast<uint4*>(x);
      float* factors = reinterpret_cast<float*>(x + R::kXBytes + R::kRawBytes);
#pragma unroll 4
      for (int token = warp - kProducerWarp - 1; token < R::kTokens; token += kXWarps) {
        uint32_t h[4];
        if constexpr (XT == kRowsMx) {
          const uint8_t* raw = x + R::kXBytes;
          decode8(reinterpret_cast<const uint32_t*>(raw + token * (kBlockK / 2))[lane], h);
          if (lane < 8) {
            const int r = (token0 + token) & 127;
            factors[token * 8 + lane] = scale_value(
                raw[R::kTokens * kBlockK / 2 + (lane >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (lane & 3)]);
          }
        } else {
          uint32_t w[4];
          if (args.x_tma) {
            const uint4 q = chunks[token * 32 + lane];
            w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
          } else {
            const uint16_t* src = static_cast<const uint16_t*>(args.x) +
                                  static_cast<long long>(token0 + token) * args.ldx;
            const int k = kb * kBlockK + lane * 8;
            const bool in = token0 + token < args.m;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t lo = in && k + 2 * i < args.k ? src[k + 2 * i] : 0u;
              const uint32_t hi = in && k + 2 * i + 1 < args.k ? src[k + 2 * i + 1] : 0u;
              w[i] = lo | hi << 16;
            }
          }
          const float factor = x_fragment<XT>(w, h);
          if (lane == 0) factors[token] = factor;
          __syncwarp();  // every lane has read its chunk before any is overwritten
        }
        chunks[x_chunk(token, lane)] = make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_proxy_async_smem();  // the ring's next TMA load of these bytes comes after them
      __syncwarp();
      if (lane == 0) mbar_arrive(&ready[s]);
    }
  } else {
    // ------------------------------------------------------------ consumers
    const int g = lane >> 2, t = lane & 3;
    const int r = warp * 16 + g;  // this lane's rows of the tile: r and r + 8
    for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
      const int s = it % R::kStages;
      const uint32_t phase = static_cast<uint32_t>(it / R::kStages) & 1u;
      if (!__all_sync(0xFFFFFFFFu, wait_or_abort(&loaded[s], phase, &abort_flag, args.status) &&
                                       wait_or_abort(&ready[s], phase, &abort_flag, args.status)))
        break;
      const uint8_t* stage = smem + s * R::kStageBytes;
      const uint8_t* wa = stage + r * 128 + 4 * t;
      const uint8_t* sc = stage + kWBytes + (r & 31) * 16 + (r >> 5) * 4;
      const uint4* chunks = reinterpret_cast<const uint4*>(stage + kWBytes + kScaleBytes);
      const float* factors = reinterpret_cast<const float*>(stage + kWBytes + kScaleBytes + R::kXBytes +
                                                            R::kRawBytes);
      float block[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) block[n][i] = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t s0 = *reinterpret_cast<const uint32_t*>(sc + half * 512);
        const uint32_t s1 = *reinterpret_cast<const uint32_t*>(sc + half * 512 + 8 * 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int j = half * 4 + q;
          uint32_t h0[4], h1[4];
          decode8(*reinterpret_cast<const uint32_t*>(wa + ((j ^ g) << 4)), h0);
          decode8(*reinterpret_cast<const uint32_t*>(wa + 8 * 128 + ((j ^ g) << 4)), h1);
          const float f0 = scale_value((s0 >> (8 * q)) & 255u);
          const float f1 = scale_value((s1 >> (8 * q)) & 255u);
          const uint32_t a0[4] = {h0[0], h1[0], h0[1], h1[1]};
          const uint32_t a1[4] = {h0[2], h1[2], h0[3], h1[3]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 b = chunks[x_chunk(8 * n + g, 4 * j + t)];
            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            float d[4];
            mma_f16(d, a0, b.x, b.y, zero);
            mma_f16(d, a1, b.z, b.w, d);
            if constexpr (XT == kRowsMx) {
              const float x0 = factors[(8 * n + 2 * t) * 8 + j];
              const float x1 = factors[(8 * n + 2 * t + 1) * 8 + j];
              total[n][0] = fmaf(d[0] * f0, x0, total[n][0]);
              total[n][1] = fmaf(d[1] * f0, x1, total[n][1]);
              total[n][2] = fmaf(d[2] * f1, x0, total[n][2]);
              total[n][3] = fmaf(d[3] * f1, x1, total[n][3]);
            } else {
              block[n][0] = fmaf(d[0], f0, block[n][0]);
              block[n][1] = fmaf(d[1], f0, block[n][1]);
              block[n][2] = fmaf(d[2], f1, block[n][2]);
              block[n][3] = fmaf(d[3], f1, block[n][3]);
            }
          }
        }
      }
      if constexpr (XT != kRowsMx) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float2 x = *reinterpret_cast<const float2*>(factors + 8 * n + 2 * t);
          total[n][0] = fmaf(block[n][0], x.x, total[n][0]);
          total[n][1] = fmaf(block[n][1], x.y, total[n][1]);
          total[n][2] = fmaf(block[n][2], x.x, total[n][2]);
          total[n][3] = fmaf(block[n][3], x.y, total[n][3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
  }

  // Partial sums [token][row] where the ring was: every load has landed and
  // been read (after an abort the output is void and nothing is stored).
  __syncthreads();
  if (abort_flag) {
    cluster_sync_all();
    cluster_sync_all();
    return;
  }
  float* partial = reinterpret_cast<float*>(smem);
  if (warp < kConsumerWarps) {
    const int g = lane >> 2, t = lane & 3, r = warp * 16 + g;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* p = partial + (8 * n + 2 * t) * kPartialPitch + r;
      p[0] = total[n][0];
      p[kPartialPitch] = total[n][1];
      p[8] = total[n][2];
      p[kPartialPitch + 8] = total[n][3];
    }
  }
  cluster_sync_all();
  const int tokens = min(R::kTokens, args.m - token0);
  const uint32_t base = smem_addr(partial);
  // Output i = (token, row) belongs to rank i / kRowsThreads mod split.
  for (int i = rank * kRowsThreads + threadIdx.x; i < tokens * kRowTile;
       i += args.split * kRowsThreads) {
    const int token = i / kRowTile, row = i % kRowTile;
    const long long n = static_cast<long long>(tile) * kRowTile + row;
    if (n >= args.n) continue;
    const uint32_t at = base + static_cast<uint32_t>((token * kPartialPitch + row) * 4);
    float sum = 0.0f;
    for (int q = 0; q < args.split; ++q) sum += ld_shared_cluster_f32(mapa_shared(at, q));
    const long long out = (token0 + token) * args.ldy + n;
    if (args.y_type == kRowsFp32) {
      if (args.bias) sum += static_cast<const float*>(args.bias)[n];
      static_cast<float*>(args.y)[out] = sum;
    } else if (args.y_type == kRowsBf16) {
      if (args.bias) sum += to_float(static_cast<const __nv_bfloat16*>(args.bias)[n]);
      static_cast<__nv_bfloat16*>(args.y)[out] = from_float<__nv_bfloat16>(sum);
    } else {
      if (args.bias) sum += to_float(static_cast<const __half*>(args.bias)[n]);
      static_cast<__half*>(args.y)[out] = from_float<__half>(sum);
    }
  }
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while a peer may still read its partial sums
}

// 2-D map of 128 rows of codes in the 128-byte swizzle (W), or of the X tile.
int rows_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long inner,
             long long rows, long long pitch_bytes, int box_inner, int box_rows,
             CUtensorMapSwizzle swizzle) {
  auto fn = tensor_map_encoder();
  if (fn == nullptr) return TCB_ERR_DEVICE;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch_bytes)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TCB_OK
             : TCB_ERR_INVALID_ARGUMENT;
}

template <int XT, int NT>
int launch_rows(const RowsProblem& p, int* status, const DeviceFacts& facts, cudaStream_t stream) {
  using R = Rows<XT, NT>;
  const long long kp = mx_padded(p.k);
  RowsArgs args;
  args.sw = static_cast<const uint8_t*>(p.sw);
  args.sx = static_cast<const uint8_t*>(p.sx);
  args.x = p.x;
  args.bias = p.bias;
  args.y = p.y;
  args.ldx = p.ldx;
  args.ldy = p.ldy;
  args.status = status;
  args.m = p.m;
  args.n = p.n;
  args.k = p.k;
  args.kblocks = static_cast<int>((kp + kBlockK - 1) / kBlockK);
  args.y_type = p.y_type;
  CUtensorMap map_w, map_x{};
  int rc = rows_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, kp / 2, p.n, kp / 2, kBlockK / 2,
                    kRowTile, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != TCB_OK) return rc;
  if (XT == kRowsMx) {
    args.x_tma = 1;
    rc = rows_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.x, kp / 2, p.m, kp / 2, kBlockK / 2,
                  R::kTokens, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc != TCB_OK) return rc;
  } else {
    // TMA wants 16-byte rows; other rows are read by the X warps.
    args.x_tma = aligned(p.x, 16) && p.ldx % 8 == 0 &&
                 rows_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, p.x, p.k, p.m, p.ldx * 2, kBlockK,
                          R::kTokens, CU_TENSOR_MAP_SWIZZLE_NONE) == TCB_OK;
  }
  const long long tiles = (static_cast<long long>(p.n) + kRowTile - 1) / kRowTile;
  const long long chunks = (static_cast<long long>(p.m) + R::kTokens - 1) / R::kTokens;
  // As many CTAs of a row tile as fit beside the other tiles in one round of
  // the SMs, each with at least one K block.
  long long split = static_cast<long long>(facts.sm_count) * R::kCtas / (tiles * chunks);
  split = split > kMaxSplit ? kMaxSplit : split;
  split = split > args.kblocks ? args.kblocks : split;
  args.split = split < 1 ? 1 : static_cast<int>(split);
  if (tiles * args.split > INT_MAX || chunks > 65535) return TCB_ERR_RESOURCE;
  auto fn = mx_rows_kernel<XT, NT>;
  static DeviceIntCache cap_cache;
  const int cap = cap_cache.get(facts.device, [&] {
    return raise_dynamic_smem(reinterpret_cast<const void*>(fn), facts.max_smem_optin);
  });
  if (cap < R::kSmem) return TCB_ERR_RESOURCE;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles * args.split), static_cast<unsigned>(chunks), 1);
  config.blockDim = dim3(kRowsThreads, 1, 1);
  config.dynamicSmemBytes = R::kSmem;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(args.split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  clear_stale_error();
  if (cudaLaunchKernelEx(&config, fn, map_w, map_x, args) != cudaSuccess) {
    clear_stale_error();
    return TCB_ERR_LAUNCH;
  }
  return TCB_OK;
}

template <int XT>
int run_tokens(const RowsProblem& p, int* status, const DeviceFacts& facts, cudaStream_t stream) {
  if (p.m <= 8) return launch_rows<XT, 1>(p, status, facts, stream);
  if (p.m <= 16) return launch_rows<XT, 2>(p, status, facts, stream);
  if (p.m <= 32) return launch_rows<XT, 4>(p, status, facts, stream);
  return launch_rows<XT, 8>(p, status, facts, stream);
}

}  // namespace

int mx_rows_run(const RowsProblem& p, int* status, const DeviceFacts& facts, cudaStream_t stream) {
  switch (p.x_type) {
    case kRowsBf16: return run_tokens<kRowsBf16>(p, status, facts, stream);
    case kRowsFp16: return run_tokens<kRowsFp16>(p, status, facts, stream);
    case kRowsMx: return run_tokens<kRowsMx>(p, status, facts, stream);
  }
  return TCB_ERR_UNSUPPORTED;
}

}  // namespace tcb
