// Products of a few rows with an MX FP4 weight on 5th-generation tensor cores
// (sm_100a): Y = X . W^T, W [N][K] in MX FP4, X a few rows of MX FP4, bf16 or fp16.
//
// With few rows the weight's bytes are all that counts (17/32 byte a weight,
// read once), so the weight takes the M side of the MMA -- 128 rows a CTA, all
// SMs busy -- and X the N side, 8 to 128 columns of
// tcgen05.mma kind::mxf4.block_scale: nothing is decoded by threads.
//
// 16-bit rows take part as eight or nine MX FP4 digits each (tcb_mx_digits.cuh), columns that
// the epilogue adds, and as products with what the digits leave.  (Decoding W to fp16 for
// mma.sync instead was bound by issue slots: 24 us at 1 x 16384 x 8192, 31 us for 16 MX
// rows at 8192 x 8192.)
//
// Where the digits come from.  Up to kInlineTokens rows, X warps of each CTA write
// the digits of its K slice into shared memory on the way; for more rows a
// kernel of their own writes them once (into the caller's workspace), and the
// product starts beside it: its weight loads are under way before the digits
// are there.  16 bf16 or 14 fp16 rows fill the 128 columns of a tile; column tiles share
// the weight through L2 while all of them run at once, and more digits than that become
// columns of the CTA-pair GEMM.
//
// Split over K.  With fewer row tiles than CTAs fit, up to eight CTAs of a
// cluster share a row tile, each with a part of K.  Each sends the others their
// share of its partial sums (stores into distributed shared memory) and adds
// its own share in rank order: no workspace, the same result every time, and
// one cluster barrier to wait for (the sums of up to kEarlyTokens tokens have room
// of their own; those of more go where the ring was, which all CTAs must have left).
//
// Roles of a CTA (one tile each):
//   warp 0      producer: per 256 K values, TMA loads of W (128 rows x 128 B) and X
//               (128-byte swizzle), bulk copies of their packed scales;
//   warp 1      MMA issuer: four MMAs a stage into one accumulator;
//   warps 2-5   scale writers (shared -> tensor memory), which also multiply what a
//               stage's digits leave, then the epilogue;
//   warps 6-9   X warps (inline digits only).
// What bounds it: HBM while the weights stream (25 B/clk per SM at two CTAs), and
// about 5 us around that: start, first loads, the cluster's join, the end.
// Captured and back to back, bf16 rows: 1 x 16384 x 8192 16.5 us (71 MB, 4.3 TB/s), 1 x
// 4096 x 4096 6.8, 16 x 16384 x 8192 21.2 with the digits' kernel (19.9 where they leave
// nothing); 16 MX rows at 8192 x 8192 9.7.
// Every wait is bounded; a wait that runs out raises the CTA's abort flag, all
// roles leave their loops, copies and MMAs in flight are waited for (bounded
// too), the CTA sends and stores nothing, and the status reports it.
#include <cudaTypedefs.h>
#include <type_traits>

#include "tcb_device.cuh"
#include "tcb_gemm_common.cuh"
#include "tcb_gemm_pair.h"
#include "tcb_host.h"
#include "tcb_mx_digits.cuh"
#include "tcb_mx_rows.h"

namespace tcb {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace {

using namespace mx_detail;
using gemm_detail::bulk_load_1d;
using gemm_detail::kBlockBytes;
using gemm_detail::kSfPairCols;
using gemm_detail::kSfStageCols;
using gemm_detail::kStepsPerBlock;
using gemm_detail::mbar_arrive;
using gemm_detail::sf_cols_a;
using gemm_detail::sf_cols_b;
using gemm_detail::sf_idesc;
using gemm_detail::wait_or_abort;

constexpr int kRowTile = 128;                     // weight rows of a CTA
constexpr int kBlockK = 2 * kBlockBytes;          // K values of a stage
constexpr int kWBytes = kRowTile * kBlockBytes;   // 16 KB
constexpr int kScaleBlock = 1024;                 // packed scales of 128 rows x 256 values
constexpr int kMaxStages = 8;
constexpr int kInlineTokens = 2;
constexpr int kXWarps = 4;
constexpr int kMaxSplit = 8;
constexpr int kEarlyTokens = 16;
constexpr int kSumBytes = kEarlyTokens * kRowTile * 4;
static_assert(Bf16Tile::kPerTile * Bf16Tile::kRows == kRowTile && Fp16Tile::kPerTile * Fp16Tile::kRows == kRowTile,
              "a column tile");
static_assert(Bf16Tile::kTileTokens <= kEarlyTokens && Fp16Tile::kTileTokens <= kEarlyTokens,
              "what the digits leave goes where the ring was, beside the sums");
// Two CTAs share an SM: half of its shared memory and of its tensor memory each.
// (One CTA with twice the stages has the same bytes in flight but one MMA thread
// and no second tile to cover its start and end: 28.6 us instead of 17.0 at
// 1 x 32768 x 4096.)
constexpr int kSmemBudget = 112 * 1024 + 512;  // 512 bytes below half of 228 KB less 1 KB a CTA
constexpr int kCtaTmemCols = 256;

enum XMode : int { kXRows = 0, kXDigits = 1, kXInline = 2 };
constexpr int rows_threads(int mode) { return (6 + (mode == kXInline ? kXWarps : 0)) * 32; }

struct RowsArgs {
  const uint8_t* sw;     // packed scales of W
  const uint8_t* sx;     // packed scales of X's rows or digits
  ValueRows x;           // 16-bit X
  const LeftList* lists; // what its digits leave
  const void* bias;
  void* y;
  long long pitch;       // code bytes of a row of W
  long long ldy;
  int* status;
  int m, n;
  int kblocks;
  int split;             // CTAs of a cluster
  int stages, stage_bytes;
  int cols;              // columns of the MMA (a multiple of 8, at most 128)
  int col_tiles;         // of 128 columns each, if there are more than one
  int y_type;            // RowsType of y and the bias
  uint32_t idesc;
};

// A role's place in the ring of stages.  Counted up, not divided out of a stage
// number: two divisions a stage cost the MMA thread 400 of its 900 cycles.
struct RingPlace {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int by, int stages) {
    s += by;
    if (s >= stages) s -= stages, phase ^= 1u;  // by <= stages
  }
};

__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate, uint32_t tsfa, uint32_t tsfb) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, "
      "[%5], [%6], p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tsfa), "r"(tsfb));
}

__device__ __forceinline__ void tmem_ld_8cols(uint32_t taddr, float (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_1col(uint32_t taddr, float& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=f"(r) : "r"(taddr) : "memory");
}

__device__ __forceinline__ void st_shared_cluster_f32(uint32_t cluster_addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// Digits of a list's tokens in one K block, a warp a token, and the list of what they
// leave.
template <typename Layout>
__global__ void __launch_bounds__(Layout::kTokens * 32)
    mx_digits_kernel(const __grid_constant__ ValueRows rows, long long pitch, int kblocks, uint8_t* codes,
                     uint8_t* scales, LeftList* lists) {
  __shared__ uint32_t counts[Layout::kTokens];
  // The product may start once the kernels before this one are done: its weight
  // may be theirs.
  wait_for_previous_kernels();
  let_next_kernel_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kb = static_cast<int>(blockIdx.x) % kblocks;
  const long long at = static_cast<long long>(blockIdx.x) / kblocks;  // the list
  const long long token = at * Layout::kTokens + warp;
  uint4 raw = make_uint4(0, 0, 0, 0);
  float left[8];
  int e8 = 0;
  bool any = false;
  if (token < rows.m) {
    raw = load_values(rows, token, kb * kBlockK + lane * 8);
    const long long byte = static_cast<long long>(kb) * kBlockBytes + lane * 4;
    const int group = lane >> 2;
    any = split_digits<Layout::kDigits>(raw, rows.bf16, left, e8, [&](int d, uint8_t code, uint32_t words) {
      const long long row = at * Layout::kRows + warp * Layout::kDigits + d;
      if (byte < pitch) *reinterpret_cast<uint32_t*>(codes + row * pitch + byte) = words;
      if ((lane & 3) == 0)
        scales[((row >> 7) * kblocks + kb) * kScaleBlock + (group >> 2) * 512 + (row & 31) * 16 +
               ((row & 127) >> 5) * 4 + (group & 3)] = code;
    });
  }
  if (any) left_of<Layout::kDigits>(raw, rows.bf16, left, e8);
  const uint32_t mine = any ? count_left(left) : 0u;
  const uint32_t warp_total = __reduce_add_sync(0xFFFFFFFFu, mine);
  if (lane == 0) counts[warp] = warp_total;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < Layout::kTokens; ++i) {
    const uint32_t n = counts[i];
    if (i < warp) before += n;
    total += n;
  }
  LeftList* list = lists + Layout::index(at, kb, kblocks);
  if (threadIdx.x == 0) list->count = total;
  if (warp_total != 0) append_left(list, before, mine, static_cast<uint32_t>(warp), left);
}

// What a list that is too short counts, for one of its tokens, as add_listed; out of the
// way of the stages' loop.
template <typename Layout>
__device__ __noinline__ float left_of_full_list(const RowsArgs& args, long long token, int kb, const uint8_t* codes,
                                                const uint8_t* scales, int row) {
  if (token >= args.x.m) return 0.0f;
  const uint8_t* mine = codes + row * kBlockBytes;
  const uint8_t* scale = scales + (row & 31) * 16 + (row >> 5) * 4;
  return left_again<Layout::kDigits>(
      args.x, token, kb,
      [&](int from) {
        return *reinterpret_cast<const uint32_t*>(mine + ((from >> 2 ^ (row & 7)) << 4) + (from & 3) * 4);
      },
      [&](int group) { return scale_value(scale[(group >> 2) * 512 + (group & 3)]); });
}

// sums[t] += the weight row of this lane (row 0..127 of the tile) times what the lists of
// a stage say of token t.  The warp has the lists in registers, eight lanes one (zeros: no
// list).  codes, scales: the stage's weights in shared
// memory.  A loop of few instructions: most of the time goes into fetching them, as the
// code runs once in a while (two or four entries at once took longer, in registers too:
// 33 x 5000 x 4136, three entries a stage, 16.0 us so, 16.5 and 17.9).
template <typename Layout>
__device__ __forceinline__ void add_listed(uint4 word, const uint8_t* codes, const uint8_t* scales, int row,
                                           float* sums) {
  const int lane = threadIdx.x & 31, first = 2 * (lane & 7);  // of the list's 16 words: the count, 15 entries
  const int count = static_cast<int>(__shfl_sync(0xFFFFFFFFu, word.x, lane & 24));
  const uint32_t list = static_cast<uint32_t>(lane >> 3) * LeftEntry::token(Layout::kTokens);
  const float value = decode1(lane & 15);                        // of code lane % 16
  const uint32_t mine = smem_addr(codes) + row * kBlockBytes;    // 16-byte chunk c at c ^ (row % 8)
  const uint32_t swizzle = (row & 7) << 4;
  const uint32_t scale = smem_addr(scales) + (row & 31) * 16 + (row >> 5) * 4;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const int at_word = first + half;
    uint32_t left = __ballot_sync(0xFFFFFFFFu, at_word > 0 && at_word <= count && count <= kLeftEntries);
#pragma unroll 1
    for (; left != 0; left &= left - 1) {
      const int from = __ffs(left) - 1;
      const LeftEntry at{__shfl_sync(0xFFFFFFFFu, word.x + list, from)};
      const float v = __uint_as_float(__shfl_sync(0xFFFFFFFFu, word.y, from));
      uint32_t code, e8;
      asm volatile("ld.shared.u8 %0, [%1];" : "=r"(code) : "r"(mine + (at.byte() ^ swizzle)));
      asm volatile("ld.shared.u8 %0, [%1];" : "=r"(e8) : "r"(scale + at.scale()));
      // A NaN scale may pass as infinity: the row's product is not a number already.
      sums[at.token()] += v * (__shfl_sync(0xFFFFFFFFu, value, code >> at.shift()) *
                               __uint_as_float(max(e8 << 23, 0x00400000u)));
    }
    word.x = word.z, word.y = word.w;
  }
}

// Appends what the inline digits of a token leave to a stage's list of `listed`
// entries; u, raw, e8 and any are split_digits' of the warp.  Returns how many there are
// then.  Not inlined: what runs once in a while lies out of the way of what always runs
// (which every launch fetches: 7.25 us instead of 6.7 at 1 x 4096 x 4096).
template <int DIGITS>
__device__ __noinline__ uint32_t list_left(float4 u0, float4 u1, uint4 raw, bool bf16, int e8, bool any,
                                           uint32_t token, LeftList* list, uint32_t listed) {
  float left[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
  left_of<DIGITS>(raw, bf16, left, e8);
  const uint32_t mine = any ? count_left(left) : 0u;
  append_left(list, listed, mine, token, left);
  return listed + __reduce_add_sync(0xFFFFFFFFu, mine);
}

// The last step of a CTA: its rows' sums over the ranks in order, the bias, one
// rounding.  Item i is row i % share of token i / share (share a power of two).
template <typename T, int kThreads>
__device__ __forceinline__ void finish(const float* sums, int split, int tokens, int share_log2, int rows,
                                       const T* bias, T* y, long long ldy) {
  constexpr int kBatch = 4;  // loads in flight
  const int items = tokens << share_log2;
  for (int first = static_cast<int>(threadIdx.x); first < items; first += kBatch * kThreads) {
    float v[kBatch] = {};
    for (int q = 0; q < split; ++q) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (first + u * kThreads < items) v[u] += sums[q * items + first + u * kThreads];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = first + u * kThreads;
      const int token = i >> share_log2, row = i & ((1 << share_log2) - 1);
      if (i < items && row < rows)
        y[token * ldy + row] = from_float<T>(v[u] + (bias == nullptr ? 0.0f : to_float(bias[row])));
    }
  }
}

// Layout: of the digits of 16-bit rows.
template <int XMODE, typename Layout = Bf16Tile>
__global__ void __launch_bounds__(rows_threads(XMODE), 2)
    mx_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ RowsArgs args) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t loaded[kMaxStages];  // operand and scale bytes landed
  __shared__ __align__(8) uint64_t digits[kMaxStages];  // X warps wrote the stage's digits
  __shared__ __align__(8) uint64_t full[kMaxStages];    // scales are in tensor memory
  __shared__ __align__(8) uint64_t empty[kMaxStages];   // the stage's MMAs, and what digits leave, are done
  __shared__ __align__(8) uint64_t acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  // An offset from smem_raw, so that the compiler still knows it for shared memory.
  uint8_t* smem = smem_raw + (-smem_addr(smem_raw) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Column tiles of the same weight rows side by side: the weight comes from L2.
  const int rank = blockIdx.x % args.split, both = blockIdx.x / args.split;
  const int tile = both / args.col_tiles, col_tile = both % args.col_tiles;
  const int kb0 = static_cast<int>(static_cast<long long>(args.kblocks) * rank / args.split);
  const int kb1 = static_cast<int>(static_cast<long long>(args.kblocks) * (rank + 1) / args.split);
  const int nkb = kb1 - kb0;
  constexpr int kTileTokens = XMODE == kXRows ? kRowTile : Layout::kTileTokens;
  const int token0 = col_tile * kTileTokens;
  const int tokens = min(args.m - token0, kTileTokens);
  const int x_bytes = args.cols * kBlockBytes;
  const int list_count = (tokens + Layout::kTokens - 1) / Layout::kTokens;  // of a stage
  LeftList* stage_lists = reinterpret_cast<LeftList*>(smem + args.stages * args.stage_bytes + kSumBytes);

  auto load_w = [&](int it, int s) {
    const int kb = kb0 + it;
    uint8_t* stage = smem + s * args.stage_bytes;
    mbar_arrive_expect_tx(&loaded[s], kWBytes + kScaleBlock +
                                          (XMODE == kXInline ? 0 : x_bytes + kScaleBlock) +
                                          (XMODE == kXDigits ? list_count * static_cast<int>(sizeof(LeftList)) : 0));
    tma_load_2d(stage, &map_w, kb * kBlockBytes, tile * kRowTile, &loaded[s]);
    bulk_load_1d(stage + kWBytes + x_bytes,
                 args.sw + (static_cast<long long>(tile) * args.kblocks + kb) * kScaleBlock,
                 kScaleBlock, &loaded[s]);
  };
  auto load_x = [&](int it, int s) {
    uint8_t* stage = smem + s * args.stage_bytes;
    uint64_t* bar = &loaded[s];
    const int kb = kb0 + it;
    tma_load_2d(stage + kWBytes, &map_x, kb * kBlockBytes, col_tile * kRowTile, bar);
    bulk_load_1d(stage + kWBytes + x_bytes + kScaleBlock,
                 args.sx + (static_cast<long long>(col_tile) * args.kblocks + kb) * kScaleBlock, kScaleBlock,
                 bar);
    if constexpr (XMODE == kXDigits)
      bulk_load_1d(stage_lists + s * Layout::kPerTile,
                   args.lists + Layout::index(static_cast<long long>(col_tile) * Layout::kPerTile, kb, args.kblocks),
                   list_count * static_cast<int>(sizeof(LeftList)), bar);
  };
  // An X warp's next values (inline digits): asked for one round ahead, the first
  // ones before the weights, behind whose bytes they would otherwise queue.
  [[maybe_unused]] uint4 x_next[kInlineTokens];
  auto ask_x = [&](int it) {
#pragma unroll
    for (int i = 0; i < kInlineTokens; ++i)
      if (i < tokens && it < nkb) x_next[i] = load_values(args.x, i, (kb0 + it) * kBlockK + lane * 8);
  };
  if constexpr (XMODE == kXInline) {
    if (warp >= 6) {
      wait_for_previous_kernels();
      ask_x(warp - 6);
    }
  }
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    if (XMODE != kXInline) prefetch_tensormap(&map_x);
    for (int s = 0; s < args.stages; ++s) {
      mbar_init(&loaded[s], 1);
      mbar_init(&digits[s], 1);
      mbar_init(&full[s], 4);
      mbar_init(&empty[s], XMODE == kXRows ? 1 : 5);
    }
    mbar_init(&acc_full, 1);
    abort_flag = 0;
    fence_mbar_init();
    // The first round of loads goes out before anything else is set up.  (The
    // digits' kernel has waited for the kernels before it.)
    if (XMODE != kXDigits) wait_for_previous_kernels();
    for (int it = 0; it < min(nkb, args.stages); ++it) {
      load_w(it, it);
      if constexpr (XMODE == kXRows) load_x(it, it);
    }
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kCtaTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_arrive_started();
  let_next_kernel_start();
  wait_for_previous_kernels();
  const uint32_t tbase = tmem_slot;
  const uint32_t tsf = tbase + static_cast<uint32_t>((args.cols + 31) & ~31);
  const int row_of_lane = 32 * (warp & 3) + lane;
  // A scale writer's sums of what the digits leave: its lane's row, a token each.
  constexpr int kStageLists = XMODE == kXInline ? 1 : Layout::kPerTile, kStageTokens = kStageLists * Layout::kTokens;
  [[maybe_unused]] float left_sums[kStageTokens] = {};
  [[maybe_unused]] bool any_left = false;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const int first = min(nkb, args.stages);
      if constexpr (XMODE == kXDigits) {
        for (int j = 0; j < first; ++j) load_x(j, j);
      }
      int it = first;
      RingPlace at;  // stage it's, whose previous load is of phase at.phase
      for (; it < nkb; ++it) {
        if (!wait_or_abort(&empty[at.s], at.phase, &abort_flag, args.status)) break;
        load_w(it, at.s);
        if constexpr (XMODE != kXInline) load_x(it, at.s);
        at.advance(1, args.stages);
      }
      // No load stays in flight after an abort either: each barrier of the last
      // round is in the phase that it was armed for.
      for (int j = it > args.stages ? it - args.stages : 0; j < it; ++j)
        mbar_wait(&loaded[j % args.stages], static_cast<uint32_t>(j / args.stages) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    if (lane == 0) {
      const uint64_t desc_const = smem_desc(0, 16, 8 * kBlockBytes, 2u);
      const uint32_t smem0 = smem_addr(smem) >> 4;
      RingPlace at;
      for (int it = 0; it < nkb; ++it, at.advance(1, args.stages)) {
        const int s = at.s;
        const uint32_t phase = at.phase;
        // `full` follows `loaded` (and `digits`) in the scale writers, which have
        // waited for both.
        if (!wait_or_abort(&loaded[s], phase, &abort_flag, args.status)) break;
        if (XMODE == kXInline && !wait_or_abort(&digits[s], phase, &abort_flag, args.status)) break;
        if (!wait_or_abort(&full[s], phase, &abort_flag, args.status)) break;
        tc_fence_after();
        const uint32_t w_lo = smem0 + static_cast<uint32_t>(s * args.stage_bytes >> 4);
        const uint32_t x_lo = w_lo + (kWBytes >> 4);
        const uint32_t sf = tsf + static_cast<uint32_t>(s * kSfStageCols);
#pragma unroll
        for (int k = 0; k < kStepsPerBlock; ++k)
          mma_mxf4(tbase, desc_const | (w_lo + static_cast<uint32_t>(k * 2)),
                   desc_const | (x_lo + static_cast<uint32_t>(k * 2)), sf_idesc(args.idesc, k),
                   (it | k) != 0, sf_cols_a(sf, k), sf_cols_b(sf, k));
        tc_commit(&empty[s]);
      }
      // After an abort too, nothing this thread issued runs on.
      tc_commit(&acc_full);
      if (!mbar_wait(&acc_full, 0)) {
        abort_flag = 1;
        report_status(args.status, TCB_ERR_TIMEOUT);
      }
    }
    __syncwarp();
  } else if (warp < 6) {
    // ------------------------------------------------------ scale writers
    const uint32_t lane_base = tsf + ((32u * (warp & 3)) << 16);
    RingPlace at;
    for (int it = 0; it < nkb; ++it, at.advance(1, args.stages)) {
      const int s = at.s;
      const uint32_t phase = at.phase;
      bool ok = wait_or_abort(&loaded[s], phase, &abort_flag, args.status);
      if (XMODE == kXInline) ok = ok && wait_or_abort(&digits[s], phase, &abort_flag, args.status);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;  // tcgen05.st needs the whole warp
      const uint8_t* sw = smem + s * args.stage_bytes + kWBytes + x_bytes + lane * 16;
      gemm_detail::write_scale_block(lane_base + static_cast<uint32_t>(s * kSfStageCols), sw,
                                     sw + kScaleBlock, sw + kScaleBlock);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      if constexpr (XMODE != kXRows) {
        uint4 word = make_uint4(0, 0, 0, 0);
        if (lane < 8 * list_count) word = reinterpret_cast<const uint4*>(stage_lists + s * kStageLists)[lane];
        if (__any_sync(0xFFFFFFFFu, (lane & 7) == 0 && word.x != 0)) {
          any_left = true;
          add_listed<Layout>(word, smem + s * args.stage_bytes, sw - lane * 16, row_of_lane, left_sums);
          uint32_t full = __ballot_sync(0xFFFFFFFFu, (lane & 7) == 0 && word.x > kLeftEntries);
          for (; full != 0; full &= full - 1) {
            const int first = (__ffs(full) - 1) / 8 * Layout::kTokens;
            for (int t = first; t < first + Layout::kTokens; ++t)
              left_sums[t] += left_of_full_list<Layout>(args, token0 + t, kb0 + it, smem + s * args.stage_bytes,
                                                        sw - lane * 16, row_of_lane);
          }
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&empty[s]);
      }
    }
  } else if (XMODE == kXInline) {
    // -------------------------------------------------------------- X warps
    // One warp a stage: digit d of token i is row i * kDigits + d of the X tile, whose
    // 16-byte chunk c lies at c ^ (row % 8) (the 128-byte swizzle).
    RingPlace at;
    at.advance(warp - 6, args.stages);
    for (int it = warp - 6; it < nkb; it += kXWarps, at.advance(kXWarps, args.stages)) {
      const int s = at.s;
      const bool ok = wait_or_abort(&empty[s], at.phase ^ 1u, &abort_flag, args.status);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      uint8_t* xt = smem + s * args.stage_bytes + kWBytes;
      uint8_t* sx = xt + x_bytes + kScaleBlock;
      uint32_t listed = 0;
#pragma unroll
      for (int token = 0; token < kInlineTokens; ++token) {
        if (token >= tokens) break;
        const int group = lane >> 2;
        float u[8];
        int e8;
        const bool any = split_digits<Layout::kDigits>(
            x_next[token], args.x.bf16, u, e8, [&](int d, uint8_t code, uint32_t words) {
              const int row = token * Layout::kDigits + d;
              *reinterpret_cast<uint32_t*>(xt + row * kBlockBytes + ((group ^ (row & 7)) << 4) + (lane & 3) * 4) = words;
              if ((lane & 3) == 0)
                sx[(group >> 2) * 512 + (row & 31) * 16 + (row >> 5) * 4 + (group & 3)] = code;
            });
        if (__any_sync(0xFFFFFFFFu, any))
          listed = list_left<Layout::kDigits>(make_float4(u[0], u[1], u[2], u[3]), make_float4(u[4], u[5], u[6], u[7]), x_next[token],
                             args.x.bf16, e8, any, token, stage_lists + s, listed);
      }
      if (lane == 0) stage_lists[s].count = listed;
      fence_proxy_async_smem();  // the MMA reads the tile through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(&digits[s]);
      ask_x(it + kXWarps);  // after the fence, which waits for loads in flight too
    }
  }
  __syncthreads();  // the abort flag is final and the ring is free

  const bool aborted = abort_flag != 0;
  // Row r of the tile belongs to the cluster's rank r / share; the sums of its
  // rows lie in that CTA as [rank of origin][token][r % share].
  const int share_log2 = 31 - __clz(kRowTile / args.split);  // split is a power of two
  const int share = 1 << share_log2;
  const bool early = tokens <= kEarlyTokens;
  float* sums = reinterpret_cast<float*>(smem + (early ? args.stages * args.stage_bytes : 0));
  cluster_wait_started();  // long past by now
  if (!early) cluster_sync_all();
  if (!aborted && warp >= 2 && warp < 6) {
    tc_fence_after();
    const int row = row_of_lane;
    float* left_in_ring = reinterpret_cast<float*>(smem);  // [token][row]
    if constexpr (XMODE != kXRows) {
      // Sixteen local loads side by side instead of one a token, each of them slow (9.3
      // instead of 10.7 us at 16 x 4096 x 4096).
      if (any_left) {
#pragma unroll
        for (int t = 0; t < kStageTokens; ++t) left_in_ring[t * kRowTile + row] = left_sums[t];
      }
    }
    const uint32_t taddr = tbase + ((32u * (warp & 3)) << 16);
    const int owner = row >> share_log2;
    const uint32_t to =
        mapa_shared(smem_addr(sums + rank * tokens * share + (row - owner * share)), owner);
    auto send = [&](int token, float v) {
      st_shared_cluster_f32(to + static_cast<uint32_t>(token * share * 4), v);
    };
    if constexpr (XMODE == kXRows) {
      for (int c = 0; c < tokens; c += 8) {
        float r[8];
        tmem_ld_8cols(taddr + static_cast<uint32_t>(c), r);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < tokens) send(c + i, r[i]);
      }
    } else {
      for (int token = 0; token < tokens; ++token) {
        static_assert(Layout::kDigits == 8 || Layout::kDigits == 9, "columns of a token");
        const uint32_t at = taddr + static_cast<uint32_t>(Layout::column(token));
        float r[9];
        tmem_ld_8cols(at, reinterpret_cast<float(&)[8]>(r));
        if constexpr (Layout::kDigits == 9) tmem_ld_1col(at + 8, r[8]);
        tmem_wait_ld();
        float sum = sum_digits<Layout::kDigits>(r);
        if (any_left) sum += left_in_ring[token * kRowTile + row];
        send(token, sum);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();
  if (!aborted) {
    const long long n0 = static_cast<long long>(tile) * kRowTile + rank * share;
    const int rows = static_cast<int>(min(static_cast<long long>(min(share, kRowTile - rank * share)),
                                          args.n - n0));
    constexpr int kThreads = rows_threads(XMODE);
    auto run = [&](auto* y) {
      using T = std::remove_pointer_t<decltype(y)>;
      const T* bias = static_cast<const T*>(args.bias);
      finish<T, kThreads>(sums, args.split, tokens, share_log2, rows, bias == nullptr ? bias : bias + n0,
                          y + token0 * args.ldy + n0, args.ldy);
    };
    if (args.y_type == kRowsFp32)
      run(static_cast<float*>(args.y));
    else if (args.y_type == kRowsBf16)
      run(static_cast<__nv_bfloat16*>(args.y));
    else
      run(static_cast<__half*>(args.y));
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, kCtaTmemCols);
  }
}

// Codes [rows][pitch bytes] as boxes of box_rows x 128 bytes in the 128-byte swizzle.
int rows_map(CUtensorMap* map, const void* base, long long rows, long long pitch, int box_rows) {
  auto fn = tensor_map_encoder();
  if (fn == nullptr) return TCB_ERR_DEVICE;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(pitch), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kBlockBytes), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TCB_OK
             : TCB_ERR_INVALID_ARGUMENT;
}

// The digits of m rows of k values as an MX tensor, and what they leave:
// [scales][lists][codes].
struct DigitSpace {
  long long rows, lists, lists_at, codes_at, bytes;
  template <typename Layout>
  DigitSpace(Layout, long long m, long long k) : rows(Layout::rows(m)), lists(Layout::lists(m)) {
    const long long kblocks = (mx_padded(k) + kBlockK - 1) / kBlockK;
    const long long tiles = (lists + Layout::kPerTile - 1) / Layout::kPerTile;
    lists_at = (rows + 255) / 256 * 2 * kScaleBlock * kblocks;
    const long long list_bytes = tiles * Layout::kPerTile * kblocks * static_cast<long long>(sizeof(LeftList));
    codes_at = lists_at + (list_bytes + 255) / 256 * 256;
    bytes = codes_at + rows * (mx_padded(k) / 2);
  }
};

template <typename Layout>
int launch_digits(const RowsArgs& args, const DigitSpace& space, uint8_t* base, cudaStream_t stream) {
  const long long blocks = space.lists * args.kblocks;
  if (blocks > INT_MAX || space.rows > INT_MAX / 2) return TCB_ERR_RESOURCE;
  return launch_overlapping(mx_digits_kernel<Layout>, dim3(static_cast<unsigned>(blocks)), 32 * Layout::kTokens, 0, 1,
                            stream, args.x, args.pitch, args.kblocks, base + space.codes_at, base,
                            reinterpret_cast<LeftList*>(base + space.lists_at));
}

template <int XMODE, typename Layout = Bf16Tile>
int launch_rows(const CUtensorMap& map_w, const CUtensorMap& map_x, RowsArgs args, const DeviceFacts& facts,
                cudaStream_t stream) {
  args.col_tiles = (args.cols + kRowTile - 1) / kRowTile;
  if (args.cols > kRowTile) args.cols = kRowTile;
  const long long tiles = (static_cast<long long>(args.n) + kRowTile - 1) / kRowTile * args.col_tiles;
  args.stage_bytes = kWBytes + args.cols * kBlockBytes + 2 * kScaleBlock;
  // A power of two of CTAs to a row tile, each with at least one K block, such
  // that all run at once, two on an SM: a cluster left over for a second round costs
  // more than the split saves.  Clusters of four and eight leave places of a GPC
  // over: of the 296 places of 148 SMs they fill 284 and 264 at most (16 MX rows, K
  // = 4096: 71 tiles as clusters of four 6.6 us, 72 tiles 10.6, 72 as pairs 7.4; 33
  // tiles as clusters of eight 5.6, 34 tiles 8.3, 34 as fours 5.4).  Clusters of
  // eight stop a little earlier, where their join costs more than they save (30
  // tiles: 5.0 with eight, 5.3 with four; 32 tiles: 5.6 and 5.3), and more CTAs of
  // them than SMs want two K blocks each (K = 2048, 30 tiles: 4.4 and 4.0).
  const long long places = 2ll * facts.sm_count;
  const long long most_in_eights = args.kblocks >= 2 * kMaxSplit ? places - 56 : places / 2;
  args.split = 1;
  if (args.kblocks >= 2 && tiles * 2 <= places) args.split = 2;
  if (args.kblocks >= 4 && tiles * 4 <= places - 16) args.split = 4;
  if (args.kblocks >= kMaxSplit && tiles * kMaxSplit <= most_in_eights) args.split = kMaxSplit;
  if (tiles * args.split > INT_MAX) return TCB_ERR_RESOURCE;
  constexpr int kLists = XMODE == kXRows ? 0 : XMODE == kXInline ? 1 : Layout::kPerTile;
  constexpr int list_bytes = kLists * static_cast<int>(sizeof(LeftList));
  args.stages = (kSmemBudget - 1024 - kSumBytes) / (args.stage_bytes + list_bytes);
  if (args.stages > kMaxStages) args.stages = kMaxStages;
  const int acc_cols = (args.cols + 31) / 32 * 32;
  while (acc_cols + args.stages * kSfStageCols > kCtaTmemCols) --args.stages;
  // The ring's places: X warps step kXWarps of them at a time.
  if (args.stages < (XMODE == kXInline ? kXWarps : 2)) return TCB_ERR_RESOURCE;
  const int smem = args.stages * (args.stage_bytes + list_bytes) + kSumBytes + 1024;
  // N of the instruction; M = 128, E2M1 x E2M1, E8M0 scales as the pair MMA.
  args.idesc = (gemm_pair_idesc() & ~(0x3Fu << 17 | 0x1Fu << 24)) |
               static_cast<uint32_t>(args.cols >> 3) << 17 | static_cast<uint32_t>(kRowTile >> 4) << 24;
  auto fn = mx_rows_kernel<XMODE, Layout>;
  static DeviceIntCache cap_cache;
  const int cap = cap_cache.get(facts.device, [&] {
    return raise_dynamic_smem(reinterpret_cast<const void*>(fn), facts.max_smem_optin);
  });
  if (cap < smem) return TCB_ERR_RESOURCE;
  return launch_overlapping(fn, dim3(static_cast<unsigned>(tiles * args.split)),
                            rows_threads(XMODE), static_cast<size_t>(smem), args.split, stream, map_w, map_x,
                            args);
}

// 16-bit rows.
template <typename Layout>
int run_16bit(const RowsProblem& p, RowsArgs args, const CUtensorMap& map_w, void* workspace, int* status,
              const DeviceFacts& facts, cudaStream_t stream) {
  CUtensorMap map_x{};
  if (p.m <= kInlineTokens) {
    args.cols = Layout::columns(p.m);
    return launch_rows<kXInline, Layout>(map_w, map_x, args, facts, stream);
  }
  uint8_t* base = static_cast<uint8_t*>(workspace);
  int rc;
  // Column tiles while all of them run at once (two to an SM), unless there are more than
  // SMs, three or more to a row tile (fewer stream the weight better) and the pairs' tiles
  // are one round.  Measured (us, column tiles / pairs; tiles of either): 33 x 8192 x 4096
  // bf16 (192, 64) 16.8/15.6, 96 x 4096 x 8192 bf16 (192, 64) 27.9/24.0, 64 x 4096 x 4096 fp16
  // (160, 48) 16.5/17.2, 28 x 16384 x 4096 fp16 (256, 64; two to a row tile) 17.9/19.9, 128 x
  // 4096 x 4096 bf16 (256, 80) 22.0/22.8, 48 x 12288 x 4096 bf16 (288, 96) 21.7/23.6, 64 x
  // 12288 x 4096 bf16 (384, 144) 29.4/24.2, 64 x 16384 x 4096 bf16 (512, 192) 33.2/30.9.
  const long long row_tiles = (static_cast<long long>(p.n) + kRowTile - 1) / kRowTile;
  const long long col_tiles = (static_cast<long long>(p.m) + Layout::kTileTokens - 1) / Layout::kTileTokens;
  const long long pair_tiles = (row_tiles + 1) / 2 * ((SliceDigits::rows(p.m) + 255) / 256);
  const bool one_round = col_tiles > 2 && pair_tiles <= facts.sm_count / 2;
  if (col_tiles > 1 && col_tiles * row_tiles > (one_round ? 1 : 2) * static_cast<long long>(facts.sm_count)) {
    // Columns of the CTA-pair GEMM, whose M side is the weight.
    const DigitSpace space(SliceDigits{}, p.m, p.k);
    if ((rc = launch_digits<SliceDigits>(args, space, base, stream)) != TCB_OK) return rc;
    PairProblem q = {};
    q.a = p.w;
    q.b = base + space.codes_at;
    q.sa = p.sw;
    q.sb = base;
    q.bias = p.bias;
    q.c = p.y;
    q.ldc = p.ldy;
    q.m = p.n;
    q.n = static_cast<int>(space.rows);
    q.k = static_cast<int>(mx_padded(p.k));
    q.out = p.y_type == kRowsFp32 ? kPairFp32 : p.y_type == kRowsBf16 ? kPairBf16 : kPairFp16;
    q.idesc = gemm_pair_idesc();
    q.overlap = true;
    q.digits_of = &args.x;
    q.digits_left = reinterpret_cast<const LeftList*>(base + space.lists_at);
    return gemm_pair_run(q, 0, status, facts, stream);
  }
  const DigitSpace space(Layout{}, p.m, p.k);
  if ((rc = launch_digits<Layout>(args, space, base, stream)) != TCB_OK) return rc;
  args.cols = Layout::columns(p.m);
  args.sx = base;
  args.lists = reinterpret_cast<const LeftList*>(base + space.lists_at);
  rc = rows_map(&map_x, base + space.codes_at, args.cols, args.pitch, args.cols < kRowTile ? args.cols : kRowTile);
  if (rc != TCB_OK) return rc;
  return launch_rows<kXDigits, Layout>(map_w, map_x, args, facts, stream);
}

}  // namespace

// X's type decides the digits, N whether they are column tiles of the few-row kernel or
// columns of the CTA-pair GEMM: room for any.
long long mx_rows_workspace(long long m, long long k) {
  if (m <= kInlineTokens) return 0;
  const long long bf16 = DigitSpace(Bf16Tile{}, m, k).bytes, fp16 = DigitSpace(Fp16Tile{}, m, k).bytes;
  const long long slice = DigitSpace(SliceDigits{}, m, k).bytes;
  const long long most = bf16 > fp16 ? bf16 : fp16;
  return most > slice ? most : slice;
}

int mx_rows_run(const RowsProblem& p, void* workspace, int* status, const DeviceFacts& facts,
                cudaStream_t stream) {
  RowsArgs args = {};
  args.sw = static_cast<const uint8_t*>(p.sw);
  args.sx = static_cast<const uint8_t*>(p.sx);
  args.x = {static_cast<const uint16_t*>(p.x), p.ldx, p.m, p.k, p.x_type == kRowsBf16,
            aligned(p.x, 16) && (p.ldx % 8 == 0 || p.m == 1)};
  args.bias = p.bias;
  args.y = p.y;
  args.pitch = mx_padded(p.k) / 2;
  args.ldy = p.ldy;
  args.status = status;
  args.m = p.m;
  args.n = p.n;
  args.kblocks = static_cast<int>((args.pitch + kBlockBytes - 1) / kBlockBytes);
  args.y_type = p.y_type;
  CUtensorMap map_w, map_x{};
  int rc = rows_map(&map_w, p.w, p.n, args.pitch, kRowTile);
  if (rc != TCB_OK) return rc;
  if (p.x_type == kRowsMx) {
    args.cols = (p.m + 7) / 8 * 8;
    if ((rc = rows_map(&map_x, p.x, p.m, args.pitch, args.cols < kRowTile ? args.cols : kRowTile)) != TCB_OK) return rc;
    return launch_rows<kXRows>(map_w, map_x, args, facts, stream);
  }
  return args.x.bf16 ? run_16bit<Bf16Tile>(p, args, map_w, workspace, status, facts, stream)
                     : run_16bit<Fp16Tile>(p, args, map_w, workspace, status, facts, stream);
}

}  // namespace tcb
