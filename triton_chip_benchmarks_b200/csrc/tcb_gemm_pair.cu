// MX FP4 GEMM on CTA pairs (tcgen05 cta_group::2, sm_100a): C = A . B^T.
//
// Two CTAs of a cluster (one per SM of a TPC) compute one 256 x 256 output
// tile together.  Each CTA loads only its half of the operands -- 128 rows of
// A and 128 rows of B -- and the pair MMA (tcgen05.mma.cta_group::2, M = 256,
// N = 256, issued by the leader CTA) reads both CTAs' shared memory.
//
// Feeding the tensor cores.  At the MX FP4 rate one SM consumes 32 KB of
// operands per 512 cycles.  Measured on B200 (a loads-only TMA probe, one CTA
// per SM), what a CTA can pull from L2 depends on how the bytes are asked
// for, not on how many are in flight: stages of 32 KB made of 16 KB boxes
// reach 45-52 B/clk per SM however deep the ring, 64 KB stages of four boxes
// 66-81, and 64 KB stages of two 3-D boxes (two 128-byte K panels per box)
// 85.  So an operand stage here holds two K blocks (256 bytes of K): A and B
// arrive as one 3-D box each (128 rows x 2 panels, 32 KB), in a ring of
// three.  A stage whose K blocks run past the last whole panel (a ragged K)
// loads 2-D boxes instead, whose out-of-bounds columns TMA fills with zeros.
//
// Scales run ahead.  The E8M0 scales of a stage (6 KB: own 128 A rows and all
// 256 B rows, two K blocks) have their own ring of four slots, in shared
// memory and in tensor memory, filled by a loader warp of their own as soon
// as a slot frees.  Moving a stage's scales into tensor memory (tcgen05.st)
// takes about 460 cycles after they land; issued with the operands by the
// operand producer, the MMA waited on them 9-10 % of its time, and a single
// thread issuing five TMA operations per stage (about 100 cycles each) could
// not keep three operand stages in flight.  (Measured on 8192^3: 3.9 to 5.8
// PFLOP/s across these steps; the breakdown is in the design notes.)  Copying
// the scales with tcgen05.cp from the MMA thread instead (six per K block,
// ordered with the MMAs, as the single-CTA kernel does) removes the writer
// warps and their wait, but each copy takes tensor-pipe time: 5.3 against
// 5.9 PFLOP/s here.
//
// The accumulator (128 rows x 256 fp32 columns per CTA) is drained by 16
// epilogue warps that each load their whole 32 x 64 slice into registers and
// release it at once, so the next tile's MMAs start while C is written.  C
// leaves through shared memory and TMA tensor stores: two 4 KB staging
// buffers, each taken in a fixed turn order by the 8 warps of one group; on a
// pair's last tile, when the operand ring is idle, each warp stages its slice
// in the ring and stores it without turns.
// Direct stores of these rows (32 rows x 16 bytes per instruction, or shuffle-
// transposed to whole lines) slowed the scale writers and the MMA issue; TMA
// stores did not.
//
// Tensor memory per CTA: accumulator columns 0-255, then four scale slots of
// 48 columns (per K block: own A rows in 4 columns and all B rows in 8 per
// pair of K steps).
//
// Roles (736 threads per CTA, both CTAs unless noted):
//   warp 0       operand producer: TMA-loads its A and B halves of each stage
//                (waiting empty, completing on the LEADER's loaded, which
//                expects the bytes of both CTAs);
//   warp 1       (leader only) MMA issuer: waits acc_empty, loaded and full,
//                issues four pair MMAs per K block, commits empty and tfree
//                to both CTAs, and acc_full to both CTAs after each tile;
//   warps 2-17   epilogue (see above), arriving on the leader's acc_empty;
//   warps 18-21  scale writers: wait sloaded and tfree, move this CTA's
//                staged scales into their tensor-memory slot (warp w writes
//                lane quarter w % 4), arrive on this CTA's sfree and the
//                leader's full;
//   warp 22      scale loader: bulk-copies each stage's scales into its slot
//                (waiting sfree, completing on this CTA's sloaded).
// Every wait is bounded; a wait that fails raises the abort flag of both
// CTAs, so the pair leaves its loops together.  A cluster barrier follows
// barrier set-up and precedes teardown, so neither CTA exits while its peer
// may still signal its barriers or read its shared memory.
//
// C's type (tcb_mx_gemm).  The epilogue rounds a 64-column slice once to 16 bits
// (one staging chunk instead of two) and adds the bias in fp32 before that; a
// lane asks for two bias values ahead of the accumulator and the columns get
// theirs by shuffle (64 broadcast loads after it: 12.9 instead of 12.0 us at
// 1000 x 4104 x 2072 fp32).  DIGITS: B's rows are the MX FP4 digits of 16-bit rows
// (tcb_mx_linear with many rows), whose columns the epilogue adds nine by nine; while a
// tile's MMAs run its warps multiply what the digits leave.
// Measured (captured, back to back): 4096^3 to bf16 31 us, 4.4 PFLOP/s; 1024^3 6.6.
//
// Counterpart in the reference suite: none (FP4 GEMM is refused at
// bench_tensor.py:1406-1407); same contract as the single-CTA tcb_gemm path.
#include <cudaTypedefs.h>
#include <type_traits>

#include "tcb_device.cuh"
#include "tcb_gemm_common.cuh"
#include "tcb_gemm_pair.h"
#include "tcb_host.h"
#include "tcb_mx_digits.cuh"
#include "tcb_registry.h"

namespace tcb {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace {

using namespace gemm_detail;

constexpr int kPairRows = 128;                                 // A rows and B rows per CTA
constexpr int kPairPanels = 2;                                 // 128-byte K blocks per stage
constexpr int kPairPanelBytes = kPairRows * kBlockBytes;       // 16 KB
constexpr int kPairStageA = kPairPanels * kPairPanelBytes;     // 32 KB
constexpr int kPairStageBytes = 2 * kPairStageA;               // A and B halves, 64 KB
constexpr int kPairStages = 3;
constexpr int kPairScaleBlock = (kPairRows + kTileN) * 8;      // own A + all B scales, one K block
constexpr int kPairSlotBytes = kPairPanels * kPairScaleBlock;  // 6 KB
constexpr int kPairSlots = 4;
constexpr int kPairEpiWarps = 16;
// Back-off of the waits off the critical path (epilogue, scale writers,
// staging turns), in ns, so that 20 warps polling do not take issue slots
// from the producer and MMA warps (measured neutral at 0-256 ns).
constexpr unsigned kPairIdleSleepNs = 64;
constexpr unsigned kPairTurnSleepNs = 128;
constexpr int kPairEpiCols = kTileN / (kPairEpiWarps / 4);     // 64 columns per epilogue warp
constexpr int kPairEpiGroups = 2;
constexpr int kPairEpiGroupWarps = kPairEpiWarps / kPairEpiGroups;
constexpr int kPairScaleWarps = 4;
constexpr int kPairLoaderWarp = 2 + kPairEpiWarps + kPairScaleWarps;  // scale loader
constexpr int kPairThreads = (kPairLoaderWarp + 1) * 32;
constexpr int kPairSlotOffset = kPairStages * kPairStageBytes;
constexpr int kPairStagingOffset = kPairSlotOffset + kPairSlots * kPairSlotBytes;
constexpr int kPairSmem = kPairStagingOffset + kPairEpiGroups * kEpiChunkBytes + 1024;
constexpr int kPairSfCols = kPairPanels * kSfStageCols;        // tensor-memory columns per slot
static_assert(kAccCols + kPairSlots * kPairSfCols <= kTmemCols, "tensor memory overflow");
static_assert(kPairSmem <= 227 * 1024 - 256, "shared memory overflow");
static_assert(kPairSlotOffset % 1024 == 0 && kPairStagingOffset % 1024 == 0,
              "operand stages and staging buffers keep the 1024-byte swizzle alignment");
constexpr int kPlainBytes = kPairEpiGroups * kEpiChunkBytes / kPairEpiWarps;  // staging of a warp
static_assert(kPlainBytes == 512, "plain stores turn four rows of 128 bytes round");
static_assert(kPairEpiCols == 64, "an epilogue warp drains two 32-column loads");
static_assert(mx_detail::SliceDigits::kRows == kPairEpiCols, "a slice is a list's tokens");
static_assert(kPairEpiWarps * 2 * kEpiChunkBytes <= kPairStages * kPairStageBytes,
              "the last tile's C slices fit in the operand ring");

struct PairArgs {
  const uint8_t* sa;  // packed E8M0 scales of A (tcb_mx_scales_pack layout)
  const uint8_t* sb;  // packed E8M0 scales of B
  void* c;            // [M][N], row pitch ldc elements
  const void* bias;   // [N] of C's type (BIAS kernels)
  long long ldc;
  int* status;
  int m, n;
  int tiles_m, tiles_n;
  int kblocks;      // 128-byte K blocks (the last may be ragged)
  int full_panels;  // whole 128-byte K blocks reachable through the 3-D maps (0: none)
  uint32_t idesc;
  mx_detail::ValueRows x;            // DIGITS kernels: the 16-bit rows,
  const mx_detail::LeftList* lists;  // what their digits leave,
  const uint8_t* a;                  // A's codes and their row bytes
  long long pitch;
};

__device__ __forceinline__ void pair_mma_mxf4(uint32_t d, uint64_t adesc, uint64_t bdesc,
                                              uint32_t idesc, uint32_t accumulate, uint32_t tsfa,
                                              uint32_t tsfb) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], "
      "p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tsfa), "r"(tsfb));
}

// Walks this pair's stages in order (its tiles t = pair, pair + pairs, ...,
// each in stage_blocks stages of two K blocks).  Advancing is an increment;
// the tile's coordinates are recomputed once per tile.  (A single thread
// recomputing them from a stage index with runtime divisions every stage
// kept the producer too busy to issue loads on time: 44 % of the MMA
// thread's time went to waiting for operands.)
struct PairCursor {
  int t, sb, tm, tn, kb0, nkb;

  __device__ __forceinline__ void start(int first, const PairArgs& a) {
    t = first;
    sb = 0;
    tile_coords(t, a.tiles_m, a.tiles_n, &tm, &tn);
    kb0 = 0;
    nkb = min(kPairPanels, a.kblocks);
  }

  __device__ __forceinline__ void next(int pairs, int stage_blocks, int tiles, const PairArgs& a) {
    if (++sb == stage_blocks) {
      sb = 0;
      t += pairs;
      if (t < tiles) tile_coords(t, a.tiles_m, a.tiles_n, &tm, &tn);
    }
    kb0 = sb * kPairPanels;
    nkb = min(kPairPanels, a.kblocks - kb0);
  }
};

// The type of C: the accumulator itself, or one rounding to 16 bits (after the
// bias, which is added in fp32).
template <int OUT>
struct PairOut;
template <>
struct PairOut<kPairFp32> { using type = float; };
template <>
struct PairOut<kPairBf16> { using type = __nv_bfloat16; };
template <>
struct PairOut<kPairFp16> { using type = __half; };

// acc += bias over this warp's 64 columns; lane l holds the bias of columns l and
// 32 + l (asked for before the accumulator was ready).
__device__ __forceinline__ void add_bias(uint32_t (&r)[2][32], float lo, float hi) {
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    r[0][e] = __float_as_uint(__uint_as_float(r[0][e]) + __shfl_sync(0xffffffffu, lo, e));
    r[1][e] = __float_as_uint(__uint_as_float(r[1][e]) + __shfl_sync(0xffffffffu, hi, e));
  }
}

// 64 fp32 columns as 32 words of two 16-bit values.
template <typename T>
__device__ __forceinline__ void to_pairs(const uint32_t (&r)[2][32], uint32_t (&h)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    h[i] = mx_detail::pack2<T>(__uint_as_float(r[i >> 4][2 * (i & 15)]),
                               __uint_as_float(r[i >> 4][2 * (i & 15) + 1]));
}

// 32 words of a row a lane (32 fp32 or 64 16-bit columns) to rows of C that TMA
// cannot write.  STEP rows at a time go through shared memory of the warp's own
// (128 bytes a row), so that a row leaves as 128 bytes side by side: lane l the word
// l.  Where a 16-bit row starts between two words, lane l stores the aligned word
// of columns 2l - 1 and 2l.  `rows` and `cols`: how many there are from the first
// to C's edge (any number, negative too).  Predicated stores: branches around a
// row's stores cost about 100 cycles a row.  (4096 x 4095 x 4096 bf16: 180 us with
// every lane storing its own row, 88 through the two staging buffers in turns, 40
// so; 31 through the tensor map at N = 4096.)
template <int STEP, typename T>
__device__ __forceinline__ void store_plain(const uint32_t (&h)[32], uint8_t* buf, T* c, long long ldc,
                                            int rows, int cols, int lane) {
  constexpr int kRows = 4;  // shared loads in flight
  constexpr int kCols = 128 / static_cast<int>(sizeof(T));
  // Chunk i of row j at i ^ swizzle(j): neither side has bank conflicts.
  auto swizzle = [](int j) { return STEP == 4 ? (j & 3) << 1 : j & 7; };
#pragma unroll 1
  for (int r = 0; r < 32; r += kRows, c += kRows * ldc, rows -= kRows) {
    if (r % STEP == 0) {
      __syncwarp();  // the rows before these have been read
      if (lane / STEP == r / STEP) {
        uint8_t* mine = buf + lane % STEP * 128;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4*>(mine + ((i ^ swizzle(lane)) << 4)) =
              make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
      }
      __syncwarp();
    }
    uint32_t v[kRows], before[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int at = (r + j) % STEP;
      v[j] = *reinterpret_cast<const uint32_t*>(buf + at * 128 + (((lane >> 2) ^ swizzle(at)) << 4) +
                                                (lane & 3) * 4);
      if constexpr (sizeof(T) == 2) before[j] = __shfl_up_sync(0xffffffffu, v[j], 1);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (j < rows && lane < cols) *reinterpret_cast<uint32_t*>(c + j * ldc + lane) = v[j];
    } else {
      const bool whole = cols >= kCols;
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        uint16_t* row = reinterpret_cast<uint16_t*>(c + j * ldc);
        const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 1;
        const uint32_t w = odd ? __byte_perm(before[j], v[j], 0x5432) : v[j];
        const bool in = j < rows && whole;
        if (in && lane >= odd) *reinterpret_cast<uint32_t*>(row + 2 * lane - odd) = w;
        // The two halves that no whole word holds: column 0 and the last.
        const uint16_t half = static_cast<uint16_t>(lane == 0 ? v[j] : v[j] >> 16);
        if (in && odd && (lane == 0 || lane == 31)) row[lane == 0 ? 0 : kCols - 1] = half;
      }
      if (!whole) {  // C's right edge
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          uint16_t* row = reinterpret_cast<uint16_t*>(c + j * ldc) + 2 * lane;
          if (j < rows && 2 * lane < cols) row[0] = static_cast<uint16_t>(v[j]);
          if (j < rows && 2 * lane + 1 < cols) row[1] = static_cast<uint16_t>(v[j] >> 16);
        }
      }
    }
  }
}

// DIGITS: a slice of 64 columns is the digits of seven tokens.  A lane (a row n of A)
// adds each token's columns, and what the digits leave (null: nothing), and stores
// C[token][n]: 32 neighbours a store.
template <typename T>
__device__ __forceinline__ void store_digits(const PairArgs& args, const uint32_t (&r)[2][32], int n, int token0,
                                             const float* left) {
  using mx_detail::SliceDigits;
  if (n >= args.m) return;
  const T* bias = static_cast<const T*>(args.bias);
  const float b = bias == nullptr ? 0.0f : mx_detail::to_float(bias[n]);
#pragma unroll
  for (int i = 0; i < SliceDigits::kTokens; ++i) {
    float v[SliceDigits::kDigits];
#pragma unroll
    for (int d = 0; d < SliceDigits::kDigits; ++d) {
      const int column = i * SliceDigits::kDigits + d;
      v[d] = __uint_as_float(r[column >> 5][column & 31]);
    }
    float sum = mx_detail::sum_digits<SliceDigits::kDigits>(v);
    const int token = token0 + i;
    if (token >= args.x.m) break;
    if (left != nullptr) sum += left[i];
    static_cast<T*>(args.c)[token * args.ldc + n] = mx_detail::from_float<T>(sum + b);
  }
}

// How C leaves: through the C tensor map (rows on 16-byte boundaries), by plain
// stores through the same shared memory, or as a digit product.  A kernel each:
// the epilogue has 64 of 80 registers in the accumulator slice, and what else it holds
// spills (bytes a thread stored: through the map 12 to 16, 68 with a 16-bit bias; plain
// stores 20 to 148; digits 48).  Measured, it does not show: fp32 through the map takes
// 41.9 us at 4096^3 (42.6 with the 8 bytes of a kernel of its own).
enum StoreMode : int { kStoreTma = 0, kStorePlain = 1, kStoreDigits = 2 };

template <int OUT, bool BIAS, int STORE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    gemm_pair_mxf4_kernel(const __grid_constant__ CUtensorMap map_a,
                          const __grid_constant__ CUtensorMap map_b,
                          const __grid_constant__ CUtensorMap map_a3,
                          const __grid_constant__ CUtensorMap map_b3,
                          const __grid_constant__ CUtensorMap map_c,
                          const __grid_constant__ PairArgs args) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t loaded[kPairStages];   // leader: both operand halves landed
  __shared__ __align__(8) uint64_t empty[kPairStages];    // pair MMAs done with the stage
  __shared__ __align__(8) uint64_t sloaded[kPairSlots];   // this CTA's scales landed
  __shared__ __align__(8) uint64_t sfree[kPairSlots];     // this CTA's writers done with the slot
  __shared__ __align__(8) uint64_t full[kPairSlots];      // leader: both CTAs' scales written
  __shared__ __align__(8) uint64_t tfree[kPairSlots];     // pair MMAs done with the tensor-memory slot
  __shared__ __align__(8) uint64_t acc_full;
  __shared__ __align__(8) uint64_t acc_empty;             // leader: both epilogues drained
  __shared__ __align__(8) uint64_t drained;               // leader: every issued MMA finished
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ volatile int store_turn[kPairEpiGroups];     // next staging turn of each group

  // An offset from smem_raw, so that the compiler still knows it for shared memory.
  uint8_t* smem = smem_raw + (-smem_addr(smem_raw) & 1023u);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int pairs = static_cast<int>(gridDim.x >> 1);
  const int tiles = args.tiles_m * args.tiles_n;
  const int stage_blocks = (args.kblocks + kPairPanels - 1) / kPairPanels;
  const int my_tiles = pair < tiles ? (tiles - pair + pairs - 1) / pairs : 0;
  const int my_stages = my_tiles * stage_blocks;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
    if (args.full_panels > 0) {
      prefetch_tensormap(&map_a3);
      prefetch_tensormap(&map_b3);
    }
    if (STORE == kStoreTma) prefetch_tensormap(&map_c);
    for (int g = 0; g < kPairEpiGroups; ++g) store_turn[g] = 0;
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&loaded[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kPairSlots; ++s) {
      mbar_init(&sloaded[s], 1);
      mbar_init(&sfree[s], kPairScaleWarps);
      mbar_init(&full[s], 2 * kPairScaleWarps);
      mbar_init(&tfree[s], 1);
    }
    mbar_init(&acc_full, 1);
    mbar_init(&acc_empty, 2 * kPairEpiWarps);
    mbar_init(&drained, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc_pair(&tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers initialised and tensor memory allocated
  tc_fence_after();
  let_next_kernel_start();
  wait_for_previous_kernels();
  const uint32_t tbase = tmem_slot;
  // An abort on either CTA stops both: a wait that fails also raises the
  // peer's flag (a store into its shared memory, which stays valid until the
  // teardown cluster barrier), so neither CTA sits out a full timeout on
  // barriers the other no longer signals.
  const uint32_t peer_abort = mapa_shared(smem_addr(const_cast<int*>(&abort_flag)), rank ^ 1u);
  auto pair_wait = [&](uint64_t* bar, uint32_t parity, unsigned sleep_ns = 0) {
    if (wait_or_abort(bar, parity, &abort_flag, args.status, sleep_ns)) return true;
    st_shared_cluster_u32(peer_abort, 1u);
    return false;
  };
  if (threadIdx.x == 0 && rank != 0) {
    // The pair MMA addresses both CTAs' tensor memory with the leader's column base.
    if (ld_shared_cluster_u32(mapa_shared(smem_addr(&tmem_slot), 0)) != tbase) {
      abort_flag = 1;
      st_shared_cluster_u32(peer_abort, 1u);
      report_status(args.status, TCB_ERR_DEVICE);
    }
  }
  __syncthreads();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      PairCursor op;
      op.start(pair, args);
      for (int it = 0; it < my_stages && !abort_flag; ++it) {
        const int s = it % kPairStages;
        const uint32_t phase = static_cast<uint32_t>(it / kPairStages) & 1u;
        if (!pair_wait(&empty[s], phase ^ 1u)) break;
        const int arow = op.tm * 2 * kPairRows + static_cast<int>(rank) * kPairRows;
        const int brow = op.tn * kTileN + static_cast<int>(rank) * kPairRows;
        uint8_t* stage = smem + s * kPairStageBytes;
        // Both CTAs' operand bytes complete on the leader's barrier.
        const uint32_t lead_loaded = mapa_shared(smem_addr(&loaded[s]), 0);
        if (rank == 0) mbar_arrive_expect_tx(&loaded[s], 2 * 2 * op.nkb * kPairPanelBytes);
        if (op.nkb == kPairPanels && op.kb0 + kPairPanels <= args.full_panels) {
          tma_load_3d_pair(stage, &map_a3, 0, arow, op.kb0, lead_loaded);
          tma_load_3d_pair(stage + kPairStageA, &map_b3, 0, brow, op.kb0, lead_loaded);
        } else {
          for (int q = 0; q < op.nkb; ++q) {
            const int x = (op.kb0 + q) * kBlockBytes;
            tma_load_2d_pair(stage + q * kPairPanelBytes, &map_a, x, arow, lead_loaded);
            tma_load_2d_pair(stage + kPairStageA + q * kPairPanelBytes, &map_b, x, brow,
                             lead_loaded);
          }
        }
        op.next(pairs, stage_blocks, tiles, args);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    if (lane == 0 && rank == 0) {
      const uint64_t desc_const = smem_desc(0, 16, 8 * kBlockBytes, 2u);
      const uint32_t smem0 = smem_addr(smem) >> 4;
      int it = 0;
      for (int ti = 0; ti < my_tiles && !abort_flag; ++ti) {
        if (!pair_wait(&acc_empty, (static_cast<uint32_t>(ti) & 1u) ^ 1u)) break;
        tc_fence_after();
        for (int sb = 0; sb < stage_blocks; ++sb, ++it) {
          const int s = it % kPairStages;
          const int slot = it % kPairSlots;
          if (!pair_wait(&loaded[s], static_cast<uint32_t>(it / kPairStages) & 1u)) break;
          if (!pair_wait(&full[slot], static_cast<uint32_t>(it / kPairSlots) & 1u)) break;
          tc_fence_after();
          const int nkb = min(kPairPanels, args.kblocks - sb * kPairPanels);
          const uint32_t a_lo = smem0 + static_cast<uint32_t>(s * kPairStageBytes >> 4);
          const uint32_t b_lo = a_lo + (kPairStageA >> 4);
          const uint32_t sf = tbase + kAccCols + static_cast<uint32_t>(slot * kPairSfCols);
#pragma unroll
          for (int q = 0; q < kPairPanels; ++q) {
            if (q >= nkb) break;
            const uint32_t panel = static_cast<uint32_t>(q * (kPairPanelBytes >> 4));
            const uint32_t sfq = sf + static_cast<uint32_t>(q * kSfStageCols);
#pragma unroll
            for (int k = 0; k < kStepsPerBlock; ++k) {
              pair_mma_mxf4(tbase, desc_const | (a_lo + panel + static_cast<uint32_t>(k * 2)),
                            desc_const | (b_lo + panel + static_cast<uint32_t>(k * 2)),
                            sf_idesc(args.idesc, k), (sb | q | k) != 0, sf_cols_a(sfq, k),
                            sf_cols_b(sfq, k));
            }
          }
          tc_commit_pair(&empty[s], 0x3);
          tc_commit_pair(&tfree[slot], 0x3);
        }
        if (abort_flag) break;
        tc_commit_pair(&acc_full, 0x3);
      }
      // Nothing this thread issued may still run when the pair tears down.
      tc_commit_pair(&drained, 0x1);
      if (!mbar_wait(&drained, 0)) report_status(args.status, TCB_ERR_TIMEOUT);
    }
    __syncwarp();
  } else if (warp < 2 + kPairEpiWarps) {
    // ------------------------------------------------------------ epilogue
    // Tensor-memory lanes 32(warp % 4).. are this warp's rows; its columns are
    // one 64-wide slice.  The whole slice comes into registers before the
    // accumulator is released.  C then goes out through the group's staging
    // buffer in a fixed turn order (turn = tile x 8 + slot): stage 32 columns,
    // TMA-store them, wait until the store has read the buffer, repeat, and
    // hand the buffer on.
    const int quarter = warp & 3;
    const int col0 = ((warp - 2) >> 2) * kPairEpiCols;
    const int group = (warp - 2) / kPairEpiGroupWarps;
    const int slot = (warp - 2) % kPairEpiGroupWarps;
    uint8_t* staging = smem + kPairStagingOffset + group * kEpiChunkBytes;
    const uint32_t lead_acc_empty = mapa_shared(smem_addr(&acc_empty), 0);
    const uint32_t taddr = tbase + ((32u * quarter) << 16) + static_cast<uint32_t>(col0);
    // Bounded wait for this warp's staging turn.
    auto turn_wait = [&](int mine) {
      if (store_turn[group] == mine) return true;
      const unsigned long long start = globaltimer_ns();
      while (store_turn[group] != mine) {
        __nanosleep(kPairTurnSleepNs);
        if (abort_flag) return false;
        if (globaltimer_ns() - start > kWaitTimeoutNs) {
          abort_flag = 1;
          st_shared_cluster_u32(peer_abort, 1u);
          report_status(args.status, TCB_ERR_TIMEOUT);
          return false;
        }
      }
      return true;
    };
    using Out = typename PairOut<OUT>::type;
    for (int ti = 0; ti < my_tiles; ++ti) {
      int row0, c;
      auto place = [&] {
        int tm, tn;
        tile_coords(pair + ti * pairs, args.tiles_m, args.tiles_n, &tm, &tn);
        row0 = tm * 2 * kPairRows + static_cast<int>(rank) * kPairRows + 32 * quarter;
        c = tn * kTileN + col0;
      };
      [[maybe_unused]] float bias_lo = 0.0f, bias_hi = 0.0f;
      if constexpr (BIAS) {
        place();
        const Out* bias = static_cast<const Out*>(args.bias);
        if (c + lane < args.n) bias_lo = mx_detail::to_float(bias[c + lane]);
        if (c + 32 + lane < args.n) bias_hi = mx_detail::to_float(bias[c + 32 + lane]);
      }
      // What the digits leave, while the tile's MMAs run.
      [[maybe_unused]] float left[mx_detail::SliceDigits::kTokens];
      [[maybe_unused]] bool any_left = false;
      [[maybe_unused]] int token0 = 0;
      if constexpr (STORE == kStoreDigits) {
        place();
        const int list = c / mx_detail::SliceDigits::kRows;
        token0 = list * mx_detail::SliceDigits::kTokens;
        if (token0 < args.x.m && row0 < args.m)
          any_left = mx_detail::left_products<mx_detail::SliceDigits>(
              args.lists + static_cast<long long>(list) * args.kblocks, args.x, token0,
              mx_detail::MxRows{args.a, args.pitch, args.sa, args.kblocks, args.m}, row0 + lane, left);
      }
      // Warp-uniform exits: tcgen05.ld and .st need the whole warp.
      if (!__all_sync(0xffffffffu, pair_wait(&acc_full, static_cast<uint32_t>(ti) & 1u,
                                              kPairIdleSleepNs)))
        break;
      tc_fence_after();
      uint32_t r[2][32];
      acc_load<2>(taddr, r);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(lead_acc_empty);
      if constexpr (!BIAS) place();
      // A 16-bit slice is one 4 KB staging chunk (64 columns), an fp32 slice two.
      constexpr int kChunks = OUT == kPairFp32 ? 2 : 1;
      if constexpr (STORE == kStoreDigits) {
        store_digits<Out>(args, r, row0 + lane, token0, any_left ? left : nullptr);
        __syncwarp();
        continue;
      }
      if constexpr (BIAS) add_bias(r, bias_lo, bias_hi);
      if constexpr (STORE == kStorePlain) {
        Out* dst = static_cast<Out*>(args.c) + static_cast<long long>(row0) * args.ldc + c;
        auto store_slice = [&](auto step, uint8_t* own) {
          constexpr int kStep = decltype(step)::value;
          if constexpr (OUT == kPairFp32) {
            store_plain<kStep>(r[0], own, dst, args.ldc, args.m - row0, args.n - c, lane);
            store_plain<kStep>(r[1], own, dst + 32, args.ldc, args.m - row0, args.n - c - 32, lane);
          } else {
            uint32_t h[32];
            to_pairs<Out>(r, h);
            store_plain<kStep>(h, own, dst, args.ldc, args.m - row0, args.n - c, lane);
          }
        };
        // The operand ring is idle behind the last tile (see below).
        if (ti + 1 == my_tiles)
          store_slice(std::integral_constant<int, 32>{}, smem + (warp - 2) * kEpiChunkBytes);
        else
          store_slice(std::integral_constant<int, 4>{},
                      smem + kPairStagingOffset + (warp - 2) * kPlainBytes);
        __syncwarp();
        continue;
      }
      auto stage_slice = [&](uint8_t* buf, int q) {
        if constexpr (OUT == kPairFp32) {
          stage_chunk(buf, lane, r[q]);
        } else {
          uint32_t h[32];
          to_pairs<Out>(r, h);
          stage_chunk(buf, lane, h);
        }
      };
      if (ti + 1 == my_tiles) {
        // Last tile: every MMA has finished reading the operand ring (acc_full
        // follows their completion) and no load refills it, so each warp
        // stages its whole slice in 8 KB of the ring of its own and stores it
        // at once instead of waiting for staging turns (with one or two tiles
        // per pair the turns were the critical path).
        uint8_t* own = smem + (warp - 2) * 2 * kEpiChunkBytes;
#pragma unroll
        for (int q = 0; q < kChunks; ++q) stage_slice(own + q * kEpiChunkBytes, q);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
#pragma unroll
          for (int q = 0; q < kChunks; ++q)
            tma_store_2d(&map_c, c + 32 * q, row0, own + q * kEpiChunkBytes);
          bulk_commit_group();
        }
        __syncwarp();
      } else {
        const int mine = ti * kPairEpiGroupWarps + slot;
        if (!__all_sync(0xffffffffu, turn_wait(mine))) break;
        __threadfence_block();
#pragma unroll
        for (int q = 0; q < kChunks; ++q) {
          stage_slice(staging, q);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_c, c + 32 * q, row0, staging);
            bulk_commit_group();
            bulk_wait_group_read<0>();
          }
          __syncwarp();
        }
        if (lane == 0) store_turn[group] = mine + 1;
      }
    }
    if (lane == 0) bulk_wait_group_all();  // C stores complete before the CTA retires
  } else if (warp < kPairLoaderWarp) {
    // ------------------------------------------------------ scale writers
    // Lane l writes rows 32j+l of each staged K block's scales into this
    // CTA's tensor-memory slot (two K steps per word).
    const int quarter = warp & 3;
    const uint32_t lane_base = tbase + ((32u * quarter) << 16) + kAccCols;
    int sb = 0;  // stage block of `it` within its tile
    for (int it = 0; it < my_stages; ++it) {
      const int slot = it % kPairSlots;
      // Warp-uniform exit: tcgen05.st needs the whole warp.  The stage's
      // scales have landed, and the MMAs that read the tensor-memory slot's
      // previous contents (kPairSlots stages back) have finished.
      const uint32_t round = static_cast<uint32_t>(it / kPairSlots) & 1u;
      if (!__all_sync(0xffffffffu, pair_wait(&sloaded[slot], round, kPairIdleSleepNs) &&
                                       pair_wait(&tfree[slot], round ^ 1u, kPairIdleSleepNs)))
        break;
      const int nkb = min(kPairPanels, args.kblocks - sb * kPairPanels);
      if (++sb == stage_blocks) sb = 0;
      // Packed layout: lane l's 16 bytes of each 512-byte half are exactly its
      // words for the four A columns (rows l, 32+l, 64+l, 96+l), and those of
      // B rows 0-127 and 128-255 for the eight B columns.
      const uint8_t* ss = smem + kPairSlotOffset + slot * kPairSlotBytes + lane * 16;
#pragma unroll
      for (int q = 0; q < kPairPanels; ++q) {
        if (q >= nkb) break;
        const uint8_t* h = ss + q * 1024;
        write_scale_block(lane_base + static_cast<uint32_t>(slot * kPairSfCols + q * kSfStageCols),
                          h, h + kPairPanels * 1024, h + 2 * kPairPanels * 1024);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sfree[slot]);  // the shared-memory slot may be refilled
        mbar_arrive_cluster(mapa_shared(smem_addr(&full[slot]), 0));
      }
    }
  } else if (lane == 0) {
    // -------------------------------------------------------- scale loader
    // Scales of each stage into slot j % kPairSlots as soon as this CTA's
    // writers have moved the slot's previous stage into tensor memory (not
    // when its MMAs finish, which would leave the loads only about three
    // stages of lead): [A own rows][B rows 0-127][B rows 128-255], nkb KiB
    // each (consecutive K blocks of a row block are contiguous in the packed
    // layout).  Its own warp, so neither the operand producer nor the scale
    // writers wait for these copies to be issued.
    const size_t rb_bytes = static_cast<size_t>(args.kblocks) * 1024;
    PairCursor sc;
    sc.start(pair, args);
    for (int j = 0; j < my_stages && !abort_flag; ++j) {
      const int slot = j % kPairSlots;
      if (!pair_wait(&sfree[slot], (static_cast<uint32_t>(j / kPairSlots) & 1u) ^ 1u)) break;
      uint8_t* ss = smem + kPairSlotOffset + slot * kPairSlotBytes;
      const uint32_t sbytes = static_cast<uint32_t>(sc.nkb) * 1024;
      mbar_arrive_expect_tx(&sloaded[slot], 3 * sbytes);
      bulk_load_1d(ss, args.sa + (2 * sc.tm + rank) * rb_bytes + sc.kb0 * 1024, sbytes,
                   &sloaded[slot]);
      bulk_load_1d(ss + kPairPanels * 1024, args.sb + (2 * sc.tn) * rb_bytes + sc.kb0 * 1024,
                   sbytes, &sloaded[slot]);
      bulk_load_1d(ss + 2 * kPairPanels * 1024, args.sb + (2 * sc.tn + 1) * rb_bytes + sc.kb0 * 1024,
                   sbytes, &sloaded[slot]);
      sc.next(pairs, stage_blocks, tiles, args);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the peer may still touch its shared memory
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc_pair(tbase, kTmemCols);
  }
}

// A [rows][row_bytes] as 128-byte x 128-row boxes (2-D) and, when it has at
// least two whole 128-byte K blocks, as 128-byte x 128-row x 2-block boxes
// over the whole K blocks (3-D: x in the block, y the row, z the block).
// `*full_panels` is set to 0 when no 3-D map is made (then every stage loads
// 2-D boxes).
int pair_maps(CUtensorMap* map2, CUtensorMap* map3, const void* base, long long rows,
              long long row_bytes, int* full_panels) {
  auto fn = tensor_map_encoder();
  if (fn == nullptr) return TCB_ERR_DEVICE;
  void* p = const_cast<void*>(base);
  cuuint64_t dims2[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides2[1] = {static_cast<cuuint64_t>(row_bytes)};
  cuuint32_t box2[2] = {static_cast<cuuint32_t>(kBlockBytes), static_cast<cuuint32_t>(kPairRows)};
  cuuint32_t estr[3] = {1, 1, 1};
  if (fn(map2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p, dims2, strides2, box2, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return TCB_ERR_INVALID_ARGUMENT;
  *map3 = CUtensorMap{};
  if (*full_panels < kPairPanels) {
    *full_panels = 0;
    return TCB_OK;
  }
  cuuint64_t dims3[3] = {static_cast<cuuint64_t>(kBlockBytes), static_cast<cuuint64_t>(rows),
                         static_cast<cuuint64_t>(*full_panels)};
  cuuint64_t strides3[2] = {static_cast<cuuint64_t>(row_bytes),
                            static_cast<cuuint64_t>(kBlockBytes)};
  cuuint32_t box3[3] = {static_cast<cuuint32_t>(kBlockBytes), static_cast<cuuint32_t>(kPairRows),
                        static_cast<cuuint32_t>(kPairPanels)};
  if (fn(map3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p, dims3, strides3, box3, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    *map3 = CUtensorMap{};
    *full_panels = 0;  // the 2-D boxes still cover every stage
  }
  return TCB_OK;
}

// C [rows][cols] as boxes of 32 rows x 128 bytes in the SWIZZLE_128B layout
// the epilogue stages (16-byte row pitch and base required).
int pair_map_c(CUtensorMap* map, void* base, int rows, int cols, long long ldc, int elem_bytes) {
  auto fn = tensor_map_encoder();
  if (fn == nullptr) return TCB_ERR_DEVICE;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldc) * elem_bytes};
  cuuint32_t box[2] = {128u / elem_bytes, 32};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, elem_bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TCB_OK
             : TCB_ERR_INVALID_ARGUMENT;
}

using PairFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, PairArgs);

template <int OUT>
PairFn pair_fn_of(bool bias, int store) {
  if (store == kStoreDigits) return gemm_pair_mxf4_kernel<OUT, false, kStoreDigits>;
  if (store == kStorePlain)
    return bias ? gemm_pair_mxf4_kernel<OUT, true, kStorePlain> : gemm_pair_mxf4_kernel<OUT, false, kStorePlain>;
  return bias ? gemm_pair_mxf4_kernel<OUT, true, kStoreTma> : gemm_pair_mxf4_kernel<OUT, false, kStoreTma>;
}

PairFn pair_fn(int out, bool bias, int store) {
  switch (out) {
    case kPairBf16: return pair_fn_of<kPairBf16>(bias, store);
    case kPairFp16: return pair_fn_of<kPairFp16>(bias, store);
  }
  return pair_fn_of<kPairFp32>(bias, store);
}

}  // namespace

// MX FP4 GEMM on CTA pairs: tensor maps, arguments and launch of `blocks / 2`
// persistent pairs (all the pairs that fit at once by default).
int gemm_pair_run(const PairProblem& p, int blocks, int* status, const DeviceFacts& facts,
                  cudaStream_t stream) {
  const long long kbytes = static_cast<long long>(p.k) / 2;
  const int elem_bytes = p.out == kPairFp32 ? 4 : 2;
  PairArgs args;
  args.sa = static_cast<const uint8_t*>(p.sa);
  args.sb = static_cast<const uint8_t*>(p.sb);
  args.c = p.c;
  args.bias = p.bias;
  args.ldc = p.ldc;
  args.status = status;
  args.m = p.m;
  args.n = p.n;
  const long long tiles_m = (static_cast<long long>(p.m) + 2 * kPairRows - 1) / (2 * kPairRows);
  const long long tiles_n = (static_cast<long long>(p.n) + kTileN - 1) / kTileN;
  if (tiles_m * tiles_n > INT_MAX / 2) return TCB_ERR_RESOURCE;
  args.tiles_m = static_cast<int>(tiles_m);
  args.tiles_n = static_cast<int>(tiles_n);
  args.kblocks = static_cast<int>((kbytes + kBlockBytes - 1) / kBlockBytes);
  const bool digits = p.digits_of != nullptr;
  args.x = digits ? *p.digits_of : mx_detail::ValueRows{};
  args.lists = p.digits_left;
  args.a = static_cast<const uint8_t*>(p.a);
  args.pitch = kbytes;
  args.idesc = p.idesc;
  CUtensorMap map_a, map_b, map_a3, map_b3;
  int panels_a = static_cast<int>(kbytes / kBlockBytes), panels_b = panels_a;
  int rc;
  if ((rc = pair_maps(&map_a, &map_a3, p.a, p.m, kbytes, &panels_a)) != TCB_OK) return rc;
  if ((rc = pair_maps(&map_b, &map_b3, p.b, p.n, kbytes, &panels_b)) != TCB_OK) return rc;
  args.full_panels = panels_a < panels_b ? panels_a : panels_b;
  CUtensorMap map_c{};
  // A row's end has to be on a 16-byte boundary too: the store clips whole 16-byte
  // units at C's edge, and would write zeros between it and the next boundary.
  const bool tma = p.ldc * elem_bytes % 16 == 0 && static_cast<long long>(p.n) * elem_bytes % 16 == 0 &&
                   aligned(p.c, 16) && !digits &&
                   pair_map_c(&map_c, p.c, p.m, p.n, p.ldc, elem_bytes) == TCB_OK;
  const int store = digits ? kStoreDigits : tma ? kStoreTma : kStorePlain;
  const PairFn fn = pair_fn(p.out, p.bias != nullptr, store);
  static DeviceIntCache cap_cache[3][2][3], resident_cache;
  const int cap = cap_cache[p.out][p.bias != nullptr][store].get(facts.device, [&] {
    return raise_dynamic_smem(reinterpret_cast<const void*>(fn), facts.max_smem_optin);
  });
  if (cap < kPairSmem) return TCB_ERR_RESOURCE;
  // Pairs that can be resident at once (one CTA per SM whatever C's type):
  // persistent pairs beyond that would only start when others finish,
  // serialising their tiles.
  const int resident = resident_cache.get(facts.device, [&] {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * (facts.sm_count / 2), 1, 1);
    config.blockDim = dim3(kPairThreads, 1, 1);
    config.dynamicSmemBytes = kPairSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, fn, &config) != cudaSuccess || clusters < 1) {
      clear_stale_error();
      clusters = facts.sm_count / 2;
    }
    return clusters;
  });
  const int tiles = args.tiles_m * args.tiles_n;
  int pairs = blocks > 0 ? blocks / 2 : facts.sm_count / 2;
  if (pairs < 1) pairs = 1;
  if (pairs > tiles) pairs = tiles;
  if (pairs > resident) pairs = resident;
  if (p.overlap)
    return launch_overlapping(fn, dim3(static_cast<unsigned>(2 * pairs)), kPairThreads, kPairSmem, 1, stream,
                              map_a, map_b, map_a3, map_b3, map_c, args);
  clear_stale_error();
  fn<<<2 * pairs, kPairThreads, kPairSmem, stream>>>(map_a, map_b, map_a3, map_b3, map_c, args);
  return launch_status();
}

int gemm_pair_info(tcb_kernel_info_t* out) {
  cudaFuncAttributes attr;
  if (cudaFuncGetAttributes(&attr, reinterpret_cast<const void*>(pair_fn(kPairFp32, false, kStoreTma))) !=
      cudaSuccess)
    return TCB_ERR_DEVICE;
  fill_kernel_info(attr, out);
  out->dynamic_smem_bytes = kPairSmem;
  out->threads_per_block = kPairThreads;
  out->tensor_core = 1;
  out->pipeline_stages = kPairStages;
  out->tile_m = 2 * kPairRows;
  out->tile_n = kTileN;
  out->cluster_ctas = 2;
  return TCB_OK;
}

}  // namespace tcb
