// The CTA-pair MX FP4 product behind tcb_gemm and tcb_mx_gemm.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "tcb_host.h"

namespace tcb {

namespace mx_detail {
struct ValueRows;
struct LeftList;
}  // namespace mx_detail

enum PairOutType : int { kPairFp32 = 0, kPairBf16 = 1, kPairFp16 = 2 };

struct PairProblem {
  const void* a;     // [m][k / 2] E2M1 codes
  const void* b;     // [n][k / 2]
  const void* sa;    // packed E8M0 scales of a
  const void* sb;
  const void* bias;  // [n] of C's type, or null
  void* c;           // [m][n], row pitch ldc elements
  long long ldc;
  int m, n, k;       // k a multiple of 32
  int out;           // PairOutType
  uint32_t idesc;
  bool overlap;      // may start while the kernels before it still run (launch_overlapping)
  // Non-null: b's rows are the MX FP4 digits of these 16-bit rows (SliceDigits), which
  // leave digits_left, and c is the product of the rows with a's, transposed.
  const mx_detail::ValueRows* digits_of;
  const mx_detail::LeftList* digits_left;
};

int gemm_pair_run(const PairProblem& p, int blocks, int* status, const DeviceFacts& facts,
                  cudaStream_t stream);
// Instruction descriptor of the pair MMA (M = N = 256, E2M1 x E2M1, E8M0 scales).
uint32_t gemm_pair_idesc();

}  // namespace tcb
