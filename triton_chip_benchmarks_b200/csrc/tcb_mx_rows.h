// The few-row MX FP4 product behind tcb_mx_gemm and tcb_mx_linear.
#pragma once

#include <cuda_runtime.h>

#include "tcb_host.h"

namespace tcb {

enum RowsType : int { kRowsFp32 = 0, kRowsBf16 = 1, kRowsFp16 = 2, kRowsMx = 3 };

// MX rows of a call at most (one column tile).
constexpr int kRowsMostMx = 128;

struct RowsProblem {
  const void* x;     // [m] rows of x_type, pitch ldx elements (MX: codes, whole groups)
  const void* sx;    // packed scales of x (MX)
  const void* w;     // [n] rows of E2M1 codes, whole groups
  const void* sw;    // packed scales of w
  const void* bias;  // [n] of y_type, or null
  void* y;           // [m][n], pitch ldy elements
  long long ldx, ldy;
  int m, n, k;
  int x_type, y_type;
};

// Bytes of workspace that mx_rows_run needs for m 16-bit rows of k values (MX
// rows need none).
long long mx_rows_workspace(long long m, long long k);
int mx_rows_run(const RowsProblem& p, void* workspace, int* status, const DeviceFacts& facts,
                cudaStream_t stream);

}  // namespace tcb
