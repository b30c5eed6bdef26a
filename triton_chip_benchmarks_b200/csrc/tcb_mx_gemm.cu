// Products with MX FP4 operands and a 16- or 32-bit result: the entry points
// that choose between the CTA-pair GEMM (tcb_gemm_pair.cu) and the few-row
// kernel (tcb_mx_rows.cu).
#include "tcb_gemm_pair.h"
#include "tcb_host.h"
#include "tcb_mx.cuh"
#include "tcb_mx_rows.h"

namespace tcb {
namespace {

// Up to so many rows of A the weight's bytes bound the product, and the few-row
// kernel, which spreads them over every SM, is faster than tiles of 256 rows:
// fewest where the tiles of 256 columns keep half of the SMs busy, most where K is
// long too.  Measured (us, few-row / CTA pairs, M = 8, 48, 64, 96, 128):
//   N x K   4096 x 4096   5.2/9.2   6.6/9.3   7.0/9.4   7.8/9.6   8.8/9.8
//           8192 x 8192   9.9/16.5 11.4/16.4 12.3/16.5 13.9/16.7 15.2/17.0
//           4096 x 1024   3.3/5.7   4.7/5.9   5.2/5.9   6.1/6.1   7.1/6.3
//           8192 x 1024             6.2/6.0   6.7/6.1   8.2/6.2
//          12288 x 4096          10.5/13.0 11.9/11.5 13.5/11.7
//          16384 x 4096   9.8/13.1 11.8/13.0 13.0/12.5 14.5/12.8 16.2/13.0
int few_rows(int n, int k, const DeviceFacts& facts) {
  const long long pairs = (static_cast<long long>(n) + 255) / 256;  // with work
  if (4 * pairs > facts.sm_count) return 48;
  const int most = 96;
  static_assert(most <= kRowsMostMx, "one column tile of the few-row kernel");
  return k >= 2048 ? most : 64;
}

bool out_type(int dtype, int* rows, int* pair, int* bytes) {
  switch (dtype) {
    case TCB_T_FP32: *rows = kRowsFp32, *pair = kPairFp32, *bytes = 4; return true;
    case TCB_T_BF16: *rows = kRowsBf16, *pair = kPairBf16, *bytes = 2; return true;
    case TCB_T_FP16: *rows = kRowsFp16, *pair = kPairFp16, *bytes = 2; return true;
  }
  return false;
}

}  // namespace
}  // namespace tcb

using namespace tcb;

extern "C" int tcb_mx_gemm(const void* A, const void* SA, const void* B, const void* SB,
                           const void* bias, int dtype, void* C, long long ldc, int M, int N, int K,
                           int* status_dev, tcb_stream_t stream) {
  if (M < 0 || N < 0 || K <= 0 || ldc < N) return TCB_ERR_INVALID_ARGUMENT;
  int rows_type, pair_type, bytes;
  if (!out_type(dtype, &rows_type, &pair_type, &bytes)) return TCB_ERR_UNSUPPORTED;
  if (M == 0 || N == 0) return TCB_OK;
  if (A == nullptr || SA == nullptr || B == nullptr || SB == nullptr || C == nullptr)
    return TCB_ERR_INVALID_ARGUMENT;
  if (K > INT_MAX - 256) return TCB_ERR_RESOURCE;
  if (!aligned(A, 16) || !aligned(B, 16) || !aligned(SA, 16) || !aligned(SB, 16) ||
      !aligned(C, bytes) || !aligned(bias, bytes))
    return TCB_ERR_ALIGNMENT;
  DeviceFacts facts;
  const int rc = current_device_facts(&facts);
  if (rc != TCB_OK) return rc;
  if (facts.major != 10) return TCB_ERR_UNSUPPORTED;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (M <= few_rows(N, K, facts)) {
    const RowsProblem p{A, SA, B, SB, bias, C, 0, ldc, M, N, K, kRowsMx, rows_type};
    return mx_rows_run(p, nullptr, status_dev, facts, s);
  }
  const PairProblem p{A, B, SA, SB, bias, C, ldc, M, N, static_cast<int>(mx_detail::mx_padded(K)),
                      pair_type, gemm_pair_idesc(), true, nullptr, nullptr};
  return gemm_pair_run(p, 0, status_dev, facts, s);
}

extern "C" int tcb_mx_linear(int x_dtype, const void* X, long long ldx, const void* W, const void* SW,
                             const void* bias, int dtype, void* Y, long long ldy, int M, int N, int K,
                             void* workspace, long long workspace_bytes, int* status_dev,
                             tcb_stream_t stream) {
  if (M < 0 || N < 0 || K <= 0 || ldx < K || ldy < N) return TCB_ERR_INVALID_ARGUMENT;
  int rows_type, pair_type, bytes;
  if (!out_type(dtype, &rows_type, &pair_type, &bytes)) return TCB_ERR_UNSUPPORTED;
  if (x_dtype != TCB_T_BF16 && x_dtype != TCB_T_FP16) return TCB_ERR_UNSUPPORTED;
  if (M == 0 || N == 0) return TCB_OK;
  if (X == nullptr || W == nullptr || SW == nullptr || Y == nullptr) return TCB_ERR_INVALID_ARGUMENT;
  if (K > INT_MAX - 256) return TCB_ERR_RESOURCE;
  const long long need = mx_rows_workspace(M, K);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return TCB_ERR_INVALID_ARGUMENT;
  if (!aligned(workspace, 256)) return TCB_ERR_ALIGNMENT;
  if (!aligned(X, 2) || !aligned(W, 16) || !aligned(SW, 16) || !aligned(Y, bytes) ||
      !aligned(bias, bytes))
    return TCB_ERR_ALIGNMENT;
  DeviceFacts facts;
  const int rc = current_device_facts(&facts);
  if (rc != TCB_OK) return rc;
  if (facts.major != 10) return TCB_ERR_UNSUPPORTED;
  const RowsProblem p{X, nullptr, W, SW, bias, Y, ldx, ldy, M, N, K,
                      x_dtype == TCB_T_BF16 ? kRowsBf16 : kRowsFp16, rows_type};
  return mx_rows_run(p, workspace, status_dev, facts, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" long long tcb_mx_linear_workspace_bytes(int M, int K) {
  if (M < 0 || K <= 0) return TCB_ERR_INVALID_ARGUMENT;
  return mx_rows_workspace(M, K);
}
