// Host-visible launchers of the 8-bit row kernels (fp8_rows.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace wc {

struct Fp8RowsParams {
  const void* x;      // [m][ldx]
  const void* delta;  // [m][ldd], or null
  void* sum;          // [m][ldsum] x + delta (with delta only)
  const float* w;     // [k] norm weights
  uint8_t* codes;     // [m][ldc]
  float* scales;      // [m][lds]
  int64_t m, k, ldx, ldd, ldsum, ldc, lds;
  float eps;
  bool vec_x, vec_d, vec_s, vec_w;  // rows aligned to eight elements
};

cudaError_t fp8_rows_launch(int x_type, Fp8RowsParams p, cudaStream_t st);
cudaError_t fp8_rmsnorm_launch(int x_type, int delta_type, Fp8RowsParams p, cudaStream_t st);
// p.m weight rows, p.scales one per 128 x 128 block.
cudaError_t fp8_weight_launch(int w_type, Fp8RowsParams p, cudaStream_t st);

}  // namespace wc
