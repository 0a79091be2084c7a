// Host-visible launcher of the 8-bit tcgen05 products (fp8_gemm.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace wc {

struct Fp8GemmParams {
  const uint8_t *a, *w, *up;         // codes [m][lda], [n][ldw], [n][ldup] (up: gated only)
  const float *sa, *sw, *sup;        // scales [m][ldsa], [n / 128][ldsw], [n / 128][ldsup]
  const void* residual;              // [m][ldr] of the output's type, or null
  void* out;                         // [m][ldo]
  float* out_scales;                 // [m][ldos], 8-bit output only
  int64_t lda, ldw, ldup, ldsa, ldsw, ldsup, ldr, ldo, ldos;
  int m, n, k;
  int act;                           // WC_ACT_*, gated only
  bool box_o, box_r;                 // rows of 16-byte blocks: whole ones of the output, aligned ones of the residual
};

// out_type WC_T_E4M3 only with gated.
cudaError_t fp8_gemm_launch(bool gated, int out_type, const Fp8GemmParams& p, int num_sms, cudaStream_t st);

// Which kernel fp8_gemm_launch takes: CTAs that share a tile, 0 for pairs of SMs.
cudaError_t fp8_gemm_split(bool gated, int out_type, const Fp8GemmParams& p, int num_sms, int* split);

// The products' status word on the current device, read and cleared in one
// step on st; waits for it.
cudaError_t fp8_gemm_take_status(uint32_t* status, cudaStream_t st);

// Enqueues a wait that runs out after limit_ns and says so in that word.
cudaError_t fp8_gemm_timeout_selftest(uint64_t limit_ns, cudaStream_t st);

}  // namespace wc
