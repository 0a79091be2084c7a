/*
 * 8-bit operators of the encoder's layers on a B200: rows and weights in
 * float8 e4m3 (4 exponent bits, 3 fraction bits, largest value 448, no
 * infinity) with one f32 scale per block of 128, the RMSNorm that produces
 * such rows, and the matrix products that read them.  (No counterpart in the
 * reference, whose layers run in f32, src/quantized_t5.rs:43-45.)
 *
 * A value is code * scale.  Rows (activations) have one scale per row and
 * 128 columns: scales [rows][ceil(k / 128)]; weights one per 128 x 128
 * block: scales [ceil(n / 128)][ceil(k / 128)].  The scale of a block is
 * max(max|x| / 448, 2^-126), its codes x / scale (the rounded f32 quotient)
 * rounded to the nearest e4m3 value (ties to even) and saturated.  A block that holds a NaN or an
 * infinity gets a NaN or infinite scale and stands for NaN throughout.
 *
 * Codes start at 16-byte boundaries and so do their rows (the leading
 * dimension, in elements, is a multiple of 16); every size may be odd, and
 * what lies between k and the leading dimension is neither read nor written.
 * Other leading dimensions are free as long as they cover the row.
 *
 * Device pointers on the current device; stream is a cudaStream_t (may be
 * 0).  Calls return once the work is enqueued, allocate nothing and keep
 * nothing of their arguments.  m = 0 (no rows) is valid and launches nothing.
 * Return codes are those of wc_t5cuda.h; wc_fp8_last_error() gives the
 * calling thread's last message.
 */
#ifndef WC_FP8_H
#define WC_FP8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { WC_T_F32 = 0, WC_T_F16 = 1, WC_T_BF16 = 2, WC_T_E4M3 = 3 };
enum { WC_ACT_GELU = 0 /* tanh form (gelu_new) */, WC_ACT_SILU = 1 };

/* x [m][k] of x_type (f32, f16, bf16) -> codes [m][ldc], scales [m][lds]. */
int wc_fp8_quantize_rows(const void* d_x, int x_type, int64_t m, int64_t k, int64_t ldx, void* d_codes, int64_t ldc,
                         float* d_scales, int64_t lds, void* stream);

/* w [n][k] of w_type -> codes [n][ldc], scales [ceil(n / 128)][lds]. */
int wc_fp8_quantize_weight(const void* d_w, int w_type, int64_t n, int64_t k, int64_t ldw, void* d_codes, int64_t ldc,
                           float* d_scales, int64_t lds, void* stream);

/* RMSNorm (T5LayerNorm, src/quantized_t5.rs:162-173) with the residual add
 * of the sub-layer before it and 8-bit rows out:
 *   t = x + delta; sum = t in x_type; y = t / sqrt(mean(t^2) + eps) * w;
 *   codes, scales = quantize_rows(y).
 * t stays f32 for the norm.  d_delta may be NULL (no add; d_sum is then not
 * written and may be NULL); d_sum may be d_x (in place). */
int wc_fp8_rmsnorm(const void* d_x, int x_type, int64_t ldx, const void* d_delta, int delta_type, int64_t ldd,
                   void* d_sum, int64_t ldsum, const float* d_w, int64_t m, int64_t k, float eps, void* d_codes,
                   int64_t ldc, float* d_scales, int64_t lds, void* stream);

/* out[m][n] = a . w^T (+ residual) for rows a [m][k] and weights w [n][k],
 * f32 sums, rounded once to out_type (f32, f16, bf16).  d_residual (of
 * out_type, leading dimension ldr) may be NULL, or d_out (in place). */
int wc_fp8_matmul(const void* d_a, int64_t lda, const float* d_sa, int64_t ldsa, int64_t m, int64_t k,
                  const void* d_w, int64_t ldw, const float* d_sw, int64_t ldsw, int64_t n, const void* d_residual,
                  int64_t ldr, void* d_out, int out_type, int64_t ldo, void* stream);

/* h = act(a . w^T) * (a . up^T), both weights [n][k] (the gated feed-forward,
 * src/quantized_t5.rs:231-252).  out_type f32, f16 or bf16: out = h [m][ldo];
 * WC_T_E4M3: out, out_scales = quantize_rows(h), codes [m][ldo] and
 * scales [m][ldos] (d_out_scales is ignored otherwise). */
int wc_fp8_gated_matmul(const void* d_a, int64_t lda, const float* d_sa, int64_t ldsa, int64_t m, int64_t k,
                        const void* d_w, int64_t ldw, const float* d_sw, int64_t ldsw, const void* d_up, int64_t ldup,
                        const float* d_sup, int64_t ldsup, int64_t n, int act, void* d_out, int out_type, int64_t ldo,
                        float* d_out_scales, int64_t ldos, void* stream);

/* Waits for `stream` and reports what the products' kernels could not report
 * when they were enqueued: WC_E_TIMEOUT when an in-kernel wait ran out on the
 * current device, on any of its streams, since the last call (the results of
 * that product are then incomplete).  One call reports it, of whichever thread
 * and stream: who runs products on several streams waits for all of them before
 * any result is trusted.  No other call reports it. */
int wc_fp8_sync(void* stream);

/* Failure-detection self-test: enqueues a wait that nothing ends, as a product's
 * would, and that gives up after limit_ns (1e6 .. 1e10); wc_fp8_sync reports it. */
int wc_selftest_fp8_timeout(uint64_t limit_ns, void* stream);

/* Self-test of the choice between the products' kernels: how many CTAs share a
 * tile (1, 2, 4 or 8: few rows), or 0 for tiles on pairs of SMs (many rows), in
 * wc_fp8_matmul or wc_fp8_gated_matmul (gated) with these arguments.  residual:
 * there is one; boxes: results and residual have rows of whole 16-byte blocks.
 * Negative: a return code. */
int wc_selftest_fp8_split(int gated, int64_t m, int64_t k, int64_t n, int out_type, int residual, int boxes);

const char* wc_fp8_last_error(void);

#ifdef __cplusplus
}
#endif

#endif
