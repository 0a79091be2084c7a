// The C ABI of include/wc_fp8.h: argument checks and dispatch.  Nothing here
// allocates device memory or throws across the boundary.
#include <cuda_runtime.h>
#include <stdio.h>

#include <atomic>

#include "../../include/wc_fp8.h"
#include "../../include/wc_t5cuda.h"
#include "fp8_gemm.h"
#include "fp8_rows.h"

namespace {

using namespace wc;

thread_local char g_fp8_error[256];

int refuse(int code, const char* msg) {
  snprintf(g_fp8_error, sizeof(g_fp8_error), "%s", msg);
  return code;
}
int done(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return WC_OK;
  snprintf(g_fp8_error, sizeof(g_fp8_error), "%s: %s", what, cudaGetErrorString(e));
  return WC_E_CUDA;
}

constexpr int64_t kMaxSize = 0x7FFFFF00;  // rows and weight rows are 32-bit inside the products
constexpr int64_t kMaxK = 1 << 30;        // columns: the row kernels add a few blocks to 32-bit column numbers

bool value_type(int t) { return t == WC_T_F32 || t == WC_T_F16 || t == WC_T_BF16; }
int type_size(int t) { return t == WC_T_F32 ? 4 : t == WC_T_E4M3 ? 1 : 2; }
bool aligned(const void* p, int64_t ld, int bytes, int type) {  // rows start at multiples of `bytes`
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld * type_size(type)) % bytes == 0;
}
// Whether rows of n results can be written by TMA boxes, which end a row at a
// multiple of 16 bytes: a row that ends between two would take the bytes behind
// it along (zeros there).
bool boxes(const void* p, int64_t ld, int64_t n, int type) {
  return aligned(p, ld, 16, type) && n * type_size(type) % 16 == 0;
}
// rows of eight elements at a time: 16-byte accesses
bool vec8(const void* p, int64_t ld, int type) { return aligned(p, ld, 16, type) && ld % 8 == 0; }
bool natural(const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_size(type) == 0; }
int64_t blocks(int64_t k) { return (k + 127) / 128; }

// Messages of the checks that several calls share; null when they pass.
const char* check_codes(const void* p, int64_t ld, int64_t k) {
  if (!p) return "codes are null";
  if (ld < k) return "leading dimension of codes below k";
  if (!aligned(p, ld, 16, WC_T_E4M3)) return "codes: base and leading dimension must be multiples of 16 bytes";
  return nullptr;
}
const char* check_scales(const float* p, int64_t ld, int64_t k) {
  if (!p || !natural(p, WC_T_F32)) return "scales are null or not aligned to 4 bytes";
  if (ld < blocks(k)) return "leading dimension of scales below ceil(k / 128)";
  return nullptr;
}
const char* check_values(const void* p, int type, int64_t ld, int64_t k) {
  if (!value_type(type)) return "type must be f32, f16 or bf16";
  if (!p || !natural(p, type)) return "values are null or not aligned to their type";
  if (ld < k) return "leading dimension of values below their row length";
  return nullptr;
}

int sm_count(int* n) {
  static std::atomic<int> counts[64] = {};  // calls come from any thread
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return done(e, "device");
  if (dev < 0 || dev >= 64) return refuse(WC_E_INVALID_ARG, "device ordinal above 63");
  if (!counts[dev]) {
    int c = 0, major = 0;
    if ((e = cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev)) != cudaSuccess)
      return done(e, "device attributes");
    if (major != 10) return refuse(WC_E_UNSUPPORTED, "these kernels are built for sm_100a (B200)");
    counts[dev] = c;
  }
  *n = counts[dev];
  return WC_OK;
}

int quantize(bool weight, const void* x, int type, int64_t m, int64_t k, int64_t ldx, void* codes, int64_t ldc,
             float* scales, int64_t lds, void* stream) {
  if (m < 0 || m > kMaxSize || k < 1 || k > kMaxK) return refuse(WC_E_INVALID_ARG, "sizes out of range (m >= 0, k >= 1)");
  if (!value_type(type)) return refuse(WC_E_INVALID_ARG, "type must be f32, f16 or bf16");
  if (m == 0) return WC_OK;
  const char* bad = check_values(x, type, ldx, k);
  if (!bad) bad = check_codes(codes, ldc, k);
  if (!bad) bad = check_scales(scales, lds, k);
  if (bad) return refuse(WC_E_INVALID_ARG, bad);
  Fp8RowsParams p{};
  p.x = x;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = scales;
  p.m = m;
  p.k = k;
  p.ldx = ldx;
  p.ldc = ldc;
  p.lds = lds;
  p.vec_x = vec8(x, ldx, type);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return done(weight ? fp8_weight_launch(type, p, st) : fp8_rows_launch(type, p, st), "quantisation launch");
}

// Checks shared by the two products; fills the common parameters.
int product(Fp8GemmParams& p, const void* a, int64_t lda, const float* sa, int64_t ldsa, int64_t m, int64_t k,
            const void* w, int64_t ldw, const float* sw, int64_t ldsw, int64_t n) {
  const char* bad = check_codes(a, lda, k);
  if (!bad) bad = check_scales(sa, ldsa, k);
  if (!bad) bad = check_codes(w, ldw, k);
  if (!bad) bad = check_scales(sw, ldsw, k);
  if (bad) return refuse(WC_E_INVALID_ARG, bad);
  p.a = static_cast<const uint8_t*>(a);
  p.w = static_cast<const uint8_t*>(w);
  p.sa = sa;
  p.sw = sw;
  p.lda = lda;
  p.ldw = ldw;
  p.ldsa = ldsa;
  p.ldsw = ldsw;
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  return WC_OK;
}

bool sizes_ok(int64_t m, int64_t k, int64_t n) {
  return m >= 0 && m <= kMaxSize && k >= 1 && k <= kMaxK && n >= 1 && n <= kMaxSize;
}

}  // namespace

extern "C" const char* wc_fp8_last_error(void) { return g_fp8_error; }

extern "C" int wc_fp8_quantize_rows(const void* d_x, int x_type, int64_t m, int64_t k, int64_t ldx, void* d_codes,
                                    int64_t ldc, float* d_scales, int64_t lds, void* stream) {
  return quantize(false, d_x, x_type, m, k, ldx, d_codes, ldc, d_scales, lds, stream);
}

extern "C" int wc_fp8_quantize_weight(const void* d_w, int w_type, int64_t n, int64_t k, int64_t ldw, void* d_codes,
                                      int64_t ldc, float* d_scales, int64_t lds, void* stream) {
  return quantize(true, d_w, w_type, n, k, ldw, d_codes, ldc, d_scales, lds, stream);
}

extern "C" int wc_fp8_rmsnorm(const void* d_x, int x_type, int64_t ldx, const void* d_delta, int delta_type,
                              int64_t ldd, void* d_sum, int64_t ldsum, const float* d_w, int64_t m, int64_t k,
                              float eps, void* d_codes, int64_t ldc, float* d_scales, int64_t lds, void* stream) {
  if (m < 0 || m > kMaxSize || k < 1 || k > kMaxK) return refuse(WC_E_INVALID_ARG, "sizes out of range (m >= 0, k >= 1)");
  if (!(eps >= 0.0f)) return refuse(WC_E_INVALID_ARG, "eps must not be negative");
  if (!value_type(x_type)) return refuse(WC_E_INVALID_ARG, "type must be f32, f16 or bf16");
  if (m == 0) return WC_OK;
  const char* bad = check_values(d_x, x_type, ldx, k);
  if (!bad && d_delta) bad = check_values(d_delta, delta_type, ldd, k);
  if (!bad && d_delta) bad = check_values(d_sum, x_type, ldsum, k);
  if (!bad) bad = check_values(d_w, WC_T_F32, k, k);
  if (!bad) bad = check_codes(d_codes, ldc, k);
  if (!bad) bad = check_scales(d_scales, lds, k);
  if (bad) return refuse(WC_E_INVALID_ARG, bad);
  Fp8RowsParams p{};
  p.x = d_x;
  p.delta = d_delta;
  p.sum = d_sum;
  p.w = d_w;
  p.codes = static_cast<uint8_t*>(d_codes);
  p.scales = d_scales;
  p.m = m;
  p.k = k;
  p.ldx = ldx;
  p.ldd = ldd;
  p.ldsum = ldsum;
  p.ldc = ldc;
  p.lds = lds;
  p.eps = eps;
  p.vec_x = vec8(d_x, ldx, x_type);
  p.vec_d = d_delta && vec8(d_delta, ldd, delta_type);
  p.vec_s = d_delta && vec8(d_sum, ldsum, x_type);
  p.vec_w = reinterpret_cast<uintptr_t>(d_w) % 16 == 0;
  return done(fp8_rmsnorm_launch(x_type, delta_type, p, static_cast<cudaStream_t>(stream)), "rmsnorm launch");
}

extern "C" int wc_fp8_matmul(const void* d_a, int64_t lda, const float* d_sa, int64_t ldsa, int64_t m, int64_t k,
                             const void* d_w, int64_t ldw, const float* d_sw, int64_t ldsw, int64_t n,
                             const void* d_residual, int64_t ldr, void* d_out, int out_type, int64_t ldo,
                             void* stream) {
  if (!sizes_ok(m, k, n)) return refuse(WC_E_INVALID_ARG, "sizes out of range (m >= 0, k >= 1, n >= 1)");
  if (!value_type(out_type)) return refuse(WC_E_INVALID_ARG, "type must be f32, f16 or bf16");
  if (m == 0) return WC_OK;
  Fp8GemmParams p{};
  int rc = product(p, d_a, lda, d_sa, ldsa, m, k, d_w, ldw, d_sw, ldsw, n);
  if (rc != WC_OK) return rc;
  const char* bad = check_values(d_out, out_type, ldo, n);
  if (!bad && d_residual) bad = check_values(d_residual, out_type, ldr, n);
  if (bad) return refuse(WC_E_INVALID_ARG, bad);
  int sms = 0;
  if ((rc = sm_count(&sms)) != WC_OK) return rc;
  p.residual = d_residual;
  p.out = d_out;
  p.ldr = ldr;
  p.ldo = ldo;
  p.box_o = boxes(d_out, ldo, n, out_type);
  p.box_r = d_residual && aligned(d_residual, ldr, 16, out_type);
  return done(fp8_gemm_launch(false, out_type, p, sms, static_cast<cudaStream_t>(stream)), "product launch");
}

extern "C" int wc_fp8_gated_matmul(const void* d_a, int64_t lda, const float* d_sa, int64_t ldsa, int64_t m,
                                   int64_t k, const void* d_w, int64_t ldw, const float* d_sw, int64_t ldsw,
                                   const void* d_up, int64_t ldup, const float* d_sup, int64_t ldsup, int64_t n,
                                   int act, void* d_out, int out_type, int64_t ldo, float* d_out_scales,
                                   int64_t ldos, void* stream) {
  if (!sizes_ok(m, k, n)) return refuse(WC_E_INVALID_ARG, "sizes out of range (m >= 0, k >= 1, n >= 1)");
  if (act != WC_ACT_GELU && act != WC_ACT_SILU) return refuse(WC_E_INVALID_ARG, "unknown activation");
  if (!value_type(out_type) && out_type != WC_T_E4M3) return refuse(WC_E_INVALID_ARG, "unknown output type");
  if (m == 0) return WC_OK;
  Fp8GemmParams p{};
  int rc = product(p, d_a, lda, d_sa, ldsa, m, k, d_w, ldw, d_sw, ldsw, n);
  if (rc != WC_OK) return rc;
  const char* bad = check_codes(d_up, ldup, k);
  if (!bad) bad = check_scales(d_sup, ldsup, k);
  if (!bad) bad = out_type == WC_T_E4M3 ? check_codes(d_out, ldo, n) : check_values(d_out, out_type, ldo, n);
  if (!bad && out_type == WC_T_E4M3) bad = check_scales(d_out_scales, ldos, n);
  if (bad) return refuse(WC_E_INVALID_ARG, bad);
  int sms = 0;
  if ((rc = sm_count(&sms)) != WC_OK) return rc;
  p.up = static_cast<const uint8_t*>(d_up);
  p.sup = d_sup;
  p.ldup = ldup;
  p.ldsup = ldsup;
  p.act = act;
  p.out = d_out;
  p.ldo = ldo;
  p.out_scales = d_out_scales;
  p.ldos = ldos;
  p.box_o = boxes(d_out, ldo, n, out_type);
  return done(fp8_gemm_launch(true, out_type, p, sms, static_cast<cudaStream_t>(stream)), "gated product launch");
}

extern "C" int wc_fp8_sync(void* stream) {
  uint32_t s = 0;
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = fp8_gemm_take_status(&s, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return done(e, "synchronising");
  return s ? refuse(WC_E_TIMEOUT, "an in-kernel wait timed out") : WC_OK;
}

extern "C" int wc_selftest_fp8_timeout(uint64_t limit_ns, void* stream) {
  if (limit_ns < 1000000ull || limit_ns > 10000000000ull) return refuse(WC_E_INVALID_ARG, "limit_ns must be 1e6 .. 1e10");
  return done(fp8_gemm_timeout_selftest(limit_ns, static_cast<cudaStream_t>(stream)), "self-test launch");
}

extern "C" int wc_selftest_fp8_split(int gated, int64_t m, int64_t k, int64_t n, int out_type, int residual, int boxes) {
  if (!sizes_ok(m, k, n) || m == 0) return refuse(WC_E_INVALID_ARG, "sizes out of range (m, k, n >= 1)");
  if (!value_type(out_type) && !(gated && out_type == WC_T_E4M3)) return refuse(WC_E_INVALID_ARG, "unknown output type");
  Fp8GemmParams p{};
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.residual = residual && !gated ? &p : nullptr;  // only whether there is one counts
  p.box_o = p.box_r = boxes != 0;
  int sms = 0, split = 0;
  if (const int rc = sm_count(&sms); rc != WC_OK) return rc;
  const int rc = done(fp8_gemm_split(gated != 0, out_type, p, sms, &split), "choice of a kernel");
  return rc != WC_OK ? rc : split;
}
