// Rows and weights to 8 bits, and the RMSNorm with the residual add that
// writes 8-bit rows.  All are bound by the bytes they read and write.
//
// One warp handles one block of 128 columns at a time, four consecutive
// elements per lane, so the block's maximum is one warp reduction and every
// access of the warp is one contiguous run (512 B of f32, 256 B of 16-bit
// values, 128 B of codes).
#include "fp8.cuh"
#include "fp8_rows.h"

namespace wc {

namespace {

constexpr int kWarps = 8;
constexpr int kHeld = 8;  // blocks a warp keeps in registers between the norm's two passes

__device__ __forceinline__ float max4_nan(float4 v) {
  return max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w)));
}
__device__ __forceinline__ uint32_t codes4(float4 v, float f) {
  return pack_e4m3x4(v.x * f, v.y * f, v.z * f, v.w * f);
}
__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Blocks are independent: one warp per kHeld blocks of a row, all loads
// issued first.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) fp8_rows_kernel(Fp8RowsParams p, int groups) {
  pdl_wait();
  pdl_launch_next();
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t row = unit / groups;
  if (row >= p.m) return;
  const int64_t c0 = (unit - row * groups) * (kHeld * kFp8Block) + lane * 4;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float4 v[kHeld];
#pragma unroll
  for (int g = 0; g < kHeld; ++g) v[g] = load4(x + c0 + g * kFp8Block, p.k - c0 - g * kFp8Block, p.vec_x);
  float mine = 0.f;
#pragma unroll
  for (int g = 0; g < kHeld; ++g) {
    const int64_t col = c0 + g * kFp8Block;
    if (col - lane * 4 >= p.k) break;
    const float s = fp8_scale(warp_max_nan(max4_nan(v[g])));
    if (lane == g) mine = s;
    store_codes4(p.codes + row * p.ldc + col, p.k - col, codes4(v[g], fp8_factor(s)));
  }
  const int64_t blk = (c0 - lane * 4) / kFp8Block + lane;
  if (lane < kHeld && blk * kFp8Block < p.k) p.scales[row * p.lds + blk] = mine;
}

// One row by WPR warps.  kHeld blocks per warp stay in registers between the
// sum of squares and the scaling (rows up to WPR * kHeld * 128 columns); a
// wider row (WPR = kWarps only) is read again for the second pass.
template <typename TX, typename TD, bool DELTA, int WPR, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps) fp8_rmsnorm_kernel(Fp8RowsParams p) {
  __shared__ float part[kWarps];
  pdl_wait();
  pdl_launch_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wi = warp % WPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWarps / WPR) + warp / WPR;
  const bool live = row < p.m;
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
  const TD* d = static_cast<const TD*>(p.delta) + row * p.ldd;
  const int64_t kblocks = live ? (p.k + kFp8Block - 1) / kFp8Block : 0;
  float4 v[kHeld], e[kHeld];
  float ss = 0.f;
  auto fetch = [&](int64_t b0) {  // blocks b0 + wi + WPR g
#pragma unroll
    for (int g = 0; g < kHeld; ++g) {
      const int64_t b = b0 + wi + WPR * g, col = b * kFp8Block + lane * 4;
      if (b < kblocks) {
        v[g] = load4(x + col, p.k - col, p.vec_x);
        if (DELTA) e[g] = load4(d + col, p.k - col, p.vec_d);
      } else {
        v[g] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int g = 0; g < kHeld; ++g)
      if (DELTA && b0 + wi + WPR * g < kblocks) {
        v[g].x += e[g].x;
        v[g].y += e[g].y;
        v[g].z += e[g].z;
        v[g].w += e[g].w;
      }
  };
  for (int64_t b0 = 0; b0 == 0 || (WIDE && b0 < kblocks); b0 += WPR * kHeld) {
    fetch(b0);
#pragma unroll
    for (int g = 0; g < kHeld; ++g) ss += v[g].x * v[g].x + v[g].y * v[g].y + v[g].z * v[g].z + v[g].w * v[g].w;
  }
  ss = warp_total(ss);
  if (WPR > 1) {
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) ss += part[warp / WPR * WPR + i];
  }
  if (!live) return;
  const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.k) + p.eps);
  for (int64_t b0 = 0; b0 == 0 || (WIDE && b0 < kblocks); b0 += WPR * kHeld) {
    if (WIDE) fetch(b0);
    float mine = 0.f;
#pragma unroll
    for (int g = 0; g < kHeld; ++g) {
      const int64_t b = b0 + wi + WPR * g, col = b * kFp8Block + lane * 4;
      if (b >= kblocks) break;
      const float4 w = load4(p.w + col, p.k - col, p.vec_w);
      if (DELTA) store4(static_cast<TX*>(p.sum) + row * p.ldsum + col, p.k - col, p.vec_s, v[g]);
      const float4 y = make_float4(v[g].x * inv * w.x, v[g].y * inv * w.y, v[g].z * inv * w.z, v[g].w * inv * w.w);
      const float s = fp8_scale(warp_max_nan(max4_nan(y)));
      if (lane == g) mine = s;
      store_codes4(p.codes + row * p.ldc + col, p.k - col, codes4(y, fp8_factor(s)));
    }
    const int64_t b = b0 + wi + WPR * lane;
    if (lane < kHeld && b < kblocks) p.scales[row * p.lds + b] = mine;
  }
}

// One CTA per 128 x 128 block, 16 rows per warp held in registers.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) fp8_weight_kernel(Fp8RowsParams p, int kblocks) {
  __shared__ float part[kWarps];
  pdl_wait();
  pdl_launch_next();
  constexpr int kRows = kFp8Block / kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t nb = blockIdx.x / kblocks, kb = blockIdx.x % kblocks;
  const int64_t row0 = nb * kFp8Block + warp * kRows, col = kb * kFp8Block + lane * 4, left = p.k - col;
  const T* x = static_cast<const T*>(p.x) + row0 * p.ldx + col;
  float4 v[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) v[r] = load4(x + r * p.ldx, row0 + r < p.m ? left : 0, p.vec_x);
  float a = 0.f;
#pragma unroll
  for (int r = 0; r < kRows; ++r) a = max_nan(a, max4_nan(v[r]));
  a = warp_max_nan(a);
  if (lane == 0) part[warp] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) a = max_nan(a, part[i]);
  const float s = fp8_scale(a), f = fp8_factor(s);
  if (threadIdx.x == 0) p.scales[nb * p.lds + kb] = s;
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (row0 + r < p.m) store_codes4(p.codes + (row0 + r) * p.ldc + col, left, codes4(v[r], f));
}

// Grid of at most 2^31 - 1 CTAs.
bool grid_of(int64_t n, dim3* g) {
  if (n < 1 || n > 0x7FFFFFFF) return false;
  *g = dim3(static_cast<unsigned>(n));
  return true;
}

template <typename TX, typename TD, bool DELTA>
cudaError_t rmsnorm(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t kb = (p.k + kFp8Block - 1) / kFp8Block;
  auto go = [&](auto kernel, int wpr) {
    dim3 grid;
    if (!grid_of((p.m + kWarps / wpr - 1) / (kWarps / wpr), &grid)) return cudaErrorInvalidValue;
    return launch_pdl(kernel, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p);
  };
  if (kb <= kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, 1, false>, 1);
  if (kb <= 2 * kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, 2, false>, 2);
  if (kb <= 4 * kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, 4, false>, 4);
  if (kb <= 8 * kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, 8, false>, 8);
  return go(fp8_rmsnorm_kernel<TX, TD, DELTA, 8, true>, 8);
}

template <typename TX>
cudaError_t rmsnorm_d(int delta_type, const Fp8RowsParams& p, cudaStream_t st) {
  if (!p.delta) return rmsnorm<TX, TX, false>(p, st);
  switch (delta_type) {
    case WC_T_F32: return rmsnorm<TX, float, true>(p, st);
    case WC_T_F16: return rmsnorm<TX, __half, true>(p, st);
    case WC_T_BF16: return rmsnorm<TX, __nv_bfloat16, true>(p, st);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t rows(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t groups = (p.k + kHeld * kFp8Block - 1) / (kHeld * kFp8Block);
  dim3 grid;
  if (groups > 0x7FFFFFFF || !grid_of((p.m * groups + kWarps - 1) / kWarps, &grid)) return cudaErrorInvalidValue;
  return launch_pdl(fp8_rows_kernel<T>, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p, static_cast<int>(groups));
}

template <typename T>
cudaError_t weight(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t kb = (p.k + kFp8Block - 1) / kFp8Block, nb = (p.m + kFp8Block - 1) / kFp8Block;
  dim3 grid;
  if (kb > 0x7FFFFFFF || !grid_of(kb * nb, &grid)) return cudaErrorInvalidValue;
  return launch_pdl(fp8_weight_kernel<T>, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p, static_cast<int>(kb));
}

}  // namespace

cudaError_t fp8_rows_launch(int x_type, Fp8RowsParams p, cudaStream_t st) {
  switch (x_type) {
    case WC_T_F32: return rows<float>(p, st);
    case WC_T_F16: return rows<__half>(p, st);
    case WC_T_BF16: return rows<__nv_bfloat16>(p, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t fp8_weight_launch(int w_type, Fp8RowsParams p, cudaStream_t st) {
  switch (w_type) {
    case WC_T_F32: return weight<float>(p, st);
    case WC_T_F16: return weight<__half>(p, st);
    case WC_T_BF16: return weight<__nv_bfloat16>(p, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t fp8_rmsnorm_launch(int x_type, int delta_type, Fp8RowsParams p, cudaStream_t st) {
  switch (x_type) {
    case WC_T_F32: return rmsnorm_d<float>(delta_type, p, st);
    case WC_T_F16: return rmsnorm_d<__half>(delta_type, p, st);
    case WC_T_BF16: return rmsnorm_d<__nv_bfloat16>(delta_type, p, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace wc
