// Rows and weights to 8 bits, and the RMSNorm with the residual add that
// writes 8-bit rows.  All are bound by the bytes they read and write.
//
// One warp handles one block of 128 columns at a time, four consecutive
// elements per lane, so the block's maximum is one warp reduction and every
// access of the warp is one contiguous run (512 B of f32, 256 B of 16-bit
// values, 128 B of codes).  VEC: every row is aligned to four elements and k
// is a multiple of four, so an access is either whole or absent; the other
// form takes the edge element by element.
#include "fp8.cuh"
#include "fp8_rows.h"

namespace wc {

namespace {

constexpr int kWarps = 8;
constexpr int kRowsHeld = 4;  // blocks of a row that one warp of fp8_rows_kernel loads at once

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

// Four elements as they are stored, so that a row waiting in registers takes
// no more of them than its type needs.
template <typename T>
struct Raw4 {
  T e[4];
};
template <>
struct Raw4<float> {
  float4 e;
};
template <typename T>
__device__ __forceinline__ float4 widen(const Raw4<T>& r) {
  if constexpr (sizeof(T) == 4)
    return r.e;
  else
    return make_float4(to_f32(r.e[0]), to_f32(r.e[1]), to_f32(r.e[2]), to_f32(r.e[3]));
}
template <bool VEC, typename T>
__device__ __forceinline__ Raw4<T> get4(const T* p, int left) {
  Raw4<T> r;
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      r.e = left > 0 ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      const uint2 u = left > 0 ? *reinterpret_cast<const uint2*>(p) : make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(&r) = u;
    }
  } else {
    if constexpr (sizeof(T) == 4) {
      r.e = load4(p, left, false);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r.e[i] = left > i ? p[i] : from_f32<T>(0.f);
    }
  }
  return r;
}
template <bool VEC, typename T>
__device__ __forceinline__ void put4(T* p, int left, float4 v) {
  if (!VEC) {
    store4(p, left, false, v);
  } else if (left > 0) {
    store4(p, 4, true, v);
  }
}
template <bool VEC>
__device__ __forceinline__ void put_codes(uint8_t* p, int left, uint32_t c) {
  if (!VEC) {
    store_codes4(p, left, c);
  } else if (left > 0) {
    *reinterpret_cast<uint32_t*>(p) = c;
  }
}

// Blocks are independent: one warp per kRowsHeld blocks of a row, all loads
// issued first.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) fp8_rows_kernel(const __grid_constant__ Fp8RowsParams p, int groups) {
  pdl_wait();
  pdl_launch_next();
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t row = groups == 1 ? unit : unit / groups;
  if (row >= p.m) return;
  const int b0 = static_cast<int>(unit - row * groups) * kRowsHeld;
  const int64_t c0 = static_cast<int64_t>(b0) * kFp8Block + lane * 4;
  const int left = static_cast<int>(p.k - c0);
  const T* x = static_cast<const T*>(p.x) + row * p.ldx + c0;
  uint8_t* codes = p.codes + row * p.ldc + c0;
  Raw4<T> v[kRowsHeld];
#pragma unroll
  for (int g = 0; g < kRowsHeld; ++g) v[g] = get4<VEC>(x + g * kFp8Block, left - g * kFp8Block);
  float mine = 0.f;
#pragma unroll
  for (int g = 0; g < kRowsHeld; ++g) {
    const float4 y = widen(v[g]);
    const float s = fp8_scale(warp_max_nan(max4_nan(y)));
    if (lane == g) mine = s;
    put_codes<VEC>(codes + g * kFp8Block, left - g * kFp8Block, codes4(y, fp8_factor(s)));
  }
  // lane's own block: left + 4 lane columns remain from the group's start
  if (lane < kRowsHeld && left + lane * 4 > lane * kFp8Block) p.scales[row * p.lds + b0 + lane] = mine;
}

// One row by WPR warps.  HELD blocks per warp stay in registers between the
// sum of squares and the scaling (rows up to WPR * HELD * 128 columns); a
// wider row (WIDE) is read again for the second pass.
template <typename TX, typename TD, bool DELTA, bool VEC, int WPR, int HELD, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps, WIDE ? 2 : 4)
    fp8_rmsnorm_kernel(const __grid_constant__ Fp8RowsParams p) {
  __shared__ float part[kWarps];
  pdl_wait();
  pdl_launch_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wi = warp % WPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWarps / WPR) + warp / WPR;
  const bool live = row < p.m;
  const int k = live ? static_cast<int>(p.k) : 0;
  constexpr int kStep = WPR * kFp8Block;  // columns between a warp's blocks
  const int64_t off = wi * kFp8Block + lane * 4;
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx + off;
  const TD* d = DELTA ? static_cast<const TD*>(p.delta) + row * p.ldd + off : nullptr;
  const int left0 = k - static_cast<int>(off);  // columns from this lane's first element on
  float4 v[HELD];
  float ss = 0.f;
  auto fetch = [&](int c0) {  // blocks at columns c0 + off + kStep g
    Raw4<TX> rx[HELD];
    Raw4<TD> rd[HELD];
#pragma unroll
    for (int g = 0; g < HELD; ++g) {
      rx[g] = get4<VEC>(x + c0 + g * kStep, left0 - c0 - g * kStep);
      if (DELTA) rd[g] = get4<VEC>(d + c0 + g * kStep, left0 - c0 - g * kStep);
    }
#pragma unroll
    for (int g = 0; g < HELD; ++g) {
      v[g] = widen(rx[g]);
      if (DELTA) {
        const float4 e = widen(rd[g]);
        v[g].x += e.x;
        v[g].y += e.y;
        v[g].z += e.z;
        v[g].w += e.w;
      }
    }
  };
  for (int c0 = 0; c0 == 0 || (WIDE && c0 < k); c0 += HELD * kStep) {
    fetch(c0);
#pragma unroll
    for (int g = 0; g < HELD; ++g) ss += v[g].x * v[g].x + v[g].y * v[g].y + v[g].z * v[g].z + v[g].w * v[g].w;
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
  const float inv = 1.0f / sqrtf(ss / static_cast<float>(k) + p.eps);
  TX* sum = DELTA ? static_cast<TX*>(p.sum) + row * p.ldsum + off : nullptr;
  uint8_t* codes = p.codes + row * p.ldc + off;
  float* scales = p.scales + row * p.lds + wi + WPR * lane;
  const float* wt = p.w + off;
  for (int c0 = 0; c0 == 0 || (WIDE && c0 < k); c0 += HELD * kStep) {
    if (WIDE) fetch(c0);
    float mine = 0.f;
#pragma unroll
    for (int g = 0; g < HELD; ++g) {
      const int c = c0 + g * kStep, left = left0 - c;
      if (left + lane * 4 <= 0) break;  // the whole block is past the row
      const float4 w = widen(get4<VEC>(wt + c, left));
      if (DELTA) put4<VEC>(sum + c, left, v[g]);
      const float4 y = make_float4(v[g].x * inv * w.x, v[g].y * inv * w.y, v[g].z * inv * w.z, v[g].w * inv * w.w);
      const float s = fp8_scale(warp_max_nan(max4_nan(y)));
      if (lane == g) mine = s;
      put_codes<VEC>(codes + c, left, codes4(y, fp8_factor(s)));
    }
    if (lane < HELD && left0 + lane * 4 > c0 + lane * kStep) scales[c0 / kFp8Block] = mine;
  }
}

// One CTA per 128 x 128 block, 16 rows per warp held in registers.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) fp8_weight_kernel(const __grid_constant__ Fp8RowsParams p, int kblocks) {
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

template <typename TX, typename TD, bool DELTA, bool VEC>
cudaError_t rmsnorm(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t kb = (p.k + kFp8Block - 1) / kFp8Block;
  auto go = [&](auto kernel, int wpr) {
    dim3 grid;
    if (!grid_of((p.m + kWarps / wpr - 1) / (kWarps / wpr), &grid)) return cudaErrorInvalidValue;
    return launch_pdl(kernel, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p);
  };
  if (kb <= 6) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 1, 6, false>, 1);
  if (kb <= 12) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 2, 6, false>, 2);
  if (kb <= 24) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 4, 6, false>, 4);
  if (kb <= 48) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 8, 6, false>, 8);
  return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 8, 8, true>, 8);
}

template <typename TX, typename TD, bool DELTA>
cudaError_t rmsnorm_v(const Fp8RowsParams& p, cudaStream_t st) {
  const bool vec = p.vec_x && p.vec_w && (!DELTA || (p.vec_d && p.vec_s)) && p.k % 4 == 0;
  return vec ? rmsnorm<TX, TD, DELTA, true>(p, st) : rmsnorm<TX, TD, DELTA, false>(p, st);
}

template <typename TX>
cudaError_t rmsnorm_d(int delta_type, const Fp8RowsParams& p, cudaStream_t st) {
  if (!p.delta) return rmsnorm_v<TX, TX, false>(p, st);
  switch (delta_type) {
    case WC_T_F32: return rmsnorm_v<TX, float, true>(p, st);
    case WC_T_F16: return rmsnorm_v<TX, __half, true>(p, st);
    case WC_T_BF16: return rmsnorm_v<TX, __nv_bfloat16, true>(p, st);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t rows(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t groups = (p.k + kRowsHeld * kFp8Block - 1) / (kRowsHeld * kFp8Block);
  dim3 grid;
  if (groups > 0x7FFFFFFF || !grid_of((p.m * groups + kWarps - 1) / kWarps, &grid)) return cudaErrorInvalidValue;
  auto kernel = p.vec_x && p.k % 4 == 0 ? fp8_rows_kernel<T, true> : fp8_rows_kernel<T, false>;
  return launch_pdl(kernel, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p, static_cast<int>(groups));
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
