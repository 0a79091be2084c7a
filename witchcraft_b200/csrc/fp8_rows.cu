// Rows and weights to 8 bits, and the RMSNorm with the residual add that
// writes 8-bit rows.  All are bound by the bytes they read and write, if only
// just: scaling, the maximum and the conversion are about ten instructions an
// element, so what a block costs beside them is shared by eight elements.
//
// Sixteen lanes handle one block of 128 columns, two runs of four elements
// each, and a warp two blocks at a time.  The runs of a lane adjoin for 16-bit
// values (16 bytes) and lie 64 columns apart for f32 (two accesses of 16 bytes
// of which each covers whole lines: norm m = 16384, k = 768: 29.4 -> 27.1 us).
// VEC: every row is aligned to eight elements and k is a multiple of eight, so
// an access is either whole or absent; the other form takes rows that start
// anywhere, in pieces or element by element.
//
// Measured (device time, inputs from DRAM): norm f32 16384 x 768 with an f16
// residual 26.2 us or 5.3 TB/s, bf16 4095 x 5000 32.9 us or 4.4 TB/s; rows f16
// 16384 x 768 8.0 us or 4.8 TB/s; weight f32 2048 x 768 3.7 us, 32 rows of norm
// 3.3 us, both latency.
#include "fp8.cuh"
#include "fp8_rows.h"

namespace wc {

namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 2 * kFp8Block;  // columns a warp takes at a time
constexpr int kHeld = 3;              // units of a row that a warp loads at once

// Where a lane's runs of four lie: the first one's column within a unit, and
// how far on the second is.
template <bool APART>
__device__ __forceinline__ int first_run(int lane) {
  return APART ? (lane >> 4) * kFp8Block + (lane & 15) * 4 : lane * 8;
}
template <bool APART>
constexpr int kSecond = APART ? 64 : 4;

struct Eight {
  float v[8];
};

__device__ __forceinline__ float max_abs(const Eight& x) {
  float m = max_abs3_nan(x.v[0], x.v[1], x.v[2]);
  m = max_abs3_nan(m, x.v[3], x.v[4]);
  m = max_abs3_nan(m, x.v[5], x.v[6]);
  return max_nan(m, fabsf(x.v[7]));
}
__device__ __forceinline__ float half_warp_max_nan(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Two runs of four elements as they are stored.
template <typename T>
struct Raw8 {
  uint4 u;
};
template <>
struct Raw8<float> {
  float4 a, b;
};
__device__ __forceinline__ Eight widen(const Raw8<float>& r) {
  return Eight{{r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w}};
}
__device__ __forceinline__ Eight widen(const Raw8<__half>& r) {
  const uint32_t w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    e.v[2 * i] = f.x;
    e.v[2 * i + 1] = f.y;
  }
  return e;
}
__device__ __forceinline__ Eight widen(const Raw8<__nv_bfloat16>& r) {
  const uint32_t w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e.v[2 * i] = __uint_as_float(w[i] << 16);
    e.v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  return e;
}
// Four 16-bit elements that start at any of them, in as few pieces as p's
// alignment allows.
__device__ __forceinline__ uint2 four_16bit(const uint16_t* e, int left) {
  if (left >= 4) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(e)) & 7;
    if (off == 0) return __ldcs(reinterpret_cast<const uint2*>(e));
    if (off == 4)
      return make_uint2(reinterpret_cast<const uint32_t*>(e)[0], reinterpret_cast<const uint32_t*>(e)[1]);
    const uint32_t m = *reinterpret_cast<const uint32_t*>(e + 1);
    return make_uint2(e[0] | m << 16, m >> 16 | static_cast<uint32_t>(e[3]) << 16);
  }
  return make_uint2((left > 0 ? e[0] : 0u) | (left > 1 ? e[1] : 0u) << 16, left > 2 ? e[2] : 0u);
}
// The lane's runs at p, `left` columns of the row being left from there on;
// zeros past it.  Rows are read once and marked to be evicted first (norm m =
// 16384, k = 768: 30.2 -> 28.8 us); the norm weights, which every row reads, and
// the first pass over rows wider than a CTA's registers go the same way.
template <bool VEC, bool APART, typename T>
__device__ __forceinline__ Raw8<T> get8(const T* p, int left) {
  constexpr int d = kSecond<APART>;
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    if constexpr (VEC) {
      r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f);
      if (left > 0) r.a = __ldcs(reinterpret_cast<const float4*>(p));
      if (left > d) r.b = __ldcs(reinterpret_cast<const float4*>(p + d));
    } else {
      auto at = [&](int i) { return left > i ? __ldcs(p + i) : 0.f; };
      r.a = make_float4(at(0), at(1), at(2), at(3));
      r.b = make_float4(at(d), at(d + 1), at(d + 2), at(d + 3));
    }
  } else {
    uint2 a = make_uint2(0u, 0u), b = a;
    if constexpr (!VEC) {
      a = four_16bit(reinterpret_cast<const uint16_t*>(p), left);
      b = four_16bit(reinterpret_cast<const uint16_t*>(p + d), left - d);
    } else if constexpr (APART) {
      if (left > 0) a = __ldcs(reinterpret_cast<const uint2*>(p));
      if (left > d) b = __ldcs(reinterpret_cast<const uint2*>(p + d));
    } else if (left > 0) {
      r.u = __ldcs(reinterpret_cast<const uint4*>(p));
      return r;
    }
    r.u = make_uint4(a.x, a.y, b.x, b.y);
  }
  return r;
}
// Four elements of a row that may start at any of them, in as few pieces as p's
// alignment allows (norm with a residual, m = 8000, k = 701: f32 25.3 -> 21.9 us
// and bf16 26.8 -> 22.1 against one by one).
template <typename T>
__device__ __forceinline__ void store4_pieces(T* p, int left, float4 v) {
  if (left < 4) return store4(p, left, v);
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) % (4 * sizeof(T));
  if constexpr (sizeof(T) == 4) {
    if (off == 0) {
      *reinterpret_cast<float4*>(p) = v;
    } else if (off == 8) {
      *reinterpret_cast<float2*>(p) = make_float2(v.x, v.y);
      *reinterpret_cast<float2*>(p + 2) = make_float2(v.z, v.w);
    } else {
      p[0] = v.x;
      *reinterpret_cast<float2*>(p + 1) = make_float2(v.y, v.z);
      p[3] = v.w;
    }
  } else {
    const T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
    const uint2 u = *reinterpret_cast<const uint2*>(e);
    if (off == 0) {
      *reinterpret_cast<uint2*>(p) = u;
    } else if (off == 4) {
      reinterpret_cast<uint32_t*>(p)[0] = u.x;
      reinterpret_cast<uint32_t*>(p)[1] = u.y;
    } else {
      p[0] = e[0];
      *reinterpret_cast<uint32_t*>(p + 1) = u.x >> 16 | u.y << 16;
      p[3] = e[3];
    }
  }
}
template <bool VEC, bool APART, typename T>
__device__ __forceinline__ void put8(T* p, int left, const Eight& x) {
  constexpr int d = kSecond<APART>;
  if constexpr (VEC && sizeof(T) == 2 && !APART) {
    if (left <= 0) return;
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x.v[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
  } else {
    const float4 a = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]), b = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
    if constexpr (!VEC) {
      store4_pieces(p, left, a);
      store4_pieces(p + d, left - d, b);
    } else if constexpr (sizeof(T) == 4) {
      if (left >= 4) *reinterpret_cast<float4*>(p) = a;
      if (left >= d + 4) *reinterpret_cast<float4*>(p + d) = b;
    } else {
      const T e[8] = {from_f32<T>(a.x), from_f32<T>(a.y), from_f32<T>(a.z), from_f32<T>(a.w),
                      from_f32<T>(b.x), from_f32<T>(b.y), from_f32<T>(b.z), from_f32<T>(b.w)};
      if (left > 0) *reinterpret_cast<uint2*>(p) = reinterpret_cast<const uint2*>(e)[0];
      if (left > d) *reinterpret_cast<uint2*>(p + d) = reinterpret_cast<const uint2*>(e)[1];
    }
  }
}
// The codes of eight values over their scale s, f = 1 / s.  Two quotients at a
// time where registers allow (rows of f16, m = 16384, k = 768: 8.4 -> 8.0 us; 7.7
// with products by f alone); the norm, which is out of them, takes one (bf16, m =
// 4095, k = 5000: 32.9 us, 33.7 by twos).
template <bool VEC, bool APART, bool TWO>
__device__ __forceinline__ void put_codes8(uint8_t* p, int left, const Eight& x, float s, float f) {
  constexpr int d = kSecond<APART>;
  const uint32_t a = codes4<TWO>(x.v[0], x.v[1], x.v[2], x.v[3], s, f),
                 b = codes4<TWO>(x.v[4], x.v[5], x.v[6], x.v[7], s, f);
  if (!APART && left >= 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(a, b);
  } else if (!VEC) {
    store_codes4(p, left, a);
    store_codes4(p + d, static_cast<int64_t>(left) - d, b);
  } else if (APART) {
    if (left > 0) *reinterpret_cast<uint32_t*>(p) = a;
    if (left > d) *reinterpret_cast<uint32_t*>(p + d) = b;
  }
}
// Quantises one unit of a row: this lane's eight values, `left` columns of the
// row being left from its first one on.
template <bool VEC, bool APART, bool TWO>
__device__ __forceinline__ void put_unit(uint8_t* codes, float* scale, int lane, int left, const Eight& x) {
  const float s = fp8_scale(half_warp_max_nan(max_abs(x)));
  if ((lane & 15) == 0 && left > 0) *scale = s;
  put_codes8<VEC, APART, TWO>(codes, left, x, s, fp8_factor(s));
}

// Blocks are independent: one warp per kHeld units of a row, all loads issued
// first.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) fp8_rows_kernel(const __grid_constant__ Fp8RowsParams p, int groups) {
  pdl_wait();
  pdl_launch_next();
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t row = groups == 1 ? unit : unit / groups;
  if (row >= p.m) return;
  constexpr bool kApart = sizeof(T) == 4;
  const int start = static_cast<int>(unit - row * groups) * (kHeld * kUnit), run = first_run<kApart>(lane);
  const int c0 = start + run;
  const int left = static_cast<int>(p.k) - c0;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx + c0;
  uint8_t* codes = p.codes + row * p.ldc + c0;
  float* scales = p.scales + row * p.lds + c0 / kFp8Block;
  Raw8<T> v[kHeld];
#pragma unroll
  for (int g = 0; g < kHeld; ++g) v[g] = get8<VEC, kApart>(x + g * kUnit, left - g * kUnit);
#pragma unroll
  for (int g = 0; g < kHeld; ++g) {
    if (left - g * kUnit + run <= 0) break;  // the whole unit is past the row
    put_unit<VEC, kApart, true>(codes + g * kUnit, scales + g * 2, lane, left - g * kUnit, widen(v[g]));
  }
}

// One row by WPR warps, its kHeld units per warp in registers between the sum
// of squares and the scaling (rows up to WPR * kHeld * 256 columns).  Five CTAs
// an SM at 48 registers (norm m = 16384, k = 768 with an f16 residual: 27.1 us
// with four, 26.2 with five, 34.3 with six, which spill): the loads of one row
// overlap the arithmetic of the others.  With f32 rows and an f32 residual five
// spill too, 32 to 64 bytes a thread (33.4 us, 4.9 TB/s).
template <typename TX, typename TD, bool DELTA, bool VEC, int WPR>
__global__ void __launch_bounds__(32 * kWarps, 5) fp8_rmsnorm_kernel(const __grid_constant__ Fp8RowsParams p) {
  __shared__ float part[kWarps];
  pdl_wait();
  pdl_launch_next();
  constexpr int kStep = WPR * kUnit;  // columns between a warp's units
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wi = warp % WPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWarps / WPR) + warp / WPR;
  constexpr bool kApart = sizeof(TX) == 4;
  const int run = first_run<kApart>(lane), off = wi * kUnit + run;
  const int left0 = row < p.m ? static_cast<int>(p.k) - off : 0;  // columns from this lane's first element on
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx + off;
  const TD* d = DELTA ? static_cast<const TD*>(p.delta) + row * p.ldd + off : nullptr;
  Raw8<TX> rx[kHeld];
  Raw8<TD> rd[DELTA ? kHeld : 1];
#pragma unroll
  for (int g = 0; g < kHeld; ++g) {
    rx[g] = get8<VEC, kApart>(x + g * kStep, left0 - g * kStep);
    if constexpr (DELTA) rd[g] = get8<VEC, kApart>(d + g * kStep, left0 - g * kStep);
  }
  Eight v[kHeld];
  float ss = 0.f;
#pragma unroll
  for (int g = 0; g < kHeld; ++g) {
    v[g] = widen(rx[g]);
    if constexpr (DELTA) {
      const Eight e = widen(rd[g]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g].v[i] += e.v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[g].v[i] * v[g].v[i];
  }
  ss = warp_total(ss);
  if (WPR > 1) {
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) ss += part[warp / WPR * WPR + i];
  }
  if (row >= p.m) return;
  const float inv = __frcp_rn(sqrtf(ss / static_cast<float>(p.k) + p.eps));
  TX* sum = DELTA ? static_cast<TX*>(p.sum) + row * p.ldsum + off : nullptr;
  uint8_t* codes = p.codes + row * p.ldc + off;
  float* scales = p.scales + row * p.lds + off / kFp8Block;
#pragma unroll
  for (int g = 0; g < kHeld; ++g) {
    const int left = left0 - g * kStep;
    if (left + run <= 0) break;  // the whole unit is past the row
    if (DELTA) put8<VEC, kApart>(sum + g * kStep, left, v[g]);
    const Eight w = widen(get8<VEC, kApart>(p.w + off + g * kStep, left));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[g].v[i] *= inv * w.v[i];
    put_unit<VEC, kApart, false>(codes + g * kStep, scales + g * (kStep / kFp8Block), lane, left, v[g]);
  }
}

// A row wider than the registers of a CTA: read twice, the second time from L2.
template <typename TX, typename TD, bool DELTA, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) fp8_rmsnorm_wide_kernel(const __grid_constant__ Fp8RowsParams p) {
  __shared__ float part[kWarps];
  pdl_wait();
  pdl_launch_next();
  constexpr int kStep = kWarps * kUnit;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr bool kApart = sizeof(TX) == 4;
  const int off = warp * kUnit + first_run<kApart>(lane), k = static_cast<int>(p.k);
  const int64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx + off;
  const TD* d = DELTA ? static_cast<const TD*>(p.delta) + row * p.ldd + off : nullptr;
  auto value = [&](int c) {
    Eight v = widen(get8<VEC, kApart>(x + c, k - off - c));
    if constexpr (DELTA) {
      const Eight e = widen(get8<VEC, kApart>(d + c, k - off - c));
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] += e.v[i];
    }
    return v;
  };
  float ss = 0.f;
#pragma unroll 2
  for (int c = 0; c < k; c += kStep) {
    const Eight v = value(c);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v.v[i] * v.v[i];
  }
  ss = warp_total(ss);
  if (lane == 0) part[warp] = ss;
  __syncthreads();
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) ss += part[i];
  const float inv = __frcp_rn(sqrtf(ss / static_cast<float>(k) + p.eps));
  TX* sum = DELTA ? static_cast<TX*>(p.sum) + row * p.ldsum + off : nullptr;
#pragma unroll 2
  for (int c = 0; c < k - warp * kUnit; c += kStep) {
    const int left = k - off - c;
    Eight v = value(c);
    if (DELTA) put8<VEC, kApart>(sum + c, left, v);
    const Eight w = widen(get8<VEC, kApart>(p.w + off + c, left));
#pragma unroll
    for (int i = 0; i < 8; ++i) v.v[i] *= inv * w.v[i];
    put_unit<VEC, kApart, false>(p.codes + row * p.ldc + off + c, p.scales + row * p.lds + (off + c) / kFp8Block, lane, left, v);
  }
}

// One CTA per 128 x 128 block, eight elements of eight rows per thread.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) fp8_weight_kernel(const __grid_constant__ Fp8RowsParams p, int kblocks) {
  __shared__ float part[kWarps];
  pdl_wait();
  pdl_launch_next();
  constexpr bool kApart = sizeof(T) == 4;
  constexpr int kTurns = kFp8Block / (2 * kWarps);  // a warp takes two rows at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t nb = blockIdx.x / kblocks, kb = blockIdx.x % kblocks;
  const int64_t row0 = nb * kFp8Block + warp * 2 + (lane >> 4), col = kb * kFp8Block + first_run<kApart>(lane & 15);
  const int left = static_cast<int>(p.k - col);
  const T* x = static_cast<const T*>(p.x) + row0 * p.ldx + col;
  Raw8<T> v[kTurns];
#pragma unroll
  for (int t = 0; t < kTurns; ++t)
    v[t] = get8<VEC, kApart>(x + 2 * kWarps * t * p.ldx, row0 + 2 * kWarps * t < p.m ? left : 0);
  float a = 0.f;
#pragma unroll
  for (int t = 0; t < kTurns; ++t) a = max_nan(a, max_abs(widen(v[t])));
  a = warp_max_nan(a);
  if (lane == 0) part[warp] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) a = max_nan(a, part[i]);
  const float s = fp8_scale(a), f = fp8_factor(s);
  if (threadIdx.x == 0) p.scales[nb * p.lds + kb] = s;
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const int64_t row = row0 + 2 * kWarps * t;
    if (row < p.m) put_codes8<VEC, kApart, true>(p.codes + row * p.ldc + col, left, widen(v[t]), s, f);
  }
}

// Grid of at most 2^31 - 1 CTAs.
bool grid_of(int64_t n, dim3* g) {
  if (n < 1 || n > 0x7FFFFFFF) return false;
  *g = dim3(static_cast<unsigned>(n));
  return true;
}

template <typename TX, typename TD, bool DELTA, bool VEC>
cudaError_t rmsnorm(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t units = (p.k + kUnit - 1) / kUnit;
  auto go = [&](auto kernel, int wpr) {
    dim3 grid;
    if (!grid_of((p.m + kWarps / wpr - 1) / (kWarps / wpr), &grid)) return cudaErrorInvalidValue;
    return launch_pdl(kernel, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p);
  };
  if (units <= kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 1>, 1);
  if (units <= 2 * kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 2>, 2);
  if (units <= 4 * kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 4>, 4);
  if (units <= 8 * kHeld) return go(fp8_rmsnorm_kernel<TX, TD, DELTA, VEC, 8>, 8);
  return go(fp8_rmsnorm_wide_kernel<TX, TD, DELTA, VEC>, 8);
}

template <typename TX, typename TD, bool DELTA>
cudaError_t rmsnorm_v(const Fp8RowsParams& p, cudaStream_t st) {
  const bool vec = p.vec_x && p.vec_w && (!DELTA || (p.vec_d && p.vec_s)) && p.k % 8 == 0;
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
  const int64_t groups = (p.k + kHeld * kUnit - 1) / (kHeld * kUnit);
  dim3 grid;
  if (groups > 0x7FFFFFFF || !grid_of((p.m * groups + kWarps - 1) / kWarps, &grid)) return cudaErrorInvalidValue;
  auto kernel = p.vec_x && p.k % 8 == 0 ? fp8_rows_kernel<T, true> : fp8_rows_kernel<T, false>;
  return launch_pdl(kernel, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p, static_cast<int>(groups));
}

template <typename T>
cudaError_t weight(const Fp8RowsParams& p, cudaStream_t st) {
  const int64_t kb = (p.k + kFp8Block - 1) / kFp8Block, nb = (p.m + kFp8Block - 1) / kFp8Block;
  dim3 grid;
  if (kb > 0x7FFFFFFF || !grid_of(kb * nb, &grid)) return cudaErrorInvalidValue;
  auto kernel = p.vec_x && p.k % 8 == 0 ? fp8_weight_kernel<T, true> : fp8_weight_kernel<T, false>;
  return launch_pdl(kernel, grid, dim3(32 * kWarps), 0, st, nullptr, 0, p, static_cast<int>(kb));
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
