// Shared by the 8-bit operators (fp8_rows.cu, fp8_gemm.cu): element types,
// the e4m3 conversion and the scale of a block.
#pragma once

#include <type_traits>
#include "common.cuh"

#include "../../include/wc_fp8.h"

namespace wc {

constexpr int kFp8Block = 128;      // columns (and weight rows) that share a scale
constexpr float kE4M3Max = 448.0f;  // largest finite e4m3 value

// The scale of a block whose largest magnitude is amax (NaN stays NaN): the
// product with 1 / 448 corrected by its remainder, which is the rounded quotient
// for every fraction of amax.  The floor keeps the reciprocal finite; a block of zeros
// gets codes of zero.
__device__ __forceinline__ float fp8_scale(float amax) {
  constexpr float c = 1.0f / kE4M3Max;
  float s = amax * c;
  if (amax < 3.0e38f) s = __fmaf_rn(__fmaf_rn(-kE4M3Max, s, amax), c, s);  // (not inf - inf)
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
// What the block's values are multiplied by: 1 / scale, the approximate
// reciprocal after one Newton step.  scale = inf: 0, so that finite values
// become 0 * inf and infinite ones NaN codes.
__device__ __forceinline__ float fp8_factor(float scale) {
  const float f = __fdividef(1.0f, scale);
  return f == 0.0f ? 0.0f : __fmaf_rn(__fmaf_rn(-scale, f, 1.0f), f, f);
}

// x / s and y / s, f = 1 / s: the product with f corrected by its remainder
// (Markstein's step), so the code is that of the rounded quotient and a tie
// between two codes stays one.  (With the product alone, one code in 10^5 of
// 16-bit values, and a few in 10^7 of f32 ones, is the other neighbour of a tie.)
// TWO: by packed instructions, which want the values in register pairs.
template <bool TWO>
__device__ __forceinline__ float2 quotients(float x, float y, float s, float f) {
  float2 q;
  if constexpr (TWO) {
    asm("{\n\t.reg .b64 v, s, f, q, r;\n\t"
        "mov.b64 v, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\tmov.b64 f, {%5, %5};\n\t"
        "mul.rn.f32x2 q, v, f;\n\tfma.rn.f32x2 r, q, s, v;\n\tfma.rn.f32x2 q, r, f, q;\n\t"
        "mov.b64 {%0, %1}, q;\n\t}"
        : "=f"(q.x), "=f"(q.y)
        : "f"(x), "f"(y), "f"(-s), "f"(f));
  } else {
    q = make_float2(x * f, y * f);
    q.x = __fmaf_rn(__fmaf_rn(-q.x, s, x), f, q.x);
    q.y = __fmaf_rn(__fmaf_rn(-q.y, s, y), f, q.y);
  }
  return q;
}

// Maximum that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Largest magnitude of three, keeping a NaN.
__device__ __forceinline__ float max_abs3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// max_nan over the warp, in every lane.
__device__ __forceinline__ float warp_max_nan(float v) {
  float d;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}

// Four f32 -> four e4m3 bytes (first in the low byte), nearest even, saturating.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// Codes of four values over their scale s, f = 1 / s.
template <bool TWO>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float s, float f) {
  const float2 q = quotients<TWO>(a, b, s, f), r = quotients<TWO>(c, d, s, f);
  return pack_e4m3x4(q.x, q.y, r.x, r.y);
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Four consecutive elements at p (of a row with `left` elements from p on),
// zeros past the row's end, first as loaded and then as f32, so that many loads
// are on their way before the first is used.  Rows may start at any element.
template <typename T>
struct Raw4 {
  uint32_t w[4];  // 16-bit: four elements in two words, or one in each
  bool whole = false;
  __device__ __forceinline__ void load(const T* p, int64_t left) {
    whole = left >= 4 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
    if (whole) {
      if constexpr (sizeof(T) == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
      }
    } else {
      using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
      const Bits* e = reinterpret_cast<const Bits*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = left > i ? e[i] : 0u;
    }
  }
  __device__ __forceinline__ float4 value() const {
    if constexpr (sizeof(T) == 4) {
      return make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
      const uint2 u = whole ? make_uint2(w[0], w[1]) : make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
      const T* e = reinterpret_cast<const T*>(&u);
      return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
    }
  }
};
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, float4 v) {
  if (left >= 4 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = v;
    } else {
      const T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    }
    return;
  }
  if (left > 0) p[0] = from_f32<T>(v.x);
  if (left > 1) p[1] = from_f32<T>(v.y);
  if (left > 2) p[2] = from_f32<T>(v.z);
  if (left > 3) p[3] = from_f32<T>(v.w);
}
// Four code bytes at p (4-byte aligned) of a row with `left` columns from p on.
__device__ __forceinline__ void store_codes4(uint8_t* p, int64_t left, uint32_t c) {
  if (left >= 4) {
    *reinterpret_cast<uint32_t*>(p) = c;
    return;
  }
  for (int i = 0; i < 3; ++i)
    if (left > i) p[i] = static_cast<uint8_t>(c >> (8 * i));
}

}  // namespace wc
