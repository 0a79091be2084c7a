// 8-bit products on the tensor cores (tcgen05 kind::f8f6f4), 128-row tiles.
//
//   y[m][n] = sum_b sa[m][b] sw[n / 128][b] P_b[m][n],
//   P_b[m][n] = sum over the 128 columns k of block b of qa[m][k] qw[n][k]
//
// The scales change with every block of 128 columns, so the tensor core's
// accumulator cannot run over the whole of K: each block's P_b goes to one of
// two TMEM buffers, and the epilogue warps add scale * P_b to sums that they
// keep in registers (one multiply-add per element and block, packed in
// pairs) while the tensor core fills the other buffer.
//
// Tile: 128 rows x 256 columns.  A thread of the epilogue owns one row (a
// TMEM lane) and 128 columns, so its row scale is one register and the weight
// scale of its columns one value per block.  For the gated product the 256
// columns are 64 gate, the same 64 up, the next 64 gate and up features, so a
// thread holds both factors of its 64 results.
//
// Warps (384 threads):
//   0      TMA producer: 128 rows of codes and 256 weight rows per block,
//          128-byte swizzle, ring of kStages
//   1      TMEM allocation, MMA issue (one thread)
//   4-11   epilogue: warp w reads TMEM lanes 32 (w % 4).., columns
//          128 (w / 4 - 1)..
#include "fp8.cuh"
#include "fp8_gemm.h"

#include <algorithm>
#include <mutex>

namespace wc {

namespace {

constexpr int kBM = 128;
constexpr int kBN = 256;
constexpr int kStages = 4;
constexpr int kABytes = kBM * kFp8Block;
constexpr int kBBytes = kBN * kFp8Block;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kStageOutBytes = 32 * 128;  // one warp's 32 rows x 32 f32 on the way out
constexpr int kOffOut = kStages * kStageBytes;
constexpr int kOffAmax = kOffOut + 8 * kStageOutBytes;
constexpr int kOffBar = kOffAmax + 2 * kBM * 4;
constexpr int kSmem = 1024 + kOffBar + 256;
static_assert(kSmem <= 232448, "dynamic shared memory per block");
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;  // two 256-column partials

__device__ uint32_t g_fp8_status;  // wait timeouts of launches without a status word of their own

// D[tmem] (+)= A[smem] . B[smem]^T for 8-bit floats, f32 accumulate, one CTA.
__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor for kind::f8f6f4 with e4m3 A and B (format 0), f32
// D, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// 32 lanes x 32 columns of f32: issue, and wait for everything issued.  The
// wait takes the registers so that no use of them can move before it.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld32_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// act(g) u, both activations in the form g / (1 + exp(-z)): z = g (SiLU), or
// z = 2 sqrt(2 / pi) (g + 0.044715 g^3), since (1 + tanh(z / 2)) / 2 =
// 1 / (1 + exp(-z)).  exp and the quotient are the fast f32 ones (a few ulp):
// the 11-bit hardware tanh would show in the f32 scales of 8-bit rows.
__device__ __forceinline__ float gate(float g, float u, int act) {
  const float z = act == WC_ACT_SILU ? g : 1.5957691216f * (g + 0.044715f * g * g * g);
  return g * __frcp_rn(1.0f + __expf(-z)) * u;
}

template <bool GATED, typename OutT>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmU, const __grid_constant__ Fp8GemmParams p) {
  constexpr bool kCodes = sizeof(OutT) == 1;  // 8-bit rows out (gated)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kOffBar);  // [kStages] operands landed
  uint64_t* empty = full + kStages;                              // [kStages] MMA done with them
  uint64_t* acc_full = empty + kStages;                          // [2] partial ready
  uint64_t* acc_empty = acc_full + 2;                            // [2] partial read by the 8 epilogue warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* status = p.status ? p.status : &g_fp8_status;

  constexpr int kFeat = GATED ? kBN / 2 : kBN;  // output columns per tile
  const int kblocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int m_tiles = (p.m + kBM - 1) / kBM, n_tiles = (p.n + kFeat - 1) / kFeat;
  const int64_t tiles = static_cast<int64_t>(m_tiles) * n_tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    if (GATED) tma_prefetch_desc(&tmU);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_next();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t i = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        const int m0 = static_cast<int>(tile / n_tiles) * kBM, f0 = static_cast<int>(tile % n_tiles) * kFeat;
        for (int kb = 0; kb < kblocks; ++kb, ++i) {
          const uint32_t s = i % kStages;
          if (!(ok = mbar_wait(&empty[s], ((i / kStages) & 1) ^ 1, status))) break;
          mbar_arrive_expect_tx(&full[s], kStageBytes);
          uint8_t* sa = smem + s * kStageBytes;
          tma_load_2d(sa, &tmA, &full[s], kb * kFp8Block, m0);
#pragma unroll
          for (int c = 0; c < 4; ++c)  // 64 weight rows each
            tma_load_2d(sa + kABytes + c * 64 * kFp8Block, GATED && (c & 1) ? &tmU : &tmW, &full[s], kb * kFp8Block,
                        GATED ? f0 + (c >> 1) * 64 : f0 + c * 64);
        }
      }
      // After a timeout the loads already issued still land in this CTA's
      // shared memory: wait for them before it exits.
      if (!ok)
        for (uint32_t j = i > kStages ? i - kStages : 0; j < i; ++j)
          mbar_wait(&full[j % kStages], (j / kStages) & 1, status);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3_f32(kBM, kBN);
      uint32_t i = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < kblocks; ++kb, ++i) {
          const uint32_t s = i % kStages, buf = i & 1;
          ok = mbar_wait(&acc_empty[buf], ((i >> 1) & 1) ^ 1, status) &&
               mbar_wait(&full[s], (i / kStages) & 1, status);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * kStageBytes);
          const uint64_t adesc = sw128_kmajor_desc(sa), bdesc = sw128_kmajor_desc(sa + kABytes);
#pragma unroll
          for (int k = 0; k < kFp8Block / 32; ++k)
            tc_mma_f8(tmem_base + buf * kBN, adesc + 2 * k, bdesc + 2 * k, idesc, k > 0 ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(&acc_full[buf]);
        }
      }
    }
  } else if (warp >= 4) {
    const int q = warp & 3, h = (warp >> 2) - 1;  // TMEM lane quarter, column half
    uint8_t* stage = smem + kOffOut + (warp - 4) * kStageOutBytes;
    float* amax = reinterpret_cast<float*>(smem + kOffAmax);  // [half][row of the tile]
    const uint32_t tlane = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * 128;
    uint32_t i = 0;
    bool ok = true;
    for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      const int m0 = static_cast<int>(tile / n_tiles) * kBM, f0 = static_cast<int>(tile % n_tiles) * kFeat;
      const int row = m0 + q * 32 + lane;
      const int nb = GATED ? f0 / kFp8Block : f0 / kFp8Block + h;  // block of weight rows
      const bool live = row < p.m && nb * kFp8Block < p.n;
      const float* sa = p.sa + row * p.ldsa;
      const float* sw = p.sw + nb * p.ldsw;
      const float* sup = GATED ? p.sup + nb * p.ldsup : nullptr;
      uint64_t acc[64];  // 128 columns in pairs
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0ull;
      for (int kb = 0; kb < kblocks; ++kb, ++i) {
        const uint32_t buf = i & 1;
        float s0 = 0.f, s1 = 0.f;
        if (live) {
          const float a = sa[kb];
          s0 = a * sw[kb];
          s1 = GATED ? a * sup[kb] : s0;
        }
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[buf], (i >> 1) & 1, status));
        if (!ok) break;
        tc_fence_after();
        uint32_t r[2][32];
        tmem_ld32_issue(tlane + buf * kBN, r[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld32_wait(r[c & 1]);
          if (c < 3) {
            tmem_ld32_issue(tlane + buf * kBN + 32 * (c + 1), r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          }
          const float s = c < 2 ? s0 : s1;
          const uint64_t ss = f2(s, s);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[16 * c + j] = f2_fma((static_cast<uint64_t>(r[c & 1][2 * j + 1]) << 32) | r[c & 1][2 * j], ss,
                                     acc[16 * c + j]);
        }
      }
      if (!ok) break;

      if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          acc[j] = f2(gate(f2_lo(acc[j]), f2_lo(acc[32 + j]), p.act), gate(f2_hi(acc[j]), f2_hi(acc[32 + j]), p.act));
      }
      const int col0 = f0 + h * (GATED ? 64 : 128);  // the thread's first output column
      if constexpr (kCodes) {
        // The 64 results of this thread and those of the thread with the same
        // row in the other half are one block of 128.
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) a = max_nan(a, max_nan(fabsf(f2_lo(acc[j])), fabsf(f2_hi(acc[j]))));
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the tile before has read its maxima
        amax[h * kBM + q * 32 + lane] = a;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float sc = fp8_scale(max_nan(a, amax[(h ^ 1) * kBM + q * 32 + lane])), fac = fp8_factor(sc);
        if (row < p.m) {
          if (h == 0) p.out_scales[row * p.ldos + nb] = sc;
          uint8_t* o = static_cast<uint8_t*>(p.out) + row * p.ldo + col0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // 16 codes
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack_e4m3x4(f2_lo(acc[8 * c + 2 * e]) * fac, f2_hi(acc[8 * c + 2 * e]) * fac,
                                 f2_lo(acc[8 * c + 2 * e + 1]) * fac, f2_hi(acc[8 * c + 2 * e + 1]) * fac);
            const int left = p.n - col0 - 16 * c;
            if (left >= 16) {
              *reinterpret_cast<uint4*>(o + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) store_codes4(o + 16 * c + 4 * e, left - 4 * e, w[e]);
            }
          }
        }
      } else {
        // 32 columns at a time through shared memory, so that eight lanes
        // write 32 consecutive elements of a row.
        OutT* out = static_cast<OutT*>(p.out);
        const OutT* res = static_cast<const OutT*>(p.residual);
        const int cc = lane & 7, r0 = m0 + q * 32 + (lane >> 3);
#pragma unroll
        for (int c = 0; c < (GATED ? 2 : 4); ++c) {
          const int col = col0 + 32 * c + 4 * cc;
          float4 rv[8];
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const int64_t rr = r0 + 4 * t;
            rv[t] = res ? load4(res + rr * p.ldr + col, rr < p.m ? p.n - col : 0, p.vec_r)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint64_t lo = acc[16 * c + 2 * j], hi = acc[16 * c + 2 * j + 1];
            *reinterpret_cast<ulonglong2*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_ulonglong2(lo, hi);
          }
          __syncwarp();
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const int lr = (lane >> 3) + 4 * t;
            const int64_t rr = r0 + 4 * t;
            float4 v = *reinterpret_cast<const float4*>(stage + lr * 128 + ((cc ^ (lr & 7)) << 4));
            v.x += rv[t].x;
            v.y += rv[t].y;
            v.z += rv[t].z;
            v.w += rv[t].w;
            store4(out + rr * p.ldo + col, rr < p.m ? p.n - col : 0, p.vec_o, v);
          }
        }
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// Codes [rows][ld] of which k columns are read: box 128 x box_rows, 128-byte
// swizzle, zeros outside.
bool codes_map(CUtensorMap* m, const uint8_t* ptr, int64_t rows, int64_t k, int64_t ld, uint32_t box_rows) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {kFp8Block, box_rows};
  cuuint32_t es[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(ptr), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GATED, typename OutT>
cudaError_t launch(const Fp8GemmParams& p, int num_sms, cudaStream_t st) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!attr_set[dev]) {
    e = cudaFuncSetAttribute(fp8_gemm_kernel<GATED, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  CUtensorMap ta, tw, tu;
  if (!codes_map(&ta, p.a, p.m, p.k, p.lda, kBM) || !codes_map(&tw, p.w, p.n, p.k, p.ldw, 64) ||
      !codes_map(&tu, GATED ? p.up : p.w, p.n, p.k, GATED ? p.ldup : p.ldw, 64))
    return cudaErrorInvalidValue;
  constexpr int kFeat = GATED ? kBN / 2 : kBN;
  const int64_t tiles = static_cast<int64_t>((p.m + kBM - 1) / kBM) * ((p.n + kFeat - 1) / kFeat);
  const int grid = static_cast<int>(std::min<int64_t>(tiles, num_sms));
  return launch_pdl(fp8_gemm_kernel<GATED, OutT>, dim3(grid), dim3(kThreads), kSmem, st, nullptr, 0, ta, tw, tu, p);
}

}  // namespace

cudaError_t fp8_gemm_launch(bool gated, int out_type, const Fp8GemmParams& p, int num_sms, cudaStream_t st) {
  if (gated) {
    switch (out_type) {
      case WC_T_F32: return launch<true, float>(p, num_sms, st);
      case WC_T_F16: return launch<true, __half>(p, num_sms, st);
      case WC_T_BF16: return launch<true, __nv_bfloat16>(p, num_sms, st);
      case WC_T_E4M3: return launch<true, uint8_t>(p, num_sms, st);
      default: return cudaErrorInvalidValue;
    }
  }
  switch (out_type) {
    case WC_T_F32: return launch<false, float>(p, num_sms, st);
    case WC_T_F16: return launch<false, __half>(p, num_sms, st);
    case WC_T_BF16: return launch<false, __nv_bfloat16>(p, num_sms, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t fp8_gemm_take_status(uint32_t* status) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_fp8_status, sizeof(uint32_t));
  if (e != cudaSuccess || *status == 0) return e;
  const uint32_t zero = 0;
  return cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof(zero));
}

}  // namespace wc
