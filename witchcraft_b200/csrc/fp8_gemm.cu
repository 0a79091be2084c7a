// 8-bit products on the tensor cores (tcgen05 kind::f8f6f4).
//
//   y[m][n] = sum_b sa[m][b] sw[n / 128][b] P_b[m][n],
//   P_b[m][n] = sum over the 128 columns k of block b of qa[m][k] qw[n][k]
//
// The scales change with every block of 128 columns, so the tensor core's
// accumulator cannot run over the whole of K: each block's P_b goes to one of
// a few TMEM buffers, and the epilogue warps add scale * P_b to sums that they
// keep in registers (one multiply-add per element and block) while the tensor
// core fills the next buffer.  A thread of the epilogue owns
// one row (a TMEM lane) and half of the tile's columns, so its row scale is
// one register and the weight scale of its columns one value per block.
// For the gated product the 256 columns of a tile are 64 gate features, the
// same 64 up features, the next 64 gate and the next 64 up: a thread holds
// both factors of its 64 results.
//
// Two kernels:
//   fp8_pair_kernel  many rows: persistent, 256 x 256 tiles on pairs of SMs,
//                    results from registers through a small staging buffer
//   fp8_tile_kernel  few rows: one 128-row tile per CTA or, with K split, per
//                    cluster, whose CTAs join their sums through distributed
//                    shared memory in rank order
//
// What bounds them (device time, inputs from DRAM).  Many rows: the epilogue
// warps, which both add up the partials and finish the tile before.  8192 x 4096
// x 8192, f16: 240 to 270 us, 2.0 to 2.3 PFLOP/s as the clock under power
// allows; 2048 x 4096 x 4096: 33.5 us, 28.3 if the tensor core could sum all of
// K (no scales).  Gated 16384 x 768 x 2048 to 8-bit rows: 68 to 76 us, where the
// tensor pipe works 35 % and the schedulers issue 57 % of the time.  Few rows:
// latency (32 x 768 x 2304: 4.2 us, of which 1 is a launch that does nothing much), and
// for one row of 4096 x 12288 the 96 CTAs (of 148 SMs) that its tiles make,
// 12.9 us or 3.9 TB/s of weights.
//
// Warps of both (384 threads):
//   0      TMA producer, 128-byte swizzle, ring of operand stages
//   1      TMEM allocation, MMA issue (one thread; of the even CTA of a pair)
//   4-11   epilogue: warp w reads TMEM lanes 32 (w % 4).., and the column
//          half w / 4 - 1
// Registers: 168 a thread at launch; the first four warps give back all but
// 56 and the epilogue takes 224 (4 x 32 x 56 + 8 x 32 x 224 = 384 x 168).
#include "cluster.cuh"
#include "fp8.cuh"
#include "fp8_gemm.h"
#include "fp8_span.h"

#include <algorithm>
#include <atomic>
#include <mutex>

namespace wc {

namespace {

constexpr int kRows = 128;      // rows of a CTA's tile (TMEM lanes)
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr int kABytes = kRows * kFp8Block;

__device__ uint32_t g_fp8_status;  // wait timeouts

// Instruction descriptor for kind::f8f6f4 with e4m3 A and B (format 0), f32
// D, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// D[tmem] (+)= A[smem] . B[smem]^T for 8-bit floats, f32 accumulate.
template <bool PAIR>
__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}

// Waits for a barrier of the operand ring or of the partials: on pairs of SMs the
// other CTA's loads, its epilogue or the even CTA's MMAs arrive there.
template <bool PAIR>
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
  if constexpr (PAIR)
    return mbar_wait_cluster_relaxed(bar, parity, status);
  else
    return mbar_wait(bar, parity, status);
}

// The MMA warp's loop over `steps` blocks: STAGES operand stages of
// STAGE_BYTES (A, then B) and BUFS partials of BN columns.  The whole warp
// runs it and one lane issues, so that descriptors stay in uniform registers:
// the warp shares its scheduler with two epilogue warps that are busy with
// multiply-adds, and every instruction in this loop is slow.
template <bool PAIR, int STAGES, int STAGE_BYTES, int B_OFFSET, int BUFS, int BN, typename Commit>
__device__ __forceinline__ void mma_loop(uint32_t tmem, uint32_t idesc, uint32_t smem, uint64_t* full, uint64_t* done,
                                         uint64_t* acc_empty, uint32_t steps, uint32_t* status, Commit commit) {
  const uint64_t a0 = sw128_kmajor_desc(smem), b0 = sw128_kmajor_desc(smem + B_OFFSET);
  uint32_t s = 0, round = 0;
#pragma unroll 1
  for (uint32_t i = 0; i < steps; ++i) {
    const uint32_t buf = i % BUFS;
    const bool ok =
        ring_wait<PAIR>(&full[s], round & 1, status) && ring_wait<PAIR>(&acc_empty[buf], ((i / BUFS) & 1) ^ 1, status);
    if (!__all_sync(0xFFFFFFFFu, ok)) return;  // one way out for the whole warp
    if (PAIR) acquire_cluster_shared();  // operands
    tc_fence_after();
    const uint64_t a = a0 + s * (STAGE_BYTES >> 4), b = b0 + s * (STAGE_BYTES >> 4);
    const uint32_t d = tmem + buf * BN;
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < kFp8Block / 32; ++k) tc_mma_f8<PAIR>(d, a + 2 * k, b + 2 * k, idesc, k > 0 ? 1u : 0u);
      commit(&done[s]);
    }
    __syncwarp();
    if (++s == STAGES) {
      s = 0;
      ++round;
    }
  }
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

// The scales of one thread's row and columns, fetched one block ahead of
// their use.  The loads are volatile, or the compiler moves them down to it;
// the first one brings the next 64 scales of its row into L2.
// Rows and columns outside the matrix use the last ones' scales (their results
// are not stored).
struct Scales {
  const float *a, *w, *u;  // the row's, the columns', the up columns' next scale
  float va, vw, vu;
};
__device__ __forceinline__ float load_ahead(const float* p) {
  float v;
  asm volatile("ld.global.nc.L2::256B.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
template <bool GATED>
__device__ __forceinline__ void fetch_scales(Scales& s, int step) {
  s.va = load_ahead(s.a);
  s.vw = load_ahead(s.w);
  s.a += step;
  s.w += step;
  if (GATED) {
    s.vu = load_ahead(s.u);
    s.u += step;
  }
}
template <bool GATED>
__device__ __forceinline__ Scales scales_at(const Fp8GemmParams& p, int row, int nb, int kb) {
  row = min(row, p.m - 1);
  nb = min(nb, (p.n - 1) / kFp8Block);
  Scales s{};
  s.a = p.sa + row * p.ldsa + kb;
  s.w = p.sw + nb * p.ldsw + kb;
  if (GATED) s.u = p.sup + nb * p.ldsup + kb;
  return s;
}

// Position in the ring of operand stages, whose `done` barriers also say that
// a block's partial is complete.
template <int STAGES>
struct Ring {
  uint32_t i = 0, stage = 0, parity = 0;  // blocks so far, and where the next one is
  __device__ __forceinline__ void next() {
    ++i;
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
  }
};

// acc[] = sum over `blocks` (>= 1) blocks, `step` apart, of scale * partial for
// this thread's row and 32 CHUNKS columns (taddr of partial 0; the others lie
// BN columns apart).  sc holds the first block's scales.  The columns come 32 at
// a time, the next 32 loading while these are added.  The multiply-adds are
// scalar: the packed form needs register pairs that a TMEM load's results have
// to be moved into.  What matters most here is that nothing spills: keeping
// the next block's first columns in flight across the loop's end made the
// whole product twice as slow.  `read(buf)` once a partial is in registers.
// False if a wait ran out.
template <bool PAIR, bool GATED, int CHUNKS, int STAGES, int BUFS, int BN, typename Read>
__device__ __forceinline__ bool sum_blocks(float (&acc)[32 * CHUNKS], Scales& sc, int blocks, int step, uint32_t taddr,
                                           uint64_t* done, Ring<STAGES>& ring, uint32_t* status, Read read) {
  static_assert(CHUNKS == 2 || CHUNKS == 4, "two register sets");
  uint32_t r[2][32];
#pragma unroll
  for (int j = 0; j < 32 * CHUNKS; ++j) acc[j] = 0.f;
#pragma unroll 1
  for (int left = blocks; left > 0; --left) {
    const float s0 = sc.va * sc.vw, s1 = GATED ? sc.va * sc.vu : s0;
    if (left > 1) fetch_scales<GATED>(sc, step);
    if (!__all_sync(0xFFFFFFFFu, ring_wait<PAIR>(&done[ring.stage], ring.parity, status))) return false;
    tc_fence_after();
    const uint32_t at = taddr + ring.i % BUFS * BN;
    auto add = [&](int c) {
      const float s = 2 * c < CHUNKS ? s0 : s1;
#pragma unroll
      for (int e = 0; e < 32; ++e) acc[32 * c + e] = __fmaf_rn(__uint_as_float(r[c & 1][e]), s, acc[32 * c + e]);
    };
    tmem_ld32_issue(at, r[0]);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      tmem_ld32_wait(r[c & 1]);
      if (c + 1 < CHUNKS) {
        tmem_ld32_issue(at + 32 * (c + 1), r[(c + 1) & 1]);
      } else {
        tc_fence_before();
        __syncwarp();
        read(ring.i % BUFS);
      }
      add(c);
    }
    ring.next();
  }
  return true;
}

// act(g) u, both activations in the form g / (1 + exp(-z)): z = g (SiLU), or
// z = 2 sqrt(2 / pi) (g + 0.044715 g^3), since (1 + tanh(z / 2)) / 2 =
// 1 / (1 + exp(-z)).  So -z log2(e) = g (c1 + c3 g^2) with two constants, and
// the exponential and the quotient are the hardware's f32 approximations (a
// few ulp): its 11-bit tanh would show in the f32 scales of 8-bit rows.  g^2
// is kept finite so that SiLU's c3 = 0 does not meet an infinity.
struct Gate {
  float c1, c3;
  __device__ __forceinline__ explicit Gate(int act) {
    constexpr float log2e = 1.4426950409f;
    c1 = act == WC_ACT_SILU ? -log2e : -1.5957691216f * log2e;
    c3 = act == WC_ACT_SILU ? 0.0f : -1.5957691216f * 0.044715f * log2e;
  }
  __device__ __forceinline__ float operator()(float g, float u) const {
    const float z = g * __fmaf_rn(c3, fminf(g * g, 1e30f), c1);
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * r * u;
  }
};

__device__ __forceinline__ void regs_for_epilogue() { asm volatile("setmaxnreg.inc.sync.aligned.u32 224;"); }
__device__ __forceinline__ void regs_given_back() { asm volatile("setmaxnreg.dec.sync.aligned.u32 56;"); }

// After a wait ran out, the loads already issued still land in shared memory:
// wait (again with a limit) for the last `stages` of the `issued` ones.
__device__ __forceinline__ void drain_loads(uint64_t* full, uint32_t stages, uint32_t issued, uint32_t* status) {
  for (uint32_t j = issued > stages ? issued - stages : 0; j < issued; ++j)
    mbar_wait(&full[j % stages], (j / stages) & 1, status);
}

// 16 bytes of a row of results: from f32, and added to f32.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ uint4 make(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ void add(float* v, uint4 r) {
    v[0] += __uint_as_float(r.x);
    v[1] += __uint_as_float(r.y);
    v[2] += __uint_as_float(r.z);
    v[3] += __uint_as_float(r.w);
  }
};
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { return pack_f16x2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
struct Pack {
  static constexpr int kN = 8;
  static __device__ __forceinline__ uint4 make(const float* v) {
    return make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
  }
  static __device__ __forceinline__ void add(float* v, uint4 r) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += to_f32(e[i]);
  }
};

// ---------------------------------------------------------------- pairs of SMs

// A cluster of two CTAs owns a 256 x 256 tile.  Each CTA loads its own 128
// rows of A and the 128 weight rows of one column half; the even CTA's MMA
// thread multiplies from both CTAs' shared memory into both CTAs' TMEM (each
// its 128 rows x 256 columns).  Loads of both CTAs complete on the even CTA's
// barriers, MMA completion is committed to both, and the epilogue warps of
// both report to the even CTA that they have read a partial.
namespace pair {

constexpr int kBN = 256;
constexpr int kStageBytes = kABytes + 128 * kFp8Block;
constexpr int kBoxBytes = 32 * 128;  // 32 rows x 128 bytes of results (or of the residual)
constexpr int kPitch = kTurnRoom;    // of such a row that starts inside a block of 16 bytes

// Shared memory: operand stages, then boxes of results for each epilogue warp
// (a warp's results are four boxes of f32 or two of 16-bit values).
template <bool GATED, typename OutT, bool BOXES>
struct Plan {
  static constexpr bool kCodes = sizeof(OutT) == 1;  // 8-bit rows out (gated)
  static constexpr int kFeat = GATED ? kBN / 2 : kBN;                // output columns per tile
  static constexpr int kBoxCols = kCodes ? 64 : 128 / sizeof(OutT);  // columns of a box of results
  static constexpr int kBoxes = kFeat / 2 / kBoxCols;                // boxes of a warp
  // boxes it has room for: a third for f32, at the cost of a stage (16384 x 768
  // x 768 with residual: 30.0 -> 27.1 us, 16384 x 2048 x 768: 42.5 -> 40.9)
  static constexpr int kBufs = kBoxes > 2 || !BOXES ? 3 : 2;
  static constexpr int kStages = kBufs == 3 ? 4 : 5;
  static constexpr int kOffOut = kStages * kStageBytes;
  static constexpr int kOffBar = kOffOut + 8 * kBufs * kBoxBytes;
  // block maxima of 8-bit rows, in a second box: codes need only the first
  static constexpr int kOffAmax = kOffOut + kBoxBytes;
  static constexpr int kSmem = 1024 + kOffBar + 512;
  static_assert(BOXES || 2 * 32 * kPitch <= kBufs * kBoxBytes, "two turns of rows off the 16-byte boundary");
  static_assert(kSmem <= 232448, "dynamic shared memory per block");
  static_assert(2 * 2 * kRows * 4 <= kBoxBytes, "maxima of two tiles");
};

// Of the stores that a warp committed, how many may still be reading their room
// when box c of a tile is written into room c % bufs.  The rooms start over with
// every tile, so they are not used in turn across tiles: the first box waits for
// all that the tile before stored (a whole sum ago), and the boxes that reuse a
// room of their own tile for the one that was in it.  kAnyStores: no wait.
constexpr int kAnyStores = 1 << 20;
__host__ __device__ constexpr int stores_in_flight(int c, int bufs) {
  return c == 0 ? 0 : c < bufs ? kAnyStores : bufs - 1;
}
// Several tiles of `boxes` boxes, a store (and group) each: whether every box
// finds its room read.
constexpr bool rooms_are_read(int boxes, int bufs) {
  int last[8] = {-1, -1, -1, -1, -1, -1, -1, -1}, read = 0, committed = 0;  // groups [0, read) are known to be read
  for (int tile = 0; tile < 4; ++tile)
    for (int c = 0; c < boxes; ++c) {
      if (committed - stores_in_flight(c, bufs) > read) read = committed - stores_in_flight(c, bufs);
      if (last[c % bufs] >= read) return false;
      last[c % bufs] = committed++;
    }
  return true;
}
static_assert(rooms_are_read(1, 2) && rooms_are_read(4, 3), "plans whose boxes go one at a time");

__device__ __forceinline__ uint32_t load_shared(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 load_shared4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void store_shared(uint32_t at, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// BOXES: results (and the residual) move by TMA boxes, which wants rows that
// start at multiples of 16 bytes.  The way out for other rows would cost the
// kernel registers even where it is not taken (f32 results 45.8 -> 50.9 us at
// 16384 x 768 x 2304).
template <bool GATED, typename OutT, bool BOXES>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmU, const __grid_constant__ CUtensorMap tmOut,
                    const __grid_constant__ CUtensorMap tmRes, const __grid_constant__ Fp8GemmParams p) {
  using PL = Plan<GATED, OutT, BOXES>;
  constexpr bool kCodes = PL::kCodes;
  constexpr int kStages = PL::kStages, kFeat = PL::kFeat, kBoxCols = PL::kBoxCols, kBoxes = PL::kBoxes,
                kBufs = PL::kBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + PL::kOffBar);  // [kStages] even CTA: operands of both landed
  uint64_t* done = full + kStages;       // [kStages] each CTA: MMA done (stage free, partial ready)
  uint64_t* acc_empty = done + kStages;  // [2] even CTA: partial read by 16 epilogue warps
  uint64_t* res_full = acc_empty + 2;    // [8][kBoxes] each epilogue warp's boxes of the residual
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + 8 * kBoxes);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  uint32_t* status = &g_fp8_status;
  // a cluster is two neighbours of the grid; said with blockIdx, the compiler
  // knows that what follows from it is the same for the whole warp
  const int rank = blockIdx.x & 1;

  const int kblocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int m_tiles = (p.m + 2 * kRows - 1) / (2 * kRows), n_tiles = (p.n + kFeat - 1) / kFeat;
  const int tiles = m_tiles * n_tiles;
  const int tile0 = blockIdx.x >> 1, tile_step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&done[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&acc_empty[i], 16);
    for (int i = 0; i < 8 * kBoxes; ++i) mbar_init(&res_full[i], 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    if (GATED) tma_prefetch_desc(&tmU);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch_next();

  if (warp < 4) {
    regs_given_back();
    if (warp == 0 && lane == 0) {
      uint32_t i = 0;
      bool ok = true;
      for (int tile = tile0; tile < tiles && ok; tile += tile_step) {
        const int m0 = (tile / n_tiles) * 2 * kRows + rank * kRows;
        const int f0 = (tile % n_tiles) * kFeat + rank * (kFeat / 2);
        for (int kb = 0; kb < kblocks; ++kb, ++i) {
          const uint32_t s = i % kStages;
          if (!(ok = ring_wait<true>(&done[s], ((i / kStages) & 1) ^ 1, status))) break;
          acquire_cluster_shared();
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
          uint8_t* sa = smem + s * kStageBytes;
          const uint32_t bar = map_to_rank(&full[s], 0);
          tma_load_2d_pair(sa, &tmA, bar, kb * kFp8Block, m0);
          tma_load_2d_pair(sa + kABytes, &tmW, bar, kb * kFp8Block, f0);
          tma_load_2d_pair(sa + kABytes + 64 * kFp8Block, GATED ? &tmU : &tmW, bar, kb * kFp8Block,
                           GATED ? f0 : f0 + 64);
        }
      }
      // the odd CTA's loads complete on the even CTA's barriers; the cluster
      // barrier at the end holds it until the even CTA has waited
      if (!ok && rank == 0) drain_loads(full, kStages, i, status);
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t idesc = idesc_e4m3_f32(2 * kRows, kBN);
      const int mine = tiles > tile0 ? (tiles - tile0 + tile_step - 1) / tile_step : 0;
      mma_loop<true, kStages, kStageBytes, kABytes, 2, kBN>(tmem_base, idesc, smem_u32(smem), full, done, acc_empty,
                                                static_cast<uint32_t>(mine) * kblocks,
                                                status, [](uint64_t* b) { tc_commit_pair(b); });
    }
  } else {
    regs_for_epilogue();
    const int q = warp & 3, h = (warp >> 2) - 1;  // TMEM lane quarter, column half
    uint8_t* box = smem + PL::kOffOut + (warp - 4) * kBufs * kBoxBytes;
    float* amax = reinterpret_cast<float*>(smem + PL::kOffAmax);  // [tile parity][half][row of the tile]
    const uint32_t tlane = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * 128;
    const uint32_t empty0 = map_to_rank(&acc_empty[0], 0);
    // A tile's scales, the first block's on their way (past the last tile: the last one's).
    auto open_tile = [&](int tile) {
      tile = min(tile, tiles - 1);
      const int f0 = (tile % n_tiles) * kFeat;
      Scales s = scales_at<GATED>(
          p, (tile / n_tiles) * 2 * kRows + rank * kRows + q * 32 + lane,
          f0 / kFp8Block + (GATED ? 0 : h), 0);
      fetch_scales<GATED>(s, 1);
      return s;
    };
    // Boxes of the residual, each with a barrier of its own that is used once a
    // tile (so the tile's parity is the barrier's); what lies outside the matrix
    // arrives as zeros.
    const bool res_boxes = !kCodes && !GATED && BOXES && p.residual != nullptr;
    const bool res_rows = !kCodes && !GATED && !BOXES && p.residual != nullptr;
    uint64_t* res_bar = res_full + (warp - 4) * kBoxes;
    auto fetch_residual = [&](int c, int x, int y) {  // one lane; the box's room is not in use
      mbar_arrive_expect_tx(&res_bar[c], kBoxBytes);
      tma_load_2d(box + c % kBufs * kBoxBytes, &tmRes, &res_bar[c], x + c * kBoxCols, y);
    };
    Ring<kStages> ring;
    uint32_t turn = 0;  // tiles so far
    bool ok = true;
    Scales sc = open_tile(tile0);
    // 8-bit rows meet at a barrier once a tile: a warp whose wait ran out goes on
    // meeting the others there
    for (int tile = tile0; tile < tiles && (ok || kCodes); tile += tile_step) {
      const int m0 = (tile / n_tiles) * 2 * kRows + rank * kRows;
      const int f0 = (tile % n_tiles) * kFeat;
      const int row0 = m0 + q * 32, col0 = f0 + h * (kFeat / 2);  // this warp's first row and output column
      // the residual's first boxes, once the tile before has left them
      if (res_boxes && lane == 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
#pragma unroll
        for (int c = 0; c < kBoxes; ++c) {
          if (c < kBufs)
            fetch_residual(c, col0, row0);
          else  // on its way to L2 meanwhile
            asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(
                             reinterpret_cast<uint64_t>(&tmRes)),
                         "r"(col0 + c * kBoxCols), "r"(row0)
                         : "memory");
        }
      }
      // the same for rows off the 16-byte boundary: the 16-byte blocks that hold
      // 128 bytes of a row from its start's block on, a bulk copy per row (what a
      // block holds of other rows is not used, and what a block that reaches out
      // of the residual holds of it is read by elements)
      const int res_bytes = row0 + lane < p.m ? max(0, min(p.n - col0, kFeat / 2)) * static_cast<int>(sizeof(OutT)) : 0;
      auto residual_row = [&] {
        return static_cast<const OutT*>(p.residual) + static_cast<int64_t>(row0 + lane) * p.ldr + col0;
      };
      auto fetch_rows = [&](int t) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(residual_row());
        const OutT* base = static_cast<const OutT*>(p.residual);
        const ResidualSpan span =
            residual_span(reinterpret_cast<uintptr_t>(from), res_bytes, reinterpret_cast<uintptr_t>(base),
                          reinterpret_cast<uintptr_t>(base + static_cast<int64_t>(p.m - 1) * p.ldr + p.n), t);
        const int start = static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15);
        const int lo = span.lo, size = max(0, span.hi - span.lo);
        const uint32_t to = smem_u32(box) + (t % 2 * 32 + lane) * kPitch - t * kTurnBytes;
        auto elements = [&](int block) {
          using Bits = std::conditional_t<sizeof(OutT) == 4, uint32_t, uint16_t>;
#pragma unroll 1
          for (int at = max(block, start); at < min(block + 16, start + res_bytes); at += sizeof(OutT)) {
            const Bits v = *reinterpret_cast<const Bits*>(from - start + at);
            if constexpr (sizeof(OutT) == 4)
              store_shared(to + at, static_cast<uint32_t>(v));
            else
              asm volatile("st.shared.b16 [%0], %1;" ::"r"(to + at), "h"(v) : "memory");
          }
        };
        if (span.head) elements(0);
        if (span.tail) elements(span.last);
        const uint32_t sum = __reduce_add_sync(0xFFFFFFFFu, static_cast<uint32_t>(size));
        if (lane == 0) mbar_arrive_expect_tx(&res_bar[t], sum);
        __syncwarp();
        if (size > 0)
          asm volatile(
              "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                  to + lo),
              "l"(from - start + lo), "r"(size), "r"(smem_u32(&res_bar[t]))
              : "memory");
      };
      if (res_rows) {
        fence_proxy_async_smem();
        __syncwarp();
        fetch_rows(0);
        if (kBoxes > 1) fetch_rows(1);
        for (int c = 256; c < res_bytes; c += 128)  // on its way to L2 meanwhile
          asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(residual_row()) + c));
      }
      float acc[128];
      ok = ok && sum_blocks<true, GATED, 4, kStages, 2, kBN>(
          acc, sc, kblocks, 1, tlane, done, ring, status,
          [&](uint32_t buf) {
            if (lane == 0) mbar_arrive_remote_relaxed(empty0 + buf * 8);
          });
      if (!ok && !kCodes) break;
      sc = open_tile(tile + tile_step);  // arrives while this tile is written

      const int row = row0 + lane;
      if constexpr (GATED) {
        const Gate gate(p.act);
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = gate(acc[j], acc[64 + j]);
      }
      if constexpr (kCodes) {
        // The 64 results of this thread and those of the thread with the same
        // row in the other half are one block of 128 (without what lies past the
        // last feature: 0, or NaN where a scale is infinite).
        if (col0 + 64 > p.n) {
#pragma unroll
          for (int j = 0; j < 64; ++j) acc[j] = col0 + j < p.n ? acc[j] : 0.f;
        }
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 64; j += 2) a = max_abs3_nan(a, acc[j], acc[j + 1]);
        float* shared = amax + (turn & 1) * 2 * kRows;  // the tile before may still be reading its own
        shared[h * kRows + q * 32 + lane] = a;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float os = fp8_scale(max_nan(a, shared[(h ^ 1) * kRows + q * 32 + lane])), fac = fp8_factor(os);
        if (h == 0 && row < p.m) p.out_scales[row * p.ldos + f0 / kFp8Block] = os;
        uint4 code[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // 16 codes
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = codes4<true>(acc[16 * c + 4 * e], acc[16 * c + 4 * e + 1], acc[16 * c + 4 * e + 2],
                                acc[16 * c + 4 * e + 3], os, fac);
          code[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (col0 + 64 > p.n && p.n % 16 != 0) {
          // The rows end here inside 16 bytes, which a TMA store would write to
          // their end: each lane writes its own.
          if (row < p.m) {
            uint8_t* to = static_cast<uint8_t*>(p.out) + static_cast<int64_t>(row) * p.ldo + col0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int left = p.n - col0 - 16 * c;
              const uint32_t w[4] = {code[c].x, code[c].y, code[c].z, code[c].w};
              if (left >= 16) {
                *reinterpret_cast<uint4*>(to + 16 * c) = code[c];
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) store_codes4(to + 16 * c + 4 * e, left - 4 * e, w[e]);
              }
            }
          }
        } else {
          // 32 rows x 64 codes by one TMA store (64-byte swizzle)
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) = code[c];
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (col0 < p.n && row0 < p.m)
              asm volatile(
                  "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                      reinterpret_cast<uint64_t>(&tmOut)),
                  "r"(smem_u32(box)), "r"(col0), "r"(row0)
                  : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      } else {
        if constexpr (BOXES) {
          // Boxes of results: converted into shared memory (128-byte swizzle)
          // and written by TMA stores, which clip what lies outside.  Two of
          // two boxes go together, with one fence; of four, one at a time.
          constexpr int kN = Pack<OutT>::kN, kTogether = kBoxes == 2 ? 2 : 1;
          static_assert(kTogether == 2 ? kBoxes == 2 && kBufs >= 2 : rooms_are_read(kBoxes, kBufs), "");
#pragma unroll
          for (int c0 = 0; c0 < kBoxes; c0 += kTogether) {
            if (res_boxes) {
#pragma unroll
              for (int c = c0; c < c0 + kTogether; ++c)
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&res_bar[c], turn & 1, status)) && ok;
            } else {
              constexpr int kBack = kBufs - 1;
              if (lane == 0) {
                if (stores_in_flight(c0, kBufs) == 0)
                  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                else if (stores_in_flight(c0, kBufs) == kBack)
                  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBack) : "memory");
              }
              __syncwarp();
            }
#pragma unroll
            for (int c = c0; c < c0 + kTogether; ++c)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                uint4* at = reinterpret_cast<uint4*>(box + c % kBufs * kBoxBytes + lane * 128 + ((k ^ (lane & 7)) << 4));
                float* v = acc + c * kBoxCols + k * kN;
                if (res_boxes) Pack<OutT>::add(v, *at);
                *at = Pack<OutT>::make(v);
                // not the whole box of the residual in registers at once: it would spill
                if (sizeof(OutT) == 4 && (k & 1)) asm volatile("" ::: "memory");
              }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
#pragma unroll
              for (int c = c0; c < c0 + kTogether; ++c)
                if (col0 + c * kBoxCols < p.n && row0 < p.m)
                  asm volatile(
                      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                          reinterpret_cast<uint64_t>(&tmOut)),
                      "r"(smem_u32(box + c % kBufs * kBoxBytes)), "r"(col0 + c * kBoxCols), "r"(row0)
                      : "memory");
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              // the residual of a later box into the room of the one written before this
              if (kBoxes > kBufs && res_boxes && c0 >= 1 && c0 - 1 + kBufs < kBoxes) {
                asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                fetch_residual(c0 - 1 + kBufs, col0, row0);
              }
            }
          }
        } else {
          // Rows off the 16-byte boundary.  A lane lays its row out in shared
          // memory as it will lie in global memory, counted from the 16-byte
          // block in which the row starts (so a 16-bit row may begin inside a
          // word), 128 bytes at a time; then eight lanes write a row, whole
          // blocks as such, the blocks that it owns in part by elements.  The
          // words of a block are turned by one for every eight rows, which
          // would else share their banks.  16384 x 768 x 2302, f16: 46.2 us, with
          // residual 71.8 (2304 columns in boxes: 36.2 and 46.4); element by
          // element it was 77 and 301, by a bulk copy per row 72 and 102.
          constexpr int kSize = sizeof(OutT), kPer = 4 / kSize;
          OutT* out = static_cast<OutT*>(p.out);
          const int bytes = max(0, min(p.n - col0, kFeat / 2)) * kSize;  // of a row
          auto start_of = [](const OutT* at) { return static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15); };
          const int own_start = start_of(out + static_cast<int64_t>(row0 + lane) * p.ldo + col0);
          const uint32_t rows_of_warp = smem_u32(box);
          uint32_t word[4];  // where words 0 to 3 of the row go
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = (own_start >> 2) + i;
            word[i] = rows_of_warp + lane * kPitch + ((at & 4) + ((at + (lane >> 3)) & 3)) * 4;
          }
          uint4 carry = make_uint4(0u, 0u, 0u, 0u);  // what a turn leaves to the next
#pragma unroll
          for (int t = 0; t < kBoxes; ++t) {
            const uint32_t room = t % 2 * 32 * kPitch, rows_at = rows_of_warp + room, own = rows_at + lane * kPitch;
            const int lo = t * 128, hi = t + 1 < kBoxes ? lo + 128 : lo + kPitch;  // bytes of the rows in this turn
            if (res_rows) {
              ok = __all_sync(0xFFFFFFFFu, mbar_wait(&res_bar[t], turn & 1, status)) && ok;
              const int rs = start_of(residual_row());
              uint4 u = load_shared4(own);
#pragma unroll
              for (int c = 0; c < 8; ++c) {  // four words of the row, out of two blocks
                const uint4 next = load_shared4(own + 16 * c + 16);
                uint32_t w[8] = {u.x, u.y, u.z, u.w, next.x, next.y, next.z, next.w};
#pragma unroll
                for (int i = 0; i < 6; ++i) w[i] = rs & 8 ? w[i + 2] : w[i];
#pragma unroll
                for (int i = 0; i < 5; ++i) w[i] = rs & 4 ? w[i + 1] : w[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float* v = acc + (t * 32 + c * 4 + i) * kPer;
                  if constexpr (kPer == 1) {
                    v[0] += __uint_as_float(w[i]);
                  } else {
                    const uint32_t x = __funnelshift_r(w[i], w[i + 1], (rs & 2) * 8);
                    const OutT* e = reinterpret_cast<const OutT*>(&x);
                    v[0] += to_f32(e[0]);
                    v[1] += to_f32(e[1]);
                  }
                }
                u = next;
              }
            } else {
              __syncwarp();
            }
            if (t > 0) store_shared(own, carry);
            uint32_t before = 0;
#pragma unroll
            for (int i = t > 0 && kPer == 2 ? -1 : 0; i < 32; ++i) {
              uint32_t w;
              if constexpr (kPer == 1) w = __float_as_uint(acc[t * 32 + i]);
              else w = pack2(acc[t * 64 + 2 * i], acc[t * 64 + 2 * i + 1], OutT());
              if (i >= 0)
                store_shared(word[i & 3] + room + (i & ~3) * 4, kPer == 1 ? w : __funnelshift_l(before, w, (own_start & 2) * 8));
              before = w;
            }
            if (kPer == 2 && t + 1 == kBoxes) store_shared(word[0] + room + 128, before >> 16);
            if (t + 1 < kBoxes) carry = load_shared4(own + 128);
            __syncwarp();
            const bool tails = bytes + 15 >= lo && (bytes & ~15) < hi;  // some row may end here
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 4) {
              const int r = r0 + (lane >> 3), j = lane & 7;
              OutT* to = out + static_cast<int64_t>(row0 + r) * p.ldo + col0;
              const int start = start_of(to), end = row0 + r < p.m ? start + bytes : 0;
              uint8_t* block = reinterpret_cast<uint8_t*>(to) - start;
              const uint32_t from = rows_at + r * kPitch;
              auto element = [&](int at) {
                if (at < lo || at >= hi) return;
                const uint32_t w = load_shared(from + ((at - lo) & ~15) + (((at >> 2) + (r0 >> 3)) & 3) * 4);
                if constexpr (kPer == 1)
                  *reinterpret_cast<uint32_t*>(block + at) = w;
                else
                  *reinterpret_cast<uint16_t*>(block + at) = static_cast<uint16_t>(w >> (at & 2) * 8);
              };
              if (lo + 16 * j >= start && lo + 16 * j + 16 <= end) {
                const uint4 u = load_shared4(from + 16 * j);
                const uint32_t x[4] = {u.x, u.y, u.z, u.w};
                *reinterpret_cast<uint4*>(block + lo + 16 * j) =
                    make_uint4(x[(r0 >> 3) & 3], x[((r0 >> 3) + 1) & 3], x[((r0 >> 3) + 2) & 3], x[((r0 >> 3) + 3) & 3]);
              }
              const int inner = (start + 15) & ~15;  // the first block that the row begins
              if (t == 0 && start + j * kSize < min(inner, end)) element(start + j * kSize);
              if (tails) {
                const int at = max(end & ~15, inner) + j * kSize;
                if (at < end) element(at);
              }
            }
            if (res_rows && t + 2 < kBoxes) {
              fence_proxy_async_smem();
              __syncwarp();
              fetch_rows(t + 2);
            }
          }
        }
      }
      if (ok || kCodes) ++turn;  // else what is left of this tile is waited for below
    }
    // Stores have to finish before the CTA ends; so do the residual loads that
    // a wait that ran out left behind (with a limit: some were never issued).
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (!ok && (res_boxes || res_rows))
      for (int c = 0; c < kBoxes; ++c) mbar_wait_limit(&res_bar[c], turn & 1, status, kWaitLimitNs / 1000);
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace pair

// ---------------------------------------------------------------- single tiles

// One 128 x BN tile per cluster of `split` CTAs, CTA r taking every split-th
// block of K from r on.  The sums meet in shared memory: each CTA writes its
// 128 x BN f32 over its operand stages, and after a cluster barrier CTA r
// finishes rows r, r + split, ... adding the CTAs' values in rank order, one
// warp per row (so a block of 128 results is one warp, and its maximum one
// warp reduction).  Rows past m are neither loaded nor read back.
namespace tile {

// A_ROWS: rows of A that a stage has room for.  With few rows the weights are
// what streams, and the room goes to more stages: a load from DRAM takes about
// 1.5 us, so 96 KB in flight are 64 GB/s an SM.  (The MMA still reads 128 rows:
// what follows A in the stage fills the lanes that nothing reads.)
template <int BN, int A_ROWS>
struct Plan {
  static constexpr int kA = A_ROWS * kFp8Block;
  static constexpr int kStageBytes = kA + BN * kFp8Block;
  static constexpr int kStages = (232448 - 1024 - 512) / kStageBytes < 12 ? (232448 - 1024 - 512) / kStageBytes : 12;
  static constexpr int kBufs = static_cast<int>(kTmemCols) / BN;  // partials
  static constexpr int kOffBar = kStages * kStageBytes;
  static constexpr int kSmem = 1024 + kOffBar + 512;
  static_assert(kSmem <= 232448, "dynamic shared memory per block");
  static_assert(A_ROWS * BN * 4 <= kOffBar, "the sums fit over the operand stages");
  static_assert(kStageBytes % 1024 == 0 && BN * kFp8Block >= kABytes - kA, "A's 128 rows stay inside the stage");
};

// Byte offset of the 16-byte chunk c of row r of the sums (conflict-free both
// for a thread per row and for a warp per row).
template <int BN>
__device__ __forceinline__ uint32_t sum_offset(int r, int c) {
  return static_cast<uint32_t>(r * (BN * 4) + ((c ^ (r & 31)) << 4));
}
__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <bool GATED, typename OutT, int BN, int A_ROWS>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmU, const __grid_constant__ Fp8GemmParams p, int split,
                    int a_rows) {
  using PL = Plan<BN, A_ROWS>;
  constexpr bool kCodes = sizeof(OutT) == 1;
  constexpr int kChunks = BN / 64;  // 32-column chunks of a thread's half
  static_assert(BN == (GATED ? 256 : 128), "a tile is 128 features, of both weights in the gated product");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + PL::kOffBar);
  uint64_t* done = full + PL::kStages;  // MMA done: stage free, partial ready
  uint64_t* acc_empty = done + PL::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + PL::kBufs);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  uint32_t* status = &g_fp8_status;

  constexpr int kFeat = GATED ? BN / 2 : BN;
  const int kblocks = (p.k + kFp8Block - 1) / kFp8Block;
  const int n_tiles = (p.n + kFeat - 1) / kFeat;
  const int rank = blockIdx.x % split, tile = blockIdx.x / split;  // a cluster is `split` neighbours of the grid
  const int m0 = (tile / n_tiles) * kRows, f0 = (tile % n_tiles) * kFeat;
  const int rows = min(kRows, p.m - m0);
  const int epi_warps = 2 * ((rows + 31) / 32);  // warps whose lanes hold rows of the matrix

  if (threadIdx.x == 0) {
    for (int i = 0; i < PL::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&done[i], 1);
    }
    for (int i = 0; i < PL::kBufs; ++i) mbar_init(&acc_empty[i], epi_warps);
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

  if (warp < 4) {
    regs_given_back();
    if (warp == 0 && lane == 0) {
      uint32_t i = 0;
      bool ok = true;
      for (int kb = rank; kb < kblocks; kb += split, ++i) {
        const uint32_t s = i % PL::kStages;
        if (!(ok = mbar_wait(&done[s], ((i / PL::kStages) & 1) ^ 1, status))) break;
        mbar_arrive_expect_tx(&full[s], a_rows * kFp8Block + BN * kFp8Block);
        uint8_t* sa = smem + s * PL::kStageBytes;
        tma_load_2d(sa, &tmA, &full[s], kb * kFp8Block, m0);
#pragma unroll
        for (int c = 0; c < BN / 64; ++c)  // 64 weight rows each
          tma_load_2d(sa + PL::kA + c * 64 * kFp8Block, GATED && (c & 1) ? &tmU : &tmW, &full[s], kb * kFp8Block,
                      GATED ? f0 + (c >> 1) * 64 : f0 + c * 64);
      }
      if (!ok) drain_loads(full, PL::kStages, i, status);
    } else if (warp == 1) {
      constexpr uint32_t idesc = idesc_e4m3_f32(kRows, BN);
      mma_loop<false, PL::kStages, PL::kStageBytes, PL::kA, PL::kBufs, BN>(
          tmem_base, idesc, smem_u32(smem), full, done, acc_empty,
          (kblocks - rank + split - 1) / split, status, [](uint64_t* b) { tc_commit(b); });
    }
  } else {
    regs_for_epilogue();
    const int q = warp & 3, h = (warp >> 2) - 1;
    if (q * 32 < rows) {
      const uint32_t tlane = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * (BN / 2);
      const int lrow = q * 32 + lane, row = m0 + lrow;
      const int nb = f0 / kFp8Block;  // block of weight rows
      const int blocks = (kblocks - rank + split - 1) / split;  // at least one: split <= kblocks
      Scales sc = scales_at<GATED>(p, row, nb, rank);
      float acc[32 * kChunks];
      Ring<PL::kStages> ring;
      fetch_scales<GATED>(sc, split);
      sum_blocks<false, GATED, kChunks, PL::kStages, PL::kBufs, BN>(
          acc, sc, blocks, split, tlane, done, ring, status,
          [&](uint32_t buf) {
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          });
      // The last partial was committed after every MMA of this CTA, so the
      // operand stages are free for the sums.
#pragma unroll
      for (int j = 0; j < 8 * kChunks; ++j)
        *reinterpret_cast<float4*>(smem + sum_offset<BN>(lrow, h * (BN / 8) + j)) =
            make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
    }
  }

  // the residual of a warp's next row is on its way while a row is finished (m =
  // 128, k = n = 768, a CTA per tile: 9.8 -> 7.5 us)
  const int first = rank + split * (warp - 4);  // row
  const OutT* res = GATED ? nullptr : static_cast<const OutT*>(p.residual);
  Raw4<OutT> next;
  if (warp >= 4 && res && first < rows)
    next.load(res + static_cast<int64_t>(m0 + first) * p.ldr + f0 + lane * 4, p.n - f0 - lane * 4);
  __syncwarp();
  if (split > 1)
    cluster_sync();
  else
    __syncthreads();

  if (warp >= 4) {
    const uint32_t base = smem_u32(smem);
    // the sum over the cluster of chunk c of row r
    auto total = [&](int r, int c) {
      const uint32_t at = base + sum_offset<BN>(r, c);
      if (split == 1) {
        float4 v;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "r"(at)
                     : "memory");
        return v;
      }
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < split; ++s) {
        uint32_t remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(s));
        const float4 u = load_cluster(remote);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      return v;
    };
    for (int r = first; r < rows; r += split * 8) {
      const int64_t row = m0 + r;
      if constexpr (GATED) {
        // lane: features 4 lane .. 4 lane + 3 of the tile's 128
        const int c = (lane >> 4) * 32 + (lane & 15);
        const float4 g = total(r, c), u = total(r, c + 16);
        const Gate gate(p.act);
        const int col = f0 + lane * 4, left = p.n - col;  // past the last feature: 0, whatever the scales are
        const float4 v = make_float4(left > 0 ? gate(g.x, u.x) : 0.f, left > 1 ? gate(g.y, u.y) : 0.f,
                                     left > 2 ? gate(g.z, u.z) : 0.f, left > 3 ? gate(g.w, u.w) : 0.f);
        if constexpr (kCodes) {
          const float a = max_abs3_nan(max_abs3_nan(v.x, v.y, v.z), v.w, v.w);
          const float sc = fp8_scale(warp_max_nan(a)), fac = fp8_factor(sc);
          if (lane == 0) p.out_scales[row * p.ldos + f0 / kFp8Block] = sc;
          store_codes4(static_cast<uint8_t*>(p.out) + row * p.ldo + col, p.n - col,
                       codes4<false>(v.x, v.y, v.z, v.w, sc, fac));
        } else {
          store4(static_cast<OutT*>(p.out) + row * p.ldo + col, left, v);
        }
      } else {
        const int col = f0 + lane * 4;
        float4 v = total(r, lane);
        if (res) {
          const float4 x = next.value();
          if (r + split * 8 < rows) next.load(res + (row + split * 8) * p.ldr + col, p.n - col);
          v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
        }
        store4(static_cast<OutT*>(p.out) + row * p.ldo + col, p.n - col, v);
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  if (split > 1)
    cluster_sync();  // no CTA leaves while another reads its sums
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace tile

// ---------------------------------------------------------------- status

__device__ uint32_t g_fp8_taken;  // what the last take_status_kernel found

// Reads and clears in one step: a wait of another stream that runs out meanwhile
// is either in what this one takes or left for the next.
__global__ void take_status_kernel() { g_fp8_taken = atomicExch(&g_fp8_status, 0u); }

// A wait that nothing ends, as a product's would run out.
__global__ void timeout_selftest_kernel(uint64_t limit_ns) {
  __shared__ uint64_t bar;
  mbar_init(&bar, 1);
  mbar_fence_init();
  mbar_wait_limit(&bar, 0, &g_fp8_status, limit_ns);
}

// ---------------------------------------------------------------- host

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

// Codes [rows][ld] of which k columns are meant: box `box_cols` (128 or 64)
// x box_rows, swizzled over the box's width, zeros outside.
bool codes_map(CUtensorMap* m, const uint8_t* ptr, int64_t rows, int64_t k, int64_t ld, uint32_t box_rows,
               uint32_t box_cols = kFp8Block) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t es[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(ptr), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_cols == kFp8Block ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Results or residual [rows][ld]: boxes of 32 rows x 128 bytes, 128-byte swizzle.
template <typename T>
bool values_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int64_t ld) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * sizeof(T)};
  cuuint32_t box[2] = {128 / sizeof(T), 32};
  cuuint32_t es[2] = {1, 1};
  return enc(m, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
             const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Largest dynamic shared memory, once per device and kernel.
template <auto KERNEL>
cudaError_t allow_smem(int bytes) {
  static std::atomic<bool> set[64] = {};  // calls come from any thread
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!set[dev]) {
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    set[dev] = true;
  }
  return cudaSuccess;
}

cudaLaunchAttribute cluster_of(int n) {
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeClusterDimension;
  a.val.clusterDim.x = n;
  a.val.clusterDim.y = 1;
  a.val.clusterDim.z = 1;
  return a;
}

int clusters_of(int num_sms) { return std::max(1, num_sms / 2); }

template <bool GATED, typename OutT, bool BOXES>
cudaError_t launch_pair(const Fp8GemmParams& p, int num_sms, cudaStream_t st) {
  constexpr auto kernel = pair::fp8_pair_kernel<GATED, OutT, BOXES>;
  cudaError_t e = allow_smem<kernel>(pair::Plan<GATED, OutT, BOXES>::kSmem);
  if (e != cudaSuccess) return e;
  CUtensorMap ta, tw, tu;
  if (!codes_map(&ta, p.a, p.m, p.k, p.lda, kRows) || !codes_map(&tw, p.w, p.n, p.k, p.ldw, 64) ||
      (GATED && !codes_map(&tu, p.up, p.n, p.k, p.ldup, 64)))
    return cudaErrorInvalidValue;
  if (!GATED) tu = tw;
  constexpr int kFeat = GATED ? pair::kBN / 2 : pair::kBN;
  const int64_t tiles = static_cast<int64_t>((p.m + 2 * kRows - 1) / (2 * kRows)) * ((p.n + kFeat - 1) / kFeat);
  if (tiles > 0x40000000 || tiles * ((p.k + kFp8Block - 1) / kFp8Block) > 0xFFFFFFFFll * clusters_of(num_sms))
    return cudaErrorInvalidValue;  // tile and block numbers are 32-bit
  const int clusters = static_cast<int>(std::min<int64_t>(tiles, clusters_of(num_sms)));
  // results by TMA boxes where rows (and the residual's) start at multiples of 16 bytes
  CUtensorMap to = ta, tr = ta;
  if constexpr (sizeof(OutT) == 1) {
    if (!codes_map(&to, static_cast<const uint8_t*>(p.out), p.m, p.n, p.ldo, 32, 64)) return cudaErrorInvalidValue;
  } else if constexpr (BOXES) {
    if (!values_map<OutT>(&to, p.out, p.m, p.n, p.ldo) ||
        (p.residual && !values_map<OutT>(&tr, p.residual, p.m, p.n, p.ldr)))
      return cudaErrorInvalidValue;
  }
  const cudaLaunchAttribute attr = cluster_of(2);
  return launch_pdl(kernel, dim3(2 * clusters), dim3(kThreads), pair::Plan<GATED, OutT, BOXES>::kSmem, st, &attr, 1, ta, tw, tu, to, tr,
                    p);
}

template <bool GATED, typename OutT, int BN, int A_ROWS>
cudaError_t launch_tile(const Fp8GemmParams& p, int split, cudaStream_t st) {
  constexpr auto kernel = tile::fp8_tile_kernel<GATED, OutT, BN, A_ROWS>;
  constexpr int kSmem = tile::Plan<BN, A_ROWS>::kSmem;
  cudaError_t e = allow_smem<kernel>(kSmem);
  if (e != cudaSuccess) return e;
  // rows of a box of A: as many as there are, in steps of the swizzle's eight
  const int a_rows = std::min(A_ROWS, (p.m + 7) / 8 * 8);
  CUtensorMap ta, tw, tu;
  if (!codes_map(&ta, p.a, p.m, p.k, p.lda, a_rows) || !codes_map(&tw, p.w, p.n, p.k, p.ldw, 64) ||
      (GATED && !codes_map(&tu, p.up, p.n, p.k, p.ldup, 64)))
    return cudaErrorInvalidValue;
  if (!GATED) tu = tw;
  constexpr int kFeat = GATED ? BN / 2 : BN;
  const int64_t tiles = static_cast<int64_t>((p.m + kRows - 1) / kRows) * ((p.n + kFeat - 1) / kFeat);
  if (tiles * split > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const cudaLaunchAttribute attr = cluster_of(split);
  return launch_pdl(kernel, dim3(static_cast<unsigned>(tiles * split)), dim3(kThreads), kSmem, st, &attr,
                    split > 1 ? 1 : 0, ta, tw, tu, p, split, a_rows);
}

// CTAs that run at once in clusters of `split` (a power of two up to 8): a
// cluster stays inside a group of SMs, so large ones leave some of them idle.
template <auto KERNEL>
int resident_ctas(int split, int smem, int num_sms) {
  static std::atomic<int> counts[64][4] = {};  // calls come from any thread
  int dev = 0;
  if (split == 1 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return num_sms;
  std::atomic<int>& count = counts[dev][split == 2 ? 1 : split == 4 ? 2 : 3];
  int n = count.load();
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(num_sms / split * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr = cluster_of(split);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, KERNEL, &cfg) != cudaSuccess) {
      cudaGetLastError();
      clusters = num_sms / split;
    }
    n = std::max(split, clusters * split);
    count.store(n);
  }
  return n;
}

struct Cost {  // us
  float tile, tile_rows, block, join, pair_start, pair_round, pair_block;
};

// Whether rows of results or of the residual start off the 16-byte boundary.
template <typename OutT>
bool off_boundary(const Fp8GemmParams& p) {
  return sizeof(OutT) > 1 && !(p.box_o && (!p.residual || p.box_r));
}

// Columns of a single tile's weights: 128 features, of both in the gated product.
template <bool GATED>
constexpr int kTileBN = GATED ? 256 : 128;

// CTAs that share a single tile's K, or 0 for pairs of SMs.
template <bool GATED, typename OutT>
cudaError_t choose(const Fp8GemmParams& p, int num_sms, int* chosen) {
  constexpr int BN = kTileBN<GATED>;
  constexpr int kFeat = 128;  // output columns of a single tile
  const int64_t kblocks = (static_cast<int64_t>(p.k) + kFp8Block - 1) / kFp8Block;
  const int64_t tiles = static_cast<int64_t>((p.m + kRows - 1) / kRows) * ((p.n + kFeat - 1) / kFeat);
  // Which kernel, and how many CTAs share a tile's K: whichever should end
  // first by what was measured (us, inputs from DRAM).  A single tile costs a
  // start and an end that grow with its rows, and its blocks one after the
  // other; a join over a cluster costs extra; more tiles than SMs go in rounds.
  // A pair's round is cheaper per element but starts slower, and rows off the
  // 16-byte boundary cost it more than the single tile, whose CTAs also share the
  // residual's rows.  Measured with 768 <= k <=
  // 8192 and 1 <= m <= 4096, extrapolated elsewhere; at m = 128, k = 768, n = 2304: 6.1 / 6.8 / 5.6 / 6.5 us
  // with 1, 2, 4, 8 CTAs a tile and 6.8 on pairs.
  const Cost c = GATED ? Cost{2.8f, 4.2f, 0.46f, 0.6f, 2.8f, 1.8f, 0.45f} : Cost{2.05f, 1.95f, 0.32f, 0.65f, 4.0f, 1.0f, 0.42f};
  const float rows = static_cast<float>(std::min<int64_t>(p.m, kRows)) / kRows;
  constexpr int kPairFeat = GATED ? 128 : 256;
  const int64_t pairs = static_cast<int64_t>((p.m + 2 * kRows - 1) / (2 * kRows)) * ((p.n + kPairFeat - 1) / kPairFeat);
  const bool off = off_boundary<OutT>(p);
  const float pair_off = !off ? 0.0f : (p.residual ? 3.2f : 1.3f) * (sizeof(OutT) == 4 ? 1.6f : 1.0f);
  const float tile_res = !p.residual ? 0.0f : rows * (off ? 3.0f : 1.2f) * (sizeof(OutT) == 4 ? 2.0f : 1.0f);
  float best = c.pair_start + static_cast<float>((pairs + clusters_of(num_sms) - 1) / clusters_of(num_sms)) *
                                  (c.pair_round + c.pair_block * kblocks + pair_off);
  constexpr auto kernel = tile::fp8_tile_kernel<GATED, OutT, BN, kRows>;
  constexpr int kSmem = tile::Plan<BN, kRows>::kSmem;
  if (cudaError_t e = allow_smem<kernel>(kSmem); e != cudaSuccess) return e;
  int split = 0;  // pairs
  for (int s = 1; s <= 8 && s <= kblocks; s *= 2) {
    const int fit = resident_ctas<kernel>(s, kSmem, num_sms);
    const float rounds = static_cast<float>((tiles * s + fit - 1) / fit);
    const float t = rounds * (c.tile + c.tile_rows * rows + tile_res / s + c.block * static_cast<float>((kblocks + s - 1) / s) +
                              (s > 1 ? c.join : 0.0f));
    if (t < best) {
      best = t;
      split = s;
    }
  }
  *chosen = split;
  return cudaSuccess;
}

template <bool GATED, typename OutT>
cudaError_t launch(const Fp8GemmParams& p, int num_sms, cudaStream_t st) {
  constexpr int BN = kTileBN<GATED>;
  int split = 0;
  if (cudaError_t e = choose<GATED, OutT>(p, num_sms, &split); e != cudaSuccess) return e;
  if (split == 0) {
    if constexpr (sizeof(OutT) > 1)
      if (off_boundary<OutT>(p)) return launch_pair<GATED, OutT, false>(p, num_sms, st);
    return launch_pair<GATED, OutT, true>(p, num_sms, st);
  }
  return p.m <= 32 ? launch_tile<GATED, OutT, BN, 32>(p, split, st) : launch_tile<GATED, OutT, BN, kRows>(p, split, st);
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

cudaError_t fp8_gemm_split(bool gated, int out_type, const Fp8GemmParams& p, int num_sms, int* split) {
  if (gated) {
    switch (out_type) {
      case WC_T_F32: return choose<true, float>(p, num_sms, split);
      case WC_T_F16: return choose<true, __half>(p, num_sms, split);
      case WC_T_BF16: return choose<true, __nv_bfloat16>(p, num_sms, split);
      case WC_T_E4M3: return choose<true, uint8_t>(p, num_sms, split);
      default: return cudaErrorInvalidValue;
    }
  }
  switch (out_type) {
    case WC_T_F32: return choose<false, float>(p, num_sms, split);
    case WC_T_F16: return choose<false, __half>(p, num_sms, split);
    case WC_T_BF16: return choose<false, __nv_bfloat16>(p, num_sms, split);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t fp8_gemm_take_status(uint32_t* status, cudaStream_t st) {
  static std::mutex mu;  // one caller at a time has g_fp8_taken
  std::lock_guard<std::mutex> lock(mu);
  take_status_kernel<<<1, 1, 0, st>>>();
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(status, g_fp8_taken, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

cudaError_t fp8_gemm_timeout_selftest(uint64_t limit_ns, cudaStream_t st) {
  timeout_selftest_kernel<<<1, 1, 0, st>>>(limit_ns);
  return cudaGetLastError();
}

}  // namespace wc
