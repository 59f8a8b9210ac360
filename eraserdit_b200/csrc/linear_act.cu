// Matrix product with its epilogue on the sm_100a tensor cores:
//   y = residual + gate * act(x W^T + bias)
// BF16 or FP16 operands, FP32 accumulation in TMEM, every step of the epilogue
// in FP32, one rounding.  Any row count, any n; rows of x and W start on 16
// bytes (TMA), k is free.
//
// Two kernels, chosen by the host (pick_plan):
//   pair_kernel   large products.  A persistent kernel of CTA pairs
//                 (cta_group::2), one 256 x 256 tile a pair: each CTA stages
//                 128 rows of x and 128 rows of W, so an instruction reads half
//                 of W's tile from either shared memory and a CTA loads 32 KB
//                 per 64-deep step for 128 x 256 outputs.  An accumulator is
//                 256 TMEM columns, so two fit, and the epilogue of a tile runs
//                 beside the products of the next.
//   split_kernel  few tiles (short row counts, narrow outputs).  One 128 x 64
//                 or 128 x 128 tile a CTA, the reduction split over the CTAs of
//                 a cluster, whose FP32 partial sums are added through
//                 distributed shared memory in rank order (the result does not
//                 depend on timing).  Only the rows that exist are loaded, so
//                 one token streams W and little else.
// Roles of a CTA: warp 0 TMA producer, warp 1 MMA issuer, the others epilogue.
// Every wait is bounded; one that gives up records a status bit, and every
// thread still reaches the cluster barriers, so no CTA leaves a peer behind.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/eraserdit_b200.h"
#include "host_common.h"
#include "sm100_ptx.cuh"
#include "tmem_io.cuh"

namespace erd {
namespace lact {

constexpr int kRowBytes = 128;  // 64 values of K per stage and row: one swizzle atom
constexpr int kBK = 64;

// kind::f16 instruction descriptor for BF16 (format 1) or FP16 (format 0)
// operands, both K-major, FP32 accumulation.
template <bool kBf16>
__host__ __device__ constexpr uint32_t idesc(int m, int n) {
  return (1u << 4) | ((kBf16 ? 1u : 0u) << 7) | ((kBf16 ? 1u : 0u) << 10) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// ---------------------------------------------------------------- cluster PTX
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // the barrier wants whole warps, also behind one-lane roles
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}
// Address of this CTA's shared-memory location `addr` in CTA `rank`.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}

// ------------------------------------------------------- cta_group::2 tcgen05
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void mma_pair_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc_, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc_), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` (the same offset) in both CTAs of the pair when the products
// issued so far have completed.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// 2-D load into this CTA's shared memory whose bytes are counted on a barrier
// of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* desc, uint32_t bar,
                                                 int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(desc)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

// ------------------------------------------------------------------- epilogue
template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_float<__half>(__half x) {
  return __half2float(x);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// x * sigmoid(z): the logistic function through 2^x and a reciprocal, both to
// a few units in the last place of FP32 (a tanh instruction would keep 11 bits).
__device__ __forceinline__ float times_sigmoid(float x, float z) {
  return __fdividef(x, 1.0f + ex2_approx(-1.4426950408889634f * z));
}
// gelu with tanh: (1 + tanh(u)) / 2 = sigmoid(2 u), u = sqrt(2/pi) (x + 0.044715 x^3).
__device__ __forceinline__ float gelu_tanh(float x) {
  return times_sigmoid(x, x * fmaf(0.07135481283f, x * x, 1.5957691216f));
}
// gelu with the normal distribution function; erfc keeps the small values of
// negative arguments that 1 + erf would cancel.
__device__ __forceinline__ float gelu_erf(float x) {
  return 0.5f * x * erfcf(-0.70710678118654752f * x);
}

template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == ERD_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = gelu_tanh(v[i]);
  } else if (act == ERD_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = times_sigmoid(v[i], v[i]);
  } else if (act == ERD_ACT_RELU) {
    // not fmaxf: a NaN stays one
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
  } else if (act == ERD_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = gelu_erf(v[i]);
  }
}

struct Epilogue {
  int m, n;
  int act;
  const void* bias;      // [n] or null
  const void* gate;      // [groups][n] or null
  int gate_rows;         // rows of one gate group
  const void* residual;  // [m][ld_res] or null
  long long ld_res;
  void* y;
  long long ldy;
  int vec_res, vec_y;  // rows start on 16 bytes
};

// Eight values from column `col` of row `row` (what lies behind column n is 0).
template <typename T>
__device__ __forceinline__ uint4 load8(const void* base, long long ld, int vec, int row, int col,
                                       int n) {
  const T* p = static_cast<const T*>(base) + row * ld + col;
  if (vec && col + 8 <= n) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col + i < n)
      w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void store8(void* base, long long ld, int vec, int row, int col, int n,
                                       const uint4& v) {
  T* p = static_cast<T*>(base) + row * ld + col;
  if (vec && col + 8 <= n) {
    *reinterpret_cast<uint4*>(p) = v;
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col + i < n)
      reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
}

constexpr int kPiece = 64;                    // columns an epilogue warp takes at a time
constexpr int kStageBytes = 32 * kPiece * 2;  // 32 rows of a piece, 16-byte chunks swizzled
constexpr int kSlabBytes = 2 * kPiece * 4;    // bias and gate of a piece as floats

// One warp, 32 rows from row0 (TMEM lanes) x 64 columns from col0.  The
// residual comes in and the result goes out through a staging block, 128 bytes
// of a row at a time, so that a warp's access covers four whole lines instead
// of 32 pieces of 16 bytes.
template <typename T>
__device__ __forceinline__ void epilogue_piece(const Epilogue& e, uint32_t taddr, int row0,
                                               int col0, uint8_t* stage, float* slab, int lane) {
  const int sub = lane >> 3, chunk = lane & 7;  // row within a group of 4, 16-byte chunk
  if (e.residual != nullptr) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int rr = 4 * q + sub;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row0 + rr < e.m && col0 + chunk * 8 < e.n)
        v = load8<T>(e.residual, e.ld_res, e.vec_res, row0 + rr, col0 + chunk * 8, e.n);
      *reinterpret_cast<uint4*>(stage + rr * 128 + ((chunk ^ (rr & 7)) * 16)) = v;
    }
  }
  const int row = row0 + lane;
  int group = 0;
  bool one_group = true;
  if (e.gate != nullptr) {
    group = min(row, e.m - 1) / e.gate_rows;
    one_group = __all_sync(0xffffffffu, group == __shfl_sync(0xffffffffu, group, 0));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = lane + 32 * i;
    float b = 0.f, g = 1.f;
    if (col0 + c < e.n) {
      if (e.bias != nullptr) b = to_float(static_cast<const T*>(e.bias)[col0 + c]);
      if (e.gate != nullptr && one_group)
        g = to_float(
            static_cast<const T*>(e.gate)[static_cast<long long>(group) * e.n + col0 + c]);
    }
    slab[c] = b;
    slab[kPiece + c] = g;
  }
  __syncwarp();
  uint32_t r[kPiece];
  tmem_ld_wait_64(taddr, r);
  uint8_t* own = stage + lane * 128;
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // 32 columns at a time
    float v[32];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = reinterpret_cast<const float4*>(slab)[h * 8 + i];
      v[4 * i] = __uint_as_float(r[h * 32 + 4 * i]) + b.x;
      v[4 * i + 1] = __uint_as_float(r[h * 32 + 4 * i + 1]) + b.y;
      v[4 * i + 2] = __uint_as_float(r[h * 32 + 4 * i + 2]) + b.z;
      v[4 * i + 3] = __uint_as_float(r[h * 32 + 4 * i + 3]) + b.w;
    }
    activate(v, e.act);
    if (e.gate != nullptr) {
      if (one_group) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 g = reinterpret_cast<const float4*>(slab)[16 + h * 8 + i];
          v[4 * i] *= g.x;
          v[4 * i + 1] *= g.y;
          v[4 * i + 2] *= g.z;
          v[4 * i + 3] *= g.w;
        }
      } else {  // two groups meet within these 32 rows
        const T* g = static_cast<const T*>(e.gate) + static_cast<long long>(group) * e.n;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (col0 + h * 32 + i < e.n) v[i] *= to_float(g[col0 + h * 32 + i]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4* at = reinterpret_cast<uint4*>(own + (((h * 4 + c) ^ (lane & 7)) * 16));
      if (e.residual != nullptr) {
        const uint4 w = *at;
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2<T>(ww[i]);
          v[8 * c + 2 * i] += f.x;
          v[8 * c + 2 * i + 1] += f.y;
        }
      }
      *at = make_uint4(pack2<T>(v[8 * c], v[8 * c + 1]), pack2<T>(v[8 * c + 2], v[8 * c + 3]),
                       pack2<T>(v[8 * c + 4], v[8 * c + 5]), pack2<T>(v[8 * c + 6], v[8 * c + 7]));
    }
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int rr = 4 * q + sub;
    if (row0 + rr < e.m && col0 + chunk * 8 < e.n)
      store8<T>(e.y, e.ldy, e.vec_y, row0 + rr, col0 + chunk * 8, e.n,
                *reinterpret_cast<const uint4*>(stage + rr * 128 + ((chunk ^ (rr & 7)) * 16)));
  }
  __syncwarp();
}

// ---------------------------------------------------------------- pair kernel
constexpr int kPairStages = 5;
constexpr int kPairOperandBytes = 128 * kRowBytes;  // 16 KB of x and of W per CTA and stage
constexpr int kPairEpilogueWarps = 8;
constexpr int kPairThreads = 32 * (2 + kPairEpilogueWarps);
constexpr int kPairTile = 256;  // rows and columns of a pair's tile

struct __align__(8) PairBarriers {
  uint64_t full[kPairStages];   // the leader's: bytes of both CTAs
  uint64_t empty[kPairStages];  // each CTA's own
  uint64_t acc_full[2];         // each CTA's own
  uint64_t acc_empty[2];        // the leader's: every epilogue warp of both CTAs
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

constexpr int kPairSmemA = 0;
constexpr int kPairSmemB = kPairSmemA + kPairStages * kPairOperandBytes;
constexpr int kPairSmemStage = kPairSmemB + kPairStages * kPairOperandBytes;
constexpr int kPairSmemSlab = kPairSmemStage + kPairEpilogueWarps * kStageBytes;
constexpr int kPairSmemBar = kPairSmemSlab + kPairEpilogueWarps * kSlabBytes;
constexpr int kPairSmemLaunch = kPairSmemBar + 1024 + 1024;  // + base alignment
static_assert(kPairSmemLaunch <= 227 * 1024, "shared memory budget");

struct PairParams {
  Epilogue e;
  int k, tiles_m, tiles_n;
  int* status;
};

template <typename T, bool kBf16>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmap_a,
                const __grid_constant__ CUtensorMap tmap_b, const PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  PairBarriers* bars = reinterpret_cast<PairBarriers*>(smem + kPairSmemBar);
  const uint32_t sA = smem_u32(smem + kPairSmemA);
  const uint32_t sB = smem_u32(smem + kPairSmemB);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.tiles_m * p.tiles_n;
  const int ksteps = (p.k + kBK - 1) / kBK;
  volatile int* abort = &bars->abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bars->acc_full[b]), 1);
      mbar_init(smem_u32(&bars->acc_empty[b]), 2 * kPairEpilogueWarps);
    }
    mbar_init(smem_u32(&bars->drain), 1);
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&bars->tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers and TMEM of both CTAs exist
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmap_a);
      tma_prefetch_desc(&tmap_b);
      uint32_t it = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs) {
        const int m0 = (tile / p.tiles_n) * kPairTile + static_cast<int>(rank) * 128;
        const int n0 = (tile % p.tiles_n) * kPairTile + static_cast<int>(rank) * 128;
        for (int kk = 0; kk < ksteps; ++kk, ++it) {
          const uint32_t s = it % kPairStages;
          const uint32_t ph = (it / kPairStages) & 1;
          if (!mbar_wait(smem_u32(&bars->empty[s]), ph ^ 1, abort, p.status,
                         kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t full = smem_u32(&bars->full[s]);
          // The leader announces the bytes of both CTAs.  The other CTA's may
          // land first: the phase cannot end before the leader's arrival.
          if (rank == 0) mbar_arrive_expect_tx(full, 4 * kPairOperandBytes);
          const uint32_t bar = map_rank(full, 0);
          tma_load_2d_pair(sA + s * kPairOperandBytes, &tmap_a, bar, kk * kBK, m0);
          tma_load_2d_pair(sB + s * kPairOperandBytes, &tmap_b, bar, kk * kBK, n0);
        }
      }
      if (*abort && rank == 0) {
        // Let the loads that may be in flight land before exiting.
        for (int d = 0; d < kPairStages && it > 0; ++d) {
          --it;
          mbar_wait_drain(smem_u32(&bars->full[it % kPairStages]), (it / kPairStages) & 1);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer (the leader)
    if (lane == 0 && rank == 0) {
      constexpr uint32_t id = idesc<kBf16>(256, 256);
      uint32_t it = 0, count = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++count) {
        const uint32_t buf = count & 1;
        if (!mbar_wait(smem_u32(&bars->acc_empty[buf]), ((count >> 1) & 1) ^ 1, abort, p.status,
                       kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        for (int kk = 0; kk < ksteps; ++kk, ++it) {
          const uint32_t s = it % kPairStages;
          const uint32_t ph = (it / kPairStages) & 1;
          if (!mbar_wait(smem_u32(&bars->full[s]), ph, abort, p.status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = sA + s * kPairOperandBytes, b = sB + s * kPairOperandBytes;
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4)
            mma_pair_ss(d, sdesc_sw128(a + k4 * 32, 16, 1024), sdesc_sw128(b + k4 * 32, 16, 1024),
                        id, (kk > 0 || k4 > 0) ? 1u : 0u);
          mma_commit_pair(smem_u32(&bars->empty[s]));
        }
        if (!ok) break;
        mma_commit_pair(smem_u32(&bars->acc_full[buf]));
      }
      // Every product completes before the TMEM of both CTAs is released.
      mma_commit_pair(smem_u32(&bars->drain));
      mbar_wait_drain(smem_u32(&bars->drain), 0);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int w = warp - 2, quad = warp & 3, half = w >> 2;
    uint8_t* stage = smem + kPairSmemStage + w * kStageBytes;
    float* slab = reinterpret_cast<float*>(smem + kPairSmemSlab + w * kSlabBytes);
    uint32_t count = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++count) {
      const uint32_t buf = count & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->acc_full[buf]), (count >> 1) & 1,
                                             abort, p.status, kStatusTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int row0 = (tile / p.tiles_n) * kPairTile + static_cast<int>(rank) * 128 + quad * 32;
      const int col0 = (tile % p.tiles_n) * kPairTile + half * 128;
      const uint32_t taddr =
          tmem + (static_cast<uint32_t>(quad * 32) << 16) + buf * 256 + half * 128;
      if (row0 < p.e.m) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c)
          if (col0 + c * kPiece < p.e.n)
            epilogue_piece<T>(p.e, taddr + c * kPiece, row0, col0 + c * kPiece, stage, slab, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(&bars->acc_empty[buf]), 0));
    }
  }
  tc_fence_before();
  cluster_sync();  // no CTA leaves while the other may still signal it
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// --------------------------------------------------------------- split kernel
constexpr int kSplitEpilogueWarps = 4;
constexpr int kSplitThreads = 32 * (2 + kSplitEpilogueWarps);
constexpr int kSplitMaxStages = 12;

struct __align__(8) SplitBarriers {
  uint64_t full[kSplitMaxStages];
  uint64_t empty[kSplitMaxStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort;
};

struct SplitParams {
  Epilogue e;
  int k, tiles_n;
  int a_rows;   // rows of the x box (a multiple of 8, at most 128)
  int stages;   // ring depth that fits the shared memory of this launch
  int splits;   // CTAs of a cluster: parts of the reduction
  int tail;     // offset of the staging blocks and barriers
  int* status;
};

// Shared memory: [stages][x box] [stages][W box], at p.tail staging, slabs and
// barriers; the FP32 partial sums (splits > 1) lie where the ring was.
template <int BN>
struct SplitSmem {
  static constexpr int kBBytes = BN * kRowBytes;
  static __host__ __device__ int a_bytes(int a_rows) { return (a_rows * kRowBytes + 1023) & ~1023; }
  static __host__ __device__ int ring(int a_rows, int stages) {
    return stages * (a_bytes(a_rows) + kBBytes);
  }
  static constexpr int kTail =
      kSplitEpilogueWarps * (kStageBytes + kSlabBytes) + 1024;  // staging, slabs, barriers
};

// 16-byte chunk `c4` of row `r` of the partial sums, swizzled so that the 32
// rows a warp writes at a time do not meet in the same banks.
template <int BN>
__device__ __forceinline__ int partial_offset(int r, int c4) {
  return r * (BN * 4) + ((c4 ^ (r & 7)) * 16);
}

template <typename T, bool kBf16, int BN>
__global__ void __launch_bounds__(kSplitThreads)
    split_kernel(const __grid_constant__ CUtensorMap tmap_a,
                 const __grid_constant__ CUtensorMap tmap_b, const SplitParams p) {
  using S = SplitSmem<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int a_bytes = S::a_bytes(p.a_rows);
  uint8_t* tail = smem + p.tail;
  SplitBarriers* bars = reinterpret_cast<SplitBarriers*>(
      tail + kSplitEpilogueWarps * (kStageBytes + kSlabBytes));
  const uint32_t sA = smem_u32(smem);
  const uint32_t sB = sA + p.stages * a_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits;  // also the rank in the cluster
  const int tile = blockIdx.x / p.splits;
  const int m0 = (tile / p.tiles_n) * 128, n0 = (tile % p.tiles_n) * BN;
  const int ksteps = (p.k + kBK - 1) / kBK;
  const int k_lo = static_cast<int>(static_cast<long long>(ksteps) * split / p.splits);
  const int k_hi = static_cast<int>(static_cast<long long>(ksteps) * (split + 1) / p.splits);
  volatile int* abort = &bars->abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    mbar_init(smem_u32(&bars->acc_full), 1);
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&bars->tmem_base), BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  bool have = false;  // this warp's rows of the accumulator may be read
  if (warp == 0) {
    if (lane == 0) {
      const uint32_t tx = static_cast<uint32_t>(p.a_rows * kRowBytes + S::kBBytes);
      int it = 0;
      for (int kk = k_lo; kk < k_hi; ++kk, ++it) {
        const int s = it % p.stages;
        const uint32_t ph = (it / p.stages) & 1;
        if (!mbar_wait(smem_u32(&bars->empty[s]), ph ^ 1, abort, p.status,
                       kStatusTimeoutProducer))
          break;
        const uint32_t full = smem_u32(&bars->full[s]);
        mbar_arrive_expect_tx(full, tx);
        tma_load_2d(sB + s * S::kBBytes, &tmap_b, full, kk * kBK, n0);
        tma_load_2d(sA + s * a_bytes, &tmap_a, full, kk * kBK, m0);
      }
      if (*abort) {
        for (int d = 0; d < p.stages && it > 0; ++d) {
          --it;
          mbar_wait_drain(smem_u32(&bars->full[it % p.stages]), (it / p.stages) & 1);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id = idesc<kBf16>(128, BN);
      for (int kk = k_lo, it = 0; kk < k_hi; ++kk, ++it) {
        const int s = it % p.stages;
        const uint32_t ph = (it / p.stages) & 1;
        if (!mbar_wait(smem_u32(&bars->full[s]), ph, abort, p.status, kStatusTimeoutMma)) break;
        tc_fence_after();
        const uint32_t a = sA + s * a_bytes, b = sB + s * S::kBBytes;
        // Rows of the product beyond the x box read whatever the shared memory
        // behind it holds; their accumulator lanes are never read.
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          mma_bf16_ss(tmem, sdesc_sw128(a + k4 * 32, 16, 1024), sdesc_sw128(b + k4 * 32, 16, 1024),
                      id, (it > 0 || k4 > 0) ? 1u : 0u);
        }
        mma_commit(smem_u32(&bars->empty[s]));
      }
      mma_commit(smem_u32(&bars->acc_full));
      mbar_wait_drain(smem_u32(&bars->acc_full), 0);
    }
  } else {
    have = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->acc_full), 0, abort, p.status,
                                             kStatusTimeoutEpilogue));
    // A reduction that was cut short has set the flag before it committed.
    have = have && __all_sync(0xffffffffu, *abort == 0);
    tc_fence_after();
    const int quad = warp & 3;
    const int row0 = m0 + quad * 32;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    if (have && row0 < p.e.m) {
      if (p.splits == 1) {
        uint8_t* stage = tail + (warp - 2) * kStageBytes;
        float* slab = reinterpret_cast<float*>(tail + kSplitEpilogueWarps * kStageBytes +
                                               (warp - 2) * kSlabBytes);
#pragma unroll 1
        for (int c = 0; c < BN; c += kPiece)
          if (n0 + c < p.e.n)
            epilogue_piece<T>(p.e, taddr + c, row0, n0 + c, stage, slab, lane);
      } else {
        // The ring is free: every load has been consumed by a finished product.
        const int r = quad * 32 + lane;
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          uint32_t v[32];
          tmem_ld_wait_32(taddr + c, v);
          if (m0 + r < p.e.m) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(smem + partial_offset<BN>(r, c / 4 + i)) =
                  make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  if (p.splits == 1) {
    __syncthreads();
  } else {
    cluster_sync();
    // Each CTA adds and finishes its share of the tile, eight columns a thread.
    // A split that gave up has set the status word; its partial sums are stale
    // and the tile's values are then as undefined as those of any timed-out call.
    const int rows = min(128, p.e.m - m0);
    const int total = rows * (BN / 8);
    const int lo = static_cast<int>(static_cast<long long>(total) * split / p.splits);
    const int hi = static_cast<int>(static_cast<long long>(total) * (split + 1) / p.splits);
    const uint32_t base = smem_u32(smem);
    for (int i = lo + static_cast<int>(threadIdx.x); i < hi; i += kSplitThreads) {
      const int r = i / (BN / 8), c8 = i % (BN / 8);
      const int row = m0 + r, col = n0 + c8 * 8;
      if (col >= p.e.n) continue;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
      for (int s = 0; s < p.splits; ++s) {
        const uint32_t peer = map_rank(base, static_cast<uint32_t>(s));
        const float4 a = ld_cluster(peer + partial_offset<BN>(r, c8 * 2));
        const float4 b = ld_cluster(peer + partial_offset<BN>(r, c8 * 2 + 1));
        v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
        v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
      }
      if (p.e.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < p.e.n) v[j] += to_float(static_cast<const T*>(p.e.bias)[col + j]);
      }
      activate(v, p.e.act);
      if (p.e.gate != nullptr) {
        const T* g = static_cast<const T*>(p.e.gate) +
                     static_cast<long long>(row / p.e.gate_rows) * p.e.n + col;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < p.e.n) v[j] *= to_float(g[j]);
      }
      if (p.e.residual != nullptr) {
        const uint4 w = load8<T>(p.e.residual, p.e.ld_res, p.e.vec_res, row, col, p.e.n);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<T>(ww[j]);
          v[2 * j] += f.x;
          v[2 * j + 1] += f.y;
        }
      }
      store8<T>(p.e.y, p.e.ldy, p.e.vec_y, row, col, p.e.n,
                make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                           pack2<T>(v[6], v[7])));
    }
    cluster_sync();  // the peers have read this CTA's sums
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool pair;
  int bn, splits, a_rows;
};

// Which kernel, and how a small product is cut.
Plan pick_plan(int m, int n, int k, int sms) {
  Plan pl = {};
  const long long tiles_pair = static_cast<long long>((m + 255) / 256) * ((n + 255) / 256);
  if (tiles_pair * 2 >= sms) {
    pl.pair = true;
    return pl;
  }
  const int ksteps = (k + kBK - 1) / kBK;
  const long long tm = (m + 127) / 128;
  const long long t128 = tm * ((n + 127) / 128), t64 = tm * ((n + 63) / 64);
  pl.bn = t128 >= sms ? 128 : 64;
  const long long tiles = pl.bn == 128 ? t128 : t64;
  pl.splits = 1;
  while (pl.splits < 8 && tiles * pl.splits * 2 <= 2LL * sms && ksteps / (pl.splits * 2) >= 4)
    pl.splits *= 2;
  pl.a_rows = m >= 128 ? 128 : (m + 7) / 8 * 8;
  return pl;
}

template <typename T, bool kBf16, int BN>
int launch_split(const CUtensorMap& ta, const CUtensorMap& tb, SplitParams p, const Plan& pl,
                 cudaStream_t st) {
  using S = SplitSmem<BN>;
  const int ksteps = (p.k + kBK - 1) / kBK;
  const int per_split = (ksteps + pl.splits - 1) / pl.splits;
  const int budget = 112 * 1024 - S::kTail - 1024;  // two CTAs on a multiprocessor
  p.stages = budget / S::ring(pl.a_rows, 1);
  if (p.stages > kSplitMaxStages) p.stages = kSplitMaxStages;
  if (p.stages > per_split) p.stages = per_split;
  // The ring, the 128 rows that a product reads from a stage's x box however
  // few were loaded, and the partial sums all end before the tail.
  p.tail = S::ring(pl.a_rows, p.stages);
  const int reach = (p.stages - 1) * S::a_bytes(pl.a_rows) + 128 * kRowBytes;
  if (p.tail < reach) p.tail = reach;
  if (pl.splits > 1 && p.tail < 128 * BN * 4) p.tail = 128 * BN * 4;
  const int bytes = p.tail + S::kTail + 1024;  // + base alignment
  cudaError_t e = cudaFuncSetAttribute(split_kernel<T, kBf16, BN>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e != cudaSuccess) return static_cast<int>(e);
  const long long tiles = static_cast<long long>((p.e.m + 127) / 128) * p.tiles_n;
  if (tiles * pl.splits > 0x7fffffffLL) return kErrTooLarge;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * pl.splits));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(pl.splits);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, split_kernel<T, kBf16, BN>, ta, tb, p);
  return static_cast<int>(e);
}

int operand_map(CUtensorMap* map, bool bf16, const void* base, int rows, int k, int64_t ld,
                int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld) * 2};
  const uint32_t box[2] = {kBK, static_cast<uint32_t>(box_rows)};
  return encode_tensor_map(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
      const_cast<void*>(base), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, bool kBf16>
int run(const Epilogue& e, const void* x, int64_t ldx, const void* w, int64_t ldw, int k,
        int* status, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return static_cast<int>(err);
  Plan pl = pick_plan(e.m, e.n, k, sms);
  CUtensorMap ta, tb;
  if (pl.pair) {
    const long long tm = (e.m + 255) / 256, tn = (e.n + 255) / 256;
    if (tm * tn > (1LL << 30)) return kErrTooLarge;
    if (operand_map(&ta, kBf16, x, e.m, k, ldx, 128) ||
        operand_map(&tb, kBf16, w, e.n, k, ldw, 128))
      return kErrTensorMap;
    PairParams p = {e, k, static_cast<int>(tm), static_cast<int>(tn), status};
    err = cudaFuncSetAttribute(pair_kernel<T, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kPairSmemLaunch);
    if (err != cudaSuccess) return static_cast<int>(err);
    const long long pairs = tm * tn < sms / 2 ? tm * tn : sms / 2;
    pair_kernel<T, kBf16>
        <<<static_cast<unsigned>(2 * pairs), kPairThreads, kPairSmemLaunch, st>>>(ta, tb, p);
    return static_cast<int>(cudaGetLastError());
  }
  if (operand_map(&ta, kBf16, x, e.m, k, ldx, pl.a_rows) ||
      operand_map(&tb, kBf16, w, e.n, k, ldw, pl.bn))
    return kErrTensorMap;
  SplitParams p = {};
  p.e = e;
  p.k = k;
  p.tiles_n = (e.n + pl.bn - 1) / pl.bn;
  p.a_rows = pl.a_rows;
  p.status = status;
  p.splits = pl.splits;
  return pl.bn == 128 ? launch_split<T, kBf16, 128>(ta, tb, p, pl, st)
                      : launch_split<T, kBf16, 64>(ta, tb, p, pl, st);
}

}  // namespace lact
}  // namespace erd

using namespace erd;

extern "C" int erd_linear_act(int dtype, const void* x, int64_t ldx, const void* weight,
                              int64_t ldw, const void* bias, int activation, const void* gate,
                              int gate_rows, const void* residual, int64_t ld_residual, void* y,
                              int64_t ldy, int m, int n, int k, int* status, void* stream) {
  if (x == nullptr || weight == nullptr || y == nullptr) return kErrNullPointer;
  if ((dtype != ERD_BF16 && dtype != ERD_FP16) || activation < ERD_ACT_NONE ||
      activation > ERD_ACT_GELU_TANH || m <= 0 || n <= 0 || k <= 0 || ldx < k || ldw < k ||
      ldy < n || (residual != nullptr && ld_residual < n) || (gate != nullptr && gate_rows <= 0))
    return kErrBadShape;
  const uintptr_t values = reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(gate) |
                           reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y);
  if (!aligned16(x) || !aligned16(weight) || (ldx & 7) != 0 || (ldw & 7) != 0 || (values & 1) != 0)
    return kErrMisaligned;
  if (m > 0x7fffff00 || n > 0x7fffff00 || k > 0x7fffff00) return kErrTooLarge;
  if (int rc = check_device_sm100()) return rc;
  lact::Epilogue e = {};
  e.m = m;
  e.n = n;
  e.act = activation;
  e.bias = bias;
  e.gate = gate;
  e.gate_rows = gate_rows;
  e.residual = residual;
  e.ld_res = ld_residual;
  e.y = y;
  e.ldy = ldy;
  e.vec_res = aligned16(residual) && (ld_residual & 7) == 0;
  e.vec_y = aligned16(y) && (ldy & 7) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == ERD_BF16
             ? lact::run<__nv_bfloat16, true>(e, x, ldx, weight, ldw, k, status, st)
             : lact::run<__half, false>(e, x, ldx, weight, ldw, k, status, st);
}
