// Matrix product with its epilogue on the sm_100a tensor cores:
//   y = residual + gate * act(x W^T + bias)
// BF16 or FP16 operands, FP32 accumulation in TMEM, every step of the epilogue
// in FP32, one rounding.  Any row count, any n; rows of x and W start on 16
// bytes (TMA), k is free.
//
// Three kernels, chosen by the host:
//   row_kernel    up to two rows: FP32 products of W's stream, no tensor cores.
//   pair_kernel   large products.  A persistent kernel of CTA pairs
//                 (cta_group::2), one 256 x 256 tile a pair: each CTA stages 128
//                 rows of x and half of W's tile, so an instruction reads W from
//                 both shared memories and a CTA loads 32 KB per 64-deep step
//                 for 128 x 256 outputs.  An accumulator is 256 TMEM columns, so
//                 two fit, and the epilogue of a tile runs beside the products of
//                 the next.  Where the last round of tiles would leave more than
//                 half of the pairs idle, its tiles are cut into 256 x 128.
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

// One lane of a converged warp.  The producer and issuer loops run behind this
// rather than behind `lane == 0`: the compiler then knows that one thread is
// active and keeps descriptors and barrier addresses in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// Place in a ring of shared-memory stages.
struct RingPlace {
  uint32_t s = 0, phase = 0;
  __device__ __forceinline__ void next(uint32_t stages) {
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
  __device__ __forceinline__ void back(uint32_t stages) {
    if (s == 0) {
      s = stages;
      phase ^= 1;
    }
    --s;
  }
};

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
// a few units in the last place of FP32 (a tanh instruction would keep 11 bits).  Below
// z = -87.3 the quotient's divisor passes 2^126 and the result is 0, where the value is
// under |x| 2^-126.
__device__ __forceinline__ float times_sigmoid(float x, float z) {
  return __fdividef(x, 1.0f + ex2_approx(-1.4426950408889634f * z));
}
// gelu with tanh: (1 + tanh(u)) / 2 = sigmoid(2 u), u = sqrt(2/pi) (x + 0.044715 x^3).
__device__ __forceinline__ float gelu_tanh(float x) {
  return times_sigmoid(x, x * fmaf(0.07135481283f, x * x, 1.5957691216f));
}
// exp(z^2) erfc(z) = t P(t), t = 1 / (1 + p z), z >= 0, to 2.5e-7 of itself
// (the form of Abramowitz and Stegun 7.1.25-26 with a P of degree 7 fitted by
// gen_erfcx_poly.py); kErfcxP is p / sqrt(2).
constexpr float kErfcxP = 0x1.33bb9ep-2f;
constexpr float kErfcx0 = 0x1.eae990p-3f;
constexpr float kErfcx1 = 0x1.ee7c9cp-3f;
constexpr float kErfcx2 = 0x1.a0356ap-3f;
constexpr float kErfcx3 = 0x1.f8f460p-3f;
constexpr float kErfcx4 = -0x1.638d84p-4f;
constexpr float kErfcx5 = 0x1.8ecc88p-2f;
constexpr float kErfcx6 = -0x1.35bb0ap-2f;
constexpr float kErfcx7 = 0x1.1a2760p-4f;
// gelu with the normal distribution function, x Phi(x): Phi(-|x|) =
// erfc(|x| / sqrt(2)) / 2 keeps its digits where 1 + erf would cancel, and
// costs 18 instructions and 2 MUFU where erfcf made the epilogue of a 2048-deep
// product longer than its tile's products (2.37 against 1.58 ms).
__device__ __forceinline__ float gelu_erf(float x) {
  const float t = __fdividef(1.0f, fmaf(kErfcxP, fabsf(x), 1.0f));
  float q = fmaf(kErfcx7, t, kErfcx6);
  q = fmaf(q, t, kErfcx5);
  q = fmaf(q, t, kErfcx4);
  q = fmaf(q, t, kErfcx3);
  q = fmaf(q, t, kErfcx2);
  q = fmaf(q, t, kErfcx1);
  q = fmaf(q, t, kErfcx0);
  const float below = 0.5f * q * t * ex2_approx(-0.72134752044448f * x * x);  // Phi(-|x|)
  const float y = fminf(x, 64.f) * below;  // at 64 `below` has long been 0; +inf * 0 is NaN
  return x > 0.f ? x - y : y;
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
  int vec_bias, vec_gate, vec_res, vec_y;  // rows start on 16 bytes
  int two_res, two_y;                      // rows start on 4 bytes
};

// Four values from column `col` of row `row` (what lies behind column n is 0).
template <typename T>
__device__ __forceinline__ uint2 load4(const void* base, long long ld, int vec, int row, int col,
                                       int n) {
  const T* p = static_cast<const T*>(base) + row * ld + col;
  if (vec && col + 4 <= n) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < n)
      w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
  return make_uint2(w[0], w[1]);
}
template <typename T>
__device__ __forceinline__ void store4(void* base, long long ld, int vec, int row, int col, int n,
                                       const uint2& v) {
  T* p = static_cast<T*>(base) + row * ld + col;
  if (vec && col + 4 <= n) {
    *reinterpret_cast<uint2*>(p) = v;
    return;
  }
  const uint32_t w[2] = {v.x, v.y};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < n)
      reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
}

constexpr int kPiece = 64;                    // columns an epilogue warp takes at a time
constexpr int kStageBytes = 32 * kPiece * 2;  // 32 rows of a piece, 16-byte chunks swizzled
constexpr int kSlabBytes = 2 * kPiece * 4;    // bias and gate of a piece as floats

// Byte of value (row, column) in a staging block.
__device__ __forceinline__ int staged(int r, int c) {
  return r * 128 + (((c >> 3) ^ (r & 7)) * 16) + (c & 7) * 2;
}

// What an epilogue warp reads from global memory for one piece (32 rows x 64
// columns), requested a piece ahead so that its latency lies under the products
// or the arithmetic of the piece before.  With the loads behind the wait for
// the accumulator a gated residual took 2.54 instead of 1.58 ms at 65280 x 8192
// x 2048.
template <typename T>
struct Piece {
  int row0, col0;
  bool inside;     // every row and column exists and rows start on 16 bytes
  bool one_group;  // the 32 rows share a gate
  int group;
  T b[2], g[2];  // as they are: a conversion here would wait for them
  uint32_t res[32];

  __device__ __forceinline__ void request(const Epilogue& e, int row, int col, int lane) {
    row0 = row;
    col0 = col;
    const bool whole = row + 32 <= e.m && col + kPiece <= e.n;
    inside = whole && e.vec_y && (e.residual == nullptr || e.vec_res);
    group = 0;
    one_group = true;
    if (e.gate != nullptr) {
      group = min(row + lane, e.m - 1) / e.gate_rows;
      one_group = __all_sync(0xffffffffu, group == __shfl_sync(0xffffffffu, group, 0));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = col + lane + 32 * i;
      b[i] = T(0.f);
      g[i] = T(1.f);
      if (c < e.n) {
        if (e.bias != nullptr) b[i] = static_cast<const T*>(e.bias)[c];
        if (e.gate != nullptr && one_group)
          g[i] = static_cast<const T*>(e.gate)[static_cast<long long>(group) * e.n + c];
      }
    }
    if (e.residual != nullptr) {
      const int r = row + (lane >> 3), c = col + (lane & 7) * 8;
      if (inside) {
        const T* p = static_cast<const T*>(e.residual) + r * e.ld_res + c;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * q * e.ld_res);
          res[4 * q] = v.x, res[4 * q + 1] = v.y, res[4 * q + 2] = v.z, res[4 * q + 3] = v.w;
        }
      } else if (e.two_res) {  // a row an instruction, two values a lane
        const int c2 = col + 2 * lane, rows = min(32, e.m - row);
        const uint16_t* p = static_cast<const uint16_t*>(e.residual) + row * e.ld_res + c2;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          res[q] = 0u;
          if (q < rows) {
            if (c2 + 1 < e.n)
              res[q] = *reinterpret_cast<const uint32_t*>(p + q * e.ld_res);
            else if (c2 < e.n)
              res[q] = p[q * e.ld_res];
          }
        }
      }
    }
  }

  // First half: the requested values move to shared memory, which frees the
  // registers for the next request.
  __device__ __forceinline__ void park(const Epilogue& e, uint8_t* stage, float* slab, int lane) {
    const int sub = lane >> 3, chunk = lane & 7;  // row within a group of 4, 16-byte chunk
    if (e.residual != nullptr && inside) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int rr = 4 * q + sub;
        *reinterpret_cast<uint4*>(stage + rr * 128 + ((chunk ^ (rr & 7)) * 16)) =
            make_uint4(res[4 * q], res[4 * q + 1], res[4 * q + 2], res[4 * q + 3]);
      }
    } else if (e.residual != nullptr && e.two_res) {
#pragma unroll
      for (int q = 0; q < 32; ++q)
        *reinterpret_cast<uint32_t*>(stage + staged(q, 2 * lane)) = res[q];
    } else if (e.residual != nullptr) {
      // rows on odd values: one by one, 32 neighbouring ones a warp, 32 requests at a
      // time (four at a time took 184 us at 9907 x 1447 x 1184)
      const int rows = min(32, e.m - row0);
      const uint16_t* p =
          static_cast<const uint16_t*>(e.residual) + row0 * e.ld_res + col0 + lane;
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 16) {
        uint16_t v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int rr = r0 + (i >> 1), c = 32 * (i & 1);
          v[i] = rr < rows && col0 + lane + c < e.n ? p[rr * e.ld_res + c] : 0;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i)
          *reinterpret_cast<uint16_t*>(stage + staged(r0 + (i >> 1), lane + 32 * (i & 1))) = v[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      slab[lane + 32 * i] = to_float(b[i]);
      slab[kPiece + lane + 32 * i] = to_float(g[i]);
    }
    __syncwarp();
  }
};

// One piece: a lane owns a row of it, adds up its 64 columns from TMEM and the
// parked values, and leaves the result in the staging block, from where the
// warp stores 128 bytes of a row at a time (four whole lines an instruction
// instead of 32 pieces of 16 bytes).
template <typename T>
__device__ __forceinline__ void finish_piece(const Epilogue& e, uint32_t taddr, int row0, int col0,
                                             bool inside, bool one_group, int group,
                                             uint8_t* stage, const float* slab, int lane) {
  const int sub = lane >> 3, chunk = lane & 7;
  uint8_t* own = stage + lane * 128;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {  // 32 columns at a time
    uint32_t r[32];
    tmem_ld_wait_32(taddr + h * 32, r);
    float v[32];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = reinterpret_cast<const float4*>(slab)[h * 8 + i];
      v[4 * i] = __uint_as_float(r[4 * i]) + b.x;
      v[4 * i + 1] = __uint_as_float(r[4 * i + 1]) + b.y;
      v[4 * i + 2] = __uint_as_float(r[4 * i + 2]) + b.z;
      v[4 * i + 3] = __uint_as_float(r[4 * i + 3]) + b.w;
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
        const T* g = static_cast<const T*>(e.gate) + static_cast<long long>(group) * e.n + col0;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (col0 + h * 32 + i < e.n) v[i] *= to_float(g[h * 32 + i]);
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
  const int r = row0 + sub, c = col0 + chunk * 8;
  if (inside) {
    T* p = static_cast<T*>(e.y) + r * e.ldy + c;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<uint4*>(p + 4 * q * e.ldy) = *reinterpret_cast<const uint4*>(
          stage + (4 * q + sub) * 128 + ((chunk ^ ((4 * q + sub) & 7)) * 16));
  } else if (e.two_y) {
    const int c2 = col0 + 2 * lane, rows = min(32, e.m - row0);
    uint16_t* p = static_cast<uint16_t*>(e.y) + row0 * e.ldy + c2;
#pragma unroll 4
    for (int q = 0; q < rows; ++q) {
      const uint32_t v = *reinterpret_cast<const uint32_t*>(stage + staged(q, 2 * lane));
      if (c2 + 1 < e.n)
        *reinterpret_cast<uint32_t*>(p + q * e.ldy) = v;
      else if (c2 < e.n)
        p[q * e.ldy] = static_cast<uint16_t>(v);
    }
  } else {
    // rows on odd values: one by one, 32 neighbouring ones a warp (pieces of 16
    // bytes, whose values are apart by lanes, took twice the time of the products)
    const int rows = min(32, e.m - row0);
#pragma unroll 4
    for (int i = 0; i < 2 * rows; ++i) {
      const int rr = i >> 1, cc = lane + 32 * (i & 1);
      if (col0 + cc < e.n)
        static_cast<uint16_t*>(e.y)[(row0 + rr) * e.ldy + col0 + cc] =
            *reinterpret_cast<const uint16_t*>(stage + staged(rr, cc));
    }
  }
  __syncwarp();
}

// ---------------------------------------------------------------- pair kernel
constexpr int kPairEpilogueWarps = 8;
constexpr int kPairThreads = 32 * (2 + kPairEpilogueWarps);
constexpr int kPairRows = 256;                      // rows of a pair's tile
constexpr int kPairABytes = 128 * kRowBytes;        // x of one CTA and stage
constexpr int kPairStages = 5;
constexpr int kPairBBytes = 128 * kRowBytes;        // W of one CTA and stage (wide tile)

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
constexpr int kPairSmemB = kPairSmemA + kPairStages * kPairABytes;
constexpr int kPairSmemStage = kPairSmemB + kPairStages * kPairBBytes;
constexpr int kPairSmemSlab = kPairSmemStage + kPairEpilogueWarps * kStageBytes;
constexpr int kPairSmemBar = kPairSmemSlab + kPairEpilogueWarps * kSlabBytes;
constexpr int kPairSmemLaunch = kPairSmemBar + 1024 + 1024;  // + base alignment
static_assert(kPairSmemLaunch <= 227 * 1024, "shared memory budget");

struct PairParams {
  Epilogue e;
  int k, tiles_m, tiles_n;
  int wide;   // tiles that are taken whole
  int items;  // these and the halves of the others
  int* status;
};

// The tile of an item: its first row and column, and whether it is 256 or 128
// columns wide.  Pairs take tiles in bands of kBand tile rows, column by column
// within a band, so that the tiles in flight form a block that reads few distinct
// rows of x and of W.
constexpr int kBand = 8;
struct PairTile {
  int m0, n0;
  bool wide;
};
__device__ __forceinline__ PairTile pair_tile(const PairParams& p, int item) {
  const bool whole = item < p.wide;
  const int tile = whole ? item : p.wide + ((item - p.wide) >> 1);
  const int band = tile / (kBand * p.tiles_n);
  const int rows = min(kBand, p.tiles_m - band * kBand);
  const int r = tile - band * kBand * p.tiles_n;
  const int tn = r / rows;
  PairTile t;
  t.m0 = (band * kBand + r - tn * rows) * kPairRows;
  t.n0 = tn * 256 + (whole ? 0 : ((item - p.wide) & 1) * 128);
  t.wide = whole && p.e.n - t.n0 > 128;  // a narrow last column is a narrow tile
  return t;
}

template <typename T, bool kBf16>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmap_a,
                const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_b_half, const PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  PairBarriers* bars = reinterpret_cast<PairBarriers*>(smem + kPairSmemBar);
  const uint32_t sA = smem_u32(smem + kPairSmemA);
  const uint32_t sB = smem_u32(smem + kPairSmemB);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
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
    if (elect_one()) {
      tma_prefetch_desc(&tmap_a);
      tma_prefetch_desc(&tmap_b);
      tma_prefetch_desc(&tmap_b_half);
      RingPlace at;
      uint32_t issued = 0;
      bool ok = true;
      const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
      const uint32_t leader0 = map_rank(full0, 0);
      for (int item = pair; ok && item < p.items; item += pairs) {
        const PairTile t = pair_tile(p, item);
        const int m0 = t.m0 + static_cast<int>(rank) * 128;
        const int n0 = t.n0 + static_cast<int>(rank) * (t.wide ? 128 : 64);
        const CUtensorMap* map_w = t.wide ? &tmap_b : &tmap_b_half;
        const uint32_t bytes = 2 * (kPairABytes + (t.wide ? kPairBBytes : kPairBBytes / 2));
        for (int k0 = 0; k0 < p.k; k0 += kBK) {
          if (!mbar_wait(empty0 + 8 * at.s, at.phase ^ 1, abort, p.status,
                         kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          // The leader announces the bytes of both CTAs.  The other CTA's may
          // land first: the phase cannot end before the leader's arrival.
          if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * at.s, bytes);
          const uint32_t bar = leader0 + 8 * at.s;
          tma_load_2d_pair(sA + at.s * kPairABytes, &tmap_a, bar, k0, m0);
          tma_load_2d_pair(sB + at.s * kPairBBytes, map_w, bar, k0, n0);
          at.next(kPairStages);
          ++issued;
        }
      }
      if (*abort && rank == 0) {
        // Let the loads that may be in flight land before exiting.
        for (uint32_t d = 0; d < kPairStages && d < issued; ++d) {
          at.back(kPairStages);
          mbar_wait_drain(full0 + 8 * at.s, at.phase);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer (the leader)
    if (rank == 0 && elect_one()) {
      // Descriptors of stage 0; a stage or 32 bytes of K further is an addition
      // to the address field (16-byte units).
      const uint64_t da0 = sdesc_sw128(sA, 16, 1024), db0 = sdesc_sw128(sB, 16, 1024);
      const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
      RingPlace at;
      uint32_t count = 0;
      bool ok = true;
      for (int item = pair; ok && item < p.items; item += pairs, ++count) {
        const uint32_t id =
            pair_tile(p, item).wide ? idesc<kBf16>(256, 256) : idesc<kBf16>(256, 128);
        const uint32_t buf = count & 1;
        if (!mbar_wait(smem_u32(&bars->acc_empty[buf]), ((count >> 1) & 1) ^ 1, abort, p.status,
                       kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        uint32_t acc = 0;
        for (int k0 = 0; k0 < p.k; k0 += kBK) {
          if (!mbar_wait(full0 + 8 * at.s, at.phase, abort, p.status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = da0 + at.s * (kPairABytes / 16);
          const uint64_t db = db0 + at.s * (kPairBBytes / 16);
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            mma_pair_ss(d, da + 2 * k4, db + 2 * k4, id, acc);
            acc = 1;
          }
          mma_commit_pair(empty0 + 8 * at.s);
          at.next(kPairStages);
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
    // This warp's corner of a tile: 32 rows, half of the columns.  Pieces without
    // rows or columns are skipped.
    PairTile t;
    int row0, col0;
    auto corner = [&](int item) {
      t = pair_tile(p, item);
      row0 = t.m0 + static_cast<int>(rank) * 128 + quad * 32;
      col0 = t.n0 + half * (t.wide ? 128 : 64);
    };
    Piece<T> piece;
    if (pair < p.items) {
      corner(pair);
      if (row0 < p.e.m && col0 < p.e.n) piece.request(p.e, row0, col0, lane);
    }
    uint32_t count = 0;
    for (int item = pair; item < p.items; item += pairs, ++count) {
      const uint32_t buf = count & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->acc_full[buf]), (count >> 1) & 1,
                                             abort, p.status, kStatusTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int pieces = t.wide ? 2 : 1;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + buf * 256 +
                             half * (t.wide ? 128 : 64);
#pragma unroll 1
      for (int c = 0; c < pieces; ++c) {
        const bool any = row0 < p.e.m && col0 + c * kPiece < p.e.n;
        const int row = row0, col = col0 + c * kPiece;
        const bool inside = piece.inside, one_group = piece.one_group;
        const int group = piece.group;
        if (any) piece.park(p.e, stage, slab, lane);
        // the next piece, of this tile or the next
        const bool last = c == pieces - 1;
        if (last && item + pairs < p.items) corner(item + pairs);
        if (!last || item + pairs < p.items) {
          const int next = col0 + (last ? 0 : kPiece);
          if (row0 < p.e.m && next < p.e.n) piece.request(p.e, row0, next, lane);
        }
        if (any)
          finish_piece<T>(p.e, taddr + c * kPiece, row, col, inside, one_group, group, stage, slab,
                          lane);
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
constexpr int kSplitEpilogueWarps = 8;  // two for each quarter of the rows
constexpr int kSplitThreads = 32 * (2 + kSplitEpilogueWarps);
constexpr int kSplitMaxStages = 20;
// Clusters of eight leave multiprocessors of a group idle (15 fit at a time
// with one CTA each), so their CTAs came in two waves.
constexpr int kMaxSplits = 4;

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
  int direct;   // one part whose warps finish their rows from TMEM
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

// Bias, gate and residual of four columns of one row.
template <typename T>
struct Side {
  uint2 bias, gate, res;
  __device__ __forceinline__ void request(const Epilogue& e, int row, int col) {
    bias = gate = res = make_uint2(0u, 0u);
    if (e.bias != nullptr) bias = load4<T>(e.bias, 0, e.vec_bias, 0, col, e.n);
    if (e.gate != nullptr)
      gate = load4<T>(e.gate, e.n, e.vec_gate, row / e.gate_rows, col, e.n);
    if (e.residual != nullptr) res = load4<T>(e.residual, e.ld_res, e.vec_res, row, col, e.n);
  }
};

// 16-byte chunk `c4` of row `r` of the partial sums, swizzled so that the 32
// rows a warp writes at a time do not meet in the same banks.
template <int BN>
__device__ __forceinline__ int partial_offset(int r, int c4) {
  return r * (BN * 4) + ((c4 ^ (r & 7)) * 16);
}

template <typename T, bool kBf16, int BN>
__global__ void __launch_bounds__(kSplitThreads, 1)
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
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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

  // Unless the accumulator is finished in place: the four-column chunks of the
  // tile that this CTA finishes; what a thread's first one needs is requested now.
  constexpr int kRowChunks = BN / 4;
  const int chunks = min(128, p.e.m - m0) * kRowChunks;
  const int share_lo = static_cast<int>(static_cast<long long>(chunks) * split / p.splits);
  const int share_hi = static_cast<int>(static_cast<long long>(chunks) * (split + 1) / p.splits);
  Side<T> side;
  if (!p.direct) {
    const int i = share_lo + static_cast<int>(threadIdx.x);
    if (i < share_hi && n0 + i % kRowChunks * 4 < p.e.n)
      side.request(p.e, m0 + i / kRowChunks, n0 + i % kRowChunks * 4);
  }

  bool have = false;  // this warp's rows of the accumulator may be read
  if (warp == 0) {
    if (elect_one()) {
      const uint32_t tx = static_cast<uint32_t>(p.a_rows * kRowBytes + S::kBBytes);
      const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
      const uint32_t stages = static_cast<uint32_t>(p.stages);
      RingPlace at;
      uint32_t issued = 0;
      for (int kk = k_lo; kk < k_hi; ++kk) {
        if (!mbar_wait(empty0 + 8 * at.s, at.phase ^ 1, abort, p.status, kStatusTimeoutProducer))
          break;
        const uint32_t full = full0 + 8 * at.s;
        mbar_arrive_expect_tx(full, tx);
        tma_load_2d(sB + at.s * S::kBBytes, &tmap_b, full, kk * kBK, n0);
        tma_load_2d(sA + at.s * a_bytes, &tmap_a, full, kk * kBK, m0);
        at.next(stages);
        ++issued;
      }
      if (*abort) {
        for (uint32_t d = 0; d < stages && d < issued; ++d) {
          at.back(stages);
          mbar_wait_drain(full0 + 8 * at.s, at.phase);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t id = idesc<kBf16>(128, BN);
      const uint64_t da0 = sdesc_sw128(sA, 16, 1024), db0 = sdesc_sw128(sB, 16, 1024);
      const uint32_t full0 = smem_u32(&bars->full[0]), empty0 = smem_u32(&bars->empty[0]);
      const uint32_t stages = static_cast<uint32_t>(p.stages);
      RingPlace at;
      uint32_t acc = 0;
      for (int kk = k_lo; kk < k_hi; ++kk) {
        if (!mbar_wait(full0 + 8 * at.s, at.phase, abort, p.status, kStatusTimeoutMma)) break;
        tc_fence_after();
        const uint64_t da = da0 + at.s * static_cast<uint32_t>(a_bytes / 16);
        const uint64_t db = db0 + at.s * (S::kBBytes / 16);
        // Rows of the product beyond the x box read whatever the shared memory
        // behind it holds; their accumulator lanes are never read.
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          mma_bf16_ss(tmem, da + 2 * k4, db + 2 * k4, id, acc);
          acc = 1;
        }
        mma_commit(empty0 + 8 * at.s);
        at.next(stages);
      }
      mma_commit(smem_u32(&bars->acc_full));
      mbar_wait_drain(smem_u32(&bars->acc_full), 0);
    }
  } else {
    // A quarter of the rows and, of the columns, one half (a 64-column tile that is
    // finished in place is one piece, and the second warp has none).
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int row0 = m0 + quad * 32, piece_col = half * kPiece;
    const bool mine = row0 < p.e.m && piece_col < BN && n0 + piece_col < p.e.n;
    Piece<T> piece;
    if (p.direct && mine) piece.request(p.e, row0, n0 + piece_col, lane);
    have = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->acc_full), 0, abort, p.status,
                                             kStatusTimeoutEpilogue));
    // A reduction that was cut short has set the flag before it committed.
    have = have && __all_sync(0xffffffffu, *abort == 0);
    tc_fence_after();
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    if (have && p.direct && mine) {
      uint8_t* stage = tail + (warp - 2) * kStageBytes;
      float* slab = reinterpret_cast<float*>(tail + kSplitEpilogueWarps * kStageBytes +
                                             (warp - 2) * kSlabBytes);
      piece.park(p.e, stage, slab, lane);
      finish_piece<T>(p.e, taddr + piece_col, row0, n0 + piece_col, piece.inside, piece.one_group,
                      piece.group, stage, slab, lane);
    } else if (have && !p.direct && row0 < p.e.m) {
      // The ring is free: every load has been consumed by a finished product.
      const int r = quad * 32 + lane;
#pragma unroll 1
      for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
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
  tc_fence_before();
  if (p.direct) {
    __syncthreads();
  } else {
    cluster_sync();
    // Each CTA adds and finishes its share of the tile, four columns a thread, so
    // that a warp reads 512 neighbouring bytes of a peer.  A split that gave up has
    // set the status word; its partial sums are stale and the tile's values are then
    // as undefined as those of any timed-out call.
    const uint32_t base = smem_u32(smem);
    for (int i = share_lo + static_cast<int>(threadIdx.x); i < share_hi; i += kSplitThreads) {
      const int r = i / kRowChunks, c4 = i % kRowChunks;
      const int row = m0 + r, col = n0 + c4 * 4;
      if (col >= p.e.n) continue;
      // All requests first: one round trip over the cluster, not one per part.
      float4 a[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        if (s < p.splits)
          a[s] = ld_cluster(map_rank(base, static_cast<uint32_t>(s)) + partial_offset<BN>(r, c4));
      if (i >= share_lo + kSplitThreads) side.request(p.e, row, col);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        if (s < p.splits) v[0] += a[s].x, v[1] += a[s].y, v[2] += a[s].z, v[3] += a[s].w;
      const uint32_t bias[2] = {side.bias.x, side.bias.y};
      const uint32_t gate[2] = {side.gate.x, side.gate.y};
      const uint32_t res[2] = {side.res.x, side.res.y};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 f = unpack2<T>(bias[j]);
        v[2 * j] += f.x;
        v[2 * j + 1] += f.y;
      }
      activate(v, p.e.act);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (p.e.gate != nullptr) {
          const float2 g = unpack2<T>(gate[j]);
          v[2 * j] *= g.x;
          v[2 * j + 1] *= g.y;
        }
        const float2 f = unpack2<T>(res[j]);
        v[2 * j] += f.x;
        v[2 * j + 1] += f.y;
      }
      store4<T>(p.e.y, p.e.ldy, p.e.vec_y, row, col, p.e.n,
                make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])));
    }
    cluster_sync();  // the peers have read this CTA's sums
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

// ----------------------------------------------------------------- row kernel
// A few rows (at most 2) are a stream over W: a warp takes four columns (rows
// of W), its lanes 16 bytes of each at a time, and multiplies them with every
// row of x in FP32.  No barrier, TMEM or cluster set-up stands before the first
// load.  The reduction may be shared by several warps of the block (their sums
// are added in warp order).
constexpr int kRowWarps = 8;
constexpr int kRowCols = 4;
constexpr int kRowMax = 2;

template <typename T, int M>
__global__ void __launch_bounds__(32 * kRowWarps)
    row_kernel(const Epilogue e, const T* __restrict__ x, long long ldx, const T* __restrict__ w,
               long long ldw, int k, int share) {
  constexpr int V = M * kRowCols;  // sums of a warp
  __shared__ float sums[kRowWarps][V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % share;
  const int col0 =
      static_cast<int>(blockIdx.x * (kRowWarps / share) + warp / share) * kRowCols;
  const T* wr[kRowCols];
  const T* xr[M];
#pragma unroll
  for (int r = 0; r < kRowCols; ++r) wr[r] = w + min(col0 + r, e.n - 1) * ldw;
#pragma unroll
  for (int i = 0; i < M; ++i) xr[i] = x + min(i, e.m - 1) * ldx;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;

  auto add = [&](const uint4 (&wv)[kRowCols], const uint4 (&xv)[M]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float2 wf[kRowCols];
#pragma unroll
      for (int r = 0; r < kRowCols; ++r)
        wf[r] = unpack2<T>(q == 0 ? wv[r].x : q == 1 ? wv[r].y : q == 2 ? wv[r].z : wv[r].w);
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const float2 xf =
            unpack2<T>(q == 0 ? xv[i].x : q == 1 ? xv[i].y : q == 2 ? xv[i].z : xv[i].w);
#pragma unroll
        for (int r = 0; r < kRowCols; ++r)
          acc[i * kRowCols + r] =
              fmaf(xf.y, wf[r].y, fmaf(xf.x, wf[r].x, acc[i * kRowCols + r]));
      }
    }
  };
  const int chunks = k / 8, step = 32 * share;
  int c = part * 32 + lane;
  constexpr int U = 4;  // chunks requested at a time
#pragma unroll 1
  for (; c + (U - 1) * step < chunks; c += U * step) {
    uint4 wv[U][kRowCols], xv[U][M];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int r = 0; r < kRowCols; ++r)
        wv[u][r] = *reinterpret_cast<const uint4*>(wr[r] + (c + u * step) * 8LL);
#pragma unroll
      for (int i = 0; i < M; ++i)
        xv[u][i] = *reinterpret_cast<const uint4*>(xr[i] + (c + u * step) * 8LL);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) add(wv[u], xv[u]);
  }
#pragma unroll 1
  for (; c < chunks; c += step) {
    uint4 wv[kRowCols], xv[M];
#pragma unroll
    for (int r = 0; r < kRowCols; ++r) wv[r] = *reinterpret_cast<const uint4*>(wr[r] + c * 8LL);
#pragma unroll
    for (int i = 0; i < M; ++i) xv[i] = *reinterpret_cast<const uint4*>(xr[i] + c * 8LL);
    add(wv, xv);
  }
  if (part == 0 && lane < k - chunks * 8) {  // what lies behind k may not be read
    const int kk = chunks * 8 + lane;
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int r = 0; r < kRowCols; ++r)
        acc[i * kRowCols + r] =
            fmaf(to_float(xr[i][kk]), to_float(wr[r][kk]), acc[i * kRowCols + r]);
  }
  // Sums over the lanes: halve the values a lane is responsible for while there
  // are several, then add what is left; value i ends in the lanes whose top
  // log2(V) bits are i.
  int left = V, mine = 0;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    if (left > 1) {
      left /= 2;
      const bool hi = (lane & d) != 0;
      mine += hi ? left : 0;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if (i < left) {
          const float keep = hi ? acc[i + left] : acc[i];
          const float give = hi ? acc[i] : acc[i + left];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
        }
      }
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], d);
    }
  }
  constexpr int kDup = 32 / V;  // lanes that hold the same value
  if (share > 1) {
    if (lane % kDup == 0) sums[warp][mine] = acc[0];
    __syncthreads();
    if (part != 0) return;
    acc[0] = 0.f;
    for (int s = 0; s < share; ++s) acc[0] += sums[warp + s][mine];
  }
  const int row = mine / kRowCols, col = col0 + mine % kRowCols;
  if (lane % kDup != 0 || row >= e.m || col >= e.n) return;
  float v[1] = {acc[0]};
  if (e.bias != nullptr) v[0] += to_float(static_cast<const T*>(e.bias)[col]);
  activate(v, e.act);
  if (e.gate != nullptr)
    v[0] *= to_float(static_cast<const T*>(e.gate)[static_cast<long long>(row / e.gate_rows) * e.n +
                                                   col]);
  if (e.residual != nullptr) v[0] += to_float(static_cast<const T*>(e.residual)[row * e.ld_res + col]);
  const uint32_t packed = pack2<T>(v[0], 0.f);
  static_cast<uint16_t*>(e.y)[row * e.ldy + col] = static_cast<uint16_t>(packed);
}

// ------------------------------------------------------------------ host side
struct Plan {
  bool pair;
  int bn, splits, a_rows;
};

// Which kernel for more than kRowMax rows, and how a small product is cut: the
// least estimated time, in clocks, of
//   the pair kernel: 512 a 64-deep step and round of sms / 2 tiles, 300 for a last
//   round of half tiles;
//   the split kernel with 64 or 128 columns and 1, 2 or 4 parts, one wave of CTAs
//   (its steps wait for L2, and parts add a round trip through the cluster).
Plan pick_plan(int m, int n, int k, int sms) {
  const long long ksteps = (k + kBK - 1) / kBK;
  auto waves = [](long long tiles, long long at_once) { return (tiles + at_once - 1) / at_once; };
  Plan best = {};
  long long least = -1;
  auto offer = [&](bool pair, int bn, int splits, long long cost) {
    if (least >= 0 && cost >= least) return;
    least = cost;
    best.pair = pair;
    best.bn = bn;
    best.splits = splits;
  };
  {
    const long long tiles = ((m + 255LL) / 256) * ((n + 255LL) / 256), pairs = sms / 2;
    const long long whole = tiles / pairs, rest = tiles % pairs;
    const long long last = rest == 0 ? 0 : 2 * rest <= pairs ? 300 : 512;
    offer(true, 256, 1, ksteps * (whole * 512 + last) + 9000);
  }
  for (int bn = 64; bn <= 128; bn += 64) {
    const long long tiles = ((m + 127LL) / 128) * ((n + bn - 1LL) / bn);
    for (int splits = 1; splits <= kMaxSplits; splits *= 2) {
      if (splits > 1 && (ksteps < 4 * splits || tiles * splits > sms)) break;
      const long long steps = (ksteps + splits - 1) / splits;
      offer(false, bn, splits,
            waves(tiles * splits, sms) * (steps * (bn == 64 ? 270 : 300) + 3000) + 3000 +
                (splits > 1 ? 2500 : 0));
    }
  }
  best.a_rows = m >= 128 ? 128 : (m + 7) / 8 * 8;
  return best;
}

template <typename T, bool kBf16>
int launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb_half,
                PairParams p, int sms, cudaStream_t st) {
  const long long tm = (p.e.m + 255LL) / 256, tn = (p.e.n + 255LL) / 256, tiles = tm * tn;
  if (tiles > (1LL << 29)) return kErrTooLarge;
  const int pairs = sms / 2;
  const int rest = static_cast<int>(tiles % pairs);
  p.tiles_m = static_cast<int>(tm);
  p.tiles_n = static_cast<int>(tn);
  p.wide = static_cast<int>(tiles) - (2 * rest <= pairs ? rest : 0);
  p.items = p.wide + 2 * (static_cast<int>(tiles) - p.wide);
  cudaError_t e = cudaFuncSetAttribute(pair_kernel<T, kBf16>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmemLaunch);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int used = p.items < pairs ? p.items : pairs;
  pair_kernel<T, kBf16><<<static_cast<unsigned>(2 * used), kPairThreads, kPairSmemLaunch, st>>>(
      ta, tb, tb_half, p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, bool kBf16, int BN>
int launch_split(const CUtensorMap& ta, const CUtensorMap& tb, SplitParams p, const Plan& pl,
                 cudaStream_t st) {
  using S = SplitSmem<BN>;
  // Few rows or several parts: all threads finish four-column chunks of the sums
  // in shared memory (few rows would leave a whole piece to one or two warps,
  // some 3500 clocks).
  p.direct = pl.splits == 1 && p.e.m > 64;
  const int ksteps = (p.k + kBK - 1) / kBK;
  const int per_split = (ksteps + pl.splits - 1) / pl.splits;
  // One CTA a multiprocessor with as deep a ring as fits: three stages (two CTAs
  // a multiprocessor) left 0.47 us of load latency in every 64-deep step.
  const int budget = 227 * 1024 - S::kTail - 1024;
  p.stages = budget / S::ring(pl.a_rows, 1);
  if (p.stages > kSplitMaxStages) p.stages = kSplitMaxStages;
  if (p.stages > per_split) p.stages = per_split;
  // The ring, the 128 rows that a product reads from a stage's x box however
  // few were loaded, and the partial sums all end before the tail.
  p.tail = S::ring(pl.a_rows, p.stages);
  const int reach = (p.stages - 1) * S::a_bytes(pl.a_rows) + 128 * kRowBytes;
  if (p.tail < reach) p.tail = reach;
  if (!p.direct && p.tail < 128 * BN * 4) p.tail = 128 * BN * 4;
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
  if (e.m <= kRowMax) {
    // Enough warps to fill the device, each with two chunks a lane at least.
    const int groups = (e.n + kRowCols - 1) / kRowCols;
    int share = 1;
    while (share < kRowWarps && static_cast<long long>(groups) * share < 16LL * sms &&
           k >= 32 * 8 * 4 * share)
      share *= 2;
    const unsigned blocks =
        static_cast<unsigned>((groups + kRowWarps / share - 1) / (kRowWarps / share));
    const T* xt = static_cast<const T*>(x);
    const T* wt = static_cast<const T*>(w);
    if (e.m == 1)
      row_kernel<T, 1><<<blocks, 32 * kRowWarps, 0, st>>>(e, xt, ldx, wt, ldw, k, share);
    else
      row_kernel<T, 2><<<blocks, 32 * kRowWarps, 0, st>>>(e, xt, ldx, wt, ldw, k, share);
    return static_cast<int>(cudaGetLastError());
  }
  const Plan pl = pick_plan(e.m, e.n, k, sms);
  CUtensorMap ta, tb;
  if (pl.pair) {
    CUtensorMap tb_half;
    if (operand_map(&ta, kBf16, x, e.m, k, ldx, 128) ||
        operand_map(&tb, kBf16, w, e.n, k, ldw, 128) ||
        operand_map(&tb_half, kBf16, w, e.n, k, ldw, 64))
      return kErrTensorMap;
    const PairParams p = {e, k, 0, 0, 0, 0, status};
    return launch_pair<T, kBf16>(ta, tb, tb_half, p, sms, st);
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

extern "C" int erd_linear_act(const erd_linear_act_args* args, int* status, void* stream) {
  if (args == nullptr) return kErrNullPointer;
  const erd_linear_act_args& a = *args;
  if (a.struct_bytes != static_cast<int64_t>(sizeof(a))) return kErrBadShape;
  if (a.x == nullptr || a.weight == nullptr || a.y == nullptr) return kErrNullPointer;
  if ((a.dtype != ERD_BF16 && a.dtype != ERD_FP16) || a.activation < ERD_ACT_NONE ||
      a.activation > ERD_ACT_GELU_TANH || a.m <= 0 || a.n <= 0 || a.k <= 0 || a.ldx < a.k ||
      a.ldw < a.k || a.ldy < a.n || (a.residual != nullptr && a.ld_residual < a.n) ||
      (a.gate != nullptr && a.gate_rows <= 0))
    return kErrBadShape;
  auto address = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const uintptr_t values = address(a.bias) | address(a.gate) | address(a.residual) | address(a.y);
  if (!aligned16(a.x) || !aligned16(a.weight) || (a.ldx & 7) != 0 || (a.ldw & 7) != 0 ||
      (values & 1) != 0)
    return kErrMisaligned;
  if (a.m > 0x7fffff00 || a.n > 0x7fffff00 || a.k > 0x7fffff00) return kErrTooLarge;
  if (int rc = check_device_sm100()) return rc;
  lact::Epilogue e = {};
  e.m = a.m;
  e.n = a.n;
  e.act = a.activation;
  e.bias = a.bias;
  e.gate = a.gate;
  e.gate_rows = a.gate_rows;
  e.residual = a.residual;
  e.ld_res = a.ld_residual;
  e.y = a.y;
  e.ldy = a.ldy;
  e.vec_bias = aligned16(a.bias);
  e.two_res = (reinterpret_cast<uintptr_t>(a.residual) & 3) == 0 && (a.ld_residual & 1) == 0;
  e.two_y = (reinterpret_cast<uintptr_t>(a.y) & 3) == 0 && (a.ldy & 1) == 0;
  e.vec_gate = aligned16(a.gate) && (a.n & 7) == 0;
  e.vec_res = aligned16(a.residual) && (a.ld_residual & 7) == 0;
  e.vec_y = aligned16(a.y) && (a.ldy & 7) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.dtype == ERD_BF16
             ? lact::run<__nv_bfloat16, true>(e, a.x, a.ldx, a.weight, a.ldw, a.k, status, st)
             : lact::run<__half, false>(e, a.x, a.ldx, a.weight, a.ldw, a.k, status, st);
}
