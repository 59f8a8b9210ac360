// Attention over key blocks that a cheap score selects, head_dim 64, BF16 or
// FP16 on sm_100a:
//   score(I, J) = (sum_{i in I} q_i) . mean_{j in J, j < length} k_j     (FP64)
//   each query block I keeps its `topk` highest-scoring key blocks (ties: the
//   lowest index), and its queries attend the valid keys of those blocks.
// A query block is 128 queries (one tile of the tensor cores) or one query.
//
// The scores are sums in 64 bits so that the choice does not depend on the
// order of summation: sums of 64 or 128 16-bit values are exact or nearly so,
// and two blocks change places only where their scores agree to 1e-15.
//
// Steps (all on the caller's stream):
//   pool_kernel     one pass over k (and, for blocks of 128, q): block sums.
//                   Bound by memory; a caller that keeps the key means next to
//                   its keys (key_pool) skips it for single queries.
//   few_blocks_kernel   blocks of 128, at most 64 key blocks: scores and choice.
//   score_kernel    blocks of 128: scores = sums times means, FP64 tiles.
//   select_kernel   blocks of 128: one warp a row finds the topk-th key by
//                   bisection over the bits of the scores.
//   tile_attn_kernel    blocks of 128: tcgen05 attention over the chosen blocks.
//   row_kernel      single queries: scores, choice and a stream over the chosen
//                   blocks, split over a cluster when there are few rows.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <math_constants.h>

#include "../../include/eraserdit_b200.h"
#include "host_common.h"
#include "sm100_ptx.cuh"
#include "tmem_io.cuh"

namespace erd {
namespace btk {

constexpr int kDim = 64;       // head_dim
constexpr int kTile = 128;     // queries of a tile and keys of a step
constexpr int kHalf = 64;      // keys that are loaded (and chosen) together at least

// Most queries, keys and chosen blocks: the kernels' int indices step past these
// by at most 128.
constexpr int kMaxCount = 0x7fff0000;
constexpr float kMaxScale = 2.3e38f;  // times log2(e) it is finite

// ------------------------------------------------------------ small helpers
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
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = unpack2<T>(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

struct Strides {
  long long token, head, batch;
};

// Valid keys of a batch entry.
__device__ __forceinline__ int key_length(const int* lengths, int b, int kv_len) {
  return lengths == nullptr ? kv_len : min(max(__ldg(lengths + b), 0), kv_len);
}

// The kernels of one call follow each other by programmatic dependent launch: a
// kernel lets the next one start as soon as all of its own CTAs have, and the next
// one sets itself up and then waits here for the whole of the one before (and so,
// in turn, of those before that) before it touches what they write.
__device__ __forceinline__ void start_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------- block sums
struct PoolParams {
  const void* x;
  Strides st;
  int heads, len, block, blocks;
  const int* lengths;  // keys only; null: all
  int mean;            // divide by the number of summed tokens
  double* out;         // [batch][heads][blocks][64]
};

// One CTA sums one block of four heads: a lane eight channels (16 bytes) of a
// token, the warps take turns and their sums are added in order.  Eight warps
// where there are few blocks (3 x 2005 tokens: 31 us with one warp a block, 10
// with four, 7 with eight), four where the device is full anyway (32640 tokens x
// 32 heads: 54 against 59 us).
constexpr int kPoolWarps = 8;
template <typename T>
__device__ __forceinline__ void pool_block(const PoolParams& p, long long item,
                                           double (*part)[32][8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int hg = (p.heads + 3) / 4;
  const int h = static_cast<int>(item % hg) * 4 + lane / 8;
  const long long bn = item / hg;
  const int n = static_cast<int>(bn % p.blocks), b = static_cast<int>(bn / p.blocks);
  const int len = key_length(p.lengths, b, p.len);
  const int t0 = n * p.block, t1 = min(t0 + p.block, len);
  double sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.0;
  if (h < p.heads) {
    const T* src = static_cast<const T*>(p.x) + b * p.st.batch + h * p.st.head + (lane & 7) * 8;
    constexpr int U = 8;  // tokens requested together
    for (int t = t0 + warp; t < t1; t += U * warps) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tu = t + u * warps;
        v[u] = make_uint4(0u, 0u, 0u, 0u);  // adds zeros behind the end
        if (tu < t1) v[u] = *reinterpret_cast<const uint4*>(src + tu * p.st.token);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[8];
        unpack8<T>(v[u], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += static_cast<double>(f[i]);
      }
    }
  }
  if (warp > 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) part[warp - 1][lane][i] = sum[i];
  }
  __syncthreads();
  if (warp > 0 || h >= p.heads) return;
  for (int w = 0; w < warps - 1; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += part[w][lane][i];
  if (p.mean && t1 > t0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] /= static_cast<double>(t1 - t0);
  }
  double2* dst = reinterpret_cast<double2*>(
      p.out + ((static_cast<long long>(b) * p.heads + h) * p.blocks + n) * kDim + (lane & 7) * 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = make_double2(sum[2 * i], sum[2 * i + 1]);
}

template <typename T>
__global__ void __launch_bounds__(32 * kPoolWarps)
    pool_kernel(const PoolParams a, const PoolParams b, long long items_a) {
  __shared__ double part[kPoolWarps - 1][32][8];
  start_next();
  const long long item = blockIdx.x;
  if (item < items_a)
    pool_block<T>(a, item, part);
  else
    pool_block<T>(b, item - items_a, part);
}

// ------------------------------------------------------------------- scores
// scores[b][h][g][n] = q_sum[b][h][g] . k_mean[b][h / per][n] on the FP64 matrix
// instruction (m8n8k4): 64 x 64 a CTA, 32 x 32 a warp.  Rows are padded to 68
// doubles, so the fragments' reads meet no bank twice.
constexpr int kScoreTile = 64, kScorePitch = kDim + 4;
constexpr int kScoreSmem = 2 * kScoreTile * kScorePitch * 8;

__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
               : "+d"(d[0]), "+d"(d[1])
               : "d"(a), "d"(b));
}

__global__ void __launch_bounds__(128)
    score_kernel(const double* q_sum, const double* k_mean, double* scores, int heads, int per,
                 int groups, int blocks) {
  extern __shared__ double tiles[];  // [64 groups][68], [64 blocks][68]
  double* sq = tiles;
  double* sk = tiles + kScoreTile * kScorePitch;
  const int n0 = blockIdx.x * kScoreTile, g0 = blockIdx.y * kScoreTile;
  const int bh = blockIdx.z;
  const int b = bh / heads, h = bh - b * heads;
  const long long kv = static_cast<long long>(b) * (heads / per) + h / per;
  const double* qg = q_sum + static_cast<long long>(bh) * groups * kDim;
  const double* kg = k_mean + kv * blocks * kDim;
  start_next();
  wait_previous();
  for (int i = threadIdx.x; i < kScoreTile * kDim / 2; i += 128) {
    const int r = i / (kDim / 2), c = i % (kDim / 2) * 2;
    double2 q = make_double2(0.0, 0.0), k = make_double2(0.0, 0.0);
    if (g0 + r < groups)
      q = *reinterpret_cast<const double2*>(qg + (g0 + r) * static_cast<long long>(kDim) + c);
    if (n0 + r < blocks)
      k = *reinterpret_cast<const double2*>(kg + (n0 + r) * static_cast<long long>(kDim) + c);
    *reinterpret_cast<double2*>(sq + r * kScorePitch + c) = q;
    *reinterpret_cast<double2*>(sk + r * kScorePitch + c) = k;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wm = (warp & 1) * 32, wn = (warp >> 1) * 32;
  double acc[4][4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = 0.0;
  const double* qa = sq + (wm + lane / 4) * kScorePitch + lane % 4;
  const double* kb = sk + (wn + lane / 4) * kScorePitch + lane % 4;
#pragma unroll 4
  for (int d = 0; d < kDim; d += 4) {
    double a[4], k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = qa[i * 8 * kScorePitch + d];
      k[i] = kb[i * 8 * kScorePitch + d];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_f64(acc[i][j], a[i], k[j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int g = g0 + wm + i * 8 + lane / 4;
    if (g >= groups) continue;
    double* dst = scores + (static_cast<long long>(bh) * groups + g) * blocks;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + wn + j * 8 + lane % 4 * 2;
      if (n < blocks) dst[n] = acc[i][j][0];
      if (n + 1 < blocks) dst[n + 1] = acc[i][j][1];
    }
  }
}

// ---------------------------------------------------------------- selection
// Order-preserving key of a score: greater score, greater key; -0 is 0, NaN is
// below every number.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) return 0ull;
  const unsigned long long u =
      static_cast<unsigned long long>(__double_as_longlong(s + 0.0));
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// One warp writes the indices of the `take` greatest of n scores (ties: lowest
// index; NaN below every number) in ascending order, then -1 up to topk.
// `score(i)` gives score i.
//
// With kPer > 0 (n <= 32 kPer) the scores stay in registers, rounded to FP32, and
// the threshold is bisected between the smallest and the greatest: rounding keeps
// the order, so a threshold that exactly `take` rounded scores reach splits the
// scores as they are.  That ends after about log2 of (range / gap at the
// threshold) steps, ten at 510 blocks, where the bits of the scores from the top
// took twenty.  Where FP32 cannot split them (ties, infinities, n > 32 kPer) the
// bits of the keys decide, upper words first, lower words where those tie.
template <int kPer, typename Score>
__device__ __forceinline__ void select_topk(Score score, int n, int take, int topk, int* out,
                                            int lane) {
  const int rounds = (n + 31) / 32;
  const uint32_t before = (1u << lane) - 1;
  for (int i = take + lane; i < topk; i += 32) out[i] = -1;
  if (take >= n) {
    for (int i = lane; i < n; i += 32) out[i] = i;
    return;
  }
  if (kPer > 0) {
    float f[kPer > 0 ? kPer : 1];
    float lo = CUDART_INF_F, hi = -CUDART_INF_F;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = j * 32 + lane;
      f[j] = -CUDART_INF_F;
      if (i < n) {
        f[j] = __double2float_rn(score(i));
        finite = finite && fabsf(f[j]) < CUDART_INF_F;  // false for NaN
        lo = fminf(lo, f[j]);
        hi = fmaxf(hi, f[j]);
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    if (__all_sync(0xffffffffu, finite)) {
      // take < n scores reach no threshold above hi, all n reach lo
      for (int step = 0; step < 40; ++step) {
        const float mid = 0.5f * lo + 0.5f * hi;
        if (!(mid > lo && mid < hi)) break;
        int c = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) c += f[j] >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c == take) {
          int count = 0;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const bool yes = f[j] >= mid;
            const uint32_t mask = __ballot_sync(0xffffffffu, yes);
            if (yes) out[count + __popc(mask & before)] = j * 32 + lane;
            count += __popc(mask);
          }
          return;
        }
        (c > take ? lo : hi) = mid;
      }
    }
  }
  // Keys of the scores: the greatest t whose upper word at least `take` keys
  // reach, then the greatest lower word that as many reach as are still wanted.
  auto count_keys = [&](auto reaches) {
    int c = 0;
    for (int j = 0; j < rounds; ++j) {
      const int i = j * 32 + lane;
      c += i < n && reaches(score_key(score(i)));
    }
    return __reduce_add_sync(0xffffffffu, c);
  };
  uint32_t t = 0, low = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t up = t | (1u << bit);
    if (count_keys([&](unsigned long long k) { return static_cast<uint32_t>(k >> 32) >= up; }) >=
        take)
      t = up;
  }
  const int want =
      take - count_keys([&](unsigned long long k) { return static_cast<uint32_t>(k >> 32) > t; });
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t up = low | (1u << bit);
    if (count_keys([&](unsigned long long k) {
          return static_cast<uint32_t>(k >> 32) == t && static_cast<uint32_t>(k) >= up;
        }) >= want)
      low = up;
  }
  const unsigned long long bound = (static_cast<unsigned long long>(t) << 32) | low;
  // keys equal to the bound that are taken
  const int ties = take - count_keys([&](unsigned long long k) { return k > bound; });
  int count = 0, tied = 0;
  for (int j = 0; j < rounds; ++j) {
    const int i = j * 32 + lane;
    const unsigned long long k = i < n ? score_key(score(i)) : 0ull;
    const bool tie = i < n && k == bound;
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    const bool yes =
        (i < n && k > bound) || (tie && tied + __popc(tie_mask & before) < ties);
    tied += __popc(tie_mask);
    const uint32_t mask = __ballot_sync(0xffffffffu, yes);
    if (yes) out[count + __popc(mask & before)] = i;
    count += __popc(mask);
  }
}

constexpr int kSelectWarps = 4;
template <int kPer>
__global__ void __launch_bounds__(32 * kSelectWarps)
    select_kernel(const double* scores, int* selection, const int* lengths, long long rows,
                  long long rows_per_batch, int blocks, int kv_len, int key_block, int topk) {
  start_next();
  wait_previous();
  const long long row = static_cast<long long>(blockIdx.x) * kSelectWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int len = key_length(lengths, static_cast<int>(row / rows_per_batch), kv_len);
  const int n = (len + key_block - 1) / key_block;
  const double* s = scores + row * blocks;
  select_topk<kPer>([&](int i) { return s[i]; }, n, min(topk, n), topk,
                    selection + row * topk, threadIdx.x & 31);
}

// Scores and choice in one kernel where a row's scores are one tile (64 blocks): 16
// query blocks a CTA, 16 x 16 scores and then four rows a warp.  One launch and one
// round trip through memory less: the whole call for 3 x 2005 queries and keys of 8
// heads with 16 blocks 38.4 -> 34.0 us, for 3 x 128 queries of 32 heads and 64 blocks
// 31.6 -> 24.8.  (With 64 rows a CTA each warp would choose for 16 rows in turn.)
constexpr int kFewGroups = 16;
__global__ void __launch_bounds__(128)
    few_blocks_kernel(const double* q_sum, const double* k_mean, int* selection,
                      const int* lengths, int heads, int per, int groups, int blocks, int kv_len,
                      int key_block, int topk) {
  __shared__ double sq[kFewGroups * kScorePitch], sk[kScoreTile * kScorePitch];
  const int g0 = blockIdx.x * kFewGroups, bh = blockIdx.y;
  const int b = bh / heads, h = bh - b * heads;
  const long long kv = static_cast<long long>(b) * (heads / per) + h / per;
  const double* qg = q_sum + static_cast<long long>(bh) * groups * kDim;
  const double* kg = k_mean + kv * blocks * kDim;
  start_next();
  wait_previous();
  for (int i = threadIdx.x; i < (kFewGroups + kScoreTile) * kDim / 2; i += 128) {
    const int r = i / (kDim / 2), c = i % (kDim / 2) * 2;
    double2 v = make_double2(0.0, 0.0);
    if (r < kFewGroups) {
      if (g0 + r < groups)
        v = *reinterpret_cast<const double2*>(qg + (g0 + r) * static_cast<long long>(kDim) + c);
      *reinterpret_cast<double2*>(sq + r * kScorePitch + c) = v;
    } else {
      const int n = r - kFewGroups;
      if (n < blocks) v = *reinterpret_cast<const double2*>(kg + n * kDim + c);
      *reinterpret_cast<double2*>(sk + n * kScorePitch + c) = v;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double acc[2][2][2] = {};
  const double* qa = sq + lane / 4 * kScorePitch + lane % 4;
  const double* kb = sk + (warp * 16 + lane / 4) * kScorePitch + lane % 4;
#pragma unroll 4
  for (int d = 0; d < kDim; d += 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        mma_f64(acc[i][j], qa[i * 8 * kScorePitch + d], kb[j * 8 * kScorePitch + d]);
  }
  __syncthreads();  // the query sums give way to the scores
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      *reinterpret_cast<double2*>(sq + (i * 8 + lane / 4) * kScorePitch + warp * 16 + j * 8 +
                                  lane % 4 * 2) = make_double2(acc[i][j][0], acc[i][j][1]);
  __syncthreads();
  const int n = (key_length(lengths, b, kv_len) + key_block - 1) / key_block;
  for (int r = warp; r < kFewGroups && g0 + r < groups; r += 4) {
    const double* s = sq + r * kScorePitch;
    select_topk<2>([&](int i) { return s[i]; }, n, min(topk, n), topk,
                   selection + (static_cast<long long>(bh) * groups + g0 + r) * topk, lane);
  }
}

// -------------------------------------------------- attention of 128-row tiles
// One CTA a query tile, four CTAs a multiprocessor.  A step is one 64-key piece
// of a chosen block.  Warps 0-3 softmax, one thread a row; one thread of warp 4
// loads (TMA) and issues the products.  TMEM: scores 64 columns, O 64; P is
// written over the scores it came from.
//
// A CTA's steps are a chain (S ready -> softmax -> P V and the next Q K -> S
// ready).  Its exponentials take 384 clocks at least (8192 a step, of which MUFU
// does three quarters at 16 a clock and multiprocessor).  Two chains, with their
// buffers doubled, had MUFU at 65 % and the tensor cores at 32 % and took 1.59 ms
// at 32640 tokens x 32 heads, 64 of 510 blocks; four take 1.24 ms with 61 % and
// 40 %.  So no unit is full: with one score buffer a CTA's products and its softmax
// never run together, and four CTAs do not cover each other's waits.  Where there
// are fewer tiles than slots, one chain's length is the time: about 2 us a step.
//
// The chain also orders everything else.  When every row's P of step j has
// arrived, S(j) had been ready, so Q K(j) and P V(j - 1) had completed: their
// stages of K and V are free without further barriers, and O may be rescaled.
constexpr int kTileThreads = 160;
constexpr int kStages = 2;                     // 64-key pieces of K and of V
constexpr int kTileBytes = kTile * kDim * 2;   // Q, 16 KB
constexpr int kPieceBytes = kHalf * kDim * 2;  // 8 KB
constexpr float kRescale = 8.0f;  // log2 units the running maximum may lag behind

struct __align__(8) TileBarriers {
  uint64_t q_full, k_full[kStages], v_full[kStages];
  uint64_t s_full, p_full, o_done;
  uint32_t tmem_base;
  int abort;
};
constexpr int kTileSmemK = kTileBytes;
constexpr int kTileSmemV = kTileSmemK + kStages * kPieceBytes;
constexpr int kTileSmemBar = kTileSmemV + kStages * kPieceBytes;
constexpr int kTileSmemLaunch = kTileSmemBar + 256 + 1024;  // + base alignment
static_assert(4 * (kTileSmemLaunch + 1024) <= 228 * 1024, "four CTAs a multiprocessor");
static_assert(sizeof(TileBarriers) <= 256, "barrier block");

struct TileParams {
  int q_len, kv_len, per;  // per: query heads of a key head
  int key_block, topk;
  const int* lengths;
  const int* selection;  // [batch][heads][tiles][topk], ascending, -1 behind
  float scale_log2;
  void* out;
  Strides o_st;
  int* status;
};

// Maximum of three, NaN if one is.
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Loads 16 TMEM columns of this thread's lane and waits for them.
__device__ __forceinline__ void tmem_ld_wait_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// 2^x for a pair of x <= kRescale on the FMA pipe: exp2_poly2 (a cubic, 7.5e-5 of
// the value, against BF16's 2^-9), and for FP16 weights (2^-12) the same split
// with the quartic that minimises the relative error on [0, 1) (2.7e-6,
// minimax_exp2(4) of gen_exp2_poly.py).  Below 2^-126 both give 2^-126.
template <typename T>
__device__ __forceinline__ void exp2_fma(float x0, float x1, float& y0, float& y1) {
  exp2_poly2(x0, x1, y0, y1);
}
template <>
__device__ __forceinline__ void exp2_fma<__half>(float x0, float x1, float& y0, float& y1) {
  constexpr float c0 = 0x1.00002cp+0f, c1 = 0x1.62d164p-1f, c2 = 0x1.ee79bep-3f,
                  c3 = 0x1.aa12a4p-5f, c4 = 0x1.bb7f6ep-7f;
  x0 = fmaxf(x0, -126.0f);
  x1 = fmaxf(x1, -126.0f);
  float t0, t1, j0, j1, f0, f1, p0, p1;
  add2_rm(t0, t1, x0, x1, kRoundMagic, kRoundMagic);  // t = magic + floor(x)
  sub2(j0, j1, t0, t1, kRoundMagic, kRoundMagic);     // floor(x), exact
  sub2(f0, f1, x0, x1, j0, j1);                       // f in [0, 1), exact
  fma2(p0, p1, c4, c4, f0, f1, c3, c3);
  fma2(p0, p1, p0, p1, f0, f1, c2, c2);
  fma2(p0, p1, p0, p1, f0, f1, c1, c1);
  fma2(p0, p1, p0, p1, f0, f1, c0, c0);
  y0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  y1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

// Of every four pairs of a row's weights one takes the FMA pipe and three MUFU,
// whose work four chains are bound by first: 32640 tokens x 16 heads took 805 us
// with none, 756 with one in eight, 727 with two, 773 with three.
constexpr int kFmaEvery = 4;

// Weights of one row's 64 scores, of which the first n count: P = 2^(S c - m) as
// 16-bit pairs, their FP32 sum, and the maximum of S c.  What is masked or -inf
// weighs 2^-126 in an FMA pair and 0 in the others (V's masked rows are zeros,
// and a row that has met only -inf, m = -inf, is cleared at the end).  A score
// that is NaN or +inf makes the sum NaN, as it makes the softmax.
template <typename T>
__device__ __forceinline__ void weigh(uint32_t tS, float c, float m, int n, uint32_t (&pk)[32],
                                      float& sum, float& m_tile) {
  uint32_t sr[kHalf];
  tmem_ld_wait_64(tS, sr);
  if (n < kHalf) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
      if (i >= n) sr[i] = __float_as_uint(-CUDART_INF_F);
  }
  const float neg_m = m == -CUDART_INF_F ? 0.f : -m;
  float sum0 = 0.f, sum1 = 0.f, mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float s0 = __uint_as_float(sr[2 * i]), s1 = __uint_as_float(sr[2 * i + 1]);
    float x0, x1, p0, p1;
    fma2(x0, x1, s0, s1, c, c, neg_m, neg_m);
    if (i & 1)
      mx1 = fmax3_nan(mx1, s0, s1);
    else
      mx0 = fmax3_nan(mx0, s0, s1);
    if (i % kFmaEvery == 0) {
      exp2_fma<T>(x0, x1, p0, p1);
    } else {
      p0 = ex2_approx(x0);
      p1 = ex2_approx(x1);
    }
    add2(sum0, sum1, sum0, sum1, p0, p1);
    pk[i] = pack2<T>(p0, p1);
  }
  m_tile = fmax3_nan(mx0, mx1, mx1) * c;
  sum = m_tile < CUDART_INF_F ? sum0 + sum1 : CUDART_NAN_F;
}

// First key of 64-key piece `i` of a tile's list.  (An ordinary read: the kernel that
// writes the list may still run when this one starts.)
__device__ __forceinline__ int piece_key(const TileParams& p, const int* list, int i) {
  const int shift = p.key_block >> 7;  // pieces of a block: 1 << shift
  return list[i >> shift] * p.key_block + (i & shift) * kHalf;
}

// kind::f16 instruction descriptor with BF16 (format 1) or FP16 (format 0)
// operands, FP32 accumulation; b_mn_major: B's rows are the reduction (V).
template <bool kBf16>
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool b_mn_major) {
  return (1u << 4) | ((kBf16 ? 1u : 0u) << 7) | ((kBf16 ? 1u : 0u) << 10) |
         ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

template <typename T, bool kBf16>
__global__ void __launch_bounds__(kTileThreads, 4)
    tile_attn_kernel(const __grid_constant__ CUtensorMap tmap_q,
                     const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const TileParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  TileBarriers* bars = reinterpret_cast<TileBarriers*>(smem + kTileSmemBar);
  const uint32_t sQ = smem_u32(smem), sK = sQ + kTileSmemK, sV = sQ + kTileSmemV;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int tile = blockIdx.x, head = blockIdx.y, batch = blockIdx.z;
  const int len = key_length(p.lengths, batch, p.kv_len);
  const int kept = min(p.topk, (len + p.key_block - 1) / p.key_block);
  const int steps = kept << (p.key_block >> 7);  // 64-key pieces
  const int* list =
      p.selection +
      ((static_cast<long long>(batch) * gridDim.y + head) * gridDim.x + tile) * p.topk;
  const int row = threadIdx.x & 127;
  // this thread's row of the result, or null (computed where it is needed: the
  // softmax has no registers to spare)
  auto out_row = [&]() -> uint4* {
    const int tok = static_cast<int>(blockIdx.x) * kTile + static_cast<int>(threadIdx.x);
    if (threadIdx.x >= kTile || tok >= p.q_len) return nullptr;
    return reinterpret_cast<uint4*>(static_cast<T*>(p.out) + blockIdx.z * p.o_st.batch +
                                    blockIdx.y * p.o_st.head + tok * p.o_st.token);
  };
  if (steps == 0) {  // no valid key: zeros
    wait_previous();
    if (uint4* dst = out_row()) {
#pragma unroll
      for (int i = 0; i < 8; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  volatile int* abort = &bars->abort;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bars->q_full), 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&bars->k_full[i]), 1);
      mbar_init(smem_u32(&bars->v_full[i]), 1);
    }
    mbar_init(smem_u32(&bars->s_full), 1);
    mbar_init(smem_u32(&bars->p_full), 4);  // one arrival a softmax warp
    mbar_init(smem_u32(&bars->o_done), 1);
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == 4) {
    tmem_alloc(smem_u32(&bars->tmem_base), 2 * kHalf);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  if (threadIdx.x == kTile) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  wait_previous();  // the choice

  if (warp == 4) {
    // --------------------------------------------------- loads and products
    if (elect_one()) {
      constexpr uint32_t id_qk = idesc<kBf16>(kTile, kHalf, false);
      constexpr uint32_t id_pv = idesc<kBf16>(kTile, kDim, true);
      const uint32_t tO = tmem + kHalf;
      const uint64_t dq = sdesc_sw128(sQ, 16, 1024);
      const uint64_t dk0 = sdesc_sw128(sK, 16, 1024), dv0 = sdesc_sw128(sV, 1024, 1024);
      const int kv_head = head / p.per;
      int k_issued = 0, v_issued = 0;
      auto load_k = [&](int j, int key) {
        const uint32_t bar = smem_u32(&bars->k_full[j & 1]);
        mbar_arrive_expect_tx(bar, kPieceBytes);
        tma_load_5d(sK + (j & 1) * kPieceBytes, &tmap_k, bar, 0, key, kv_head, batch, 0);
        k_issued = j + 1;
      };
      auto load_v = [&](int j, int key) {
        const uint32_t bar = smem_u32(&bars->v_full[j & 1]);
        mbar_arrive_expect_tx(bar, kPieceBytes);
        tma_load_5d(sV + (j & 1) * kPieceBytes, &tmap_v, bar, 0, key, kv_head, batch, 0);
        v_issued = j + 1;
      };
      auto issue_qk = [&](int j) {
        const uint64_t dk = dk0 + (j & 1) * (kPieceBytes / 16);
#pragma unroll
        for (int k = 0; k < kDim / 16; ++k)
          mma_bf16_ss(tmem, dq + 2 * k, dk + 2 * k, id_qk, k > 0);
        mma_commit(smem_u32(&bars->s_full));
      };
      const uint32_t q_bar = smem_u32(&bars->q_full);
      // keys of the steps ahead, read before they are needed
      const int key0 = piece_key(p, list, 0);
      int key1 = steps > 1 ? piece_key(p, list, 1) : 0;
      int key2 = steps > 2 ? piece_key(p, list, 2) : 0;
      mbar_arrive_expect_tx(q_bar, kTileBytes);
      tma_load_5d(sQ, &tmap_q, q_bar, 0, tile * kTile, head, batch, 0);
      load_k(0, key0);
      load_v(0, key0);
      if (steps > 1) {
        load_k(1, key1);
        load_v(1, key1);
      }
      bool ok = mbar_wait(q_bar, 0, abort, p.status, kStatusTimeoutMma) &&
                mbar_wait(smem_u32(&bars->k_full[0]), 0, abort, p.status, kStatusTimeoutMma);
      if (ok) {
        tc_fence_after();
        issue_qk(0);
      }
      for (int j = 0; ok && j < steps; ++j) {
        const bool more = j + 1 < steps;
        const int key3 = j + 3 < steps ? piece_key(p, list, j + 3) : 0;
        ok = mbar_wait(smem_u32(&bars->v_full[j & 1]), (j >> 1) & 1, abort, p.status,
                       kStatusTimeoutMma) &&
             (!more || mbar_wait(smem_u32(&bars->k_full[(j + 1) & 1]), ((j + 1) >> 1) & 1, abort,
                                 p.status, kStatusTimeoutMma)) &&
             mbar_wait(smem_u32(&bars->p_full), j & 1, abort, p.status, kStatusTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = dv0 + (j & 1) * (kPieceBytes / 16);
#pragma unroll
        for (int k = 0; k < kHalf / 16; ++k)
          mma_bf16_ts(tO, tmem + k * 8, dv + k * (2048 / 16), id_pv,
                      (j > 0 || k > 0) ? 1u : 0u);
        if (more) issue_qk(j + 1);
        if (j + 2 < steps) load_k(j + 2, key2);
        if (j > 0 && more) load_v(j + 1, key1);
        key1 = key2;
        key2 = key3;
      }
      // Every product completes before TMEM is released, and every load lands.
      mma_commit(smem_u32(&bars->o_done));
      mbar_wait_drain(smem_u32(&bars->o_done), 0);
      if (*abort) {
        mbar_wait_drain(q_bar, 0);
        for (int d = max(0, k_issued - 2); d < k_issued; ++d)
          mbar_wait_drain(smem_u32(&bars->k_full[d & 1]), (d >> 1) & 1);
        for (int d = max(0, v_issued - 2); d < v_issued; ++d)
          mbar_wait_drain(smem_u32(&bars->v_full[d & 1]), (d >> 1) & 1);
      }
    }
  } else {
    // ------------------------------------------------------------- softmax
    const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tS = tmem + lane_off, tO = tS + kHalf;
    const float c = p.scale_log2;
    float m_run = -CUDART_INF_F, l_run = 0.f;  // running maximum (log2 domain) and sum
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      // Valid keys of the piece: the list ascends, so only the last block's
      // pieces can be short.
      int n = kHalf;
      if (j + 2 >= steps) n = min(len - piece_key(p, list, j), kHalf);
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->s_full), j & 1, abort, p.status,
                                             kStatusTimeoutSoftmax))) {
        ok = false;
        break;
      }
      tc_fence_after();
      // P against the maximum so far, the step's own maximum taken along the way
      // (the exponentials, not the comparisons, set the pace).  P is bounded by
      // 2^kRescale as long as no row's maximum has grown by more; where one has
      // (and in the first step) the step is done over: the scores are still there.
      uint32_t pk[32];
      float sum, m_tile;
      weigh<T>(tS, c, m_run, n, pk, sum, m_tile);
      const bool raise = m_tile > m_run + kRescale;
      if (__any_sync(0xffffffffu, raise)) {
        const float m_new = raise ? m_tile : m_run;
        if (j > 0) {  // O holds the products up to step j - 1
          const float alpha = raise ? ex2_approx(m_run - m_new) : 1.0f;
          l_run *= alpha;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t o[16];
            tmem_ld_wait_16(tO + h * 16, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(tO + h * 16, o);
          }
        }
        m_run = m_new;
        weigh<T>(tS, c, m_run, n, pk, sum, m_tile);
      }
      tmem_st32(tS, pk);
      l_run += sum;
      // Rows of V behind the sequence's end may hold anything (0 * NaN is NaN):
      // they are cleared before the product reads them.
      if (n < kHalf && len < p.kv_len) {
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->v_full[j & 1]), (j >> 1) & 1, abort,
                                               p.status, kStatusTimeoutSoftmax))) {
          ok = false;
          break;
        }
        if (row < kHalf && row >= n) {
          uint4* v =
              reinterpret_cast<uint4*>(smem + kTileSmemV + (j & 1) * kPieceBytes + row * 128);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (elect_one()) mbar_arrive(smem_u32(&bars->p_full));
    }
    if (ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->o_done), 0, abort, p.status,
                                                kStatusTimeoutEpilogue))) {
      tc_fence_after();
      if (__all_sync(0xffffffffu, *abort == 0)) {
        uint4* dst = out_row();
        // every score was -inf: weights of nothing
        const float inv = m_run == -CUDART_INF_F && l_run == l_run ? 0.f : 1.0f / l_run;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          tmem_ld_wait_32(tO + h * 32, o);
          if (dst != nullptr) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = pack2<T>(__uint_as_float(o[8 * i + 2 * k]) * inv,
                                __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
              dst[h * 4 + i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kHalf);
  }
}

// -------------------------------------------------------------- single queries
// A row (batch, head, query) is the work of a cluster of 1 to 8 CTAs, in one
// launch.  Its CTAs share the blocks' scores (eight lanes a block, eight channels
// each, FP64) and write each score into every CTA's shared memory; each makes the
// choice by itself and attends its part of it: eight lanes a key (16 bytes each of
// its K and V rows), four neighbouring keys a lane group at a time and four more
// on the way, with running maximum and sum.  Groups, warps and CTAs are merged in
// a fixed order.  Bound by the bytes of the means and the chosen blocks.
constexpr int kRowWarps = 8;
constexpr int kRowKeys = 4;
constexpr int kMaxSplits = 8;
// Shared memory: arrays of fixed size (2376 bytes and their alignment), scores and choice.
constexpr int kRowStatic = 4096;
constexpr int kRowSmemMax = 220 * 1024;
static_assert(kRowStatic + kRowSmemMax <= 227 * 1024, "shared memory of a CTA");

struct RowParams {
  const void *q, *k, *v;
  Strides q_st, k_st, v_st, o_st;
  void* out;
  const int* lengths;
  const double* k_mean;
  int* selection;
  int heads, per, q_len, kv_len, key_block, blocks, topk, splits;
  int follows;  // launched behind the kernel that computes the means
  float scale_log2;
};

__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ float ld_cluster_f32(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Weight that a part with maximum m has under the common maximum `top`.
__device__ __forceinline__ float part_weight(float m, float top) {
  return m == -CUDART_INF_F ? 0.f : ex2_approx(m - top);
}

template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps, 2) row_kernel(const RowParams p) {
  __shared__ float part_m[kRowWarps], part_l[kRowWarps], part_o[kRowWarps][kDim];
  __shared__ float cta[kDim + 2];  // this CTA's O, maximum, sum
  extern __shared__ double scores[];  // [blocks], then the choice
  int* list = reinterpret_cast<int*>(scores + p.blocks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x % p.splits);  // also the rank in the cluster
  const long long row = blockIdx.x / p.splits;                // (batch, head, query)
  const int qi = static_cast<int>(row % p.q_len);
  const int bh = static_cast<int>(row / p.q_len);
  const int b = bh / p.heads, h = bh - b * p.heads;
  const int len = key_length(p.lengths, b, p.kv_len);
  const int n = (len + p.key_block - 1) / p.key_block;
  const int take = min(p.topk, n);
  const int group = lane >> 3, c8 = (lane & 7) * 8;
  float q[8];
  {
    const T* src = static_cast<const T*>(p.q) + b * p.q_st.batch + h * p.q_st.head +
                   qi * p.q_st.token + c8;
    unpack8<T>(*reinterpret_cast<const uint4*>(src), q);
  }
  // ---------------------------------------------------------------- scores
  if (p.follows) wait_previous();  // the means of this call
  // No CTA's shared memory is written before it has started.
  if (p.splits > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if (take < n) {
    double qd[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) qd[i] = static_cast<double>(q[i]);
    const double* mean =
        p.k_mean +
        (static_cast<long long>(b) * (p.heads / p.per) + h / p.per) * p.blocks * kDim + c8;
    const int stride = p.splits * kRowWarps * 4;
    constexpr int U = 4;  // blocks of a lane group requested together
    for (int i0 = (split * kRowWarps + warp) * 4; i0 < n; i0 += stride * U) {
      double2 v[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * stride + group;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[u][j] = i < n ? *reinterpret_cast<const double2*>(
                                mean + i * static_cast<long long>(kDim) + 2 * j)
                          : make_double2(0.0, 0.0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * stride + group;
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s = fma(qd[2 * j], v[u][j].x, s);
          s = fma(qd[2 * j + 1], v[u][j].y, s);
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        // lane r of the group writes into CTA r
        if ((lane & 7) < p.splits && i < n)
          asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(map_rank(scores + i, lane & 7)),
                       "d"(s)
                       : "memory");
      }
    }
  }
  if (p.splits > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  // ---------------------------------------------------------------- choice
  if (warp == 0) {
    auto score = [&](int i) { return scores[i]; };
    if (n <= 32 * 4)
      select_topk<4>(score, n, take, take, list, lane);
    else if (n <= 32 * 16)
      select_topk<16>(score, n, take, take, list, lane);
    else if (n <= 32 * 48)
      select_topk<48>(score, n, take, take, list, lane);
    else
      select_topk<0>(score, n, take, take, list, lane);
    __syncwarp();
    if (split == 0) {
      int* out = p.selection + row * p.topk;
      for (int i = lane; i < p.topk; i += 32) out[i] = i < take ? list[i] : -1;
    }
  }
  __syncthreads();
  // ------------------------------------------------------------- attention
  const int shift = p.key_block >> 7;
  const int pieces = take << shift;
  const int lo = static_cast<int>(static_cast<long long>(pieces) * split / p.splits);
  const int hi = static_cast<int>(static_cast<long long>(pieces) * (split + 1) / p.splits);
  const T* kp = static_cast<const T*>(p.k) + b * p.k_st.batch + h / p.per * p.k_st.head + c8;
  const T* vp = static_cast<const T*>(p.v) + b * p.v_st.batch + h / p.per * p.v_st.head + c8;
  float m = -CUDART_INF_F, l = 0.f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  // units of 16 keys: a quarter of a 64-key piece, four keys a lane group; the
  // next unit is requested before the current one is used
  uint4 kv[2][kRowKeys], vv[2][kRowKeys];
  int first = 0, next_first = 0;
  auto request = [&](int u, uint4 (&kk)[kRowKeys], uint4 (&v_)[kRowKeys], int& f0) {
    f0 = list[(u >> 2) >> shift] * p.key_block + ((u >> 2) & shift) * kHalf + (u & 3) * 16 +
         group * kRowKeys;
#pragma unroll
    for (int i = 0; i < kRowKeys; ++i) {
      kk[i] = v_[i] = make_uint4(0u, 0u, 0u, 0u);
      if (f0 + i < len) kk[i] = *reinterpret_cast<const uint4*>(kp + (f0 + i) * p.k_st.token);
    }
#pragma unroll
    for (int i = 0; i < kRowKeys; ++i)
      if (f0 + i < len) v_[i] = *reinterpret_cast<const uint4*>(vp + (f0 + i) * p.v_st.token);
  };
  auto use = [&](const uint4 (&kk)[kRowKeys], const uint4 (&v_)[kRowKeys], int f0) {
    float s[kRowKeys], top = m;
#pragma unroll
    for (int i = 0; i < kRowKeys; ++i) {
      float f[8], d = 0.f;
      unpack8<T>(kk[i], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) d = fmaf(q[j], f[j], d);
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
      s[i] = f0 + i < len ? d * p.scale_log2 : -CUDART_INF_F;
      top = fmaxf(top, s[i]);
    }
    const float zero = top == -CUDART_INF_F ? 0.f : top;
    const float alpha = ex2_approx(m - zero);
    l *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] *= alpha;
#pragma unroll
    for (int i = 0; i < kRowKeys; ++i) {
      const float w = ex2_approx(s[i] - zero);
      l += w;
      float f[8];
      unpack8<T>(v_[i], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(w, f[j], o[j]);
    }
    m = top;
  };
  {
    const int end = 4 * hi;
    int u = 4 * lo + warp;
    if (u < end) request(u, kv[0], vv[0], first);
    while (u < end) {
      if (u + kRowWarps < end) request(u + kRowWarps, kv[1], vv[1], next_first);
      use(kv[0], vv[0], first);
      u += kRowWarps;
      if (u >= end) break;
      if (u + kRowWarps < end) request(u + kRowWarps, kv[0], vv[0], first);
      use(kv[1], vv[1], next_first);
      u += kRowWarps;
    }
  }
  // ----------------------------------------------------------------- merge
  // the four lane groups of the warp
#pragma unroll
  for (int x = 8; x < 32; x <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, x), top = fmaxf(m, m2);
    const float mine = part_weight(m, top), theirs = part_weight(m2, top);
    l = l * mine + __shfl_xor_sync(0xffffffffu, l, x) * theirs;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = o[j] * mine + __shfl_xor_sync(0xffffffffu, o[j], x) * theirs;
    m = top;
  }
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part_o[warp][c8 + j] = o[j];
    if (lane == 0) {
      part_m[warp] = m;
      part_l[warp] = l;
    }
  }
  __syncthreads();
  const int d = threadIdx.x;
  float om = 0.f, lm = 0.f, top = -CUDART_INF_F;
  if (d < kDim) {
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, part_m[w]);
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float weight = part_weight(part_m[w], top);
      om += part_o[w][d] * weight;
      lm += part_l[w] * weight;
    }
  }
  if (p.splits > 1) {
    if (d < kDim) cta[d] = om;
    if (d == 0) {
      cta[kDim] = top;
      cta[kDim + 1] = lm;
    }
    cluster_arrive();
    cluster_wait();
    if (split == 0 && d < kDim) {
      float ms[kMaxSplits], ls[kMaxSplits], os[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) {
        if (s < p.splits) {
          ms[s] = ld_cluster_f32(&cta[kDim], s);
          ls[s] = ld_cluster_f32(&cta[kDim + 1], s);
          os[s] = ld_cluster_f32(&cta[d], s);
        }
      }
      top = -CUDART_INF_F;
      om = lm = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        if (s < p.splits) top = fmaxf(top, ms[s]);
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) {
        if (s < p.splits) {
          const float weight = part_weight(ms[s], top);
          om += os[s] * weight;
          lm += ls[s] * weight;
        }
      }
    }
    cluster_arrive();  // the others' sums have been read
    cluster_wait();
  }
  if (split == 0 && d < kDim) {
    const float y = lm == 0.f ? 0.f : om / lm;
    uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.o_st.batch + h * p.o_st.head +
                    qi * p.o_st.token + d;
    *dst = static_cast<uint16_t>(pack2<T>(y, 0.f));
  }
}

// ---------------------------------------------------------------- host side
struct Sizes {
  long long blocks, groups;
  size_t pool, q_sum, scores, total;
};

Sizes workspace_sizes(long long batch, long long q_heads, long long kv_heads, long long q_len,
                      long long kv_len, int query_block, int key_block, bool has_pool) {
  Sizes s = {};
  s.blocks = (kv_len + key_block - 1) / key_block;
  s.groups = (q_len + query_block - 1) / query_block;
  s.pool = has_pool ? 0 : static_cast<size_t>(batch * kv_heads * s.blocks * kDim) * 8;
  if (query_block == kTile) {
    s.q_sum = static_cast<size_t>(batch * q_heads * s.groups * kDim) * 8;
    s.scores = static_cast<size_t>(batch * q_heads * s.groups * s.blocks) * 8;
  }
  s.total = s.pool + s.q_sum + s.scores;
  return s;
}

bool strides_ok(const Strides& s) { return ((s.token | s.head | s.batch) & 7) == 0; }

int operand_map(CUtensorMap* map, bool bf16, const void* base, int len, int heads, int batch,
                const Strides& st, int rows) {
  const uint64_t dims[5] = {static_cast<uint64_t>(kDim), static_cast<uint64_t>(len),
                            static_cast<uint64_t>(heads), static_cast<uint64_t>(batch), 1};
  // a dimension of one still needs a valid stride
  auto stride = [](long long s, uint64_t n) -> uint64_t {
    return n > 1 ? static_cast<uint64_t>(s) * 2 : 16;
  };
  const uint64_t strides[4] = {stride(st.token, dims[1]), stride(st.head, dims[2]),
                               stride(st.batch, dims[3]), 16};
  const uint32_t box[5] = {kDim, static_cast<uint32_t>(rows), 1, 1, 1};
  return encode_tensor_map(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
      const_cast<void*>(base), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

long long pool_items(const PoolParams& p, int batch) {
  return static_cast<long long>(batch) * p.blocks * ((p.heads + 3) / 4);
}

template <typename T>
int launch_pool(const PoolParams* a, const PoolParams* b, int batch, cudaStream_t st) {
  const long long items_a = a == nullptr ? 0 : pool_items(*a, batch);
  const long long items = items_a + (b == nullptr ? 0 : pool_items(*b, batch));
  if (items > 0x7fffffffLL) return kErrTooLarge;
  const PoolParams none = {};
  const int warps = items < 16 * 148 ? kPoolWarps : kPoolWarps / 2;
  pool_kernel<T><<<static_cast<unsigned>(items), 32 * warps, 0, st>>>(
      a == nullptr ? none : *a, b == nullptr ? none : *b, items_a);
  return static_cast<int>(cudaGetLastError());
}

// Launch configuration of a kernel that may start while the call's previous one
// still runs, or of a cluster launch.
struct Config {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[2];
  Config(dim3 grid, int threads, size_t smem, cudaStream_t st) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attrs;
    cfg.numAttrs = 0;
  }
  Config& follow() {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    return *this;
  }
  Config& cluster(int ctas) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(ctas);
    attrs[cfg.numAttrs].val.clusterDim.y = attrs[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
    return *this;
  }
  Config(const Config&) = delete;
};

struct Call {
  const void *q, *k, *v;
  Strides q_st, k_st, v_st, o_st;
  int batch, q_heads, kv_heads, q_len, kv_len;
  const int* lengths;
  const double* pool;
  int topk, query_block, key_block;
  float scale;
  void* out;
  int* selection;
  char* workspace;
  int* status;
};

template <typename T, bool kBf16>
int run(const Call& c, cudaStream_t st) {
  const Sizes sz = workspace_sizes(c.batch, c.q_heads, c.kv_heads, c.q_len, c.kv_len,
                                   c.query_block, c.key_block, c.pool != nullptr);
  const bool tiles = c.query_block == kTile;
  const int blocks = static_cast<int>(sz.blocks), groups = static_cast<int>(sz.groups);
  double* own_pool = reinterpret_cast<double*>(c.workspace);
  double* q_sum = reinterpret_cast<double*>(c.workspace + sz.pool);
  double* scores = reinterpret_cast<double*>(c.workspace + sz.pool + sz.q_sum);
  const double* pool = c.pool != nullptr ? c.pool : own_pool;
  const int per = c.q_heads / c.kv_heads;
  const float scale_log2 = c.scale * 1.4426950408889634f;

  const PoolParams kp = {c.k, c.k_st, c.kv_heads, c.kv_len, c.key_block, blocks, c.lengths, 1,
                         own_pool};
  const PoolParams qp = {c.q, c.q_st, c.q_heads, c.q_len, kTile, groups, nullptr, 0, q_sum};
  if (c.pool == nullptr || tiles) {
    if (int rc = launch_pool<T>(c.pool == nullptr ? &kp : nullptr, tiles ? &qp : nullptr, c.batch,
                                st))
      return rc;
  }
  if (tiles) {
    cudaError_t e;
    if (blocks <= kScoreTile) {
      Config choose(dim3((groups + kFewGroups - 1) / kFewGroups,
                         static_cast<unsigned>(c.batch * c.q_heads)),
                    128, 0, st);
      e = cudaLaunchKernelEx(&choose.follow().cfg, few_blocks_kernel,
                             static_cast<const double*>(q_sum), pool, c.selection, c.lengths,
                             c.q_heads, per, groups, blocks, c.kv_len, c.key_block, c.topk);
      if (e != cudaSuccess) return static_cast<int>(e);
    } else {
      e = cudaFuncSetAttribute(
          score_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kScoreSmem);
      if (e != cudaSuccess) return static_cast<int>(e);
      const dim3 grid((blocks + kScoreTile - 1) / kScoreTile,
                      (groups + kScoreTile - 1) / kScoreTile,
                      static_cast<unsigned>(c.batch * c.q_heads));
      Config score(grid, 128, kScoreSmem, st);
      e = cudaLaunchKernelEx(&score.follow().cfg, score_kernel, static_cast<const double*>(q_sum),
                             pool, scores, c.q_heads, per, groups, blocks);
      if (e != cudaSuccess) return static_cast<int>(e);
      const long long per_batch = static_cast<long long>(c.q_heads) * groups;
      const long long rows = c.batch * per_batch;
      const unsigned ctas = static_cast<unsigned>((rows + kSelectWarps - 1) / kSelectWarps);
      auto select = blocks <= 32 * 8 ? select_kernel<8>
                    : blocks <= 32 * 16 ? select_kernel<16>
                    : blocks <= 32 * 32 ? select_kernel<32> : select_kernel<0>;
      Config choose(dim3(ctas), 32 * kSelectWarps, 0, st);
      e = cudaLaunchKernelEx(&choose.follow().cfg, select, static_cast<const double*>(scores),
                             c.selection, c.lengths, rows, per_batch, blocks, c.kv_len, c.key_block,
                             c.topk);
      if (e != cudaSuccess) return static_cast<int>(e);
    }
    CUtensorMap tq, tk, tv;
    if (operand_map(&tq, kBf16, c.q, c.q_len, c.q_heads, c.batch, c.q_st, kTile) ||
        operand_map(&tk, kBf16, c.k, c.kv_len, c.kv_heads, c.batch, c.k_st, kHalf) ||
        operand_map(&tv, kBf16, c.v, c.kv_len, c.kv_heads, c.batch, c.v_st, kHalf))
      return kErrTensorMap;
    e = cudaFuncSetAttribute(tile_attn_kernel<T, kBf16>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmemLaunch);
    if (e != cudaSuccess) return static_cast<int>(e);
    const TileParams p = {c.q_len, c.kv_len, per, c.key_block, c.topk, c.lengths, c.selection,
                          scale_log2, c.out, c.o_st, c.status};
    Config attend(dim3(groups, c.q_heads, c.batch), kTileThreads, kTileSmemLaunch, st);
    return static_cast<int>(
        cudaLaunchKernelEx(&attend.follow().cfg, tile_attn_kernel<T, kBf16>, tq, tk, tv, p));
  }

  const long long rows = static_cast<long long>(c.batch) * c.q_heads * c.q_len;
  const int most = c.topk < blocks ? c.topk : blocks;  // chosen blocks of a row
  const int smem = blocks * 8 + most * 4;
  // Above 48 KB, the kernel's own arrays among them, the size has to be allowed first.
  // That is a property of the function, which calls of other threads set too: always
  // the largest size, so that no call takes back what another one needs.
  if (smem + kRowStatic > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        row_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmemMax);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  RowParams p = {c.q, c.k, c.v, c.q_st, c.k_st, c.v_st, c.o_st, c.out, c.lengths, pool,
                 c.selection, c.q_heads, per, c.q_len, c.kv_len, c.key_block, blocks, c.topk, 1,
                 c.pool == nullptr, scale_log2};
  // As many CTAs as two a multiprocessor hold at once, each with two 64-key pieces
  // at least.
  const long long pieces = static_cast<long long>(most) << (c.key_block >> 7);
  while (p.splits < kMaxSplits && rows * p.splits * 2 <= 2 * 148 && pieces >= p.splits * 4)
    p.splits *= 2;
  Config attend(dim3(static_cast<unsigned>(rows * p.splits)), 32 * kRowWarps,
                static_cast<size_t>(smem), st);
  attend.cluster(p.splits);
  if (p.follows) attend.follow();
  return static_cast<int>(cudaLaunchKernelEx(&attend.cfg, row_kernel<T>, p));
}

}  // namespace btk
}  // namespace erd

using namespace erd;

extern "C" size_t erd_block_topk_workspace_bytes(int batch, int q_heads, int kv_heads, int q_len,
                                                 int kv_len, int query_block, int key_block,
                                                 int has_pool) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_len <= 0 || kv_len <= 0 ||
      (query_block != 1 && query_block != btk::kTile) || (key_block != 64 && key_block != 128))
    return 0;
  return btk::workspace_sizes(batch, q_heads, kv_heads, q_len, kv_len, query_block, key_block,
                              has_pool != 0)
      .total;
}

extern "C" int erd_block_key_means(int dtype, const void* k, int64_t k_token_stride,
                                   int64_t k_head_stride, int64_t k_batch_stride, int batch,
                                   int kv_heads, int kv_len, int key_block,
                                   const int32_t* key_lengths, double* means, void* stream) {
  if (k == nullptr || means == nullptr) return kErrNullPointer;
  if ((dtype != ERD_BF16 && dtype != ERD_FP16) || batch <= 0 || kv_heads <= 0 || kv_len <= 0 ||
      (key_block != 64 && key_block != 128))
    return kErrBadShape;
  const btk::Strides st = {k_token_stride, k_head_stride, k_batch_stride};
  if (!aligned16(k) || !aligned16(means) || !btk::strides_ok(st) ||
      (reinterpret_cast<uintptr_t>(key_lengths) & 3) != 0)
    return kErrMisaligned;
  if (kv_len > btk::kMaxCount) return kErrTooLarge;
  if (int rc = check_device_sm100()) return rc;
  const btk::PoolParams p = {k, st, kv_heads, kv_len, key_block,
                             (kv_len + key_block - 1) / key_block, key_lengths, 1, means};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == ERD_BF16 ? btk::launch_pool<__nv_bfloat16>(&p, nullptr, batch, s)
                           : btk::launch_pool<__half>(&p, nullptr, batch, s);
}

extern "C" int erd_block_topk_attn(const erd_block_topk_args* args, int* status, void* stream) {
  if (args == nullptr) return kErrNullPointer;
  const erd_block_topk_args& a = *args;
  if (a.struct_bytes != static_cast<int64_t>(sizeof(a))) return kErrBadShape;
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.out == nullptr ||
      a.selection == nullptr)
    return kErrNullPointer;
  if ((a.dtype != ERD_BF16 && a.dtype != ERD_FP16) || a.head_dim != btk::kDim || a.batch <= 0 ||
      a.q_heads <= 0 || a.kv_heads <= 0 || a.q_heads % a.kv_heads != 0 || a.q_len <= 0 ||
      a.kv_len <= 0 || a.topk <= 0 || (a.query_block != 1 && a.query_block != btk::kTile) ||
      (a.key_block != 64 && a.key_block != 128) ||
      !(a.softmax_scale > 0.f && a.softmax_scale <= btk::kMaxScale))
    return kErrBadShape;
  if (a.batch > 65535 || a.q_heads > 65535 ||
      static_cast<long long>(a.batch) * a.q_heads > 65535 || a.kv_len > btk::kMaxCount ||
      a.q_len > btk::kMaxCount || a.topk > btk::kMaxCount)
    return kErrTooLarge;
  const btk::Sizes sz =
      btk::workspace_sizes(a.batch, a.q_heads, a.kv_heads, a.q_len, a.kv_len, a.query_block,
                           a.key_block, a.key_means != nullptr);
  const long long rows = static_cast<long long>(a.batch) * a.q_heads * sz.groups;
  if (rows > (1LL << 27) || (a.query_block == 1 && sz.blocks * 12 > btk::kRowSmemMax) ||
      (sz.groups + 63) / 64 > 65535)
    return kErrTooLarge;
  if (sz.total > 0 && a.workspace == nullptr) return kErrNullPointer;
  if (a.workspace_bytes < 0 || static_cast<size_t>(a.workspace_bytes) < sz.total)
    return kErrBadShape;
  btk::Call c = {};
  c.q = a.q;
  c.k = a.k;
  c.v = a.v;
  c.q_st = {a.q_stride[0], a.q_stride[1], a.q_stride[2]};
  c.k_st = {a.k_stride[0], a.k_stride[1], a.k_stride[2]};
  c.v_st = {a.v_stride[0], a.v_stride[1], a.v_stride[2]};
  c.o_st = {a.out_stride[0], a.out_stride[1], a.out_stride[2]};
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) ||
      !aligned16(a.workspace) || !aligned16(a.key_means) || !btk::strides_ok(c.q_st) ||
      !btk::strides_ok(c.k_st) || !btk::strides_ok(c.v_st) || !btk::strides_ok(c.o_st) ||
      ((reinterpret_cast<uintptr_t>(a.key_lengths) | reinterpret_cast<uintptr_t>(a.selection)) &
       3) != 0)
    return kErrMisaligned;
  if (int rc = check_device_sm100()) return rc;
  c.batch = a.batch;
  c.q_heads = a.q_heads;
  c.kv_heads = a.kv_heads;
  c.q_len = a.q_len;
  c.kv_len = a.kv_len;
  c.lengths = a.key_lengths;
  c.pool = a.key_means;
  c.topk = a.topk;
  c.query_block = a.query_block;
  c.key_block = a.key_block;
  c.scale = a.softmax_scale;
  c.out = a.out;
  c.selection = a.selection;
  c.workspace = static_cast<char*>(a.workspace);
  c.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.dtype == ERD_BF16 ? btk::run<__nv_bfloat16, true>(c, st)
                             : btk::run<__half, false>(c, st);
}
