// Rotary positions of query and key heads, alone or behind an RMS norm of
// each head, in one pass over the data:
//   y = x * rsqrt(mean_d(x^2) + eps) * w            (with the norm)
//   (y0, y1) -> (y0 c - y1 s, y0 s + y1 c)          for each rotated pair
// with c = a cos(2 pi t), s = a sin(2 pi t) and t = position * turns[pair].
// Pairs are channels (i, i + rotary_dim / 2) ("half") or (2 i, 2 i + 1)
// ("interleaved"); channels from rotary_dim on are not turned.
//
// Numerics: t is computed and reduced to [-1/2, 1/2] in 64 bits, so that a
// far position loses nothing (position 2^31 leaves 22 bits behind the point);
// what is left goes to sincospif in 32 bits.  Norm and rotation are FP32 and
// the result is rounded once.
//
// Bound by memory: each value is read once and written once.  A warp takes one
// token (or, when there are few tokens, some of its heads), computes each
// pair's cosine and sine once, one pair a lane, shares them through shared
// memory, and then walks over the heads; the angles cost one 64-bit product
// per token and pair and no table is read.  A lane owns two 16-byte chunks of
// a head that hold whole pairs in either layout, so loads and stores are
// 16 bytes wide and the norm's sum needs log2(lanes per head) shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/eraserdit_b200.h"
#include "host_common.h"

namespace erd {
namespace rot {

constexpr int kWarps = 8;
constexpr int kMaxHeadDim = 1024;
// Heads that one lane group loads before it computes: with 8 warps of two
// 16-byte chunks a lane this keeps 8 KB a warp in flight.
constexpr int kUnroll = 4;

struct Params {
  const void* in[2];  // queries, keys
  void* out[2];
  const void* weight[2];  // null: 1
  long long in_ts[2], in_hs[2], in_bs[2];
  long long out_ts[2], out_hs[2], out_bs[2];
  int heads[2];
  float eps[2];
  int weight_fp32;
  int batch, tokens, dim, rotary;
  int lanes, log2_lanes;  // lanes of a warp for one head (vector kernel)
  int iters[2];           // head groups of queries and of keys
  int chunk, chunks;      // head groups of one warp, warps of one token
  const double* turns;    // [rotary / 2] turns per position step
  float amplitude, sin_sign;
  int axis1, axis2;  // first pair of the second and third position axis
  const void* pos;   // null: start + token
  int pos_wide;
  long long pos_as, pos_bs, pos_ts, start;
};

// Cosine and sine of every rotated pair of one token into this warp's slab.
__device__ __forceinline__ void angles(const Params& p, int b, int tok, int lane, float2* slab) {
  for (int i = lane; i < p.rotary / 2; i += 32) {
    long long where = p.start + tok;
    if (p.pos != nullptr) {
      const int axis = (i >= p.axis1) + (i >= p.axis2);
      const long long at = axis * p.pos_as + b * p.pos_bs + tok * p.pos_ts;
      where = p.pos_wide ? static_cast<const long long*>(p.pos)[at]
                         : static_cast<long long>(static_cast<const int*>(p.pos)[at]);
    }
    double t = static_cast<double>(where) * p.turns[i];
    t -= rint(t);
    float s, c;
    sincospif(2.0f * static_cast<float>(t), &s, &c);
    slab[i] = make_float2(c * p.amplitude, s * p.amplitude * p.sin_sign);
  }
  __syncwarp();
}

template <typename T>
struct Vec;  // 16 bytes of T as floats
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16(x); }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = h.x;
      f[2 * i + 1] = h.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ float round(float x) { return x; }
};

// Weights of channels [c, c + kN) of one norm.
template <typename T>
__device__ __forceinline__ void load_weight(const Params& p, int which, int c, float* w) {
  constexpr int N = Vec<T>::kN;
  if (p.weight_fp32) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = static_cast<const float*>(p.weight[which])[c + i];
  } else {
    const T* base = static_cast<const T*>(p.weight[which]) + c;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = Vec<T>::one(base[i]);
  }
}

template <typename T, bool kNorm, bool kInterleaved>
__global__ void __launch_bounds__(32 * kWarps) head_rotary_kernel(const Params p) {
  constexpr int N = Vec<T>::kN;  // channels of a 16-byte chunk
  extern __shared__ float2 slabs[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const long long token = item / p.chunks;
  if (token >= static_cast<long long>(p.batch) * p.tokens) return;
  const int part = static_cast<int>(item - token * p.chunks);
  const int b = static_cast<int>(token / p.tokens);
  const int tok = static_cast<int>(token - static_cast<long long>(b) * p.tokens);
  float2* slab = slabs + warp * (p.rotary / 2);
  angles(p, b, tok, lane, slab);

  // This lane's two chunks of every head it meets.
  const int sub = lane & (p.lanes - 1), slot = lane >> p.log2_lanes, per = 32 >> p.log2_lanes;
  int c0, c1;
  if (kInterleaved || sub >= p.rotary / (2 * N)) {
    c0 = 2 * N * sub;  // also behind the rotated channels of the half layout
    c1 = c0 + N;
  } else {
    c0 = N * sub;
    c1 = p.rotary / 2 + N * sub;
  }
  const bool has0 = c0 < p.dim, has1 = c1 < p.dim;
  const bool turn0 = c0 < p.rotary, turn1 = c1 < p.rotary;
  float2 cs[N];  // of this lane's N pairs
#pragma unroll
  for (int i = 0; i < N; ++i) {
    cs[i] = make_float2(1.f, 0.f);
    if (kInterleaved) {
      const int c = i < N / 2 ? c0 : c1;
      if (c < p.rotary) cs[i] = slab[c / 2 + (i & (N / 2 - 1))];
    } else if (turn0) {
      cs[i] = slab[c0 + i];
    }
  }

  const int first = part * p.chunk, last = min(first + p.chunk, p.iters[0] + p.iters[1]);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int lo = max(first - (which ? p.iters[0] : 0), 0);
    const int hi = min(last - (which ? p.iters[0] : 0), p.iters[which]);
    if (lo >= hi) continue;
    float w[2 * N];
    if (kNorm) {
#pragma unroll
      for (int i = 0; i < 2 * N; ++i) w[i] = 1.f;
      if (p.weight[which] != nullptr) {
        if (has0) load_weight<T>(p, which, c0, w);
        if (has1) load_weight<T>(p, which, c1, w + N);
      }
    }
    const T* src = static_cast<const T*>(p.in[which]) + b * p.in_bs[which] + tok * p.in_ts[which];
    T* dst = static_cast<T*>(p.out[which]) + b * p.out_bs[which] + tok * p.out_ts[which];
    const long long in_hs = p.in_hs[which], out_hs = p.out_hs[which];
    const int heads = p.heads[which];
#pragma unroll 1
    for (int it = lo; it < hi; it += kUnroll) {
      uint4 v0[kUnroll], v1[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int head = (it + u) * per + slot;
        v0[u] = v1[u] = make_uint4(0u, 0u, 0u, 0u);
        if (it + u < hi && head < heads) {
          if (has0) v0[u] = *reinterpret_cast<const uint4*>(src + head * in_hs + c0);
          if (has1) v1[u] = *reinterpret_cast<const uint4*>(src + head * in_hs + c1);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int head = (it + u) * per + slot;
        if (it + u >= hi) break;  // the same for the whole warp
        float x[2 * N];
        Vec<T>::unpack(v0[u], x);
        Vec<T>::unpack(v1[u], x + N);
        if (kNorm) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * N; ++i) sum = fmaf(x[i], x[i], sum);
          for (int d = 1; d < p.lanes; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const float r = rsqrtf(sum / static_cast<float>(p.dim) + p.eps[which]);
#pragma unroll
          for (int i = 0; i < 2 * N; ++i) x[i] = x[i] * r * w[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float& a = kInterleaved ? x[2 * i] : x[i];
          float& d = kInterleaved ? x[2 * i + 1] : x[N + i];
          if (kInterleaved ? (i < N / 2 ? turn0 : turn1) : turn0) {
            const float a0 = a, d0 = d;
            a = a0 * cs[i].x - d0 * cs[i].y;
            d = a0 * cs[i].y + d0 * cs[i].x;
          }
        }
        if (head < heads) {
          if (has0) *reinterpret_cast<uint4*>(dst + head * out_hs + c0) = Vec<T>::pack(x);
          if (has1) *reinterpret_cast<uint4*>(dst + head * out_hs + c1) = Vec<T>::pack(x + N);
        }
      }
    }
  }
}

// The same for sizes and strides that 16-byte chunks do not fit: a warp takes
// one head at a time, a lane every 32nd pair and every 32nd channel behind the
// pairs, value by value.  The norm reads the head twice (the second time from
// L1); every lane has the sum before any lane writes, so in-place calls hold.
template <typename T, bool kNorm, bool kInterleaved>
__global__ void __launch_bounds__(32 * kWarps) head_rotary_scalar_kernel(const Params p) {
  extern __shared__ float2 slabs[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const long long token = item / p.chunks;
  if (token >= static_cast<long long>(p.batch) * p.tokens) return;
  const int part = static_cast<int>(item - token * p.chunks);
  const int b = static_cast<int>(token / p.tokens);
  const int tok = static_cast<int>(token - static_cast<long long>(b) * p.tokens);
  float2* slab = slabs + warp * (p.rotary / 2);
  angles(p, b, tok, lane, slab);
  const int first = part * p.chunk, last = min(first + p.chunk, p.heads[0] + p.heads[1]);
#pragma unroll 1
  for (int h = first; h < last; ++h) {
    const int which = h >= p.heads[0], head = which ? h - p.heads[0] : h;
    const T* src = static_cast<const T*>(p.in[which]) + b * p.in_bs[which] +
                   tok * p.in_ts[which] + head * p.in_hs[which];
    T* dst = static_cast<T*>(p.out[which]) + b * p.out_bs[which] + tok * p.out_ts[which] +
             head * p.out_hs[which];
    float r = 1.f;
    if (kNorm) {
      float sum = 0.f;
      for (int c = lane; c < p.dim; c += 32) {
        const float x = Vec<T>::one(src[c]);
        sum = fmaf(x, x, sum);
      }
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      r = rsqrtf(sum / static_cast<float>(p.dim) + p.eps[which]);
    }
    auto value = [&](int c) {
      float x = Vec<T>::one(src[c]);
      if (kNorm) {
        float w = 1.f;
        if (p.weight[which] != nullptr)
          w = p.weight_fp32 ? static_cast<const float*>(p.weight[which])[c]
                            : Vec<T>::one(static_cast<const T*>(p.weight[which])[c]);
        x = x * r * w;
      }
      return x;
    };
    for (int i = lane; i < p.rotary / 2; i += 32) {
      const int a = kInterleaved ? 2 * i : i, d = kInterleaved ? 2 * i + 1 : i + p.rotary / 2;
      const float x0 = value(a), x1 = value(d);
      const float2 cs = slab[i];
      dst[a] = Vec<T>::round(x0 * cs.x - x1 * cs.y);
      dst[d] = Vec<T>::round(x0 * cs.y + x1 * cs.x);
    }
    for (int c = p.rotary + lane; c < p.dim; c += 32) dst[c] = Vec<T>::round(value(c));
  }
}

template <typename T, bool kNorm, bool kInterleaved>
int launch(Params p, bool vector, cudaStream_t stream) {
  constexpr int N = Vec<T>::kN;
  if (vector) {
    const int tasks = (p.dim + 2 * N - 1) / (2 * N);
    p.lanes = 1;
    p.log2_lanes = 0;
    while (p.lanes < tasks) p.lanes *= 2, ++p.log2_lanes;
    const int per = 32 / p.lanes;
    for (int w = 0; w < 2; ++w) p.iters[w] = (p.heads[w] + per - 1) / per;
  } else {
    p.lanes = 32;
    p.log2_lanes = 5;
    for (int w = 0; w < 2; ++w) p.iters[w] = p.heads[w];
  }
  // A warp walks over all heads of a token, unless that leaves the device
  // short of warps (32 on each of 148 multiprocessors).
  const long long tokens = static_cast<long long>(p.batch) * p.tokens;
  const int iters = p.iters[0] + p.iters[1];
  const long long share = tokens * iters / (148 * 32);
  p.chunk = static_cast<int>(share < 1 ? 1 : share > iters ? iters : share);
  p.chunks = (iters + p.chunk - 1) / p.chunk;
  const long long blocks = (tokens * p.chunks + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffffLL) return kErrTooLarge;
  const size_t smem = static_cast<size_t>(kWarps) * (p.rotary / 2) * sizeof(float2);
  if (vector)
    head_rotary_kernel<T, kNorm, kInterleaved>
        <<<static_cast<unsigned>(blocks), 32 * kWarps, smem, stream>>>(p);
  else
    head_rotary_scalar_kernel<T, kNorm, kInterleaved>
        <<<static_cast<unsigned>(blocks), 32 * kWarps, smem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int dispatch(const Params& p, bool norm, bool interleaved, bool vector, cudaStream_t stream) {
  if (norm)
    return interleaved ? launch<T, true, true>(p, vector, stream)
                       : launch<T, true, false>(p, vector, stream);
  return interleaved ? launch<T, false, true>(p, vector, stream)
                     : launch<T, false, false>(p, vector, stream);
}

}  // namespace rot
}  // namespace erd

using namespace erd;

extern "C" int erd_head_norm_rotary(const erd_head_norm_rotary_args* args, void* stream) {
  if (args == nullptr) return kErrNullPointer;
  const erd_head_norm_rotary_args& a = *args;
  if (a.struct_bytes != static_cast<int64_t>(sizeof(a))) return kErrBadShape;
  if (a.q == nullptr || a.q_out == nullptr ||
      (a.k_heads > 0 && (a.k == nullptr || a.k_out == nullptr)) ||
      (a.rotary_dim > 0 && a.turns == nullptr))
    return kErrNullPointer;
  if (a.dtype < ERD_BF16 || a.dtype > ERD_FP32 || a.batch <= 0 || a.tokens <= 0 ||
      a.q_heads <= 0 || a.k_heads < 0 || a.head_dim <= 0 || a.rotary_dim < 0 ||
      a.rotary_dim > a.head_dim || (a.rotary_dim & 1) != 0)
    return kErrBadShape;
  if (a.head_dim > rot::kMaxHeadDim) return kErrTooLarge;
  auto address = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const uintptr_t elem = a.dtype == ERD_FP32 ? 4 : 2;
  const uintptr_t all = address(a.q) | address(a.q_out) |
                        (a.k_heads > 0 ? address(a.k) | address(a.k_out) : 0);
  const uintptr_t weights = address(a.q_weight) | address(a.k_weight);
  if ((all & (elem - 1)) != 0 || (weights & (a.weight_fp32 ? 3 : elem - 1)) != 0 ||
      (address(a.turns) & 7) != 0 || (address(a.positions) & (a.positions_int64 ? 7 : 3)) != 0)
    return kErrMisaligned;
  if (int rc = check_device_sm100()) return rc;
  rot::Params p = {};
  p.in[0] = a.q;
  p.in[1] = a.k;
  p.out[0] = a.q_out;
  p.out[1] = a.k_out;
  p.weight[0] = a.norm ? a.q_weight : nullptr;
  p.weight[1] = a.norm ? a.k_weight : nullptr;
  p.in_ts[0] = a.q_stride[0], p.in_hs[0] = a.q_stride[1], p.in_bs[0] = a.q_stride[2];
  p.in_ts[1] = a.k_stride[0], p.in_hs[1] = a.k_stride[1], p.in_bs[1] = a.k_stride[2];
  p.out_ts[0] = a.q_out_stride[0], p.out_hs[0] = a.q_out_stride[1];
  p.out_bs[0] = a.q_out_stride[2], p.out_ts[1] = a.k_out_stride[0];
  p.out_hs[1] = a.k_out_stride[1], p.out_bs[1] = a.k_out_stride[2];
  p.heads[0] = a.q_heads;
  p.heads[1] = a.k_heads;
  p.eps[0] = a.q_eps;
  p.eps[1] = a.k_eps;
  p.weight_fp32 = a.weight_fp32;
  p.batch = a.batch;
  p.tokens = a.tokens;
  p.dim = a.head_dim;
  p.rotary = a.rotary_dim;
  p.turns = a.turns;
  p.amplitude = a.amplitude;
  p.sin_sign = a.inverse ? -1.f : 1.f;
  p.axis1 = a.second_axis;
  p.axis2 = a.third_axis;
  p.pos = a.positions;
  p.pos_wide = a.positions_int64;
  p.pos_as = a.pos_stride[0];
  p.pos_bs = a.pos_stride[1];
  p.pos_ts = a.pos_stride[2];
  p.start = a.start;
  // Chunks of 16 bytes fit when every head starts on 16 bytes, the head is a
  // whole number of chunks (at most two a lane) and no chunk holds both turned
  // and other channels or, in the half layout, channels of both halves.
  const int n = static_cast<int>(16 / elem);
  int64_t strides = 0;
  for (int i = 0; i < 3; ++i) {
    strides |= a.q_stride[i] | a.q_out_stride[i];
    if (a.k_heads > 0) strides |= a.k_stride[i] | a.k_out_stride[i];
  }
  const bool vector = (all & 15) == 0 && (strides & (n - 1)) == 0 && a.head_dim % n == 0 &&
                      a.head_dim <= 64 * n && a.rotary_dim % (a.interleaved ? n : 2 * n) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case ERD_BF16: return rot::dispatch<__nv_bfloat16>(p, a.norm, a.interleaved, vector, st);
    case ERD_FP16: return rot::dispatch<__half>(p, a.norm, a.interleaved, vector, st);
    default: return rot::dispatch<float>(p, a.norm, a.interleaved, vector, st);
  }
}
