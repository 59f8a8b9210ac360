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
// per token and pair and no table is read.  A lane owns two chunks of a head that
// hold whole pairs in either layout, so accesses are wide and the norm's sum needs
// log2(lanes per head) shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/eraserdit_b200.h"
#include "host_common.h"

namespace erd {
namespace rot {

constexpr int kWarps = 4;
constexpr int kMaxHeadDim = 1024;
// Head groups that a warp requests together; the next ones are on the way while
// these are turned, and the first ones while the angles are computed.
constexpr int kUnroll = 1;

struct Params {
  const void* in[2];  // queries, keys
  void* out[2];
  const void* weight[2];  // null: 1
  long long in_ts[2], in_hs[2], in_bs[2];
  long long out_ts[2], out_hs[2], out_bs[2];
  int heads[2];
  float eps[2], inv_dim;
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
  unsigned long long addresses;  // all data pointers and all strides, or-ed (host)
  long long strides;
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

// One value, and 32-bit words of one or two values, as floats.
template <typename T>
struct Value;
template <>
struct Value<__nv_bfloat16> {
  static constexpr int kPerWord = 2;
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t pack(const float* f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16(x); }
};
template <>
struct Value<__half> {
  static constexpr int kPerWord = 2;
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
    f[0] = h.x;
    f[1] = h.y;
  }
  static __device__ __forceinline__ uint32_t pack(const float* f) {
    const __half2 h = __floats2half2_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};
template <>
struct Value<float> {
  static constexpr int kPerWord = 1;
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t pack(const float* f) { return __float_as_uint(f[0]); }
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ float round(float x) { return x; }
};

// A chunk of N values, read and written at once.
template <typename T, int N>
struct __align__(sizeof(T) * N) Chunk {
  static constexpr int kWords = N / Value<T>::kPerWord;
  uint32_t w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) Value<T>::unpack(w[i], f + i * Value<T>::kPerWord);
  }
  __device__ __forceinline__ void pack(const float* f) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = Value<T>::pack(f + i * Value<T>::kPerWord);
  }
};

// Weights of channels [c, c + N) of one norm.
template <typename T, int N>
__device__ __forceinline__ void load_weight(const Params& p, int which, int c, float* w) {
  if (p.weight_fp32) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = static_cast<const float*>(p.weight[which])[c + i];
  } else {
    const T* base = static_cast<const T*>(p.weight[which]) + c;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = Value<T>::one(base[i]);
  }
}

// N: channels of a chunk.  With 16-byte chunks 32 warps a multiprocessor hold the
// rotation (64 registers; 6.5 TB/s), 24 the norm with it (80 registers, a lane's
// coefficients double; 5.1 TB/s).  Two head groups at a time, more or fewer warps,
// larger blocks, and 8-byte chunks for the norm (265 us, twice the sums to wait
// for) were slower at 2 x 32640 tokens x 64 heads x 64.
template <typename T, int N, bool kNorm, bool kInterleaved>
__global__ void __launch_bounds__(32 * kWarps, kNorm ? 6 : 8) head_rotary_kernel(const Params p) {
  using V = Chunk<T, N>;
  extern __shared__ float2 slabs[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const long long token = item / p.chunks;
  if (token >= static_cast<long long>(p.batch) * p.tokens) return;
  const int part = static_cast<int>(item - token * p.chunks);
  const int b = static_cast<int>(token / p.tokens);
  const int tok = static_cast<int>(token - static_cast<long long>(b) * p.tokens);

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
  const int first = part * p.chunk, last = min(first + p.chunk, p.iters[0] + p.iters[1]);
  // Head group i of queries, then keys: its tensor and this lane's head.
  auto place = [&](int i, int& which, int& head) {
    which = i >= p.iters[0];
    head = (which ? i - p.iters[0] : i) * per + slot;
  };
  auto request = [&](int it, V (&v0)[kUnroll], V (&v1)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      v0[u].clear();
      v1[u].clear();
      int which, head;
      place(it + u, which, head);
      if (it + u < last && head < p.heads[which]) {
        const T* src = static_cast<const T*>(p.in[which]) + b * p.in_bs[which] +
                       tok * p.in_ts[which] + head * p.in_hs[which];
        if (has0) v0[u] = *reinterpret_cast<const V*>(src + c0);
        if (has1) v1[u] = *reinterpret_cast<const V*>(src + c1);
      }
    }
  };
  V va0[kUnroll], va1[kUnroll], vb0[kUnroll], vb1[kUnroll];
  request(first, va0, va1);

  float2* slab = slabs + warp * (p.rotary / 2);
  angles(p, b, tok, lane, slab);
  // Of this lane's N pairs (a, d): a' = a ca - d sd, d' = a sa + d cd, with the
  // norm's weights of their channels multiplied in (plain channels: 1, 0, 0, 1).
  float ca[N], sd[kNorm ? N : 1], sa[N], cd[kNorm ? N : 1];
  auto coefficients = [&](int which) {
    float w[2 * N];
    if (kNorm) {
#pragma unroll
      for (int i = 0; i < 2 * N; ++i) w[i] = 1.f;
      if (p.weight[which] != nullptr) {
        if (has0) load_weight<T, N>(p, which, c0, w);
        if (has1) load_weight<T, N>(p, which, c1, w + N);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float2 cs = make_float2(1.f, 0.f);
      if (kInterleaved) {
        const int c = i < N / 2 ? c0 : c1;
        if (c < p.rotary) cs = slab[c / 2 + (i & (N / 2 - 1))];
      } else if (c0 < p.rotary) {
        cs = slab[c0 + i];
      }
      ca[i] = cs.x;
      sa[i] = cs.y;
      if (kNorm) {
        const float wa = w[kInterleaved ? 2 * i : i], wd = w[kInterleaved ? 2 * i + 1 : N + i];
        ca[i] = cs.x * wa;
        sa[i] = cs.y * wa;
        cd[i] = cs.x * wd;
        sd[i] = cs.y * wd;
      }
    }
  };
  int have = -1;
  auto turn = [&](int it, const V (&v0)[kUnroll], const V (&v1)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (it + u >= last) break;  // the same for the whole warp
      int which, head;
      place(it + u, which, head);
      if (kNorm ? which != have : have < 0) {
        coefficients(which);
        have = which;
      }
      float x[2 * N];
      v0[u].unpack(x);
      v1[u].unpack(x + N);
      float r = 1.f;
      if (kNorm) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) sum = fmaf(x[i], x[i], sum);
        for (int d = 1; d < p.lanes; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        r = rsqrtf(fmaf(sum, p.inv_dim, p.eps[which]));
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float& a = kInterleaved ? x[2 * i] : x[i];
        float& d = kInterleaved ? x[2 * i + 1] : x[N + i];
        if (kNorm) {
          a *= r;
          d *= r;
        }
        // channels that are not turned pass as they are (0 * inf is NaN)
        const bool turned = kInterleaved ? (i < N / 2 ? c0 : c1) < p.rotary : c0 < p.rotary;
        const float a0 = a, d0 = d;
        if (turned) {
          a = a0 * ca[i] - d0 * (kNorm ? sd[kNorm ? i : 0] : sa[i]);
          d = a0 * sa[i] + d0 * (kNorm ? cd[kNorm ? i : 0] : ca[i]);
        } else if (kNorm) {
          a = a0 * ca[i];
          d = d0 * cd[kNorm ? i : 0];
        }
      }
      if (head < p.heads[which]) {
        T* dst = static_cast<T*>(p.out[which]) + b * p.out_bs[which] + tok * p.out_ts[which] +
                 head * p.out_hs[which];
        V y;
        y.pack(x);
        if (has0) *reinterpret_cast<V*>(dst + c0) = y;
        y.pack(x + N);
        if (has1) *reinterpret_cast<V*>(dst + c1) = y;
      }
    }
  };
#pragma unroll 1
  for (int it = first; it < last; it += 2 * kUnroll) {
    request(it + kUnroll, vb0, vb1);
    turn(it, va0, va1);
    request(it + 2 * kUnroll, va0, va1);
    turn(it + kUnroll, vb0, vb1);
  }
}

// The same for sizes and strides that no chunk fits: a warp takes
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
        const float x = Value<T>::one(src[c]);
        sum = fmaf(x, x, sum);
      }
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      r = rsqrtf(fmaf(sum, p.inv_dim, p.eps[which]));
    }
    auto value = [&](int c) {
      float x = Value<T>::one(src[c]);
      if (kNorm) {
        float w = 1.f;
        if (p.weight[which] != nullptr)
          w = p.weight_fp32 ? static_cast<const float*>(p.weight[which])[c]
                            : Value<T>::one(static_cast<const T*>(p.weight[which])[c]);
        x = x * r * w;
      }
      return x;
    };
    for (int i = lane; i < p.rotary / 2; i += 32) {
      const int a = kInterleaved ? 2 * i : i, d = kInterleaved ? 2 * i + 1 : i + p.rotary / 2;
      const float x0 = value(a), x1 = value(d);
      const float2 cs = slab[i];
      dst[a] = Value<T>::round(x0 * cs.x - x1 * cs.y);
      dst[d] = Value<T>::round(x0 * cs.y + x1 * cs.x);
    }
    for (int c = p.rotary + lane; c < p.dim; c += 32) dst[c] = Value<T>::round(value(c));
  }
}

// Chunks of N fit when every head starts on their size, the head is a whole number
// of them (at most two a lane) and no chunk holds both turned and other channels or,
// in the half layout, channels of both halves.
template <typename T, int N>
bool chunks_fit(const Params& p, bool interleaved) {
  return (p.addresses & (N * sizeof(T) - 1)) == 0 && (p.strides & (N - 1)) == 0 && p.dim % N == 0 &&
         p.dim <= 64 * N && p.rotary % (interleaved ? N : 2 * N) == 0;
}

// A warp walks over all head groups of a token, unless that leaves the device short
// of warps (32 on each of 148 multiprocessors).
int share_tokens(Params& p, unsigned* blocks) {
  const long long tokens = static_cast<long long>(p.batch) * p.tokens;
  const int iters = p.iters[0] + p.iters[1];
  const long long share = tokens * iters / (148 * 32);
  p.chunk = static_cast<int>(share < 1 ? 1 : share > iters ? iters : share);
  p.chunks = (iters + p.chunk - 1) / p.chunk;
  const long long n = (tokens * p.chunks + kWarps - 1) / kWarps;
  if (n > 0x7fffffffLL) return kErrTooLarge;
  *blocks = static_cast<unsigned>(n);
  return kErrOk;
}

template <typename T, int N, bool kNorm, bool kInterleaved>
int launch_chunks(Params p, size_t smem, cudaStream_t stream) {
  const int tasks = (p.dim + 2 * N - 1) / (2 * N);
  p.lanes = 1;
  p.log2_lanes = 0;
  while (p.lanes < tasks) p.lanes *= 2, ++p.log2_lanes;
  const int per = 32 / p.lanes;
  for (int w = 0; w < 2; ++w) p.iters[w] = (p.heads[w] + per - 1) / per;
  unsigned blocks;
  if (int rc = share_tokens(p, &blocks)) return rc;
  head_rotary_kernel<T, N, kNorm, kInterleaved><<<blocks, 32 * kWarps, smem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// The widest chunks that fit (16, 8 or 4 bytes), else value by value.
template <typename T, bool kNorm, bool kInterleaved>
int launch(Params p, cudaStream_t stream) {
  constexpr int N = static_cast<int>(16 / sizeof(T));
  const size_t smem = static_cast<size_t>(kWarps) * (p.rotary / 2) * sizeof(float2);
  if (chunks_fit<T, N>(p, kInterleaved))
    return launch_chunks<T, N, kNorm, kInterleaved>(p, smem, stream);
  if (chunks_fit<T, N / 2>(p, kInterleaved))
    return launch_chunks<T, N / 2, kNorm, kInterleaved>(p, smem, stream);
  if constexpr (N > 4) {
    if (chunks_fit<T, N / 4>(p, kInterleaved))
      return launch_chunks<T, N / 4, kNorm, kInterleaved>(p, smem, stream);
  }
  p.lanes = 32;
  p.log2_lanes = 5;
  for (int w = 0; w < 2; ++w) p.iters[w] = p.heads[w];
  unsigned blocks;
  if (int rc = share_tokens(p, &blocks)) return rc;
  head_rotary_scalar_kernel<T, kNorm, kInterleaved>
      <<<blocks, 32 * kWarps, smem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int dispatch(const Params& p, bool norm, bool interleaved, cudaStream_t stream) {
  if (norm) return interleaved ? launch<T, true, true>(p, stream) : launch<T, true, false>(p, stream);
  return interleaved ? launch<T, false, true>(p, stream) : launch<T, false, false>(p, stream);
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
  p.inv_dim = 1.0f / static_cast<float>(a.head_dim);
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
  p.addresses = all;
  for (int i = 0; i < 3; ++i) {
    p.strides |= a.q_stride[i] | a.q_out_stride[i];
    if (a.k_heads > 0) p.strides |= a.k_stride[i] | a.k_out_stride[i];
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case ERD_BF16: return rot::dispatch<__nv_bfloat16>(p, a.norm, a.interleaved, st);
    case ERD_FP16: return rot::dispatch<__half>(p, a.norm, a.interleaved, st);
    default: return rot::dispatch<float>(p, a.norm, a.interleaved, st);
  }
}
