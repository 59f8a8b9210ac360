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
  long long items;        // warps with work
  // Bytes from one token, head and head group to the next (vector kernel).
  unsigned in_token[2], out_token[2], in_head[2], out_head[2], in_step[2], out_step[2];
  const double* turns;    // [rotary / 2] turns per position step
  float amplitude, sin_sign;
  int axis1, axis2;  // first pair of the second and third position axis
  const void* pos;   // null: start + token
  int pos_wide;
  long long pos_as, pos_bs, pos_ts, start;
  unsigned long long addresses;  // all data pointers and all strides, or-ed (host)
  long long strides;
  unsigned long long weights;  // the norm's weight pointers, or-ed (host)
};

// Cosines of all rotated pairs of a warp's token, then sines; each part is as long as
// eight-value reads from any chunk's first pair need.
__host__ __device__ __forceinline__ int slab_part(int rotary) { return (rotary / 2 + 7) & ~7; }

// Cosine and sine of every rotated pair of one token into this warp's slab.
__device__ __forceinline__ void angles(const Params& p, int b, int tok, int lane, float* slab) {
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
    slab[i] = c * p.amplitude;
    slab[slab_part(p.rotary) + i] = s * p.amplitude * p.sin_sign;
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

// N (2, 4 or 8) neighbouring floats of shared or global memory, in reads of 16 bytes
// at most.
template <int N>
__device__ __forceinline__ void load_floats(const float* src, float* f) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(src + i);
      f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
    }
  } else {
    const float2 v = *reinterpret_cast<const float2*>(src);
    f[0] = v.x, f[1] = v.y;
  }
}

// Weights of channels [c, c + N) of one norm.
template <typename T, int N>
__device__ __forceinline__ void load_weight(const Params& p, int which, int c, float* w) {
  if (p.weight_fp32)
    load_floats<N>(static_cast<const float*>(p.weight[which]) + c, w);
  else
    reinterpret_cast<const Chunk<T, N>*>(static_cast<const T*>(p.weight[which]) + c)->unpack(w);
}

// Two floats in one register pair: one instruction does both.
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float lo, float hi) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.v) : "f"(lo), "f"(hi));
  return t;
}
__device__ __forceinline__ void split(Two t, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(t.v));
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two t;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
  return t;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two t;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return t;
}

// N: channels of a chunk.  A warp walks over head groups, the next group's values on
// the way while this one is turned, the first one's while the angles are computed.
//
// Besides memory, instructions bound it: counted at 213 a head group and 256 with the
// norm, three quarters of all issue slots went to them.  So the norm and its
// coefficients are computed two values at a time (the rotation alone is not: a factor's
// sign is free in the plain form, and eight registers fewer let 32 warps reside),
// addresses advance by a constant, and weights and angles are read 16 bytes at a time:
// 121 and 167 a group.  The norm with 16-byte chunks is held at 80 registers, so that 24
// warps reside; that spills one to three of them (4 to 12 bytes a thread).
//
// kAhead, the norm with eight groups or more a warp: it also asks L2 for the group
// behind the next, which costs no registers: what 24 warps have requested at a time
// does not cover the memory's latency.  64 heads below 100 -> 90 us, in calls back to
// back for a tenth of a second 202 -> 200 for two such clips.  With fewer groups the
// instructions weigh more (4 heads of queries and of keys 35.4 -> 36.7 us), and the
// rotation alone, whose 32 warps fill the memory, loses in a row of calls (169 -> 173).
//
// 32640 tokens with 64 values a head, rotation and norm with it: 64 heads 84 and 90 us
// (6.4 and 5.9 TB/s; 86 and 107 before all this), 8 heads 22 and 35 us (3.0 and 1.9
// TB/s; 25 and 40 before; here the angles and coefficients of a token, used once or
// twice, are most of the instructions).  Two head groups at a time, more or fewer
// warps, larger blocks, several tokens a warp, and 8-byte chunks for the norm (twice
// the sums to wait for) were slower.
template <typename T, int N, bool kNorm, bool kInterleaved, bool kAhead>
__global__ void __launch_bounds__(32 * kWarps, kNorm ? 6 : 8) head_rotary_kernel(const Params p) {
  using V = Chunk<T, N>;
  constexpr int P = N / 2;  // couples of this lane's N pairs
  extern __shared__ __align__(16) float slabs[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (item >= p.items) return;
  int part = 0, b, tok;
  if (p.items <= 0x7fffffffLL) {  // divisions of 64 bits are long
    unsigned token = static_cast<unsigned>(item);
    if (p.chunks > 1) {
      token /= static_cast<unsigned>(p.chunks);
      part = static_cast<int>(item) - static_cast<int>(token) * p.chunks;
    }
    b = static_cast<int>(token / static_cast<unsigned>(p.tokens));
    tok = static_cast<int>(token) - b * p.tokens;
  } else {
    const long long token = item / p.chunks;
    part = static_cast<int>(item - token * p.chunks);
    b = static_cast<int>(token / p.tokens);
    tok = static_cast<int>(token - static_cast<long long>(b) * p.tokens);
  }

  // This lane's two chunks of every head it meets: N pairs from N * sub on, or plain
  // channels.  In the interleaved layout the second chunk may be plain alone.
  const int sub = lane & (p.lanes - 1), slot = lane >> p.log2_lanes, per = 32 >> p.log2_lanes;
  const bool adjoin = kInterleaved || sub >= p.rotary / (2 * N);
  auto first_of = [](int i) { return kInterleaved ? 2 * i : i; };  // pair i in a lane's values
  auto second_of = [](int i) { return kInterleaved ? 2 * i + 1 : N + i; };
  const int c0 = adjoin ? 2 * N * sub : N * sub;
  const int c1 = adjoin ? c0 + N : p.rotary / 2 + c0;
  const bool has0 = c0 < p.dim, has1 = c1 < p.dim;
  const bool turned0 = c0 < p.rotary, turned1 = kInterleaved ? c1 < p.rotary : turned0;
  const int apart = (c1 - c0) * static_cast<int>(sizeof(T));
  const int first = part * p.chunk, last = min(first + p.chunk, p.iters[0] + p.iters[1]);

  int which = first >= p.iters[0], head = (first - (which ? p.iters[0] : 0)) * per + slot;
  auto place = [&](const void* base, const long long* bs, const unsigned* ts,
                   const unsigned* hs) {
    const unsigned long long at = static_cast<unsigned long long>(static_cast<unsigned>(tok)) *
                                      ts[which] +
                                  static_cast<unsigned long long>(static_cast<unsigned>(head)) *
                                      hs[which];
    return static_cast<const char*>(base) + at + b * bs[which] * static_cast<int>(sizeof(T)) +
           c0 * static_cast<int>(sizeof(T));
  };
  const char* src = place(p.in[which], p.in_bs, p.in_token, p.in_head);
  V v0, v1;  // lanes and channels outside of a head keep the zeros
  v0.clear();
  v1.clear();
  auto request = [&] {
    if (head < p.heads[which]) {
      if (has0) v0 = *reinterpret_cast<const V*>(src);
      if (has1) v1 = *reinterpret_cast<const V*>(src + apart);
    }
  };
  request();
  // Asks L2 for group `next`, the one behind the requested one, unless it is of the
  // other tensor.
  auto prefetch = [&](int next) {
    if (kAhead && next < last && next != p.iters[0] && head + per < p.heads[which]) {
      const char* at = src + p.in_step[which];
      if (has0) asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      if (!kInterleaved && has1) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + apart));
    }
  };
  prefetch(first + 1);

  const int half = slab_part(p.rotary);
  float* slab = slabs + warp * 2 * half;
  angles(p, b, tok, lane, slab);

  // Of this lane's N pairs (a, d): a' = a ca + d nd, d' = a sa + d cd, with the
  // norm's weights of their channels multiplied in (plain channels: 1, 0, 0, 1).
  Two ca[P], nd[kNorm ? P : 1], sa[P], cd[kNorm ? P : 1];
  auto coefficients = [&] {
    float w[2 * N], c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = 1.f, s[i] = 0.f;
    if (turned0) {
      load_floats<N>(slab + N * sub, c);
      load_floats<N>(slab + half + N * sub, s);
    }
    if (!turned1) {
#pragma unroll
      for (int i = N / 2; i < N; ++i) c[i] = 1.f, s[i] = 0.f;
    }
    if (kNorm) {
#pragma unroll
      for (int i = 0; i < 2 * N; ++i) w[i] = 1.f;
      if (p.weight[which] != nullptr) {
        if (has0) load_weight<T, N>(p, which, c0, w);
        if (has1) load_weight<T, N>(p, which, c1, w + N);
      }
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const Two cc = two(c[2 * j], c[2 * j + 1]), ss = two(s[2 * j], s[2 * j + 1]);
      ca[j] = cc, sa[j] = ss;
      if (kNorm) {
        const Two ns = two(-s[2 * j], -s[2 * j + 1]);
        const Two wa = two(w[first_of(2 * j)], w[first_of(2 * j + 1)]);
        const Two wd = two(w[second_of(2 * j)], w[second_of(2 * j + 1)]);
        ca[j] = mul(cc, wa), sa[j] = mul(ss, wa), cd[j] = mul(cc, wd), nd[j] = mul(ns, wd);
      }
    }
  };

  coefficients();
  char* dst = const_cast<char*>(place(p.out[which], p.out_bs, p.out_token, p.out_head));

#pragma unroll 1
  for (int it = first; it < last; ++it) {  // the same for the whole warp
    Two a[P], d[P];
    {
      float x[2 * N];
      v0.unpack(x);
      v1.unpack(x + N);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        a[j] = two(x[first_of(2 * j)], x[first_of(2 * j + 1)]);
        d[j] = two(x[second_of(2 * j)], x[second_of(2 * j + 1)]);
      }
    }
    const bool live = head < p.heads[which];
    const float eps = kNorm ? p.eps[which] : 0.f;
    if (it + 1 < last) {
      head += per;
      src += p.in_step[which];
      if (it + 1 == p.iters[0]) {
        which = 1;
        head = slot;
        src = place(p.in[1], p.in_bs, p.in_token, p.in_head);
      }
      request();
      prefetch(it + 2);
    }
    if (kNorm) {
      Two s0 = mul(a[0], a[0]), s1 = mul(d[0], d[0]);
#pragma unroll
      for (int j = 1; j < P; ++j) s0 = fma(a[j], a[j], s0), s1 = fma(d[j], d[j], s1);
      float t0, t1, t2, t3;
      split(s0, t0, t1);
      split(s1, t2, t3);
      float sum = (t0 + t1) + (t2 + t3);
      for (int m = 1; m < p.lanes; m <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      const float r = rsqrtf(fmaf(sum, p.inv_dim, eps));
      const Two rr = two(r, r);
#pragma unroll
      for (int j = 0; j < P; ++j) a[j] = mul(a[j], rr), d[j] = mul(d[j], rr);
    }
    float y[2 * N];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      Two e = mul(a[j], ca[j]), f = mul(d[j], kNorm ? cd[kNorm ? j : 0] : ca[j]);
      // channels that are not turned pass as they are (0 * inf is NaN)
      const bool turned = j < N / 4 || N < 4 ? turned0 : turned1;
      if (kNorm && turned) f = fma(a[j], sa[j], f);
      if (kNorm && turned) e = fma(d[j], nd[kNorm ? j : 0], e);
      float &e0 = y[first_of(2 * j)], &e1 = y[first_of(2 * j + 1)];
      split(e, e0, e1);
      if (!kNorm && turned) {  // a factor's sign costs nothing here, a register above
        float d0, d1, s0, s1;
        split(d[j], d0, d1);
        split(sa[j], s0, s1);
        e0 = fmaf(d0, -s0, e0);
        e1 = fmaf(d1, -s1, e1);
      }
      float &f0 = y[second_of(2 * j)], &f1 = y[second_of(2 * j + 1)];
      split(f, f0, f1);
      if (!kNorm && turned) {
        float a0, a1, s0, s1;
        split(a[j], a0, a1);
        split(sa[j], s0, s1);
        f0 = fmaf(a0, s0, f0);
        f1 = fmaf(a1, s1, f1);
      }
    }
    if (live) {
      V out;
      out.pack(y);
      if (has0) *reinterpret_cast<V*>(dst) = out;
      out.pack(y + N);
      if (has1) *reinterpret_cast<V*>(dst + apart) = out;
    }
    dst += p.out_step[which];
    if (it + 1 == p.iters[0] && it + 1 < last) {  // keys from here on
      dst = const_cast<char*>(place(p.out[1], p.out_bs, p.out_token, p.out_head));
      if (kNorm) coefficients();
    }
  }
}

// The same for sizes and strides that no chunk fits: a warp takes
// one head at a time, a lane every 32nd pair and every 32nd channel behind the
// pairs, value by value.  The norm reads the head twice (the second time from
// L1); every lane has the sum before any lane writes, so in-place calls hold.
template <typename T, bool kNorm, bool kInterleaved>
__global__ void __launch_bounds__(32 * kWarps) head_rotary_scalar_kernel(const Params p) {
  extern __shared__ __align__(16) float slabs[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (item >= p.items) return;
  const long long token = item / p.chunks;
  const int part = static_cast<int>(item - token * p.chunks);
  const int b = static_cast<int>(token / p.tokens);
  const int tok = static_cast<int>(token - static_cast<long long>(b) * p.tokens);
  const int half_slab = slab_part(p.rotary);
  float* slab = slabs + warp * 2 * half_slab;
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
      const float c = slab[i], s = slab[half_slab + i];
      dst[a] = Value<T>::round(x0 * c - x1 * s);
      dst[d] = Value<T>::round(x0 * s + x1 * c);
    }
    for (int c = p.rotary + lane; c < p.dim; c += 32) dst[c] = Value<T>::round(value(c));
  }
}

// Chunks of N fit when every head and the norm's weights start on their size, the head
// is a whole number of them (at most two a lane) and no chunk holds both turned and
// other channels or, in the half layout, channels of both halves.  Chunks of two pairs
// in the interleaved layout are turned together, so both are or neither is.  Steps
// from token to token and from head group to head group have 32 bits.
template <typename T, int N>
bool chunks_fit(const Params& p, bool interleaved) {
  for (int w = 0; w < 2; ++w) {
    for (long long n : {p.in_ts[w], p.out_ts[w], 32 * p.in_hs[w], 32 * p.out_hs[w]})
      if (n < 0 || n > 0x7fffffffLL / 4) return false;
  }
  return (p.addresses & (N * sizeof(T) - 1)) == 0 && (p.strides & (N - 1)) == 0 && p.dim % N == 0 &&
         p.dim <= 64 * N && p.rotary % (interleaved && N != 2 ? N : 2 * N) == 0 &&
         (p.weights & (N * (p.weight_fp32 ? 4 : sizeof(T)) < 16
                           ? N * (p.weight_fp32 ? 4 : sizeof(T)) - 1
                           : 15)) == 0;
}

// A warp walks over all head groups of a token, unless that leaves the device short
// of warps (32 on each of 148 multiprocessors).
int share_tokens(Params& p, unsigned* blocks) {
  const long long tokens = static_cast<long long>(p.batch) * p.tokens;
  const int iters = p.iters[0] + p.iters[1];
  const long long share = tokens * iters / (148 * 32);
  p.chunk = static_cast<int>(share < 1 ? 1 : share > iters ? iters : share);
  p.chunks = (iters + p.chunk - 1) / p.chunk;
  p.items = tokens * p.chunks;
  const long long n = (p.items + kWarps - 1) / kWarps;
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
  for (int w = 0; w < 2; ++w) {
    p.iters[w] = (p.heads[w] + per - 1) / per;
    auto bytes = [](long long n) { return static_cast<unsigned>(n * sizeof(T)); };
    p.in_token[w] = bytes(p.in_ts[w]);
    p.out_token[w] = bytes(p.out_ts[w]);
    p.in_head[w] = bytes(p.in_hs[w]);
    p.out_head[w] = bytes(p.out_hs[w]);
    p.in_step[w] = bytes(p.in_hs[w] * per);
    p.out_step[w] = bytes(p.out_hs[w] * per);
  }
  unsigned blocks;
  if (int rc = share_tokens(p, &blocks)) return rc;
  if constexpr (kNorm && N * sizeof(T) == 16) {
    if (p.chunk >= 8) {
      head_rotary_kernel<T, N, kNorm, kInterleaved, true>
          <<<blocks, 32 * kWarps, smem, stream>>>(p);
      return static_cast<int>(cudaGetLastError());
    }
  }
  head_rotary_kernel<T, N, kNorm, kInterleaved, false><<<blocks, 32 * kWarps, smem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// The widest chunks that fit (16, 8 or 4 bytes), else value by value.
template <typename T, bool kNorm, bool kInterleaved>
int launch(Params p, cudaStream_t stream) {
  constexpr int N = static_cast<int>(16 / sizeof(T));
  const size_t smem = static_cast<size_t>(kWarps) * 2 * slab_part(p.rotary) * sizeof(float);
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
  if (norm)
    return interleaved ? launch<T, true, true>(p, stream) : launch<T, true, false>(p, stream);
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
  p.weights = a.norm ? weights : 0;
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
