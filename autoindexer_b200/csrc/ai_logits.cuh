// Rows of logits as the vocabulary kernels read them: 16-byte vectors of a row,
// and the exponent of a logit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include <cfloat>

#include "ai_common.cuh"
#include "sm100_ptx.cuh"

namespace ai {
namespace logits {

template <typename T>
__device__ __forceinline__ float at(const T* p, int64_t i) {
  return to_f32(p[i]);
}

// 16 bytes of logits: all -inf, the larger of each pair of places, the largest,
// as fp32 pairs and back (rounded once).
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ static float top(uint32_t a) { return __uint_as_float(a); }
  __device__ static void get(const uint4& r, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    f[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  __device__ static uint4 put(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr uint32_t kNone = 0xff80ff80u;
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ static float top(uint32_t a) {
    return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
  }
  __device__ static void get(const uint4& r, float2 (&f)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ static uint4 put(const float2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __float22bfloat162_rn(f[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec<__half> {
  static constexpr uint32_t kNone = 0xfc00fc00u;
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ static float top(uint32_t a) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&a));
    return fmaxf(f.x, f.y);
  }
  __device__ static void get(const uint4& r, float2 (&f)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
  __device__ static uint4 put(const float2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __float22half2_rn(f[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Slope c of a row's exponent (1 for a greedy row, which has no use for it),
// finite and above zero: a logit at the maximum keeps the exponent 0 and a
// masked one -inf at any temperature, subnormal or infinite ones included.
__device__ __forceinline__ float slope(float tau) {
  return tau > 0.f ? fminf(fmaxf(kLog2e / tau, FLT_MIN), FLT_MAX) : 1.f;
}

// 1 / tau of a temperature above zero, finite: what a difference of logits is
// times this is a difference of log-probabilities, in fp32's range where the
// logits are (in units of log 2 it may pass it).
__device__ __forceinline__ float inverse(float tau) { return fminf(1.f / tau, FLT_MAX); }

// d (a difference of logits, -inf for a masked one) times `inv`, 1 / tau or a
// probability over tau, which may be 0 (an infinite temperature) or infinite.
__device__ __forceinline__ float scaled(float d, float inv) { return d == 0.f || d == -CUDART_INF_F ? d : d * inv; }

// A finite upstream gradient over tau, short of fp32's range by 2^12: what it meets,
// weights of 0 among it, gives no NaN at the smallest temperatures.
__device__ __forceinline__ float over_tau(float up, float inv) {
  constexpr float kMost = FLT_MAX * 0x1p-12f;
  const float x = up * inv;
  return fabsf(x) > kMost && fabsf(up) < CUDART_INF_F ? copysignf(kMost, x) : x;
}

// 2^((x - m) c), 0 for a masked logit (m may be -inf then).
__device__ __forceinline__ float weight(float x, float c, float m) {
  return x == -CUDART_INF_F ? 0.f : ptx::ex2((x - m) * c);
}

// The exponent of a weight that is 0 anyway, in products with that weight.
constexpr float kNoWeight = -500.f;

// Exponentials of a part of a row.  A NaN or +inf among its logits makes s NaN.
struct Part {
  float m;  // the largest logit; -inf without an unmasked one
  float s;  // sum of the weights e = 2^y, y = (x - m) c
  float t;  // sum of e y, where it is wanted (the entropy is ln 2 (log2 s - t / s))
};

__device__ __forceinline__ Part merge(const Part& a, const Part& b, float c) {
  Part r;
  r.m = fmaxf(a.m, b.m);
  const float ya = a.m == -CUDART_INF_F ? -CUDART_INF_F : (a.m - r.m) * c, fa = ptx::ex2(ya);
  const float yb = b.m == -CUDART_INF_F ? -CUDART_INF_F : (b.m - r.m) * c, fb = ptx::ex2(yb);
  r.s = a.s * fa + b.s * fb;
  r.t = fa * fmaf(fmaxf(ya, kNoWeight), a.s, a.t) + fb * fmaf(fmaxf(yb, kNoWeight), b.s, b.t);
  return r;
}

__device__ __forceinline__ Part merge_lanes(Part p, float c) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    Part q;
    q.m = __shfl_xor_sync(0xffffffffu, p.m, d);
    q.s = __shfl_xor_sync(0xffffffffu, p.s, d);
    q.t = __shfl_xor_sync(0xffffffffu, p.t, d);
    p = merge(p, q, c);
  }
  return p;
}

// The largest of vectors [u0, u1) (NaN counts as -inf).
template <typename T, int U>
__device__ __forceinline__ float largest(const uint4 (&raw)[U], int u0, int u1) {
  uint32_t big = Vec<T>::kNone;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u >= u0 && u < u1)
      big = Vec<T>::larger(big, Vec<T>::larger(Vec<T>::larger(raw[u].x, raw[u].y), Vec<T>::larger(raw[u].z, raw[u].w)));
  return Vec<T>::top(big);
}

// Adds U vectors of logits, `largest` among them, to a thread's part (vectors past
// the row's end are all -inf, which adds nothing).  kT: with t.
template <typename T, int U, bool kT>
__device__ __forceinline__ void accumulate(Part& p, const uint4 (&raw)[U], float c, float largest) {
  constexpr int E = 16 / sizeof(T);
  // (without an unmasked logit the maximum stays -inf and nothing is added)
  const float top = fmaxf(p.m, largest), o = top == -CUDART_INF_F ? 0.f : top;
  const float2 no = make_float2(-o, -o), cc = make_float2(c, c);
  float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float2 f[E / 2];
    Vec<T>::get(raw[u], f);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      const float2 y = __fmul2_rn(__fadd2_rn(f[k], no), cc);
      const float2 e = make_float2(ptx::ex2(y.x), ptx::ex2(y.y));
      s = __fadd2_rn(s, e);
      if constexpr (kT) t = __ffma2_rn(e, make_float2(fmaxf(y.x, kNoWeight), fmaxf(y.y, kNoWeight)), t);
    }
  }
  const float y = p.m == -CUDART_INF_F ? -CUDART_INF_F : (p.m - top) * c, f = ptx::ex2(y);
  if constexpr (kT) p.t = f * fmaf(fmaxf(y, kNoWeight), p.s, p.t) + (t.x + t.y);
  p.s = p.s * f + (s.x + s.y);
  p.m = top;
}

template <typename T, int U, bool kT>
__device__ __forceinline__ void accumulate(Part& p, const uint4 (&raw)[U], float c) {
  accumulate<T, U, kT>(p, raw, c, largest<T, U>(raw, 0, U));
}

// The temperature of a batch row; one that is not above zero is reported and
// counts as 1.
__device__ __forceinline__ float row_tau(const float* temperature, int64_t b, int32_t* status) {
  if (!temperature) return 1.f;
  const float tau = __ldg(temperature + b);
  if (tau > 0.f) return tau;
  report(status, AI_ERR_DEV_BOUNDS);
  return 1.f;
}

// A row cut for `splits` CTAs, in units of `unit` vectors: whole 16-byte vectors [i0, i1) of
// the row from its first boundary (element `head`), in the CTA's slice, and the
// elements [e0, e1) that the slice covers with the row's ragged ends, which the
// first and the last slice have.
struct Slice {
  int head, tail;  // elements before the first vector; first element behind the last one
  int i0, i1;
  int e0, e1;
};

template <typename T>
__device__ __forceinline__ Slice slice_of(const T* row, int vocab, int split, int splits, int unit) {
  constexpr int E = 16 / sizeof(T);
  Slice r;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  r.head = min(vocab, (E - mis) % E);
  const int vecs = (vocab - r.head) / E;
  r.tail = r.head + vecs * E;
  const int per = ((vecs + splits - 1) / splits + unit - 1) / unit * unit;
  r.i0 = min(vecs, split * per);
  r.i1 = min(vecs, r.i0 + per);
  r.e0 = split == 0 ? 0 : r.head + r.i0 * E;
  r.e1 = split == splits - 1 ? vocab : r.head + r.i1 * E;
  return r;
}

}  // namespace logits
}  // namespace ai
