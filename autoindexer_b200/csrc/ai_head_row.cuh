// One head row (D elements of one head of one token) held by D / 16 lanes:
// lane l has dims [8 l, 8 l + 8) and their rotate-half partners
// [D/2 + 8 l, D/2 + 8 l + 8), so the norm's sum is log2(D / 16) shuffles and
// the rotation needs no exchange.  fp32 arithmetic throughout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/ai_attn.h"
#include "ai_common.cuh"

namespace ai {
namespace headrow {

// Eight elements as they lie in memory (16 bytes of a 16-bit type, 32 of fp32).
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};

// kVec: rows start on 16-byte boundaries (wide loads); otherwise element by element.
template <typename T, bool kVec>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
    memcpy(&r, e, sizeof(r));
  }
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T* p, const Raw8<T>& r) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.v[i];
  } else {
    T e[8];
    memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e[i];
  }
}

// Eight values as four pairs, for the packed fp32 instructions.
struct F8 {
  float2 v[4];
};

__device__ __forceinline__ F8 fill8(float x) {
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = make_float2(x, x);
  return r;
}

__device__ __forceinline__ F8 unpack(const Raw8<float>& r) {
  F8 f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f.v[2 * i] = make_float2(__uint_as_float(r.v[i].x), __uint_as_float(r.v[i].y));
    f.v[2 * i + 1] = make_float2(__uint_as_float(r.v[i].z), __uint_as_float(r.v[i].w));
  }
  return f;
}
__device__ __forceinline__ F8 unpack(const Raw8<__nv_bfloat16>& r) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  F8 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  return f;
}
__device__ __forceinline__ F8 unpack(const Raw8<__half>& r) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  F8 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  return f;
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack(const F8& f) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[2 * i] = from_f32<T>(f.v[i].x), e[2 * i + 1] = from_f32<T>(f.v[i].y);
  Raw8<T> r;
  memcpy(&r, e, sizeof(r));
  return r;
}

// The lane's 16 weights (dims 8 l + i in lo, D/2 + 8 l + i in hi); 1 without a weight.
template <typename T>
__device__ __forceinline__ void load_weight(const void* w, bool w_f32, int D, int l, F8& lo, F8& hi) {
  lo = hi = fill8(1.f);
  if (!w) return;
  const int a = 8 * l, b = D / 2 + 8 * l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (w_f32) {
      const float* p = static_cast<const float*>(w) + 2 * i;
      lo.v[i] = make_float2(__ldg(p + a), __ldg(p + a + 1));
      hi.v[i] = make_float2(__ldg(p + b), __ldg(p + b + 1));
    } else {
      const T* p = static_cast<const T*>(w) + 2 * i;
      lo.v[i] = make_float2(to_f32(p[a]), to_f32(p[a + 1]));
      hi.v[i] = make_float2(to_f32(p[b]), to_f32(p[b + 1]));
    }
  }
}

// cos and sin of the lane's eight slots; the identity without tables.
__device__ __forceinline__ void load_angles(const float* cos, const float* sin, int64_t row, int half, int l, F8& c,
                                            F8& s) {
  if (!cos) {
    c = fill8(1.f);
    s = fill8(0.f);
    return;
  }
  const float4* pc = reinterpret_cast<const float4*>(cos + row * half + 8 * l);
  const float4* ps = reinterpret_cast<const float4*>(sin + row * half + 8 * l);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 x = __ldg(pc + i), y = __ldg(ps + i);
    c.v[2 * i] = make_float2(x.x, x.y), c.v[2 * i + 1] = make_float2(x.z, x.w);
    s.v[2 * i] = make_float2(y.x, y.y), s.v[2 * i + 1] = make_float2(y.z, y.w);
  }
}

// Table row of (row b, token t)'s position id.  The id is compared in 64 bits
// (an int64 id must not wrap into the table).
__device__ __forceinline__ int64_t table_row(const AiPositions& p, int64_t b, int64_t t, int n_pos, int32_t* status) {
  const int64_t at = b * p.stride_b + t;
  const int64_t id = p.is_int64 ? __ldg(static_cast<const long long*>(p.ptr) + at)
                                : (int64_t)__ldg(static_cast<const int32_t*>(p.ptr) + at);
  if (id < 0 || id >= n_pos) {
    report(status, AI_ERR_DEV_BOUNDS);
    return 0;
  }
  return id;
}

// Sum over the kLanes lanes of a row (every lane of the warp takes part).
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float dot8(const F8& a, const F8& b, const F8& c, const F8& d) {
  float2 s = __fmul2_rn(a.v[0], b.v[0]);
  float2 u = __fmul2_rn(c.v[0], d.v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    s = __ffma2_rn(a.v[i], b.v[i], s);
    u = __ffma2_rn(c.v[i], d.v[i], u);
  }
  s = __fadd2_rn(s, u);
  return s.x + s.y;
}

// 1 / sqrt(mean(x^2) + eps) of the row.
template <int D>
__device__ __forceinline__ float inv_rms(const F8& lo, const F8& hi, float eps) {
  return rsqrtf(row_sum<D / 16>(dot8(lo, lo, hi, hi)) * (1.f / D) + eps);
}

__device__ __forceinline__ void scale8(F8& f, float r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = __fmul2_rn(f.v[i], make_float2(r, r));
}
__device__ __forceinline__ void mul8(F8& f, const F8& g) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = __fmul2_rn(f.v[i], g.v[i]);
}

// (lo, hi) -> (lo c - hi s, hi c + lo s); kBack: the transpose.
template <bool kBack>
__device__ __forceinline__ void rotate(F8& lo, F8& hi, const F8& c, const F8& s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = lo.v[i], b = hi.v[i], n = make_float2(-s.v[i].x, -s.v[i].y);
    lo.v[i] = __ffma2_rn(a, c.v[i], __fmul2_rn(b, kBack ? s.v[i] : n));
    hi.v[i] = __ffma2_rn(b, c.v[i], __fmul2_rn(a, kBack ? n : s.v[i]));
  }
}

// A row normalised (if it has a weight) and rotated.
template <int D>
__device__ __forceinline__ void norm_rotate(F8& lo, F8& hi, bool normed, const F8& wlo, const F8& whi, const F8& c,
                                            const F8& s, float eps) {
  if (normed) {
    const float r = inv_rms<D>(lo, hi, eps);
    mul8(lo, wlo);
    mul8(hi, whi);
    scale8(lo, r);
    scale8(hi, r);
  }
  rotate<false>(lo, hi, c, s);
}

// Whether every row of a (B, H, T, D) tensor starts on a 16-byte boundary.
inline bool rows_aligned(const AiTensor4& t, int dtype) {
  const int64_t per16 = dtype == AI_DTYPE_F32 ? 4 : 8;
  return (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0 &&
         t.stride_b % per16 == 0 && t.stride_h % per16 == 0 && t.stride_t % per16 == 0;
}

}  // namespace headrow
}  // namespace ai
