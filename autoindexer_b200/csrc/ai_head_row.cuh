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

template <typename T>
__device__ __forceinline__ void unpack(const Raw8<T>& r, float (&f)[8]) {
  T e[8];
  memcpy(e, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack(const float (&f)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
  Raw8<T> r;
  memcpy(&r, e, sizeof(r));
  return r;
}

// The lane's 16 weights (dims 8 l + i in lo, D/2 + 8 l + i in hi); 1 without a weight.
template <typename T>
__device__ __forceinline__ void load_weight(const void* w, bool w_f32, int D, int l, float (&lo)[8], float (&hi)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 1.f;
  if (!w) return;
  const int a = 8 * l, b = D / 2 + 8 * l;
  if (w_f32) {
    const float* p = static_cast<const float*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = __ldg(p + a + i), hi[i] = __ldg(p + b + i);
  } else {
    const T* p = static_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = to_f32(p[a + i]), hi[i] = to_f32(p[b + i]);
  }
}

// cos and sin of the lane's eight slots; the identity without tables.
__device__ __forceinline__ void load_angles(const float* cos, const float* sin, int64_t row, int half, int l,
                                            float (&c)[8], float (&s)[8]) {
  if (!cos) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    return;
  }
  const float4* pc = reinterpret_cast<const float4*>(cos + row * half + 8 * l);
  const float4* ps = reinterpret_cast<const float4*>(sin + row * half + 8 * l);
  const float4 c0 = __ldg(pc), c1 = __ldg(pc + 1), s0 = __ldg(ps), s1 = __ldg(ps + 1);
  c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
  s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
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

// x -> 1 / sqrt(mean(x^2) + eps) of the row.
template <int D>
__device__ __forceinline__ float inv_rms(const float (&lo)[8], const float (&hi)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(lo[i], lo[i], fmaf(hi[i], hi[i], ss));
  return rsqrtf(row_sum<D / 16>(ss) * (1.f / D) + eps);
}

__device__ __forceinline__ void rotate(float (&lo)[8], float (&hi)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = lo[i], b = hi[i];
    lo[i] = a * c[i] - b * s[i];
    hi[i] = b * c[i] + a * s[i];
  }
}

// Whether every row of a (B, H, T, D) tensor starts on a 16-byte boundary.
inline bool rows_aligned(const AiTensor4& t, int dtype) {
  const int64_t per16 = dtype == AI_DTYPE_F32 ? 4 : 8;
  return (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0 &&
         t.stride_b % per16 == 0 && t.stride_h % per16 == 0 && t.stride_t % per16 == 0;
}

}  // namespace headrow
}  // namespace ai
