// New keys and values into the paged cache in 4 bits, and the values back from
// it (declared in include/ai_attn.h, the format at AiPool4).
//
// A head row sits in eight lanes: lane g has dims 32 c + 4 g + {0 .. 3} of every
// group c, whose codes are its D / 16 consecutive bytes of the row, so a row's
// bytes leave in one piece and a group's extremes are three shuffles.  A warp
// takes four heads of a token at a time, K rows and V rows alike.
//
// A code is the whole number nearest to x / d, halves to even, as the quotient's
// exact value has it: x times the reciprocal gives a candidate c, the remainder
// x - c d is exact in fp32 (c is off by less than one, so it has no more bits
// than x and d together leave), and where it is not below half of d the candidate
// moves.

#include <cuda_runtime.h>

#include <cstring>

#include "ai_head_row.cuh"
#include "ai_kernels.h"
#include "ai_kv4.cuh"

namespace ai {
namespace kv4 {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kRows = 4;  // head rows of a warp

// Four consecutive elements.
template <typename T, bool kVec>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (kVec && sizeof(T) == 4) {
    return __ldg(reinterpret_cast<const float4*>(p));
  } else if constexpr (kVec) {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
    T e[4];
    memcpy(e, &r, 8);
    return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
  } else {
    return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ void store4(T* p, float4 f) {
  T e[4] = {from_f32<T>(f.x), from_f32<T>(f.y), from_f32<T>(f.z), from_f32<T>(f.w)};
  if constexpr (kVec && sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = f;
  } else if constexpr (kVec) {
    uint2 r;
    memcpy(&r, e, 8);
    *reinterpret_cast<uint2*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = e[i];
  }
}

__device__ __forceinline__ int code(float x, float d, float inv) {
  constexpr float kShift = 12582912.f;  // 1.5 2^23: the sum's last bit counts ones
  float c = fmaf(x, inv, kShift) - kShift;
  const float rest = fmaf(-c, d, x), half = 0.5f * fabsf(d);
  if (!(fabsf(rest) < half)) {
    // Past the half: on to the neighbour; on it: to the even one.
    const float step = (rest < 0.f) == (d < 0.f) ? 1.f : -1.f;
    if (fabsf(rest) > half || (fabsf(rest) == half && ((int)c & 1))) c += step;
  }
  return (int)fminf(fmaxf(c, -8.f), 7.f) + 8;
}

// The lane's codes and the scales of a row of which it has f[c] (eight lanes).
template <int C>
__device__ __forceinline__ void quantize(const float4 (&f)[C], uint16_t (&codes)[C], __half (&scales)[C]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float top = fmaxf(fmaxf(f[c].x, f[c].y), fmaxf(f[c].z, f[c].w));
    float low = fminf(fminf(f[c].x, f[c].y), fminf(f[c].z, f[c].w));
    // (0 times a NaN or an infinity is NaN)
    float bad = f[c].x * 0.f + f[c].y * 0.f + (f[c].z * 0.f + f[c].w * 0.f);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      bad += __shfl_xor_sync(0xffffffffu, bad, o);
    }
    const float want = fminf(fmaxf((top > -low ? top : low) * -0.125f, -65504.f), 65504.f);
    __half h = __float2half_rn(want);
    const float d = __half2float(h), inv = 1.f / d;
    uint32_t q = 0x8888u;
    if (bad != 0.f) {
      h = __ushort_as_half((unsigned short)0x7fffu);
    } else if (d != 0.f) {
      q = code(f[c].x, d, inv) | code(f[c].y, d, inv) << 4 | code(f[c].z, d, inv) << 8 | code(f[c].w, d, inv) << 12;
    }
    codes[c] = (uint16_t)q;
    scales[c] = h;
  }
}

// Which token and heads an item is about.
struct Item {
  int64_t b;
  int t, h0, h1;
};

__device__ __forceinline__ Item item_of(const AiPaged4Args& a, uint32_t it, int per, int chunks) {
  const uint32_t tok = it / (uint32_t)chunks, seq = tok / (uint32_t)a.seq_len;
  Item r;
  r.b = seq;
  r.t = (int)(tok - seq * (uint32_t)a.seq_len);
  r.h0 = (int)(it - tok * (uint32_t)chunks) * per;
  r.h1 = min(a.num_kv_heads, r.h0 + per);
  return r;
}

template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads, 6) append_kernel(const AiPaged4Args a, const int per, const int chunks,
                                                             const uint32_t items) {
  constexpr int C = D / kGroup;
  const int lane = threadIdx.x % 32, sub = lane / 8, g = lane % 8;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const Item i = item_of(a, it, per, chunks);
  if (i.t >= new_tokens(a.n, i.b, a.seq_len, a.status)) return;
  const Place p = place(a.pool, i.b, (int64_t)__ldg(a.lens + i.b) + i.t);
  if (p.page < 0) {
    report(a.status, AI_ERR_DEV_BOUNDS);
    return;
  }
  for (int hb = i.h0; hb < i.h1; hb += kRows) {
    const int64_t h = min(hb + sub, i.h1 - 1);  // (rows past the last head repeat it, unstored)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const AiTensor4 &src = kv ? a.v : a.k, &cd = kv ? a.pool.v_codes : a.pool.k_codes,
                      &sc = kv ? a.pool.v_scales : a.pool.k_scales;
      const T* x = static_cast<const T*>(src.ptr) + i.b * src.stride_b + h * src.stride_h + i.t * src.stride_t + 4 * g;
      float4 f[C];
#pragma unroll
      for (int c = 0; c < C; ++c) f[c] = load4<T, kVec>(x + kGroup * c);
      uint16_t codes[C];
      __half scales[C];
      quantize<C>(f, codes, scales);
      if (hb + sub < i.h1) {
        uint8_t* co = static_cast<uint8_t*>(const_cast<void*>(cd.ptr)) + p.page * cd.stride_b + h * cd.stride_h +
                      p.slot * cd.stride_t + g * 2 * C;
        __half* so = static_cast<__half*>(const_cast<void*>(sc.ptr)) + p.page * sc.stride_b + h * sc.stride_h +
                     p.slot * sc.stride_t;
        if constexpr (C == 4) {
          uint2 r;
          memcpy(&r, codes, 8);
          *reinterpret_cast<uint2*>(co) = r;
          if (g == 0) {
            memcpy(&r, scales, 8);
            *reinterpret_cast<uint2*>(so) = r;
          }
        } else if constexpr (C == 2) {
          uint32_t r;
          memcpy(&r, codes, 4);
          *reinterpret_cast<uint32_t*>(co) = r;
          if (g == 0) {
            memcpy(&r, scales, 4);
            *reinterpret_cast<uint32_t*>(so) = r;
          }
        } else {
          *reinterpret_cast<uint16_t*>(co) = codes[0];
          if (g == 0) *so = scales[0];
        }
      }
    }
  }
}

template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads, 6) read_kernel(const AiPaged4Args a, const int per, const int chunks,
                                                           const uint32_t items) {
  constexpr int C = D / kGroup;
  const int lane = threadIdx.x % 32, sub = lane / 8, g = lane % 8;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const Item i = item_of(a, it, per, chunks);
  const bool wanted = i.t < new_tokens(a.n, i.b, a.seq_len, a.status);
  Place p{-1, 0};
  if (wanted) {
    p = place(a.pool, i.b, (int64_t)__ldg(a.lens + i.b) + i.t);
    if (p.page < 0) report(a.status, AI_ERR_DEV_BOUNDS);
  }
  for (int hb = i.h0; hb < i.h1; hb += kRows) {
    const int64_t h = hb + sub;
    if (h >= i.h1) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const AiTensor4 &dst = kv ? a.v : a.k, &cd = kv ? a.pool.v_codes : a.pool.k_codes,
                      &sc = kv ? a.pool.v_scales : a.pool.k_scales;
      uint16_t codes[C] = {};
      __half scales[C] = {};
      if (p.page >= 0) {
        const uint8_t* co = static_cast<const uint8_t*>(cd.ptr) + p.page * cd.stride_b + h * cd.stride_h +
                            p.slot * cd.stride_t + g * 2 * C;
        const __half* so = static_cast<const __half*>(sc.ptr) + p.page * sc.stride_b + h * sc.stride_h +
                           p.slot * sc.stride_t;
        if constexpr (C == 4) {
          uint2 r = *reinterpret_cast<const uint2*>(co);
          memcpy(codes, &r, 8);
          r = *reinterpret_cast<const uint2*>(so);
          memcpy(scales, &r, 8);
        } else if constexpr (C == 2) {
          uint32_t r = *reinterpret_cast<const uint32_t*>(co);
          memcpy(codes, &r, 4);
          r = *reinterpret_cast<const uint32_t*>(so);
          memcpy(scales, &r, 4);
        } else {
          codes[0] = *reinterpret_cast<const uint16_t*>(co);
          scales[0] = *so;
        }
      }
      T* x = static_cast<T*>(const_cast<void*>(dst.ptr)) + i.b * dst.stride_b + h * dst.stride_h + i.t * dst.stride_t + 4 * g;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float d = __half2float(scales[c]);
        const int q = codes[c];
        auto value = [&](int j) { return (float)((q >> (4 * j) & 15) - 8) * d; };
        store4<T, kVec>(x + kGroup * c, p.page >= 0 ? make_float4(value(0), value(1), value(2), value(3)) : make_float4(0.f, 0.f, 0.f, 0.f));
      }
    }
  }
}

int check(const AiPaged4Args* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->num_kv_heads <= 0) return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  for (const AiTensor4* t : {&a->k, &a->v}) {
    if (!t->ptr) return AI_ERR_NULL;
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < 0) return AI_ERR_STRIDE;
  }
  if (!a->lens) return AI_ERR_NULL;
  return check_pool(a->pool, a->head_dim);
}

template <typename T, int D>
int launch(const AiPaged4Args& a, bool read, cudaStream_t st) {
  // One row group per item while that gives every SM at most a few warps; then
  // a token's heads stay together, so its page is looked up once.
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  const int per = tokens <= 4096 ? (kRows < a.num_kv_heads ? kRows : a.num_kv_heads) : a.num_kv_heads;
  const int chunks = (a.num_kv_heads + per - 1) / per;
  const int64_t items = tokens * chunks, blocks = (items + kWarps - 1) / kWarps;
  if (items > 0x7fffffff) return AI_ERR_SHAPE;
  const bool vec = headrow::rows_aligned(a.k, a.dtype) && headrow::rows_aligned(a.v, a.dtype);
  const auto kernel = read ? (vec ? read_kernel<T, D, true> : read_kernel<T, D, false>)
                           : (vec ? append_kernel<T, D, true> : append_kernel<T, D, false>);
  ProfScope ps(AI_PROF_PAGED4, st);
  kernel<<<(unsigned)blocks, kThreads, 0, st>>>(a, per, chunks, (uint32_t)items);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int dispatch(const AiPaged4Args& a, bool read, cudaStream_t st) {
  if (a.head_dim == 128) return launch<T, 128>(a, read, st);
  if (a.head_dim == 64) return launch<T, 64>(a, read, st);
  return launch<T, 32>(a, read, st);
}

int run(const AiPaged4Args* a, bool read, void* stream) {
  const int rc = check(a);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == AI_DTYPE_BF16) return dispatch<__nv_bfloat16>(*a, read, st);
  if (a->dtype == AI_DTYPE_F16) return dispatch<__half>(*a, read, st);
  return dispatch<float>(*a, read, st);
}

}  // namespace kv4
}  // namespace ai

extern "C" int ai_paged_append_4bit(const AiPaged4Args* args, void* stream) { return ai::kv4::run(args, false, stream); }
extern "C" int ai_paged_read_4bit(const AiPaged4Args* args, void* stream) { return ai::kv4::run(args, true, stream); }
