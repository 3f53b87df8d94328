// New keys and values into the paged cache in 4 bits, and the values back from
// it (declared in include/ai_attn.h, the format at AiPool4).
//
// Sixteen consecutive dims of a head row, half a group, sit in a lane, so a
// group's extremes are one shuffle; their codes are four pairs of bytes of the row.
// A warp takes K and V of 512 dims of a token at a time.
//
// A code is the whole number nearest to x / d, halves to even, as the quotient's
// exact value has it.  16-bit values: x times the reciprocal of d is good to 2^-20,
// and a quotient that is not a half exactly is at least 2^-13 from one (x has 8 or
// 11 bits, d 11), so it is rounded to 2^-16 first, which makes exact halves exact.
// fp32: the remainder x - c d of a candidate c is exact, and where it is not below
// half of d the candidate moves.
//
// Measured, for an append and a read of what it wrote (8 KV heads of 128): 64
// sequences by a token 5.3 us, two launches' latency; 8 by up to 2047 tokens of fp16
// 30 us for 115 MB (3.9 TB/s): about 550 instructions a warp for K and V of 512 dims in
// the append (the extremes, the checks for what is no number), 400 in the read, share
// the time with memory.

#include <cuda_runtime.h>

#include <cstring>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_kv4.cuh"
#include "sm100_ptx.cuh"

namespace ai {
namespace kv4 {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kDims = 16;  // of a lane

// Sixteen consecutive elements as they lie in memory: words of 32 bits.
template <typename T>
struct Raw {
  uint32_t w[4 * sizeof(T)];
};

// kAlign: the boundaries that rows start on, 32 or 16 bytes (wide accesses; with 32
// whole sectors each), or 0: element by element.
template <typename T, int kAlign>
__device__ __forceinline__ Raw<T> load(const T* p) {
  Raw<T> r;
  if constexpr (kAlign == 32) {
#pragma unroll
    for (int i = 0; i < (int)(4 * sizeof(T)); i += 8)
      asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]), "=r"(r.w[i + 4]), "=r"(r.w[i + 5]),
                     "=r"(r.w[i + 6]), "=r"(r.w[i + 7])
                   : "l"(reinterpret_cast<const uint32_t*>(p) + i));
  } else if constexpr (kAlign == 16) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
  } else {
    T e[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) e[i] = p[i];
    memcpy(&r, e, sizeof(r));
  }
  return r;
}

template <typename T, int kAlign>
__device__ __forceinline__ void store(T* p, const Raw<T>& r) {
  if constexpr (kAlign == 32) {
#pragma unroll
    for (int i = 0; i < (int)(4 * sizeof(T)); i += 8) {
      uint32_t w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = r.w[i + k];
      ptx::st_global_v8(reinterpret_cast<uint32_t*>(p) + i, w);
    }
  } else if constexpr (kAlign == 16) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
  } else {
    T e[kDims];
    memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < kDims; ++i) p[i] = e[i];
  }
}

// Sums with 2^23 + 2^22 keep whole numbers in their last bits, sums with 192 keep
// 2^-16.
constexpr float kWhole = 12582912.f, kSixteenth = 192.f;

// The bits of 2^23 + 2^22 + code.
template <typename T>
__device__ __forceinline__ uint32_t code(float x, float d, float inv) {
  float t;
  if constexpr (sizeof(T) == 2) {
    t = fmaf(x, inv, kSixteenth) - kSixteenth + (kWhole + 8.f);
  } else {
    float c = fmaf(x, inv, kWhole) - kWhole;
    const float rest = fmaf(-c, d, x), half = 0.5f * fabsf(d);
    if (!(fabsf(rest) < half)) {
      // Past the half: on to the neighbour; on it: to the even one.
      const float step = (rest < 0.f) == (d < 0.f) ? 1.f : -1.f;
      if (fabsf(rest) > half || (fabsf(rest) == half && ((int)c & 1))) c += step;
    }
    t = c + (kWhole + 8.f);
  }
  return __float_as_uint(fminf(fmaxf(t, kWhole), kWhole + 15.f));
}

// The lane's codes, a word of four per four dims, and its group's scale.
template <typename T>
__device__ __forceinline__ void quantize(const Raw<T>& raw, uint16_t (&codes)[4], __half& scale) {
  T e[kDims];
  memcpy(e, &raw, sizeof(raw));
  float f[kDims], top = -CUDART_INF_F, low = CUDART_INF_F, bad = 0.f;
#pragma unroll
  for (int i = 0; i < kDims; ++i) {
    f[i] = to_f32(e[i]);
    top = fmaxf(top, f[i]);
    low = fminf(low, f[i]);
    bad = fmaf(f[i], 0.f, bad);  // (0 times a NaN or an infinity is NaN)
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  low = fminf(low, __shfl_xor_sync(0xffffffffu, low, 1));
  bad += __shfl_xor_sync(0xffffffffu, bad, 1);
  scale = __float2half_rn(fminf(fmaxf((top > -low ? top : low) * -0.125f, -65504.f), 65504.f));
  const float d = __half2float(scale), inv = 1.f / d;
  if (bad != 0.f) scale = __ushort_as_half((unsigned short)0x7fffu);
  const bool plain = bad == 0.f && d != 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c0 = code<T>(f[4 * i], d, inv), c1 = code<T>(f[4 * i + 1], d, inv), c2 = code<T>(f[4 * i + 2], d, inv),
                   c3 = code<T>(f[4 * i + 3], d, inv);
    const uint32_t w = (c0 + (c1 << 4)) + ((c2 + (c3 << 4)) << 8);
    codes[i] = plain ? (uint16_t)w : (uint16_t)0x8888u;
  }
}

// The values of a lane's codes.
template <typename T>
__device__ __forceinline__ Raw<T> values(const uint16_t (&codes)[4], __half scale) {
  const float d = __half2float(scale);
  T e[kDims];
#pragma unroll
  for (int i = 0; i < kDims; ++i) {
    const uint32_t c = codes[i / 4] >> (4 * (i % 4)) & 15u;
    e[i] = from_f32<T>((__uint_as_float(0x4b400000u | c) - (kWhole + 8.f)) * d);
  }
  Raw<T> r;
  memcpy(&r, e, sizeof(r));
  return r;
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

// Head h of an item's token in K or V.
template <typename T>
__device__ __forceinline__ T* row(const AiTensor4& x, const Item& i, int64_t h) {
  return static_cast<T*>(const_cast<void*>(x.ptr)) + i.b * x.stride_b + h * x.stride_h + i.t * x.stride_t;
}

// Where a lane's sixteen dims of head h lie in a pool: their codes, their scale.
// (Dims 16 l + 4 i + j: group l / 2, byte pairs 4 (l % 2) + i.)
template <int D>
struct Spot {
  static constexpr int C = D / kGroup;
  uint8_t* codes;
  __half* scale;
  __device__ __forceinline__ Spot(const AiTensor4& tc, const AiTensor4& ts, const Place& p, int64_t h, int l) {
    codes = static_cast<uint8_t*>(const_cast<void*>(tc.ptr)) + p.page * tc.stride_b + h * tc.stride_h + p.slot * (D / 2) +
            (l % 2 * 4) * 2 * C + l / 2 * 2;
    scale = static_cast<__half*>(const_cast<void*>(ts.ptr)) + p.page * ts.stride_b + h * ts.stride_h + p.slot * C + l / 2;
  }
  __device__ __forceinline__ void advance(const AiTensor4& tc, const AiTensor4& ts, int heads) {
    codes += heads * tc.stride_h, scale += heads * ts.stride_h;
  }
};

// (a turn: K and V of as many heads as 512 dims are, R)
template <typename T, int D, int kAlign>
__global__ void __launch_bounds__(kThreads) append_kernel(const AiPaged4Args a, const int per, const int chunks, const uint32_t items) {
  constexpr int L = D / kDims, R = 32 / L, C = D / kGroup;  // lanes of a row
  const int lane = threadIdx.x % 32, sub = lane / L, l = lane % L;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const Item i = item_of(a, it, per, chunks);
  const int len = __ldg(a.lens + i.b);
  if (i.t >= new_tokens(a.n, i.b, a.seq_len, a.status)) return;
  // (the first turn's loads do not wait for the page, nor a turn's for the one before)
  int h = i.h0 + sub;
  const T* x[2] = {row<T>(a.k, i, h) + kDims * l, row<T>(a.v, i, h) + kDims * l};
  Raw<T> next[2] = {};
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (h < i.h1) next[u] = load<T, kAlign>(x[u]);
  const Place p = place(a.pool, i.b, (int64_t)len + i.t);
  if (p.page < 0) {
    report(a.status, AI_ERR_DEV_BOUNDS);
    return;
  }
  Spot<D> at[2] = {{a.pool.k_codes, a.pool.k_scales, p, h, l}, {a.pool.v_codes, a.pool.v_scales, p, h, l}};
  for (int h0 = i.h0; h0 < i.h1; h0 += R, h += R) {
    Raw<T> raw[2] = {next[0], next[1]};
    x[0] += R * a.k.stride_h, x[1] += R * a.v.stride_h;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (h + R < i.h1) next[u] = load<T, kAlign>(x[u]);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint16_t codes[4];
      __half scale;
      quantize<T>(raw[u], codes, scale);
      if (h < i.h1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint16_t*>(at[u].codes + k * 2 * C) = codes[k];
        if (l % 2 == 0) *at[u].scale = scale;
      }
    }
    at[0].advance(a.pool.k_codes, a.pool.k_scales, R);
    at[1].advance(a.pool.v_codes, a.pool.v_scales, R);
  }
}

template <typename T, int D, int kAlign>
__global__ void __launch_bounds__(kThreads) read_kernel(const AiPaged4Args a, const int per, const int chunks, const uint32_t items) {
  constexpr int L = D / kDims, R = 32 / L, C = D / kGroup;
  const int lane = threadIdx.x % 32, sub = lane / L, l = lane % L;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const Item i = item_of(a, it, per, chunks);
  Place p{-1, 0};
  const int len = __ldg(a.lens + i.b);
  if (i.t < new_tokens(a.n, i.b, a.seq_len, a.status)) {
    p = place(a.pool, i.b, (int64_t)len + i.t);
    if (p.page < 0) report(a.status, AI_ERR_DEV_BOUNDS);
  }
  const bool held = p.page >= 0;
  p.page = max(p.page, 0);
  T* x[2] = {row<T>(a.k, i, i.h0 + sub) + kDims * l, row<T>(a.v, i, i.h0 + sub) + kDims * l};
  Spot<D> at[2] = {{a.pool.k_codes, a.pool.k_scales, p, i.h0 + sub, l}, {a.pool.v_codes, a.pool.v_scales, p, i.h0 + sub, l}};
  for (int h = i.h0 + sub; h < i.h1; h += R) {
    if (held) {
      uint16_t codes[2][4];
      __half scale[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) codes[u][k] = *reinterpret_cast<const uint16_t*>(at[u].codes + k * 2 * C);
        scale[u] = *at[u].scale;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) store<T, kAlign>(x[u], values<T>(codes[u], scale[u]));
    } else {
      store<T, kAlign>(x[0], Raw<T>{});
      store<T, kAlign>(x[1], Raw<T>{});
    }
    x[0] += R * a.k.stride_h, x[1] += R * a.v.stride_h;
    at[0].advance(a.pool.k_codes, a.pool.k_scales, R);
    at[1].advance(a.pool.v_codes, a.pool.v_scales, R);
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
  // One turn per item while that gives every SM at most a few warps; then a
  // token's heads stay together, so its page is looked up once.
  constexpr int kTurn = 32 / (D / kDims);
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  const int per = tokens <= 4096 && kTurn < a.num_kv_heads ? kTurn : a.num_kv_heads;
  const int chunks = (a.num_kv_heads + per - 1) / per;
  const int64_t items = tokens * chunks, blocks = (items + kWarps - 1) / kWarps;
  if (items > 0x7fffffff) return AI_ERR_SHAPE;
  int align = 32;
  for (const AiTensor4* t : {&a.k, &a.v})
    while (align >= 16 && ((reinterpret_cast<uintptr_t>(t->ptr) | (uintptr_t)((t->stride_b | t->stride_h | t->stride_t) * (int64_t)sizeof(T))) & (align - 1)))
      align /= 2;
  const auto kernel = read ? (align == 32   ? read_kernel<T, D, 32>
                              : align == 16 ? read_kernel<T, D, 16>
                                            : read_kernel<T, D, 0>)
                           : (align == 32   ? append_kernel<T, D, 32>
                              : align == 16 ? append_kernel<T, D, 16>
                                            : append_kernel<T, D, 0>);
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
