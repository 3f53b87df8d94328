// New keys and values into the paged cache in 4 bits, and the values back from
// it (declared in include/ai_attn.h, the format at AiPool4).
//
// Sixteen consecutive dims of a head row, half a group, sit in a lane, so a
// group's extremes are one shuffle; their codes are four pairs of bytes of the row.
// A warp takes a token's K and V rows 512 dims at a time, two such turns' loads in
// flight together.
//
// A code is the whole number nearest to x / d, halves to even, as the quotient's
// exact value has it.  16-bit values: x times the reciprocal of d is good to 2^-20,
// and a quotient that is not a half exactly is at least 2^-13 from one (x has 8 or
// 11 bits, d 11), so it is rounded to 2^-16 first, which makes exact halves exact.
// fp32: the remainder x - c d of a candidate c is exact, and where it is not below
// half of d the candidate moves.

#include <cuda_runtime.h>

#include <cstring>

#include "ai_head_row.cuh"
#include "ai_kernels.h"
#include "ai_kv4.cuh"

namespace ai {
namespace kv4 {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kDims = 16;  // of a lane

// Sixteen consecutive elements as they lie in memory.
template <typename T>
struct Raw {
  uint4 v[sizeof(T)];
};

template <typename T, bool kVec>
__device__ __forceinline__ Raw<T> load(const T* p) {
  Raw<T> r;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T e[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) e[i] = p[i];
    memcpy(&r, e, sizeof(r));
  }
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store(T* p, const Raw<T>& r) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(p)[i] = r.v[i];
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

// Which token and rows (K rows, then V rows) an item is about.
struct Item {
  int64_t b;
  int t, r0, r1;
};

__device__ __forceinline__ Item item_of(const AiPaged4Args& a, uint32_t it, int per, int chunks) {
  const uint32_t tok = it / (uint32_t)chunks, seq = tok / (uint32_t)a.seq_len;
  Item r;
  r.b = seq;
  r.t = (int)(tok - seq * (uint32_t)a.seq_len);
  r.r0 = (int)(it - tok * (uint32_t)chunks) * per;
  r.r1 = min(2 * a.num_kv_heads, r.r0 + per);
  return r;
}

// A lane's sixteen dims of a row: of the tensor, of the codes, of the scales.
template <typename T>
struct Spot {
  T* x;
  uint8_t* codes;
  __half* scale;
};

template <typename T, int D>
__device__ __forceinline__ Spot<T> spot_of(const AiPaged4Args& a, const Item& i, const Place& p, int row, int l) {
  constexpr int C = D / kGroup;
  const bool v = row >= a.num_kv_heads;
  const int64_t h = v ? row - a.num_kv_heads : row;
  const AiTensor4 &x = v ? a.v : a.k, &cd = v ? a.pool.v_codes : a.pool.k_codes, &sc = v ? a.pool.v_scales : a.pool.k_scales;
  Spot<T> r;
  r.x = static_cast<T*>(const_cast<void*>(x.ptr)) + i.b * x.stride_b + h * x.stride_h + i.t * x.stride_t + kDims * l;
  // (dims 16 l + 4 i + j: group l / 2, byte pairs 4 (l % 2) + i)
  r.codes = static_cast<uint8_t*>(const_cast<void*>(cd.ptr)) + p.page * cd.stride_b + h * cd.stride_h + p.slot * (D / 2) +
            (l % 2 * 4) * 2 * C + l / 2 * 2;
  r.scale = static_cast<__half*>(const_cast<void*>(sc.ptr)) + p.page * sc.stride_b + h * sc.stride_h + p.slot * C + l / 2;
  return r;
}

template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads) append_kernel(const AiPaged4Args a, const int per, const int chunks, const uint32_t items) {
  constexpr int L = D / kDims, R = 32 / L, C = D / kGroup;  // lanes of a row, rows of a turn
  const int lane = threadIdx.x % 32, sub = lane / L, l = lane % L;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const Item i = item_of(a, it, per, chunks);
  if (i.t >= new_tokens(a.n, i.b, a.seq_len, a.status)) return;
  const Place p = place(a.pool, i.b, (int64_t)__ldg(a.lens + i.b) + i.t);
  if (p.page < 0) {
    report(a.status, AI_ERR_DEV_BOUNDS);
    return;
  }
  for (int r0 = i.r0; r0 < i.r1; r0 += 2 * R) {
    Spot<T> at[2];
    Raw<T> raw[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      at[u] = spot_of<T, D>(a, i, p, min(r0 + u * R + sub, i.r1 - 1), l);  // (rows past the last repeat it, unstored)
      if (u == 0 || r0 + R < i.r1) raw[u] = load<T, kVec>(at[u].x);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && r0 + R >= i.r1) break;
      uint16_t codes[4];
      __half scale;
      quantize<T>(raw[u], codes, scale);
      if (r0 + u * R + sub >= i.r1) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) *reinterpret_cast<uint16_t*>(at[u].codes + k * 2 * C) = codes[k];
      if (l % 2 == 0) *at[u].scale = scale;
    }
  }
}

template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads) read_kernel(const AiPaged4Args a, const int per, const int chunks, const uint32_t items) {
  constexpr int L = D / kDims, R = 32 / L, C = D / kGroup;
  const int lane = threadIdx.x % 32, sub = lane / L, l = lane % L;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const Item i = item_of(a, it, per, chunks);
  Place p{-1, 0};
  if (i.t < new_tokens(a.n, i.b, a.seq_len, a.status)) {
    p = place(a.pool, i.b, (int64_t)__ldg(a.lens + i.b) + i.t);
    if (p.page < 0) report(a.status, AI_ERR_DEV_BOUNDS);
  }
  for (int r0 = i.r0; r0 < i.r1; r0 += 2 * R) {
    Spot<T> at[2];
    uint16_t codes[2][4];
    __half scale[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      at[u] = spot_of<T, D>(a, i, p, min(r0 + u * R + sub, i.r1 - 1), l);
#pragma unroll
      for (int k = 0; k < 4; ++k) codes[u][k] = p.page < 0 ? (uint16_t)0x8888u : *reinterpret_cast<const uint16_t*>(at[u].codes + k * 2 * C);
      scale[u] = p.page < 0 ? __ushort_as_half((unsigned short)0) : *at[u].scale;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (r0 + u * R + sub < i.r1) store<T, kVec>(at[u].x, values<T>(codes[u], scale[u]));
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
  // Two turns of rows per item while that gives every SM at most a few warps; then
  // a token's rows stay together, so its page is looked up once.
  constexpr int kTurns = 2 * 32 / (D / kDims);
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  const int rows = 2 * a.num_kv_heads, per = tokens <= 4096 && kTurns < rows ? kTurns : rows;
  const int chunks = (rows + per - 1) / per;
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
