// Attention over the paged cache in 4 bits (declared in include/ai_attn.h).
//
// A warp per query row, fp32 arithmetic: a lane per key forms its score, a lane
// per D / 32 dims adds the weighted values.

#include <cuda_runtime.h>
#include <math_constants.h>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_kv4.cuh"
#include "sm100_ptx.cuh"

namespace ai {
namespace attn4 {

using namespace kv4;
constexpr int kWarps = 4, kThreads = 32 * kWarps;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rows_kernel(const AiPagedAttn4Args a) {
  constexpr int C = D / kGroup;
  __shared__ float s_q[kWarps][D];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= (int64_t)a.batch * a.num_q_heads * a.seq_len) return;
  const int t = (int)(row % a.seq_len), h = (int)(row / a.seq_len % a.num_q_heads);
  const int64_t b = row / a.seq_len / a.num_q_heads;
  const int64_t hk = h / (a.num_q_heads / a.num_kv_heads);
  T* out = static_cast<T*>(const_cast<void*>(a.out.ptr)) + b * a.out.stride_b + h * a.out.stride_h + t * a.out.stride_t;
  const int n = new_tokens(a.query_lens, b, a.seq_len, a.status);
  int keys = __ldg(a.lens + b);
  const int64_t most = (int64_t)a.pool.max_pages * a.pool.page_size;
  if (keys < 0 || keys > most) report(a.status, AI_ERR_DEV_BOUNDS);
  keys = max(0, (int)min((int64_t)keys, most));
  const int seen = t < n ? max(0, keys - n + t + 1) : 0;
  const T* q = static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + h * a.q.stride_h + t * a.q.stride_t;
  for (int i = lane; i < D; i += 32) s_q[warp][i] = to_f32(q[i]);
  __syncwarp();
  float m = -CUDART_INF_F, l = 0.f, o[C] = {};
  for (int k0 = 0; k0 < seen; k0 += 32) {
    const int key = k0 + lane;
    float s = -CUDART_INF_F;
    Place p{0, 0};
    if (key < seen) {
      p = place(a.pool, b, key);
      if (p.page < 0) report(a.status, AI_ERR_DEV_BOUNDS), p.page = 0;
      const AiTensor4 &cd = a.pool.k_codes, &sc = a.pool.k_scales;
      const uint8_t* co = static_cast<const uint8_t*>(cd.ptr) + p.page * cd.stride_b + hk * cd.stride_h + p.slot * cd.stride_t;
      const __half* so = static_cast<const __half*>(sc.ptr) + p.page * sc.stride_b + hk * sc.stride_h + p.slot * sc.stride_t;
      s = 0.f;
      for (int c = 0; c < C; ++c) {
        float part = 0.f;
        for (int g = 0; g < 8; ++g)
          for (int j = 0; j < 4; ++j)
            part += (float)((co[g * 2 * C + 2 * c + j / 2] >> (4 * (j % 2)) & 15) - 8) * s_q[warp][32 * c + 4 * g + j];
        s += part * __half2float(so[c]);
      }
      s *= a.scale;
    }
    float top = s;
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    top = fmaxf(top, m);
    const float base = top == -CUDART_INF_F ? 0.f : top, e = key < seen ? expf(s - base) : 0.f;
    const float down = m == -CUDART_INF_F ? 0.f : expf(m - base);
    float sum = e;
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    l = l * down + sum;
    m = top;
    for (int c = 0; c < C; ++c) o[c] *= down;
    for (int j = 0; j < min(32, seen - k0); ++j) {
      const float w = __shfl_sync(0xffffffffu, e, j);
      const int64_t page = __shfl_sync(0xffffffffu, p.page, j), slot = __shfl_sync(0xffffffffu, p.slot, j);
      const AiTensor4 &cd = a.pool.v_codes, &sc = a.pool.v_scales;
      const uint8_t* co = static_cast<const uint8_t*>(cd.ptr) + page * cd.stride_b + hk * cd.stride_h + slot * cd.stride_t;
      const __half* so = static_cast<const __half*>(sc.ptr) + page * sc.stride_b + hk * sc.stride_h + slot * sc.stride_t;
      for (int c = 0; c < C; ++c)  // (dim 32 c + lane)
        o[c] += w * ((float)((co[lane / 4 * 2 * C + 2 * c + lane % 4 / 2] >> (4 * (lane % 2)) & 15) - 8) * __half2float(so[c]));
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int c = 0; c < C; ++c) out[32 * c + lane] = from_f32<T>(o[c] * inv);
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -CUDART_INF_F : m + logf(l);
}

int check(const AiPagedAttn4Args* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->batch > 4096 || a->seq_len <= 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads)
    return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16) return AI_ERR_DTYPE;
  for (const AiTensor4* t : {&a->q, &a->out}) {
    if (!t->ptr) return AI_ERR_NULL;
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < 0) return AI_ERR_STRIDE;
  }
  if (!a->lens) return AI_ERR_NULL;
  return check_pool(a->pool, a->head_dim);
}

template <typename T, int D>
int launch(const AiPagedAttn4Args& a, cudaStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.num_q_heads * a.seq_len, blocks = (rows + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff) return AI_ERR_SHAPE;
  ProfScope ps(AI_PROF_ATTN4, st);
  rows_kernel<T, D><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int dispatch(const AiPagedAttn4Args& a, cudaStream_t st) {
  if (a.head_dim == 128) return launch<T, 128>(a, st);
  if (a.head_dim == 64) return launch<T, 64>(a, st);
  return launch<T, 32>(a, st);
}

}  // namespace attn4
}  // namespace ai

extern "C" int ai_paged_attn_4bit_workspace(const AiPagedAttn4Args* args, size_t* bytes) {
  const int rc = ai::attn4::check(args);
  if (rc != AI_OK) return rc;
  if (!bytes) return AI_ERR_NULL;
  *bytes = 0;
  return AI_OK;
}

extern "C" int ai_paged_attn_4bit(const AiPagedAttn4Args* args, void* stream) {
  const int rc = ai::attn4::check(args);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::attn4::dispatch<__nv_bfloat16>(*args, st);
  return ai::attn4::dispatch<__half>(*args, st);
}
