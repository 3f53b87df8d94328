// Attention over a paged cache of a batch whose sequences share a prefix
// (declared in include/ai_attn.h): argument checks, the one-row kernel for
// the types and layouts the tensor-core kernels do not take, and dispatch.
//
// simt: a CTA per (sequence, query token, query head).  128 keys at a time,
// prefix first: a thread per key forms its score, the CTA's running maximum
// and sum are updated, and a thread per (dim, key group) adds the weighted
// values.  fp32 throughout; bound by the K rows, which neighbouring threads
// read at a row's stride.

#include <cuda_runtime.h>
#include <math_constants.h>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_prefix_attn.h"

namespace ai {
namespace prefix {

constexpr int kThreads = 128;

__device__ __forceinline__ float block_max(float v, float* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  v = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  __syncthreads();
  return v;
}

__device__ __forceinline__ float block_sum(float v, float* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  v = (sm[0] + sm[1]) + (sm[2] + sm[3]);
  __syncthreads();
  return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) simt_kernel(const AiPrefixAttnArgs a) {
  const int tid = threadIdx.x, t = blockIdx.x % a.seq_len, h = blockIdx.x / a.seq_len, b = blockIdx.y;
  const int hk = h / (a.num_q_heads / a.num_kv_heads);
  __shared__ float s_q[D], s_p[kThreads], s_red[4], s_acc[kThreads];
  __shared__ int64_t s_v[kThreads];
  const Lens len = seq_lens(a, b);
  const int own = t < len.n ? max(0, len.keys - len.n + t + 1) : 0;
  const int shared = t < len.n ? a.prefix_len : 0;
  if (tid < D)
    s_q[tid] = to_f32(static_cast<const T*>(a.q.ptr)[b * a.q.stride_b + h * a.q.stride_h + t * a.q.stride_t + tid]) *
               a.scale;
  constexpr int kGroups = kThreads / D;
  const int d = tid % D, grp = tid / D;
  float m = -CUDART_INF_F, l = 0.f, acc = 0.f;
  __syncthreads();
  for (int64_t k0 = 0; k0 < (int64_t)shared + own; k0 += kThreads) {
    const int64_t j = k0 + tid;
    float s = -CUDART_INF_F;
    s_v[tid] = -1;
    if (j < (int64_t)shared + own) {
      const bool pre = j < shared;
      const int64_t at = pre ? j : j - shared;
      const int page = page_of(a, pre ? a.prefix_pages : a.page_table + b * a.page_table_stride, at / a.page_size);
      const T* k = static_cast<const T*>(a.k_pages.ptr) + page * a.k_pages.stride_b + hk * a.k_pages.stride_h +
                   (at % a.page_size) * a.k_pages.stride_t;
      s = 0.f;
#pragma unroll 8
      for (int i = 0; i < D; ++i) s = fmaf(s_q[i], to_f32(k[i]), s);
      s_v[tid] = page * a.v_pages.stride_b + hk * a.v_pages.stride_h + (at % a.page_size) * a.v_pages.stride_t;
    }
    const float m_new = fmaxf(m, block_max(s, s_red));
    const float base = m_new == -CUDART_INF_F ? 0.f : m_new;
    const float p = expf(s - base);
    s_p[tid] = p;
    const float alpha = expf(m - base);  // 0 while m is -inf
    l = l * alpha + block_sum(p, s_red);  // (its barriers publish s_p and s_v)
    m = m_new;
    acc *= alpha;
    for (int i = grp; i < kThreads; i += kGroups)
      if (s_v[i] >= 0) acc = fmaf(s_p[i], to_f32(static_cast<const T*>(a.v_pages.ptr)[s_v[i] + d]), acc);
    __syncthreads();
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < D) {
#pragma unroll
    for (int g = 1; g < kGroups; ++g) acc += s_acc[tid + g * D];
    T* o = static_cast<T*>(a.out.ptr) + b * a.out.stride_b + h * a.out.stride_h + t * a.out.stride_t;
    o[tid] = from_f32<T>(l > 0.f ? acc / l : 0.f);
  }
  if (tid == 0 && a.lse)
    a.lse[((int64_t)b * a.num_q_heads + h) * a.seq_len + t] = l > 0.f ? m + logf(l) : -CUDART_INF_F;
}

int check(const AiPrefixAttnArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads != 0 || a->n_pages <= 0 || a->page_size <= 0 || a->max_pages < 0 ||
      a->prefix_len < 0)
    return AI_ERR_SHAPE;
  if (a->batch > 65535 || (int64_t)a->seq_len * a->num_q_heads > 0x7fffffff ||
      (int64_t)a->max_pages * a->page_size > 0x7fffffff)
    return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  for (const AiTensor4* t : {&a->q, &a->out, &a->k_pages, &a->v_pages}) {
    if (!t->ptr) return AI_ERR_NULL;
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < 0) return AI_ERR_STRIDE;
  }
  if (!a->lens || (a->max_pages > 0 && !a->page_table) || (a->prefix_len > 0 && !a->prefix_pages)) return AI_ERR_NULL;
  if (a->page_table_stride < 0) return AI_ERR_STRIDE;
  return AI_OK;
}

template <typename T>
int simt_launch(const AiPrefixAttnArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)(a.seq_len * a.num_q_heads), a.batch);
  ProfScope ps(AI_PROF_PREFIX, st);
  if (a.head_dim == 128)
    simt_kernel<T, 128><<<grid, kThreads, 0, st>>>(a);
  else if (a.head_dim == 64)
    simt_kernel<T, 64><<<grid, kThreads, 0, st>>>(a);
  else
    simt_kernel<T, 32><<<grid, kThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace prefix
}  // namespace ai

extern "C" int ai_prefix_attn_workspace(const AiPrefixAttnArgs* args, size_t* bytes) {
  const int rc = ai::prefix::check(args);
  if (rc != AI_OK) return rc;
  if (!bytes) return AI_ERR_NULL;
  *bytes = ai::prefix::sm100_fits(*args) ? ai::prefix::sm100_workspace(*args) : 0;
  return AI_OK;
}

extern "C" int ai_prefix_attn(const AiPrefixAttnArgs* args, void* stream) {
  const int rc = ai::prefix::check(args);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ai::prefix::sm100_fits(*args)) return ai::prefix::sm100_launch(*args, st);
  if (args->dtype == AI_DTYPE_BF16) return ai::prefix::simt_launch<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::prefix::simt_launch<__half>(*args, st);
  return ai::prefix::simt_launch<float>(*args, st);
}
