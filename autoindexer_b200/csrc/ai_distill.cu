// Distillation from a teacher's likeliest words: the divergence of every row and
// the gradient of the student's logits, in one launch (declared in
// include/ai_attn.h).
//
// With y = (x - m) c, c = log2(e) / tau, over the words that the teacher does not
// list (m their largest logit, s the sum of 2^y), and the listed ones beside
// them: ln q_k, ln q_r and the loss follow from the two sums, and
//   dx_v = w / tau 2^y (M 2^((m - m_all) c) / s_all - p_r / s)   (not listed)
//   dx_k = w / tau (M q_k - p_k)                                 (listed).
// The others' sum is gathered without the listed words, not as a difference, so
// q_r keeps its digits where the student is sure of the listed ones.
//
// HBM-bound: a row is read and its gradient written.  A row is cut for a cluster
// of CTAs, which exchange their sums through distributed shared memory.

#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstring>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_logits.cuh"
#include "sm100_ptx.cuh"

namespace ai {
namespace distill {

using namespace logits;
namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32, U = 4;
constexpr int kMaxTop = AI_DISTILL_MAX_TOP;
constexpr int kMaxSplit = 16;
constexpr int kLeast = 8192;  // logits of a slice, at least (half for fp32)
static_assert(kMaxTop <= kThreads, "a thread per entry");
// A remainder of the teacher's probability below 2^-20 is what the rounding of
// its fp32 log-probabilities may leave.
constexpr float kLeastRest = 0x1p-20f;

// The teacher's entries of a row and what they sum up to.
struct Entries {
  int word[kMaxTop];   // -1: left out
  float x[kMaxTop];    // the student's logit
  float p[kMaxTop];    // the teacher's probability
  float logp[kMaxTop];
};

// Sum and maximum over the CTA's first kMaxTop threads' values, in a fixed order.
struct Reduce {
  float v[kWarps];
};
__device__ __forceinline__ float cta_sum(Reduce& r, float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  if (threadIdx.x % 32 == 0) r.v[threadIdx.x / 32] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < kMaxTop / 32; ++w) s += r.v[w];
  return s;
}
__device__ __forceinline__ float cta_max(Reduce& r, float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if (threadIdx.x % 32 == 0) r.v[threadIdx.x / 32] = v;
  __syncthreads();
  float s = -CUDART_INF_F;
#pragma unroll
  for (int w = 0; w < kMaxTop / 32; ++w) s = fmaxf(s, r.v[w]);
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) distill_kernel(const AiDistillArgs a, const int splits) {
  constexpr int E = 16 / sizeof(T);
  __shared__ Entries e;
  __shared__ Reduce red;
  __shared__ Part s_part[kWarps], s_slice;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, K = a.n_top;
  const int64_t row = blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const int64_t b = row / a.seq_len, t = row - b * a.seq_len;
  const T* x = static_cast<const T*>(a.logits) + b * a.stride_b + t * a.stride_t;
  T* d = a.dlogits ? static_cast<T*>(a.dlogits) + b * a.dstride_b + t * a.dstride_t : nullptr;
  const float wgt = a.weights ? __ldg(a.weights + row) : 1.f;
  const bool first = split == 0 && tid == 0;

  // The entries: those left out are found first (each thread has one).
  int word = -1;
  float logp = -CUDART_INF_F;
  if (tid < K && wgt != 0.f) {
    const long long w = a.top_tokens[row * K + tid];
    logp = a.top_logprobs[row * K + tid];
    if (w >= a.vocab) {
      if (split == 0) report(a.status, AI_ERR_DEV_BOUNDS);
    } else if (w >= 0 && logp != -CUDART_INF_F) {
      word = (int)w;
    }
  }
  if (tid < kMaxTop) e.word[tid] = word;
  __syncthreads();
  if (word >= 0) {
    bool again = false;
    for (int j = 0; j < tid; ++j) again |= e.word[j] == word;
    if (again) {
      word = -1;
      if (split == 0) report(a.status, AI_ERR_DEV_BOUNDS);
    }
  }
  const bool any = __syncthreads_or(word >= 0);
  if (!any) {
    if (first && a.losses) a.losses[row] = 0.f;
    if (d) {
      const Slice sl = slice_of(d, a.vocab, split, splits, kThreads);
      uint4* dv = reinterpret_cast<uint4*>(d + sl.head);
      for (int i = sl.i0 + tid; i < sl.i1; i += kThreads) __stcs(dv + i, make_uint4(0u, 0u, 0u, 0u));
      if (tid < E) {
        if (sl.e0 + tid < sl.head) d[tid] = from_f32<T>(0.f);
        if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) d[sl.tail + tid] = from_f32<T>(0.f);
      }
    }
    return;
  }
  const float tau = row_tau(a.temperature, b, first ? a.status : nullptr), c = slope(tau), inv = inverse(tau);
  const float xk = word >= 0 ? at(x, word) : -CUDART_INF_F;
  const bool renorm = a.tail == AI_TAIL_RENORMALIZE;
  if (renorm) {
    const float top = cta_max(red, word >= 0 ? logp : -CUDART_INF_F);
    const float sum = cta_sum(red, word >= 0 ? expf(logp - top) : 0.f);
    logp -= top + logf(sum);
  }
  const float p = word >= 0 ? expf(logp) : 0.f;
  if (tid < kMaxTop) e.word[tid] = word, e.x[tid] = xk, e.p[tid] = p, e.logp[tid] = logp;
  const float p_top = cta_sum(red, p);  // (also: the entries are written)
  float p_rest = renorm || 1.f - p_top < kLeastRest ? 0.f : 1.f - p_top;
  if (p_top != p_top) p_rest = p_top;

  // The sum over the words that are not listed.
  const bool alike = d && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const Slice sl = slice_of(x, a.vocab, split, splits, kThreads);
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  const uint4 none = make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
  Part part{-CUDART_INF_F, 0.f, 0.f};
  for (int i0 = sl.i0; i0 < sl.i1; i0 += kThreads * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = i0 + tid + u * kThreads < sl.i1 ? xv[i0 + tid + u * kThreads] : none;
    // Listed words among the warp's vectors are masked.
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v0 = sl.head + (i0 + u * kThreads + warp * 32) * E;
      for (int j0 = 0; j0 < K; j0 += 32) {
        const int mine = e.word[j0 + lane];
        uint32_t in = __ballot_sync(0xffffffffu, mine >= v0 && mine < v0 + 32 * E);
        while (in) {
          const int at_ = __shfl_sync(0xffffffffu, mine, __ffs(in) - 1) - v0;
          in &= in - 1;
          if (lane == at_ / E) {
            T el[E];
            memcpy(el, &raw[u], 16);
#pragma unroll
            for (int q = 0; q < E; ++q)
              if (q == at_ % E) el[q] = from_f32<T>(-CUDART_INF_F);
            memcpy(&raw[u], el, 16);
          }
        }
      }
    }
    accumulate<T, U, false>(part, raw, c);
  }
  if (tid < E) {
    auto one = [&](int v) {
      for (int j = 0; j < K; ++j)
        if (e.word[j] == v) return;
      const float f = at(x, v);
      part = merge(part, Part{f, f == -CUDART_INF_F ? 0.f : f - f + 1.f, 0.f}, c);
    };
    if (sl.e0 + tid < sl.head) one(tid);
    if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) one(sl.tail + tid);
  }
  part = merge_lanes(part, c);
  if (lane == 0) s_part[warp] = part;
  __syncthreads();
  part = s_part[0];
  for (int w = 1; w < kWarps; ++w) part = merge(part, s_part[w], c);
  if (splits > 1) {
    const cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) s_slice = part;
    cluster.sync();
    part = *cluster.map_shared_rank(&s_slice, 0);
    for (int r = 1; r < splits; ++r) part = merge(part, *cluster.map_shared_rank(&s_slice, r), c);
  }
  // All words: the listed ones beside the others.
  const float m_top = cta_max(red, xk), m_all = fmaxf(m_top, part.m);
  const float ek = xk == -CUDART_INF_F ? 0.f : ptx::ex2((xk - m_all) * c);
  const float down = part.m == -CUDART_INF_F ? 0.f : ptx::ex2((part.m - m_all) * c);
  const float s_all = cta_sum(red, ek) + part.s * down;
  const bool empty = s_all == 0.f;
  if (part.s == 0.f) p_rest = 0.f;  // no word for the bucket
  const float l2 = log2f(s_all);
  if (split == 0 && a.losses) {
    float term = word >= 0 && p != 0.f ? p * (logp - (xk - m_all) * inv + l2 * kLn2) : 0.f;
    float loss = cta_sum(red, term);
    if (p_rest != 0.f) loss += p_rest * (logf(p_rest) - (part.m - m_all) * inv - (log2f(part.s) - l2) * kLn2);
    if (tid == 0) a.losses[row] = empty ? CUDART_INF_F : loss;
  }
  if (d) {
    const float up = wgt * inv, mass = p_top + p_rest;
    const float m = part.m == -CUDART_INF_F ? 0.f : part.m;
    const float coef = part.s == 0.f ? 0.f : up * (mass * down / s_all - p_rest / part.s);
    const float2 nm = make_float2(-m, -m), cc = make_float2(c, c), cf = make_float2(coef, coef);
    uint4* dv = reinterpret_cast<uint4*>(d + sl.head);
    for (int i = sl.i0 + tid; i < sl.i1; i += kThreads) {
      const uint4 raw = __ldcs(xv + i);  // (dlogits may be the same memory: no non-coherent loads)
      float2 f[E / 2];
      Vec<T>::get(raw, f);
#pragma unroll
      for (int q = 0; q < E / 2; ++q) {
        const float2 y = __fmul2_rn(__fadd2_rn(f[q], nm), cc);
        f[q] = __fmul2_rn(make_float2(ptx::ex2(y.x), ptx::ex2(y.y)), cf);
      }
      const uint4 out = Vec<T>::put(f);
      if (alike) {
        __stcs(dv + i, out);
      } else {
        T el[E];
        memcpy(el, &out, 16);
#pragma unroll
        for (int q = 0; q < E; ++q) d[sl.head + i * E + q] = el[q];
      }
    }
    if (tid < E) {
      auto one = [&](int v) { d[v] = from_f32<T>(ptx::ex2((at(x, v) - m) * c) * coef); };
      if (sl.e0 + tid < sl.head) one(tid);
      if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) one(sl.tail + tid);
    }
    __syncthreads();
    if (word >= sl.e0 && word < sl.e1) d[word] = from_f32<T>(empty ? 0.f : up * (mass * (ek / s_all) - p));
  }
  if (splits > 1) cg::this_cluster().sync();  // (the sums have been read)
}

int check(const AiDistillArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->vocab <= 0 || a->vocab > 0x40000000 || a->n_top <= 0 || a->n_top > kMaxTop)
    return AI_ERR_SHAPE;
  if ((int64_t)a->batch * a->seq_len > 0x7fffffff / kMaxSplit) return AI_ERR_SHAPE;
  if (a->tail != AI_TAIL_BUCKET && a->tail != AI_TAIL_RENORMALIZE) return AI_ERR_SHAPE;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  if (!a->logits || !a->top_tokens || !a->top_logprobs || (!a->losses && !a->dlogits)) return AI_ERR_NULL;
  if (a->stride_b < 0 || a->stride_t < 0 || a->dstride_b < 0 || a->dstride_t < 0) return AI_ERR_STRIDE;
  if ((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->dlogits)) &
      (a->dtype == AI_DTYPE_F32 ? 3 : 1))
    return AI_ERR_ALIGN;
  return AI_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int slices(const AiDistillArgs& a) {
  const int64_t rows = (int64_t)a.batch * a.seq_len;
  const int least = a.dtype == AI_DTYPE_F32 ? kLeast / 2 : kLeast;
  int64_t n = 4 * (int64_t)sm_count() / rows;
  if (n > (a.vocab + least - 1) / least) n = (a.vocab + least - 1) / least;
  int s = 1;
  while (2 * s <= n && 2 * s <= kMaxSplit) s *= 2;
  return s;
}

template <typename T>
int launch(const AiDistillArgs& a, cudaStream_t st) {
  const int splits = slices(a);
  if (splits > 8 &&
      cudaFuncSetAttribute(distill_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return AI_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.batch * a.seq_len * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  ProfScope ps(AI_PROF_DISTILL, st);
  if (cudaLaunchKernelEx(&cfg, distill_kernel<T>, a, splits) != cudaSuccess) return AI_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace distill
}  // namespace ai

extern "C" int ai_distill(const AiDistillArgs* args, void* stream) {
  const int rc = ai::distill::check(args);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::distill::launch<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::distill::launch<__half>(*args, st);
  return ai::distill::launch<float>(*args, st);
}
