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
// HBM-bound: a row is read once and its gradient written.  A row is cut for a
// cluster of CTAs, so that its slices stay in their shared memory between the sums
// and the gradient: one bulk copy a slice, the listed words masked there (the sums
// then need no look at the list), the sums exchanged through distributed shared
// memory.

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
constexpr int kLeast = 16 * 1024;      // bytes of a slice, at least (for more CTAs than the memory asks for)
constexpr int kSlice = 40 * 1024;      // bytes of a slice where there are rows enough: five CTAs per SM
constexpr int kWidth = 32;             // slices are whole vectors of so many lanes
static_assert(AI_DISTILL_MAX_ROW_BYTES / kMaxSplit + 16 * kWidth <= 200 * 1024, "a slice in shared memory");
constexpr long long kWait = 1000000000LL;
static_assert(kMaxTop <= kThreads, "a thread per entry");
// A remainder of the teacher's probability below 2^-20 is what the rounding of
// its fp32 log-probabilities may leave.
constexpr float kLeastRest = 0x1p-20f;

constexpr int kSets = kMaxTop / 32;  // entries of a lane

// What the first warp finds out of a row's list while the slice is on its way.
struct List {
  int live;            // whether the row has an entry (and a weight)
  int word[kMaxTop];   // -1: left out
  float p_top, p_rest; // the teacher's probability on the listed words, and beside them
  float m, s;          // the student's logits there: the largest, and the sum of 2^((x - m) c)
  float term;          // sum p (ln p - (x - m) / tau)
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// 2^((x - m) c), 0 for a masked logit and NaN for NaN and +inf (m may be -inf).
__device__ __forceinline__ float share(float x, float c, float m) {
  return x == -CUDART_INF_F ? 0.f : ptx::ex2((x - m) * c);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 5) distill_kernel(const AiDistillArgs a, const int splits) {
  constexpr int E = 16 / sizeof(T);
  __shared__ List list;
  __shared__ float2 s_parts[kMaxSplit * kWarps];  // (m, s) of each warp of the cluster
  __shared__ __align__(8) uint64_t s_bar;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, K = a.n_top;
  const int64_t row = blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const int64_t b = row / a.seq_len, t = row - b * a.seq_len;
  const T* x = static_cast<const T*>(a.logits) + b * a.stride_b + t * a.stride_t;
  T* d = a.dlogits ? static_cast<T*>(a.dlogits) + b * a.dstride_b + t * a.dstride_t : nullptr;
  const Slice sl = slice_of(x, a.vocab, split, splits, kWidth);
  const int vecs = sl.i1 - sl.i0;
  const uint32_t bar = ptx::smem_u32(&s_bar);
  // (a CTA of the cluster must run before its shared memory is written to)
  if (splits > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");
  int word[kSets];
  float logp[kSets], wgt = 1.f;
  if (warp == 0) {
    if (a.weights) wgt = __ldg(a.weights + row);
    bool any = false;
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      const int k = 32 * i + lane;
      word[i] = -1;
      logp[i] = -CUDART_INF_F;
      if (32 * i >= K) continue;  // (here and below: sets past the list take no instruction of the warp)
      if (k < K) {
        const long long w = a.top_tokens[row * K + k];
        logp[i] = a.top_logprobs[row * K + k];
        if (wgt != 0.f && w >= a.vocab && split == 0) report(a.status, AI_ERR_DEV_BOUNDS);
        if (wgt != 0.f && w >= 0 && w < a.vocab && logp[i] != -CUDART_INF_F) word[i] = (int)w;
      }
      list.word[k] = word[i];
      any |= word[i] >= 0;
    }
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) {
      ptx::mbar_init(bar, 1);
      ptx::fence_mbar_init();
      list.live = any;
      if (any && vecs > 0) {
        ptx::mbar_arrive_expect_tx(bar, 16u * vecs);
        ptx::bulk_load(ptx::smem_u32(smem), x + sl.head + (int64_t)sl.i0 * E, 16u * vecs, bar);
      }
    }
  }
  __syncthreads();
  if (!list.live) {
    if (split == 0 && tid == 0 && a.losses) a.losses[row] = 0.f;
    if (d) {
      const Slice z = slice_of(d, a.vocab, split, splits, kWidth);
      uint4* dv = reinterpret_cast<uint4*>(d + z.head);
      for (int i = z.i0 + tid; i < z.i1; i += kThreads) __stcs(dv + i, make_uint4(0u, 0u, 0u, 0u));
      if (tid < E) {
        if (z.e0 + tid < z.head) d[tid] = from_f32<T>(0.f);
        if (z.e1 > z.tail && z.tail + tid < a.vocab) d[z.tail + tid] = from_f32<T>(0.f);
      }
    }
    return;
  }
  const float tau = row_tau(a.temperature, b, split == 0 && tid == 0 ? a.status : nullptr), c = slope(tau), inv = inverse(tau);
  float p[kSets], xk[kSets];
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kSets; ++i) xk[i] = word[i] >= 0 ? at(x, word[i]) : -CUDART_INF_F;
    // A word that an earlier entry has is left out.
    bool again[kSets] = {};
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      if (32 * i >= K) continue;
      again[i] = (__match_any_sync(0xffffffffu, word[i]) & ((1u << lane) - 1)) != 0;
      for (int j = 0; j < 32 * i; ++j) again[i] |= list.word[j] == word[i];
    }
    __syncwarp();
    float top = -CUDART_INF_F, m = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      if (32 * i >= K) continue;
      if (again[i] && word[i] >= 0) {
        if (split == 0) report(a.status, AI_ERR_DEV_BOUNDS);
        word[i] = list.word[32 * i + lane] = -1;
        xk[i] = -CUDART_INF_F;
      }
      if (word[i] >= 0) top = fmaxf(top, logp[i]);
      m = fmaxf(m, xk[i]);
    }
    const bool renorm = a.tail == AI_TAIL_RENORMALIZE;
    if (renorm) {
      top = warp_max(top);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kSets; ++i)
        if (32 * i < K) sum += word[i] >= 0 ? expf(logp[i] - top) : 0.f;
      const float norm = top + logf(warp_sum(sum));
#pragma unroll
      for (int i = 0; i < kSets; ++i) logp[i] -= norm;
    }
    m = warp_max(m);
    const float o = m == -CUDART_INF_F ? 0.f : m;
    float p_top = 0.f, sum = 0.f, term = 0.f;
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      if (32 * i >= K) continue;
      p[i] = word[i] >= 0 ? expf(logp[i]) : 0.f;
      p_top += p[i];
      sum += share(xk[i], c, o);
      if (p[i] != 0.f) term += p[i] * (logp[i] - (xk[i] - o) * inv);
    }
    p_top = warp_sum(p_top);
    sum = warp_sum(sum);
    term = warp_sum(term);
    if (lane == 0) {
      list.p_top = p_top;
      list.p_rest = p_top != p_top ? p_top : renorm || 1.f - p_top < kLeastRest ? 0.f : 1.f - p_top;
      list.m = m;
      list.s = sum;
      list.term = term;
    }
  }
  if (vecs > 0 && !ptx::mbar_wait(bar, 0, kWait)) {
    report(a.status, AI_ERR_DEV_TIMEOUT);
    ptx::mbar_wait(bar, 0, kWait);  // (the copy lands before the CTA ends)
  }
  // The listed words' places become -inf, which adds nothing to the others' sum.
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      const int at_ = word[i] - sl.head - sl.i0 * E;
      if (word[i] >= 0 && at_ >= 0 && at_ < vecs * E) reinterpret_cast<T*>(smem)[at_] = from_f32<T>(-CUDART_INF_F);
    }
  }
  __syncthreads();
  const uint4* held = reinterpret_cast<const uint4*>(smem);
  const uint4 none = make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
  Part part{-CUDART_INF_F, 0.f, 0.f};
  for (int i = tid; i < vecs; i += kThreads * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = i + u * kThreads < vecs ? held[i + u * kThreads] : none;
    accumulate<T, U, false>(part, raw, c);
  }
  if (tid < E) {
    auto one = [&](int v) {
      for (int j = 0; j < K; ++j)
        if (list.word[j] == v) return;
      const float f = at(x, v);
      part = merge(part, Part{f, f == -CUDART_INF_F ? 0.f : f - f + 1.f, 0.f}, c);
    };
    if (sl.e0 + tid < sl.head) one(tid);
    if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) one(sl.tail + tid);
  }
  // The warps' sums go to every CTA of the cluster; each joins them in the same order.
  {
    const float m = warp_max(part.m), s = warp_sum(part.m == -CUDART_INF_F ? part.s : part.s * ptx::ex2((part.m - m) * c));
    if (splits > 1) {
      const cg::cluster_group cluster = cg::this_cluster();
      asm volatile("barrier.cluster.wait;" ::: "memory");
      if (lane < splits) cluster.map_shared_rank(s_parts, lane)[split * kWarps + warp] = make_float2(m, s);
      cluster.sync();
    } else {
      if (lane == 0) s_parts[warp] = make_float2(m, s);
      __syncthreads();
    }
  }
  float m_rest = -CUDART_INF_F, s_rest = 0.f;
  for (int i = lane; i < splits * kWarps; i += 32) m_rest = fmaxf(m_rest, s_parts[i].x);
  m_rest = warp_max(m_rest);
  for (int i = lane; i < splits * kWarps; i += 32) {
    const float2 q = s_parts[i];
    s_rest += q.x == -CUDART_INF_F ? q.y : q.y * ptx::ex2((q.x - m_rest) * c);
  }
  s_rest = warp_sum(s_rest);
  // All words: the listed ones beside the others.
  const float p_top = list.p_top, m_all = fmaxf(list.m, m_rest);
  const float of_top = list.m == -CUDART_INF_F ? 0.f : ptx::ex2((list.m - m_all) * c);
  const float of_rest = m_rest == -CUDART_INF_F ? 0.f : ptx::ex2((m_rest - m_all) * c);
  const float s_all = list.s * of_top + (m_rest == -CUDART_INF_F ? s_rest : s_rest * of_rest);
  const float p_rest = s_rest == 0.f ? 0.f : list.p_rest;  // (no word for the bucket)
  const bool empty = s_all == 0.f;
  const float l2 = log2f(s_all);
  if (split == 0 && tid == 0 && a.losses) {
    // sum p (ln p - ln q), the list's part having been taken from its own largest logit
    const float o = list.m == -CUDART_INF_F ? 0.f : list.m;
    float loss = list.term;
    if (p_top != 0.f) loss += p_top * ((m_all - o) * inv + l2 * kLn2);
    if (p_rest != 0.f) loss += p_rest * (logf(p_rest) - (m_rest - m_all) * inv - (log2f(s_rest) - l2) * kLn2);
    a.losses[row] = empty ? CUDART_INF_F : loss;
  }
  if (!d) return;
  const float weight = a.weights ? __ldg(a.weights + row) : 1.f;
  const float up = weight * inv, mass = p_top + p_rest, m = m_rest == -CUDART_INF_F ? 0.f : m_rest;
  const float coef = s_rest == 0.f ? 0.f : up * (mass * of_rest / s_all - p_rest / s_rest);
  const float2 nm = make_float2(-m, -m), cc = make_float2(c, c), cf = make_float2(coef, coef);
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  uint4* dv = reinterpret_cast<uint4*>(d + sl.head) + sl.i0;
#pragma unroll 2
  for (int i = tid; i < vecs; i += kThreads) {
    float2 f[E / 2];
    Vec<T>::get(held[i], f);
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
      for (int q = 0; q < E; ++q) d[sl.head + (sl.i0 + i) * E + q] = el[q];
    }
  }
  if (tid < E) {
    auto one = [&](int v) { d[v] = from_f32<T>(ptx::ex2((at(x, v) - m) * c) * coef); };
    if (sl.e0 + tid < sl.head) one(tid);
    if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) one(sl.tail + tid);
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      if (word[i] < sl.e0 || word[i] >= sl.e1) continue;
      const float q = share(xk[i], c, m_all) / s_all;
      d[word[i]] = from_f32<T>(empty ? 0.f : up * (mass * q - p[i]));
    }
  }
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
  if ((int64_t)a->vocab * (a->dtype == AI_DTYPE_F32 ? 4 : 2) > AI_DISTILL_MAX_ROW_BYTES) return AI_ERR_SHAPE;
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

// CTAs of a row: what its slices ask for, and as many as give four CTAs per SM.
int slices(const AiDistillArgs& a) {
  const int64_t rows = (int64_t)a.batch * a.seq_len, bytes = (int64_t)a.vocab * (a.dtype == AI_DTYPE_F32 ? 4 : 2);
  int s = 1;
  while (s < kMaxSplit && (s * (int64_t)kSlice < bytes || (2 * s * rows <= 4 * (int64_t)sm_count() && 2 * s * (int64_t)kLeast <= bytes))) s *= 2;
  return s;
}

// Bytes of the largest slice (slice_of's rounding included).
int64_t slice_bytes(const AiDistillArgs& a, int splits) {
  const int e = a.dtype == AI_DTYPE_F32 ? 4 : 8;
  const int64_t vecs = a.vocab / e;
  return ((vecs + splits - 1) / splits + kWidth - 1) / kWidth * kWidth * 16;
}

template <typename T>
int launch(const AiDistillArgs& a, cudaStream_t st) {
  const int splits = slices(a);
  const int64_t smem = slice_bytes(a, splits);
  if (splits > 8 &&
      cudaFuncSetAttribute(distill_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return AI_ERR_LAUNCH;
  if (cudaFuncSetAttribute(distill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return AI_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.batch * a.seq_len * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
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
