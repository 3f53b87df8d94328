// Verification of drafted tokens (declared in include/ai_attn.h): softmax
// normalisers of every target and draft row, the acceptance tests, and the
// next token by an exponential race over the residual distribution.
//
// HBM-bound: every logit is read once for its row's normaliser, and of each
// sequence one target row, one draft row and the noise row once more for the
// race (mostly from L2).  Two launches:
//   stats  a CTA per (row, vocabulary slice): running maximum, its lowest
//          index and the sum of exp((x - max) / tau), merged over the CTA;
//   pick   a CTA per (sequence, slice): every CTA of a sequence merges the
//          slices of its rows and finds the first refusal (the same
//          arithmetic in the same order, so they agree), then races its
//          slice; an atomic maximum over (value, ~index) keys keeps the
//          winner, exact in any order, and the sequence's last CTA writes
//          its results.

#include <cuda_runtime.h>
#include <math_constants.h>

#include "ai_common.cuh"
#include "ai_kernels.h"

namespace ai {
namespace verify {

constexpr int kThreads = 256;
constexpr int kMaxDraft = 64;

struct Stat {
  float m;  // largest logit (-inf for an empty or fully masked slice)
  float s;  // sum of exp((x - m) / tau)
  int at;   // lowest index of m
};

// Workspace: Stat [rows][splits], then per sequence two race keys (residual,
// target) and an arrival count.
struct Ws {
  Stat* stat;
  unsigned long long* key;  // [B][2]
  unsigned int* arrived;    // [B]
  int splits, slice;        // of the stats pass (slice: a multiple of 8)
};

template <typename T>
__device__ __forceinline__ float at(const T* p, int64_t i) {
  return to_f32(p[i]);
}

// exp((x - m) / tau); 0 for a masked logit.
__device__ __forceinline__ float weight(float x, float m, float inv_tau) {
  return x == -CUDART_INF_F ? 0.f : expf((x - m) * inv_tau);
}

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float inv_tau) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  r.at = a.m > b.m ? a.at : b.m > a.m ? b.at : min(a.at, b.at);
  r.s = (a.m == -CUDART_INF_F ? 0.f : a.s * expf((a.m - r.m) * inv_tau)) +
        (b.m == -CUDART_INF_F ? 0.f : b.s * expf((b.m - r.m) * inv_tau));
  return r;
}

__device__ __forceinline__ float tau_of(const AiVerifyArgs& a, int b) {
  return a.temperature ? __ldg(a.temperature + b) : 1.f;
}

__device__ __forceinline__ int drafted(const AiVerifyArgs& a, int b) {
  const int n = a.draft_lens ? __ldg(a.draft_lens + b) : a.n_draft;
  return max(0, min(n, a.n_draft));
}

// Row r of sequence b: the target rows, then the draft rows.
template <typename T>
__device__ __forceinline__ const T* row_ptr(const AiVerifyArgs& a, int64_t b, int r) {
  if (r <= a.n_draft) return static_cast<const T*>(a.target) + b * a.target_stride_b + r * a.target_stride_t;
  return static_cast<const T*>(a.draft) + b * a.draft_stride_b + (r - a.n_draft - 1) * a.draft_stride_t;
}

__device__ __forceinline__ int n_rows(const AiVerifyArgs& a) { return a.n_draft + 1 + (a.draft ? a.n_draft : 0); }

template <typename T>
__global__ void __launch_bounds__(kThreads) stats_kernel(const AiVerifyArgs a, const Ws w) {
  const int split = blockIdx.x, rows = n_rows(a), r = blockIdx.y % rows, b = blockIdx.y / rows;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if (r == 0 && split == 0 && tid == 0) {
    w.key[2 * b] = w.key[2 * b + 1] = 0;
    w.arrived[b] = 0;
  }
  // Rows past the sequence's drafted tokens are not needed.
  const int n = drafted(a, b);
  const int i = r <= a.n_draft ? r : r - a.n_draft - 1;
  if (i > n || (r > a.n_draft && i >= n)) return;
  const float tau = tau_of(a, b), inv = tau > 0.f ? 1.f / tau : 0.f;
  const T* x = row_ptr<T>(a, b, r);
  const int v0 = split * w.slice, v1 = min(a.vocab, v0 + w.slice);
  Stat st{-CUDART_INF_F, 0.f, 0x7fffffff};
  for (int v = v0 + tid; v < v1; v += kThreads) {
    const float f = at(x, v);
    if (f > st.m || st.at == 0x7fffffff) {
      st.s = st.s * (st.m == -CUDART_INF_F ? 0.f : expf((st.m - f) * inv));
      st.m = f;
      st.at = v;
    }
    st.s += weight(f, st.m, inv);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat t;
    t.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    t.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    t.at = __shfl_xor_sync(0xffffffffu, st.at, o);
    st = merge(st, t, inv);
  }
  __shared__ Stat sm[kThreads / 32];
  if (lane == 0) sm[warp] = st;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < kThreads / 32; ++k) st = merge(st, sm[k], inv);
    w.stat[(int64_t)blockIdx.y * w.splits + split] = st;
  }
}

// Race key: larger value first, then the lower index.
__device__ __forceinline__ unsigned long long race_key(float value, int v) {
  return ((unsigned long long)__float_as_uint(value) << 32) | (unsigned int)(~v);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pick_kernel(const AiVerifyArgs a, const Ws w, const int slice) {
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid % 32;
  const int n = drafted(a, b), rows = n_rows(a);
  const float tau = tau_of(a, b), inv = tau > 0.f ? 1.f / tau : 0.f;
  __shared__ Stat st[2 * kMaxDraft + 1];
  __shared__ int s_refused[kMaxDraft + 1];
  for (int r = tid; r < rows; r += kThreads) {
    const int i = r <= a.n_draft ? r : r - a.n_draft - 1;
    if (i > n || (r > a.n_draft && i >= n)) continue;
    const Stat* p = w.stat + ((int64_t)b * rows + r) * w.splits;
    Stat s = p[0];
    for (int k = 1; k < w.splits; ++k) s = merge(s, p[k], inv);
    st[r] = s;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    long long tok = a.tokens[(int64_t)b * a.n_draft + i];
    bool ok;
    if (tok < 0 || tok >= a.vocab) {
      report(a.status, AI_ERR_DEV_BOUNDS);
      ok = false;
    } else if (!(tau > 0.f)) {
      ok = tok == st[i].at;
    } else {
      const Stat& sp = st[i];
      const float p = sp.s > 0.f ? weight(at(row_ptr<T>(a, b, i), tok), sp.m, inv) / sp.s : 0.f;
      float q = 1.f;
      if (a.draft) {
        const Stat& sq = st[a.n_draft + 1 + i];
        q = sq.s > 0.f ? weight(at(row_ptr<T>(a, b, a.n_draft + 1 + i), tok), sq.m, inv) / sq.s : 0.f;
      }
      ok = __ldg(a.uniforms + (int64_t)b * a.n_draft + i) * q < p;
    }
    s_refused[i] = !ok;
  }
  __syncthreads();
  int stop = 0;
  while (stop < n && !s_refused[stop]) ++stop;

  if (tau > 0.f) {
    const int v0 = blockIdx.x * slice, v1 = min(a.vocab, v0 + slice);
    const T* xp = row_ptr<T>(a, b, stop);
    const bool residual = stop < n, with_q = residual && a.draft;
    const T* xq = with_q ? row_ptr<T>(a, b, a.n_draft + 1 + stop) : nullptr;
    const Stat sp = st[stop];
    const Stat sq = with_q ? st[a.n_draft + 1 + stop] : Stat{0.f, 1.f, 0};
    const long long tok = residual ? a.tokens[(int64_t)b * a.n_draft + stop] : -1;
    const float* e = a.noise + (int64_t)b * a.vocab;
    unsigned long long best = 0, best_p = 0;
    for (int v = v0 + tid; v < v1; v += kThreads) {
      const float p = sp.s > 0.f ? weight(at(xp, v), sp.m, inv) / sp.s : 0.f;
      float r = p;
      if (with_q)
        r = fmaxf(p - (sq.s > 0.f ? weight(at(xq, v), sq.m, inv) / sq.s : 0.f), 0.f);
      else if (residual && v == tok)
        r = 0.f;
      const float noise = __ldg(e + v);
      const unsigned long long k = race_key(r > 0.f ? r / noise : 0.f, v);
      const unsigned long long kp = race_key(p > 0.f ? p / noise : 0.f, v);
      best = k > best ? k : best;
      best_p = kp > best_p ? kp : best_p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o), kp = __shfl_xor_sync(0xffffffffu, best_p, o);
      best = k > best ? k : best;
      best_p = kp > best_p ? kp : best_p;
    }
    if (lane == 0) {
      atomicMax(w.key + 2 * b, best);
      atomicMax(w.key + 2 * b + 1, best_p);
    }
  }
  // The sequence's last CTA writes its results.
  __shared__ bool s_last;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(w.arrived + b, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  int next;
  if (tau > 0.f) {
    const unsigned long long k = *(volatile unsigned long long*)(w.key + 2 * b);
    const unsigned long long kp = *(volatile unsigned long long*)(w.key + 2 * b + 1);
    next = (int)~(unsigned int)((k >> 32) ? k : kp);
  } else {
    next = st[stop].at;
  }
  for (int i = tid; i <= a.n_draft; i += kThreads) {
    const int64_t o = (int64_t)b * (a.n_draft + 1) + i;
    long long word = -1;
    float lp = 0.f;
    if (i <= stop) {
      word = i < stop ? a.tokens[(int64_t)b * a.n_draft + i] : next;
      if (tau > 0.f) lp = (at(row_ptr<T>(a, b, i), word) - st[i].m) * inv - logf(st[i].s);
    }
    a.out_tokens[o] = word;
    a.logprobs[o] = lp;
  }
  if (tid == 0) a.accepted[b] = stop;
}

int check(const AiVerifyArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->vocab <= 0 || a->n_draft < 0 || a->n_draft > kMaxDraft) return AI_ERR_SHAPE;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  if (!a->target || !a->noise || !a->accepted || !a->out_tokens || !a->logprobs) return AI_ERR_NULL;
  if (a->n_draft > 0 && (!a->tokens || !a->uniforms)) return AI_ERR_NULL;
  if (a->target_stride_b < 0 || a->target_stride_t < 0 || a->draft_stride_b < 0 || a->draft_stride_t < 0)
    return AI_ERR_STRIDE;
  if ((int64_t)a->batch * (2 * a->n_draft + 1) > 65535 || a->vocab > 0x40000000) return AI_ERR_SHAPE;
  return AI_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Slices of the vocabulary for `rows` rows: enough CTAs for eight per SM,
// but at least 2048 logits each.
void cut(const AiVerifyArgs& a, int64_t rows, int* splits, int* slice) {
  const int64_t want = (8 * (int64_t)sm_count() + rows - 1) / rows;
  const int64_t most = (a.vocab + 2047) / 2048;
  int64_t n = want < most ? want : most;
  if (n < 1) n = 1;
  *slice = (int)(((a.vocab + n - 1) / n + 7) / 8 * 8);
  *splits = (a.vocab + *slice - 1) / *slice;
}

int64_t row_count(const AiVerifyArgs& a) {
  return (int64_t)a.batch * (a.n_draft + 1 + (a.draft ? a.n_draft : 0));
}

size_t layout(const AiVerifyArgs& a, Ws* w) {
  const int64_t rows = row_count(a);
  cut(a, rows, &w->splits, &w->slice);
  const size_t stat = ((size_t)rows * w->splits * sizeof(Stat) + 255) & ~size_t(255);
  const size_t key = ((size_t)a.batch * 2 * sizeof(unsigned long long) + 255) & ~size_t(255);
  char* p = static_cast<char*>(a.workspace);
  w->stat = reinterpret_cast<Stat*>(p);
  w->key = reinterpret_cast<unsigned long long*>(p + stat);
  w->arrived = reinterpret_cast<unsigned int*>(p + stat + key);
  return stat + key + (((size_t)a.batch * sizeof(unsigned int) + 255) & ~size_t(255));
}

template <typename T>
int launch(const AiVerifyArgs& a, const Ws& w, cudaStream_t st) {
  ProfScope ps(AI_PROF_VERIFY, st);
  stats_kernel<T><<<dim3(w.splits, (unsigned)row_count(a)), kThreads, 0, st>>>(a, w);
  int splits, slice;
  cut(a, a.batch, &splits, &slice);
  pick_kernel<T><<<dim3(splits, a.batch), kThreads, 0, st>>>(a, w, slice);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace verify
}  // namespace ai

extern "C" int ai_verify_draft_workspace(const AiVerifyArgs* args, size_t* bytes) {
  const int rc = ai::verify::check(args);
  if (rc != AI_OK) return rc;
  if (!bytes) return AI_ERR_NULL;
  ai::verify::Ws w;
  *bytes = ai::verify::layout(*args, &w);
  return AI_OK;
}

extern "C" int ai_verify_draft(const AiVerifyArgs* args, void* stream) {
  const int rc = ai::verify::check(args);
  if (rc != AI_OK) return rc;
  ai::verify::Ws w;
  const size_t need = ai::verify::layout(*args, &w);
  if (!args->workspace || args->workspace_bytes < need) return AI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(args->workspace) & 255) return AI_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::verify::launch<__nv_bfloat16>(*args, w, st);
  if (args->dtype == AI_DTYPE_F16) return ai::verify::launch<__half>(*args, w, st);
  return ai::verify::launch<float>(*args, w, st);
}
