// Verification of drafted tokens (declared in include/ai_attn.h): softmax
// normalisers of every target and draft row, the acceptance tests, and the
// next token by an exponential race over the residual distribution.
//
// HBM-bound: every logit is read once for its row's normaliser, and of each
// sequence one target row, one draft row and the noise row once more for the
// race (mostly from L2).  Measured with a vocabulary of 151,936: 64 sequences of
// four drafts, bf16: 51 us (4.2 TB/s of what is read once; the stats pass
// alone 35 us, 5.0 TB/s); 16 of seven, fp32, no draft logits: 22.5 us; one of
// three: 8.4 us, two launches' latency.  Two launches, the second started by programmatic
// dependent launch:
//   stats  a CTA per (row, vocabulary slice): the largest logit m and the
//          sum of 2^((x - m) c), c = log2(e) / tau, four 16-byte loads per
//          thread in flight from the row's first 16-byte boundary (the ragged
//          ends one by one); in greedy rows the maximum's lowest index
//          instead of the sum;
//   pick   a CTA per (sequence, slice): every CTA of a sequence merges the
//          slices of its rows (a warp per row) and finds the first refusal
//          (the same arithmetic in the same order, so they agree), then races
//          its slice; an atomic maximum over (value, ~index) keys keeps the
//          winner, exact in any order, and the sequence's last CTA writes
//          its results.

#include <cuda_runtime.h>
#include <math_constants.h>

#include <cfloat>
#include <cstring>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "sm100_ptx.cuh"

namespace ai {
namespace verify {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxDraft = 64;
// Logits of a slice, at least: a round of 16-byte loads of all the CTA's threads
// (stats, 16-bit logits; half for fp32), one round of the race.  One sequence of
// three drafts, vocabulary 151,936, bf16: stats 9.1 / 8.4 / 8.8 us with 4096 /
// 8192 / 16384, race 8.4 / 8.4 / 9.7 with 1024 / 2048 / 8192.
constexpr int kLeastStats = 8192, kLeastPick = 2048;

// The exponent of a logit is (x - m) c: the difference first, so that the
// largest logit's weight is 1 at every temperature.  (As x c - m c the rounding
// of m c is a factor of every weight, which leaves fp32's range once c m passes
// 2^31: temperatures below 1e-7.)
struct Stat {
  float m;  // the largest logit; -inf for an empty or fully masked slice
  float s;  // sum of 2^((x - m) c)
  int at;   // greedy rows: lowest index of the largest logit
};

// Workspace: Stat [rows][splits], then per sequence a race key and an arrival
// count.
struct Ws {
  Stat* stat;
  unsigned long long* key;
  unsigned int* arrived;
  int splits;  // of the stats pass
};

template <typename T>
__device__ __forceinline__ float at(const T* p, int64_t i) {
  return to_f32(p[i]);
}

// 16 bytes of logits: all -inf, the larger of each pair of places, the largest.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ static float top(uint32_t a) { return __uint_as_float(a); }
  __device__ static void get(const uint4& r, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    f[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr uint32_t kNone = 0xff80ff80u;
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ static float top(uint32_t a) {
    return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
  }
  __device__ static void get(const uint4& r, float2 (&f)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
template <> struct Vec<__half> {
  static constexpr uint32_t kNone = 0xfc00fc00u;
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  __device__ static float top(uint32_t a) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&a));
    return fmaxf(f.x, f.y);
  }
  __device__ static void get(const uint4& r, float2 (&f)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
};

// Slope c of a row's exponent (1 for a greedy row, which has no use for it),
// finite and above zero: a logit at the maximum keeps the exponent 0 and a
// masked one -inf at any temperature, subnormal or infinite ones included.
__device__ __forceinline__ float slope(float tau) {
  return tau > 0.f ? fminf(fmaxf(kLog2e / tau, FLT_MIN), FLT_MAX) : 1.f;
}

// 2^((x - m) c), 0 for a masked logit (m may be -inf then).
__device__ __forceinline__ float weight(float x, float c, float m) {
  return x == -CUDART_INF_F ? 0.f : ptx::ex2((x - m) * c);
}

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  r.at = a.m > b.m ? a.at : b.m > a.m ? b.at : min(a.at, b.at);
  r.s = a.s * weight(a.m, c, r.m) + b.s * weight(b.m, c, r.m);
  return r;
}

__device__ __forceinline__ Stat merge_lanes(Stat st, float c) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    Stat t;
    t.m = __shfl_xor_sync(0xffffffffu, st.m, d);
    t.s = __shfl_xor_sync(0xffffffffu, st.s, d);
    t.at = __shfl_xor_sync(0xffffffffu, st.at, d);
    st = merge(st, t, c);
  }
  return st;
}

__device__ __forceinline__ float tau_of(const AiVerifyArgs& a, int b) {
  return a.temperature ? __ldg(a.temperature + b) : 1.f;
}

__device__ __forceinline__ int drafted(const AiVerifyArgs& a, int b) {
  const int n = a.draft_lens ? __ldg(a.draft_lens + b) : a.n_draft;
  if (n < 0 || n > a.n_draft) report(a.status, AI_ERR_DEV_BOUNDS);  // (taken as the nearest in range)
  return max(0, min(n, a.n_draft));
}

// Row r of sequence b: the target rows, then the draft rows.
template <typename T>
__device__ __forceinline__ const T* row_ptr(const AiVerifyArgs& a, int64_t b, int r) {
  if (r <= a.n_draft) return static_cast<const T*>(a.target) + b * a.target_stride_b + r * a.target_stride_t;
  return static_cast<const T*>(a.draft) + b * a.draft_stride_b + (r - a.n_draft - 1) * a.draft_stride_t;
}

__device__ __forceinline__ int n_rows(const AiVerifyArgs& a) { return a.n_draft + 1 + (a.draft ? a.n_draft : 0); }

// Whether row r is needed: target rows up to the last drafted token's
// successor, draft rows of drafted tokens.
__device__ __forceinline__ bool needed(const AiVerifyArgs& a, int r, int n) {
  return r <= a.n_draft ? r <= n : r - a.n_draft - 1 < n;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) stats_kernel(const AiVerifyArgs a, const Ws w) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int E = 16 / sizeof(T), U = 4;
  const int split = blockIdx.x, rows = n_rows(a), r = blockIdx.y % rows, b = blockIdx.y / rows;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if (r == 0 && split == 0 && tid == 0) {
    w.key[b] = 0;
    w.arrived[b] = 0;
  }
  if (!needed(a, r, drafted(a, b))) return;
  const float tau = tau_of(a, b), c = slope(tau);
  const bool greedy = !(tau > 0.f);
  const T* x = row_ptr<T>(a, b, r);
  // Whole 16-byte vectors of the row, and what is left at its ends.
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(a.vocab, (E - mis) % E), vecs = (a.vocab - head) / E, tail = head + vecs * E;
  const int per = ((vecs + w.splits - 1) / w.splits + kThreads - 1) / kThreads * kThreads;
  const int i0 = min(vecs, split * per), i1 = min(vecs, i0 + per);
  Stat st{-CUDART_INF_F, 0.f, 0x7fffffff};
  auto one = [&](int v) {
    const float f = at(x, v);
    st = merge(st, Stat{f, f == -CUDART_INF_F ? 0.f : 1.f, v}, c);
  };
  if (split == 0 && tid < head) one(tid);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  // (the next round's loads are in flight while this one's are summed; a
  // vector past the slice is all -inf, which adds nothing)
  const uint4 none = make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
  uint4 next[U];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = i + u * kThreads < i1 ? __ldg(xv + i + u * kThreads) : none;
  };
  load(i0 + tid);
  for (int i = i0 + tid; i < i1; i += kThreads * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    load(i + kThreads * U);
    uint32_t big = Vec<T>::larger(Vec<T>::larger(raw[0].x, raw[0].y), Vec<T>::larger(raw[0].z, raw[0].w));
    if constexpr (sizeof(T) == 4) {
      float m = Vec<T>::top(big);
#pragma unroll
      for (int u = 1; u < U; ++u) {
        m = ptx::fmax3(m, __uint_as_float(raw[u].x), __uint_as_float(raw[u].y));
        m = ptx::fmax3(m, __uint_as_float(raw[u].z), __uint_as_float(raw[u].w));
      }
      big = __float_as_uint(m);
    } else {
#pragma unroll
      for (int u = 1; u < U; ++u)
        big = Vec<T>::larger(big, Vec<T>::larger(Vec<T>::larger(raw[u].x, raw[u].y), Vec<T>::larger(raw[u].z, raw[u].w)));
    }
    const float m = Vec<T>::top(big);
    if (greedy) {
      if (m > st.m || st.at == 0x7fffffff) {
        st.m = m;
        bool found = false;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          T e[E];
          memcpy(e, &raw[u], 16);
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (!found && !(to_f32(e[k]) < m)) {
              st.at = head + (i + u * kThreads) * E + k;
              found = true;
            }
        }
      }
    } else {
      // (without a finite logit the maximum stays -inf and nothing is added)
      const float top = fmaxf(st.m, m), o = top == -CUDART_INF_F ? 0.f : top;
      const float2 no = make_float2(-o, -o), cc = make_float2(c, c);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float2 f[E / 2];
        Vec<T>::get(raw[u], f);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          const float2 z = __fmul2_rn(__fadd2_rn(f[k], no), cc);
          sum = __fadd2_rn(sum, make_float2(ptx::ex2(z.x), ptx::ex2(z.y)));
        }
      }
      st.s = st.s * weight(st.m, c, top) + (sum.x + sum.y);
      st.m = top;
    }
  }
  if (split == w.splits - 1 && tail + tid < a.vocab) one(tail + tid);  // (fewer than E)
  st = merge_lanes(st, c);
  __shared__ Stat sm[kWarps];
  if (lane == 0) sm[warp] = st;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < kWarps; ++k) st = merge(st, sm[k], c);
    w.stat[(int64_t)blockIdx.y * w.splits + split] = st;
  }
}

// Race key: larger value first, then the lower index.
__device__ __forceinline__ unsigned long long race_key(float value, int v) {
  return ((unsigned long long)__float_as_uint(value) << 32) | (unsigned int)(~v);
}

// A sequence's distributions at the row where it stops.
template <typename T>
struct Race {
  const T* xp;
  const T* xq;      // nullptr: no draft distribution
  const float* e;   // noise
  float mp, ip, mq, iq, c;  // largest logits and reciprocal sums
  int drop;         // word that has no residual (drafted with certainty and refused), or -1

  // (finite mp, mq: a masked logit's weight is 2^-inf = 0)
  __device__ __forceinline__ float p(float x) const { return ptx::ex2((x - mp) * c) * ip; }
  __device__ __forceinline__ float q(float x) const { return ptx::ex2((x - mq) * c) * iq; }
};

// The thread's best of words [v0, v1): its index is the lowest of equal
// values.  Eight words at a time: consecutive ones as 16-byte loads (kVec: v0
// and the rows are on 16-byte boundaries), else a CTA's width apart.
template <typename T, bool kVec>
__device__ __forceinline__ void race(const Race<T>& d, int v0, int v1, float& best, int& at_) {
  constexpr int kStep = kVec ? 1 : kThreads;
  for (int v = v0 + (int)threadIdx.x * (kVec ? 8 : 1); v < v1; v += kThreads * 8) {
    T p[8], q[8];
    float noise[8];
    if (kVec && v + 8 <= v1) {
      constexpr int N = sizeof(T) / 2;  // 16-byte words of eight logits
      uint4 rp[N], rq[N] = {};
#pragma unroll
      for (int i = 0; i < N; ++i) rp[i] = __ldg(reinterpret_cast<const uint4*>(d.xp + v) + i);
      if (d.xq) {
#pragma unroll
        for (int i = 0; i < N; ++i) rq[i] = __ldg(reinterpret_cast<const uint4*>(d.xq + v) + i);
      }
      const float4 n0 = __ldg(reinterpret_cast<const float4*>(d.e + v));
      const float4 n1 = __ldg(reinterpret_cast<const float4*>(d.e + v) + 1);
      memcpy(p, rp, sizeof(p));
      memcpy(q, rq, sizeof(q));
      memcpy(noise, &n0, 16);
      memcpy(noise + 4, &n1, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int x = min(v + k * kStep, v1 - 1);  // (words past the slice repeat its last one)
        p[k] = d.xp[x];
        q[k] = d.xq ? d.xq[x] : p[k];
        noise[k] = __ldg(d.e + x);
      }
    }
    float r8[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) r8[k] = d.p(to_f32(p[k]));
    if (d.xq) {
#pragma unroll
      for (int k = 0; k < 8; ++k) r8[k] -= d.q(to_f32(q[k]));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int x = min(v + k * kStep, v1 - 1);
      float r = r8[k];
      if (x == d.drop) r = 0.f;
      const float value = __fdividef(r, noise[k]);
      if (value > best) best = value, at_ = x;
    }
  }
}

// The CTA's best as a race key (in thread 0).
__device__ __forceinline__ unsigned long long best_of(float best, int at_, unsigned long long* sm) {
  unsigned long long k = race_key(best, at_);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = k;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < kWarps; ++i) k = sm[i] > k ? sm[i] : k;
  return k;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pick_kernel(const AiVerifyArgs a, const Ws w, const int slice,
                                                        const bool vec) {
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int n = drafted(a, b), rows = n_rows(a);
  const float tau = tau_of(a, b), c = slope(tau);
  __shared__ Stat st[2 * kMaxDraft + 1];
  __shared__ int s_refused[kMaxDraft + 1];
  __shared__ unsigned long long s_key[kWarps];
  // What the stats pass has no part in is read while it runs: the drafted
  // tokens with their logits and uniforms (thread i: token i), and the slice's
  // noise on its way to L2.
  const int v0 = blockIdx.x * slice, v1 = min(a.vocab, v0 + slice);
  long long tok = -1;
  float u = 0.f, x_p = 0.f, x_q = 0.f;
  if (tid < n) {
    tok = a.tokens[(int64_t)b * a.n_draft + tid];
    u = __ldg(a.uniforms + (int64_t)b * a.n_draft + tid);
    if (tok < 0 || tok >= a.vocab) {
      report(a.status, AI_ERR_DEV_BOUNDS);
      tok = -1;
    } else {
      x_p = at(row_ptr<T>(a, b, tid), tok);
      if (a.draft) x_q = at(row_ptr<T>(a, b, a.n_draft + 1 + tid), tok);
    }
  }
  if (tau > 0.f)
    for (int v = v0 + 32 * tid; v < v1; v += 32 * kThreads)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.noise + (int64_t)b * a.vocab + v));
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int r = warp; r < rows; r += kWarps) {
    if (!needed(a, r, n)) continue;
    const Stat* p = w.stat + ((int64_t)b * rows + r) * w.splits;
    Stat s{-CUDART_INF_F, 0.f, 0x7fffffff};
    for (int k = lane; k < w.splits; k += 32) s = merge(s, p[k], c);
    s = merge_lanes(s, c);
    if (lane == 0) st[r] = s;
  }
  __syncthreads();
  if (tid < n) {  // (kMaxDraft is below a CTA's threads)
    bool ok = false;
    if (tok >= 0 && !(tau > 0.f)) {
      ok = tok == st[tid].at;
    } else if (tok >= 0) {
      const Stat& sp = st[tid];
      const float p = sp.s > 0.f ? weight(x_p, c, sp.m) / sp.s : 0.f;
      float q = 1.f;
      if (a.draft) {
        const Stat& sq = st[a.n_draft + 1 + tid];
        q = sq.s > 0.f ? weight(x_q, c, sq.m) / sq.s : 0.f;
      }
      ok = u * q < p;
    }
    s_refused[tid] = !ok;
  }
  __syncthreads();
  int stop = 0;
  while (stop < n && !s_refused[stop]) ++stop;

  Race<T> d;
  if (tau > 0.f) {
    const Stat sp = st[stop];
    d.xp = row_ptr<T>(a, b, stop);
    d.xq = stop < n && a.draft ? row_ptr<T>(a, b, a.n_draft + 1 + stop) : nullptr;
    d.e = a.noise + (int64_t)b * a.vocab;
    d.c = c;
    d.mp = sp.m == -CUDART_INF_F ? 0.f : sp.m;
    d.ip = sp.s > 0.f ? 1.f / sp.s : 0.f;
    d.drop = -1;
    if (d.xq) {
      const Stat sq = st[a.n_draft + 1 + stop];
      d.mq = sq.m == -CUDART_INF_F ? 0.f : sq.m;
      d.iq = sq.s > 0.f ? 1.f / sq.s : 0.f;
    } else if (stop < n) {
      const long long refused = a.tokens[(int64_t)b * a.n_draft + stop];
      if (refused >= 0 && refused < a.vocab) d.drop = (int)refused;
    }
    float best = 0.f;
    int best_at = 0;
    if (vec)
      race<T, true>(d, v0, v1, best, best_at);
    else
      race<T, false>(d, v0, v1, best, best_at);
    const unsigned long long k = best_of(best, best_at, s_key);
    if (tid == 0) atomicMax(w.key + b, k);
  }
  // The sequence's last CTA writes its results.
  __shared__ int s_last;
  if (tid == 0) {
    __threadfence();
    s_last = atomicAdd(w.arrived + b, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  __shared__ int s_next;
  if (tau > 0.f) {
    unsigned long long k = *(volatile unsigned long long*)(w.key + b);
    if ((k >> 32) == 0) {
      // Nothing is left of p after the draft's share: race p itself.
      d.xq = nullptr;
      d.drop = -1;
      float best = 0.f;
      int best_at = 0;
      race<T, false>(d, 0, a.vocab, best, best_at);
      __syncthreads();
      k = best_of(best, best_at, s_key);
    }
    if (tid == 0) s_next = (int)~(unsigned int)k;
  } else if (tid == 0) {
    s_next = st[stop].at;
  }
  __syncthreads();
  for (int i = tid; i <= a.n_draft; i += kThreads) {
    const int64_t o = (int64_t)b * (a.n_draft + 1) + i;
    long long word = -1;
    float lp = 0.f;
    if (i <= stop) {
      word = i < stop ? a.tokens[(int64_t)b * a.n_draft + i] : s_next;
      if (tau > 0.f) lp = ((at(row_ptr<T>(a, b, i), word) - st[i].m) * c - log2f(st[i].s)) * kLn2;
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

// Slices of the vocabulary for `rows` rows: enough CTAs for four per SM (what
// the registers of both kernels admit at once; 64 sequences of four drafts: 59 /
// 51 / 54 us with 2 / 4 / 8), but at least `least` logits each.
int slices(const AiVerifyArgs& a, int64_t rows, int least) {
  const int64_t want = (4 * (int64_t)sm_count() + rows - 1) / rows, most = (a.vocab + least - 1) / least;
  return (int)(want < most ? want : most);
}

int64_t row_count(const AiVerifyArgs& a) {
  return (int64_t)a.batch * (a.n_draft + 1 + (a.draft ? a.n_draft : 0));
}

size_t layout(const AiVerifyArgs& a, Ws* w) {
  const int64_t rows = row_count(a);
  w->splits = slices(a, rows, a.dtype == AI_DTYPE_F32 ? kLeastStats / 2 : kLeastStats);
  const size_t stat = ((size_t)rows * w->splits * sizeof(Stat) + 255) & ~size_t(255);
  const size_t key = ((size_t)a.batch * sizeof(unsigned long long) + 255) & ~size_t(255);
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
  if (cudaGetLastError() != cudaSuccess) return AI_ERR_LAUNCH;
  const int n = slices(a, a.batch, kLeastPick), slice = ((a.vocab + n - 1) / n + 7) / 8 * 8;
  // Every row the race reads starts on a 16-byte boundary.
  uintptr_t at = reinterpret_cast<uintptr_t>(a.target) | reinterpret_cast<uintptr_t>(a.noise);
  int64_t step = (a.target_stride_b | a.target_stride_t) * (int64_t)sizeof(T) | a.vocab * (int64_t)sizeof(float);
  if (a.draft) {
    at |= reinterpret_cast<uintptr_t>(a.draft);
    step |= (a.draft_stride_b | a.draft_stride_t) * (int64_t)sizeof(T);
  }
  const bool vec = ((at | (uintptr_t)step) & 15) == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.vocab + slice - 1) / slice, a.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, pick_kernel<T>, a, w, slice, vec) != cudaSuccess) return AI_ERR_LAUNCH;
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
