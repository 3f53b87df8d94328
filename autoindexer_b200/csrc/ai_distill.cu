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
// then need no look at the list; one warp gathers the list's own sums meanwhile), the
// sums exchanged through distributed shared memory.
//
// Measured: 4096 rows of 151,936 bf16, most with lists of 32, losses and gradients, 542 us
// (4.3 TB/s); 16 of 151,936 8.0 us; 1023 of 32,003 fp16 with lists of 64, the losses
// in one launch and the gradients, from the rows' totals, in another, 55 us (70 when
// the second one summed again).  Between
// it and the memory's 365 us stand the instructions (issued in 56% of the cycles; two
// exponentials a logit keep the SFU busy for 58%) and the phases of a slice, which
// the CTAs of an SM overlap as much as their shared memory holds.  Slices of 20
// or 80 KB take 640 and 650 us; rows that pass through an SM as a pipeline (warps that
// sum a row beside others that write the one before) 529, but twice the time where
// there are few rows for an SM.

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

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int U = 2;                   // vectors of a thread in flight
constexpr int kMaxTop = AI_DISTILL_MAX_TOP;
constexpr int kSets = kMaxTop / 32;    // entries of a lane
constexpr int kMaxSplit = 16;
constexpr int kLeast = 16 * 1024;      // bytes of a slice, at least (for more CTAs than the memory asks for)
constexpr int kSlice = 38 * 1024;      // bytes of a slice where there are rows enough: five CTAs per SM
constexpr int kWidth = 32;             // slices are whole vectors of so many lanes
constexpr int kMostSlice = AI_DISTILL_MAX_ROW_BYTES / kMaxSplit + 16 * kWidth;  // bytes
static_assert(kMostSlice <= 200 * 1024, "a slice in shared memory");
static_assert(kMaxTop <= kThreads - 32, "a thread per entry");
constexpr long long kWait = 1000000000LL;
constexpr float kLostSlice = -1.f;     // a warp's sum over a slice whose copy did not come: losses NaN, no gradient
// A remainder of the teacher's probability within kLostSum + kLost sum p |ln p| is
// what the rounding of its fp32 log-probabilities may leave: 2^-24 of each, and of the
// logarithm and the sum that they were taken less.
constexpr float kLost = 0x1p-24f, kLostSum = 0x1p-23f;

// What one warp finds out of a row's list.
struct List {
  int live;            // whether the row has an entry (and a weight)
  float up;            // weight / tau
  float c, inv;        // log2(e) / tau, 1 / tau
  float p_top, p_rest; // the teacher's probability on the listed words, and beside them
  float m, s;          // the student's logits there: the largest, and the sum of 2^((x - m) c)
  float norm;          // what the teacher's log-probabilities are taken less
  float term;          // sum p (ln p - (x - m) / tau)
  int word[kMaxTop];   // -1: left out
  float x[kMaxTop];    // the student's logits
  float p[kMaxTop];    // the teacher's probabilities
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// What a backward of its own needs of a row.
struct __align__(16) RowStats {
  float m, base;       // of the words that are not listed
  float m_all, s_all;  // of all
  float mass, norm;
  float live, unused;
};

// A row of the call.
template <typename T>
struct Row {
  const T* x;
  T* d;  // (no meaning for losses alone)
  uint32_t b;
  __device__ __forceinline__ Row(const AiDistillArgs& a, uint32_t row) {
    b = row / (uint32_t)a.seq_len;
    const int64_t t = row - b * (uint32_t)a.seq_len;
    x = static_cast<const T*>(a.logits) + b * a.stride_b + t * a.stride_t;
    d = static_cast<T*>(a.dlogits) + b * a.dstride_b + t * a.dstride_t;
  }
};

// A lane's entries of a row's list.
struct Entries {
  int word[kSets];
  float logp[kSets], x[kSets];
  float wgt, inv;
};

// A row's list, by one warp: its words, which the others wait for (`known` is called as
// soon as it is known whether the row is live) ...
template <typename T, typename F>
__device__ __forceinline__ void read_words(const AiDistillArgs& a, List& list, Entries& mine, uint32_t row, bool reports, F known) {
  const int lane = threadIdx.x % 32, K = a.n_top;
  const Row<T> r(a, row);
  int32_t* status = reports ? a.status : nullptr;
  const float wgt = a.weights ? __ldg(a.weights + row) : 1.f;
  const float tau = row_tau(a.temperature, r.b, nullptr);
  int(&word)[kSets] = mine.word;
  float(&logp)[kSets] = mine.logp, (&xk)[kSets] = mine.x;
  bool any = false;
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    const int k = 32 * i + lane;
    word[i] = -1;
    logp[i] = xk[i] = -CUDART_INF_F;
    if (32 * i >= K) continue;  // (here and below: sets past the list take no instruction of the warp)
    if (k < K) {
      const long long w = a.top_tokens[(int64_t)row * K + k];
      logp[i] = a.top_logprobs[(int64_t)row * K + k];
      if (wgt != 0.f && w >= a.vocab) report(status, AI_ERR_DEV_BOUNDS);
      if (wgt != 0.f && w >= 0 && w < a.vocab && logp[i] != -CUDART_INF_F) {
        word[i] = (int)w;
        xk[i] = at(r.x, word[i]);
      }
    }
    list.word[k] = word[i];
    any |= word[i] >= 0;
  }
  any = __any_sync(0xffffffffu, any);
  if (lane == 0) list.live = any;
  known(any);
  if (!any) return;
  if (lane == 0) row_tau(a.temperature, r.b, status);
  mine.wgt = wgt;
  mine.inv = inverse(tau);
  if (lane == 0) list.c = slope(tau);
  // A word that an earlier entry has is left out.
  __syncwarp();  // (votes do not order the lanes' words in shared memory)
  bool again[kSets] = {};
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    if (32 * i >= K) continue;
    again[i] = (__match_any_sync(0xffffffffu, word[i]) & ((1u << lane) - 1)) != 0;
    for (int j = 0; j < 32 * i; ++j) again[i] |= list.word[j] == word[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    if (32 * i >= K) continue;
    if (again[i] && word[i] >= 0) {
      report(status, AI_ERR_DEV_BOUNDS);
      word[i] = list.word[32 * i + lane] = -1;
      xk[i] = -CUDART_INF_F;
    }
  }
  __syncwarp();  // (list.c)
}

// ... and the sums over them, while the others go through the slice.
__device__ __forceinline__ void weigh(const AiDistillArgs& a, List& list, Entries& mine) {
  const int lane = threadIdx.x % 32, K = a.n_top;
  const int(&word)[kSets] = mine.word;
  float(&logp)[kSets] = mine.logp, (&xk)[kSets] = mine.x;
  const float c = list.c, inv = mine.inv;
  float p[kSets], top = -CUDART_INF_F, m = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    p[i] = 0.f;
    if (32 * i >= K) continue;
    if (word[i] >= 0) top = fmaxf(top, logp[i]);
    m = fmaxf(m, xk[i]);
  }
  const bool renorm = a.tail == AI_TAIL_RENORMALIZE;
  float norm = 0.f;
  if (renorm) {
    top = warp_max(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kSets; ++i)
      if (32 * i < K) sum += word[i] >= 0 ? expf(logp[i] - top) : 0.f;
    norm = top + logf(warp_sum(sum));
#pragma unroll
    for (int i = 0; i < kSets; ++i) logp[i] -= norm;
  }
  m = warp_max(m);
  const float o = m == -CUDART_INF_F ? 0.f : m;
  float p_top = 0.f, sum = 0.f, term = 0.f;
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    if (32 * i >= K) continue;
    if (word[i] >= 0) p[i] = expf(logp[i]);
    p_top += p[i];
    sum += weight(xk[i], c, o);
    if (p[i] != 0.f) term += p[i] * logp[i] - scaled(xk[i] - o, p[i] * inv);  // (p / tau first: logits may be as far apart as fp32 goes)
    list.x[32 * i + lane] = xk[i];
    list.p[32 * i + lane] = p[i];
  }
  p_top = warp_sum(p_top);
  sum = warp_sum(sum);
  term = warp_sum(term);
  // The remainder in 64 bits: a sure teacher's, 1e-5 say, is a small difference.
  float rest = 0.f;
  if (!renorm) {
    double all = 0.;
    float lost = 0.f;
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      if (32 * i >= K || word[i] < 0) continue;
      all += exp((double)logp[i]);
      lost += p[i] * fabsf(logp[i]);
    }
    all = 1. - warp_sum(all);
    lost = fmaf(kLost, warp_sum(lost), kLostSum);
    rest = (float)all;
    if (rest <= lost) rest = 0.f;  // (NaN stays)
  }
  if (lane == 0) {
    list.up = over_tau(mine.wgt, inv);
    list.inv = inv;
    list.p_top = p_top;
    list.p_rest = rest;
    list.m = m;
    list.s = sum;
    list.norm = norm;
    list.term = term;
  }
}

// Gradient of a listed word with the student's share q and the teacher's p.
__device__ __forceinline__ float listed_gradient(float up, float mass, float q, float p) { return up * (mass * q - p); }

// A warp's sum of the parts (m, s) of its lanes, with respect to their largest m.
__device__ __forceinline__ float2 join_lanes(float2 q, float c) {
  const float m = warp_max(q.x);
  return make_float2(m, warp_sum(q.x == -CUDART_INF_F ? q.y : q.y * ptx::ex2((q.x - m) * c)));
}

// The row's ragged ends (elements before the first vector and behind the last one):
// f(element) for those of a slice, one per thread.
template <int E, typename F>
__device__ __forceinline__ void ends(const Slice& sl, int vocab, int tid, F f) {
  if (tid >= E) return;
  if (sl.e0 + tid < sl.head) f(tid);
  if (sl.e1 > sl.tail && sl.tail + tid < vocab) f(sl.tail + tid);
}

// An element of the ragged ends joins a thread's sum.
__device__ __forceinline__ void add_end(Part& part, float f, float c) {
  part = merge(part, Part{f, f == -CUDART_INF_F ? 0.f : f - f + 1.f, 0.f}, c);  // (NaN for +inf and NaN)
}

// All words of a row: the listed ones beside the others (m, s).
struct Totals {
  float m, s;          // of the others
  float m_all, s_all;  // of all
  float p_rest, mass;
  bool empty;
  __device__ __forceinline__ Totals(const List& list, float2 rest) {
    m = rest.x, s = rest.y;
    m_all = fmaxf(list.m, m);
    const float of_top = list.m == -CUDART_INF_F ? 0.f : ptx::ex2((list.m - m_all) * list.c);
    s_all = list.s * of_top + (m == -CUDART_INF_F ? s : s * of_rest(list));
    p_rest = s == 0.f ? 0.f : list.p_rest;  // (no word for the bucket)
    mass = list.p_top + p_rest;
    empty = s_all == 0.f;
  }
  __device__ __forceinline__ float of_rest(const List& list) const {
    return m == -CUDART_INF_F ? 0.f : ptx::ex2((m - m_all) * list.c);
  }
  // sum p (ln p - ln q), the list's part having been taken from its own largest logit.
  __device__ __forceinline__ float loss(const List& list) const {
    const float o = list.m == -CUDART_INF_F ? 0.f : list.m, l2 = log2f(s_all);
    float r = list.term;
    if (list.p_top != 0.f) r += scaled(m_all - o, list.p_top * list.inv) + list.p_top * (l2 * kLn2);
    if (p_rest != 0.f) r += p_rest * (logf(p_rest) - (log2f(s) - l2) * kLn2) - scaled(m - m_all, p_rest * list.inv);
    return empty ? CUDART_INF_F : r;
  }
  // What the gradients of the others have in common, but for the weight.
  __device__ __forceinline__ float base(const List& list) const { return s == 0.f ? 0.f : mass * of_rest(list) / s_all - p_rest / s; }
  // Gradient of listed entry k.
  __device__ __forceinline__ float listed(const List& list, int k) const {
    return empty ? 0.f : listed_gradient(list.up, mass, weight(list.x[k], list.c, m_all) / s_all, list.p[k]);
  }
};

// Gradients of the words that are not listed: 2^((x - m) c) coef.  (Those of the
// listed ones come out as anything and are written over.)
struct Dense {
  float m, c, coef;
  __device__ __forceinline__ Dense(float largest, float slope, float up, float base) {
    m = largest == -CUDART_INF_F ? 0.f : largest;
    c = slope;
    coef = base == 0.f ? 0.f : up * base;
  }
  __device__ __forceinline__ float one(float x) const { return ptx::ex2((x - m) * c) * coef; }
  template <typename T>
  __device__ __forceinline__ uint4 vector(const uint4& raw) const {
    constexpr int E = 16 / sizeof(T);
    const float2 nm = make_float2(-m, -m), cc = make_float2(c, c), cf = make_float2(coef, coef);
    float2 f[E / 2];
    Vec<T>::get(raw, f);
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      const float2 y = __fmul2_rn(__fadd2_rn(f[q], nm), cc);
      f[q] = __fmul2_rn(make_float2(ptx::ex2(y.x), ptx::ex2(y.y)), cf);
    }
    return Vec<T>::put(f);
  }
};

// Vector `out` to elements [v, v + E) of a row of the gradient; `wide`: on a 16-byte
// boundary.
template <typename T>
__device__ __forceinline__ void put(T* d, int v, const uint4& out, bool wide) {
  constexpr int E = 16 / sizeof(T);
  if (wide) {
    __stcs(reinterpret_cast<uint4*>(d + v), out);
  } else {
    T e[E];
    memcpy(e, &out, 16);
#pragma unroll
    for (int q = 0; q < E; ++q) d[v + q] = e[q];
  }
}

template <typename T>
__device__ __forceinline__ bool lie_alike(const T* x, const T* d) {
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

template <typename T>
__device__ __forceinline__ void zero_row(T* d, int vocab, int split, int splits, int unit, int tid, int threads) {
  constexpr int E = 16 / sizeof(T);
  const Slice z = slice_of(d, vocab, split, splits, unit);
  for (int i = z.i0 + tid; i < z.i1; i += threads) put(d, z.head + i * E, make_uint4(0u, 0u, 0u, 0u), true);
  ends<E>(z, vocab, tid, [&](int v) { d[v] = from_f32<T>(0.f); });
}

__device__ __forceinline__ void finish(const AiDistillArgs& a, uint32_t row, const List& list, const Totals& all) {
  if (a.losses) a.losses[row] = all.loss(list);
  if (a.row_stats)
    *reinterpret_cast<RowStats*>(a.row_stats + 8 * (int64_t)row) =
        RowStats{all.m, all.base(list), all.m_all, all.s_all, all.mass, list.norm, 1.f, 0.f};
}
__device__ __forceinline__ void finish_dead(const AiDistillArgs& a, uint32_t row) {
  if (a.losses) a.losses[row] = 0.f;
  if (a.row_stats) *reinterpret_cast<RowStats*>(a.row_stats + 8 * (int64_t)row) = RowStats{};
}

// Losses alone, of rows enough and long ones: nothing has to stay, so a slice is streamed
// through the registers, by as many CTAs a row as there are rows too few for; the first
// of them joins the sums.  4096 rows of 151,936 bf16 252 us (4.4 TB/s), where slices held
// in shared memory take 371; 1023 rows of 65,536 words 50 (49), of 32,003 45 (33: more
// CTAs to hide the lists behind), 16 of 151,936 6.9 (6.2).
// Listed words are looked for where a bit says that a warp's vectors of a round hold
// one, and hidden there.
constexpr int kStreamed = 128 * 1024;  // bytes of a row from which losses alone are streamed
constexpr int kSum = kThreads - 32;  // threads that sum (the first warp reads and weighs the list)
constexpr int kAtOnce = 4;           // vectors of a thread in flight
constexpr int kRound = kSum * kAtOnce;
constexpr int kMaxRounds = AI_DISTILL_MAX_ROW_BYTES / 16 / kRound + 1;

// Sets element q of vector v, counted from the warp's first one of a round, to -inf.
template <typename T>
__device__ __forceinline__ void hide(uint4 (&raw)[kAtOnce], int v, int q) {
  constexpr int P = 4 / sizeof(T);  // elements of a word
  const uint32_t keep = P == 1 ? 0u : q % P ? 0xffffu : 0xffff0000u;
#pragma unroll
  for (int u = 0; u < kAtOnce; ++u) {
    if (v - u * kSum != (int)(threadIdx.x % 32)) continue;
    uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
    for (int h = 0; h < 4; ++h)
      if (q / P == h) w[h] = (w[h] & keep) | (Vec<T>::kNone & ~keep);
    raw[u] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) losses_kernel(const AiDistillArgs a, const int splits) {
  constexpr int E = 16 / sizeof(T);
  __shared__ List list;
  __shared__ float2 s_parts[kMaxSplit * kWarps];  // (m, s) of each warp of the cluster, in its first CTA
  __shared__ uint32_t s_flags[kMaxRounds];        // per round: bit kAtOnce warp + u
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, K = a.n_top, id = tid - 32;
  const uint32_t row = blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const Row<T> r(a, row);
  const Slice sl = slice_of(r.x, a.vocab, split, splits, kWidth);
  const uint4* xv = reinterpret_cast<const uint4*>(r.x + sl.head);
  const uint4 none = make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
  // (a CTA of the cluster must run before its shared memory is written to)
  if (splits > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");
  uint4 next[kAtOnce];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) next[u] = i + u * kSum < sl.i1 ? __ldg(xv + i + u * kSum) : none;
  };
  Entries entries;  // (the first warp's)
  if (warp == 0) {
    for (int i = lane; i < kMaxRounds; i += 32) s_flags[i] = 0;
    read_words<T>(a, list, entries, row, split == 0, [](bool) {});
    __syncwarp();
    if (list.live) {
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        const int w = entries.word[i];
        if (32 * i >= K || w < sl.head || w >= sl.tail) continue;
        const int v = (w - sl.head) / E - sl.i0;
        if (v >= 0 && v < sl.i1 - sl.i0) atomicOr(s_flags + v / kRound, 1u << (kAtOnce * (v % kSum / 32) + v % kRound / kSum));
      }
    }
  } else if (splits > 1) {
    load(sl.i0 + id);  // (few rows: they do not wait for the list)
  }
  __syncthreads();
  if (!list.live) {
    if (split == 0 && tid == 0) finish_dead(a, row);
    return;
  }
  const float c = list.c;
  if (warp == 0) {
    weigh(a, list, entries);
  } else {
    if (splits == 1) load(sl.i0 + id);
    Part part{-CUDART_INF_F, 0.f, 0.f};
    for (int i = sl.i0, round = 0; i < sl.i1; i += kRound, ++round) {
      uint4 raw[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) raw[u] = next[u];
      load(i + kRound + id);
      if (s_flags[round] >> (kAtOnce * (warp - 1)) & ((1u << kAtOnce) - 1)) {
        const int v0 = sl.head + (i + id - lane) * E;
        for (int k0 = 0; k0 < K; k0 += 32) {
          const int el = list.word[k0 + lane] - v0;
          uint32_t in = __ballot_sync(0xffffffffu, el >= 0 && el < kRound * E && el / E % kSum < 32);
          while (in) {
            const int e = __shfl_sync(0xffffffffu, el, __ffs(in) - 1);
            in &= in - 1;
            hide<T>(raw, e / E, e % E);
          }
        }
      }
      accumulate<T, kAtOnce, false>(part, raw, c);
    }
    ends<E>(sl, a.vocab, id, [&](int v) {
      for (int j = 0; j < K; ++j)
        if (list.word[j] == v) return;
      add_end(part, at(r.x, v), c);
    });
    const float2 mine = join_lanes(make_float2(part.m, part.s), c);
    if (splits > 1) {
      asm volatile("barrier.cluster.wait;" ::: "memory");
      if (lane == 0) cg::this_cluster().map_shared_rank(s_parts, 0)[split * kWarps + warp] = mine;
    } else if (lane == 0) {
      s_parts[warp] = mine;
    }
  }
  if (splits > 1) {
    if (warp == 0) asm volatile("barrier.cluster.wait;" ::: "memory");
    cg::this_cluster().sync();
  } else {
    __syncthreads();
  }
  if (split > 0 || warp > 0) return;
  float2 rest = make_float2(-CUDART_INF_F, 0.f);
  for (int i = lane; i < splits * kWarps; i += 32) {
    if (i % kWarps == 0) continue;
    const Part q = merge(Part{rest.x, rest.y, 0.f}, Part{s_parts[i].x, s_parts[i].y, 0.f}, c);
    rest = make_float2(q.m, q.s);
  }
  const Totals all(list, join_lanes(rest, c));
  if (lane == 0) finish(a, row, list, all);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 6) distill_kernel(const AiDistillArgs a, const int splits) {
  constexpr int E = 16 / sizeof(T);
  __shared__ List list;
  __shared__ float2 s_parts[kMaxSplit * kWarps];  // (m, s) of each warp of the cluster
  __shared__ __align__(8) uint64_t s_bar;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, K = a.n_top;
  const uint32_t row = blockIdx.x / (uint32_t)splits, bar = ptx::smem_u32(&s_bar);
  const int split = (int)(blockIdx.x - row * splits);
  const Row<T> r(a, row);
  const Slice sl = slice_of(r.x, a.vocab, split, splits, kWidth);
  const int vecs = sl.i1 - sl.i0;
  // (a CTA of the cluster must run before its shared memory is written to)
  if (splits > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");
  Entries entries;  // (the first warp's)
  if (warp == 0) {
    if (lane == 0) {
      ptx::mbar_init(bar, 1);
      ptx::fence_mbar_init();
    }
    read_words<T>(a, list, entries, row, split == 0, [&](bool live) {
      if (lane == 0 && live && vecs > 0) {
        ptx::mbar_arrive_expect_tx(bar, 16u * vecs);
        ptx::bulk_load(ptx::smem_u32(smem), r.x + sl.head + (int64_t)sl.i0 * E, 16u * vecs, bar);
      }
    });
  }
  __syncthreads();
  if (!list.live) {
    if (split == 0 && tid == 0) finish_dead(a, row);
    if (a.dlogits) zero_row(r.d, a.vocab, split, splits, kWidth, tid, kThreads);
    return;
  }
  const uint4* held = reinterpret_cast<const uint4*>(smem);
  const float c = list.c;
  float2 mine = make_float2(-CUDART_INF_F, 0.f);
  if (warp == 0) {
    weigh(a, list, entries);
  } else {
    bool lost = false;  // the slice never came
    if (vecs > 0 && !ptx::mbar_wait(bar, 0, kWait)) {
      report(a.status, AI_ERR_DEV_TIMEOUT);
      lost = !ptx::mbar_wait(bar, 0, kWait);  // (once more: the copy should land before the CTA ends)
    }
    // The listed words' places become -inf, which adds nothing to the others' sum.
    const int id = tid - 32;
    if (id < K) {
      const int w = list.word[id], at_ = w - sl.head - sl.i0 * E;
      if (w >= 0 && at_ >= 0 && at_ < vecs * E) reinterpret_cast<T*>(smem)[at_] = from_f32<T>(-CUDART_INF_F);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kSum) : "memory");
    const uint4 none = make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
    Part part{-CUDART_INF_F, 0.f, 0.f};
    for (int i = id; i < vecs; i += kSum * U) {
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = i + u * kSum < vecs ? held[i + u * kSum] : none;
      accumulate<T, U, false>(part, raw, c);
    }
    ends<E>(sl, a.vocab, id, [&](int v) {
      for (int j = 0; j < K; ++j)
        if (list.word[j] == v) return;
      add_end(part, at(r.x, v), c);
    });
    mine = join_lanes(make_float2(part.m, part.s), c);
    if (__any_sync(0xffffffffu, lost)) mine.y = kLostSlice;
  }
  // The warps' sums go to every CTA of the cluster; each joins them in the same order.
  if (splits > 1) {
    const cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (lane < splits) cluster.map_shared_rank(s_parts, lane)[split * kWarps + warp] = mine;
    cluster.sync();
  } else {
    if (lane == 0) s_parts[warp] = mine;
    __syncthreads();
  }
  float2 rest = make_float2(-CUDART_INF_F, 0.f);
  bool whole = true;
  for (int i = lane; i < splits * kWarps; i += 32) {
    whole &= s_parts[i].y != kLostSlice;
    const Part q = merge(Part{rest.x, rest.y, 0.f}, Part{s_parts[i].x, s_parts[i].y, 0.f}, c);
    rest = make_float2(q.m, q.s);
  }
  rest = join_lanes(rest, c);
  if (!__all_sync(0xffffffffu, whole)) {
    // (no gradient: it may lie over the logits)
    if (split == 0 && tid == 0) finish(a, row, list, Totals(list, make_float2(0.f, CUDART_NAN_F)));
    return;
  }
  const Totals all(list, rest);
  if (split == 0 && tid == 0) finish(a, row, list, all);
  if (!a.dlogits) return;
  const Dense dense(all.m, c, list.up, all.base(list));
  const bool alike = lie_alike(r.x, r.d);
#pragma unroll 2
  for (int i = tid; i < vecs; i += kThreads) put(r.d, sl.head + (sl.i0 + i) * E, dense.template vector<T>(held[i]), alike);
  ends<E>(sl, a.vocab, tid, [&](int v) { r.d[v] = from_f32<T>(dense.one(at(r.x, v))); });
  __syncthreads();
  if (tid < K) {
    const int w = list.word[tid];
    if (w >= sl.e0 && w < sl.e1) r.d[w] = from_f32<T>(all.listed(list, tid));
  }
}

// The gradient alone, from the rows' totals: a CTA per (row, slice).  One read and one
// write of the row, bound by them.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) distill_bwd_kernel(const AiDistillBwdArgs g, const int splits) {
  constexpr int E = 16 / sizeof(T), N = 4;  // vectors of a thread in flight
  const AiDistillArgs& a = g.fwd;
  __shared__ int s_word[kMaxTop];
  const int tid = threadIdx.x, K = a.n_top;
  const uint32_t row = blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const Row<T> r(a, row);
  const int64_t t = row - r.b * (uint32_t)a.seq_len;
  T* d = static_cast<T*>(g.dlogits) + r.b * g.dstride_b + t * g.dstride_t;
  const float wgt = __ldg(g.g_losses + row);
  const RowStats st = *reinterpret_cast<const RowStats*>(a.row_stats + 8 * (int64_t)row);
  const float tau = row_tau(a.temperature, r.b, nullptr);
  if (wgt == 0.f || st.live == 0.f) {
    zero_row(d, a.vocab, split, splits, kThreads, tid, kThreads);
    return;
  }
  const Slice sl = slice_of(r.x, a.vocab, split, splits, kThreads);
  const uint4* xv = reinterpret_cast<const uint4*>(r.x + sl.head);
  uint4 next[N];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (i + u * kThreads < sl.i1) next[u] = __ldcs(xv + i + u * kThreads);
  };
  load(sl.i0 + tid);
  // The thread's entry of the list: of its words in the slice the first.
  int word = -1;
  float p = 0.f, x = 0.f;
  if (tid < K) {
    const long long w = a.top_tokens[(int64_t)row * K + tid];
    const float logp = a.top_logprobs[(int64_t)row * K + tid];
    if (w >= sl.e0 && w < sl.e1 && logp != -CUDART_INF_F) {
      word = (int)w;
      x = at(r.x, word);
      p = expf(logp - st.norm);
    }
    s_word[tid] = word;
  }
  const float c = slope(tau), up = over_tau(wgt, inverse(tau));
  const Dense dense(st.m, c, up, st.base);
  const bool alike = lie_alike(r.x, d);
  for (int i = sl.i0 + tid; i < sl.i1; i += kThreads * N) {
    uint4 raw[N];
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u] = next[u];
    load(i + kThreads * N);
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (i + u * kThreads < sl.i1) put(d, sl.head + (i + u * kThreads) * E, dense.template vector<T>(raw[u]), alike);
  }
  ends<E>(sl, a.vocab, tid, [&](int v) { d[v] = from_f32<T>(dense.one(at(r.x, v))); });
  __syncthreads();
  if (word >= 0) {
    for (int j = 0; j < tid; ++j)
      if (s_word[j] == word) return;
    d[word] = from_f32<T>(st.s_all == 0.f ? 0.f : listed_gradient(up, st.mass, weight(x, c, st.m_all) / st.s_all, p));
  }
}

int check(const AiDistillArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->vocab <= 0 || a->vocab > 0x40000000 || a->n_top <= 0 || a->n_top > kMaxTop)
    return AI_ERR_SHAPE;
  if ((int64_t)a->batch * a->seq_len > 0x7fffffff / kMaxSplit) return AI_ERR_SHAPE;
  if (a->tail != AI_TAIL_BUCKET && a->tail != AI_TAIL_RENORMALIZE) return AI_ERR_SHAPE;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  if (!a->logits || !a->top_tokens || !a->top_logprobs) return AI_ERR_NULL;
  if (a->stride_b < 0 || a->stride_t < 0 || a->dstride_b < 0 || a->dstride_t < 0) return AI_ERR_STRIDE;
  if ((int64_t)a->vocab * (a->dtype == AI_DTYPE_F32 ? 4 : 2) > AI_DISTILL_MAX_ROW_BYTES) return AI_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->dlogits)) &
      (a->dtype == AI_DTYPE_F32 ? 3 : 1))
    return AI_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(a->row_stats) & 15) return AI_ERR_ALIGN;
  return AI_OK;
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

// CTAs of a row where they are streamed: for four per SM, at least kLeast bytes each.
int stream_slices(const AiDistillArgs& a) {
  const int64_t rows = (int64_t)a.batch * a.seq_len, bytes = (int64_t)a.vocab * (a.dtype == AI_DTYPE_F32 ? 4 : 2);
  int s = 1;
  while (2 * s <= kMaxSplit && 2 * s * rows <= 4 * (int64_t)sm_count() && s * (int64_t)kLeast < bytes) s *= 2;
  return s;
}

// `kernel` on clusters of `splits` CTAs, one per row.
int launch_rows(void (*kernel)(AiDistillArgs, int), const AiDistillArgs& a, int splits, int64_t smem, cudaStream_t st) {
  if (splits > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return AI_ERR_LAUNCH;
  // (the limit is the kernel's, not the call's: always the same, so that calls of other
  // threads never find it lower than they need)
  if (smem > 0 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSlice) != cudaSuccess)
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
  if (cudaLaunchKernelEx(&cfg, kernel, a, splits) != cudaSuccess) return AI_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int launch(const AiDistillArgs& a, cudaStream_t st) {
  ProfScope ps(AI_PROF_DISTILL, st);
  if (!a.dlogits && (int64_t)a.batch * a.seq_len >= sm_count() && (int64_t)a.vocab * (int64_t)sizeof(T) >= kStreamed)
    return launch_rows(losses_kernel<T>, a, stream_slices(a), 0, st);
  const int splits = slices(a);
  return launch_rows(distill_kernel<T>, a, splits, slice_bytes(a, splits), st);
}

template <typename T>
int launch_bwd(const AiDistillBwdArgs& g, cudaStream_t st) {
  const int64_t rows = (int64_t)g.fwd.batch * g.fwd.seq_len;
  const int splits = stream_slices(g.fwd);
  ProfScope ps(AI_PROF_DISTILL, st);
  distill_bwd_kernel<T><<<(unsigned)(rows * splits), kThreads, 0, st>>>(g, splits);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace distill
}  // namespace ai

extern "C" int ai_distill(const AiDistillArgs* args, void* stream) {
  const int rc = ai::distill::check(args);
  if (rc != AI_OK) return rc;
  if (!args->losses && !args->dlogits) return AI_ERR_NULL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::distill::launch<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::distill::launch<__half>(*args, st);
  return ai::distill::launch<float>(*args, st);
}

extern "C" int ai_distill_bwd(const AiDistillBwdArgs* args, void* stream) {
  if (!args) return AI_ERR_NULL;
  const AiDistillArgs& a = args->fwd;
  const int rc = ai::distill::check(&a);
  if (rc != AI_OK) return rc;
  if (!args->dlogits || !args->g_losses || !a.row_stats) return AI_ERR_NULL;
  if (args->dstride_b < 0 || args->dstride_t < 0) return AI_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(args->dlogits) & (a.dtype == AI_DTYPE_F32 ? 3 : 1)) return AI_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == AI_DTYPE_BF16) return ai::distill::launch_bwd<__nv_bfloat16>(*args, st);
  if (a.dtype == AI_DTYPE_F16) return ai::distill::launch_bwd<__half>(*args, st);
  return ai::distill::launch_bwd<float>(*args, st);
}
