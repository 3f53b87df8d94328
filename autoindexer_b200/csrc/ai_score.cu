// Log-probabilities of given tokens with the row's entropy and its likeliest
// words, and their gradient (declared in include/ai_attn.h).
//
// With m the row's largest logit, y = (x - m) c, c = log2(e) / tau, e = 2^y,
// s = sum e, t = sum e y:
//   logprob = (x_token - m) / tau - ln 2 log2 s,  entropy = ln 2 (log2 s - t / s),
//   dx_v = p_v (A + B log2 p_v) + (upstream of the entries that name v) / tau,
//   p_v = 2^(y - log2 s), A = -(g_l + sum_k g_k + g_h entropy) / tau, B = -g_h ln 2 / tau.
//
// HBM-bound: the forward reads a row once, the backward reads it and writes
// its gradient (upstream gradients depend on the forward's results of all rows,
// so no row can stay on the chip between the two).
//
// A row is cut for a cluster of CTAs (one where there are rows enough), whose
// first CTA joins what the others send it through distributed shared memory: one
// launch, no workspace.  The list of the largest logits needs no second pass over
// the row: k threads' own maxima, the k-th largest of all threads', are k logits,
// so no logit below the smallest of them can be in the list, and the maxima of
// 1 KB pieces, kept on the way, say where the others are (about k pieces).  A part
// whose logits crowd above that bound (ties, sorted rows) is gone through in order
// instead, keeping the best so far.
//
// Measured: 4096 rows of 151,936 bf16 with entropies, 3592 of them with a token,
// forward 188 us (5.8 TB/s), backward 366 us (6.4 TB/s): at the memory's rate.  509
// rows of fp32 with the 32 likeliest 66 us (4.6 TB/s; less than four CTAs per SM, the
// last of which find the memory idle).  8 rows of bf16 5.1 us, with the 20 likeliest
// 12.5 us, with 128 21 us: latency of the list's steps (its bound 1.5 us, the pieces
// above it 2 to 4, the slices' lists into one 3 to 5).

#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstring>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_logits.cuh"
#include "sm100_ptx.cuh"

namespace ai {
namespace score {

using namespace logits;
namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32, U = 4;
constexpr int kMaxTop = AI_SCORE_MAX_TOP, kRoom = 2048;
constexpr int kMaxSplit = 16;  // CTAs of a cluster
constexpr int kLeast = 8192;   // logits of a slice, at least (half for fp32)
constexpr int kWidth = 8;      // slices are whole groups of so many vectors
static_assert(kMaxSplit * kMaxTop <= kRoom && kMaxTop <= kThreads, "the parts' lists fit the buffer");

using Key = unsigned long long;

// Larger logit first, then the lower index; 0 stands for no entry, which is
// below every key.
__device__ __forceinline__ Key key_of(uint32_t order, int v) { return ((Key)order << 32) | (uint32_t)(~v); }
__device__ __forceinline__ int key_index(Key k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Order of float values as whole numbers (-0 equals 0), above `kMasked` for what is
// not masked.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kMasked = 0x007fffffu;  // order(-inf)

constexpr int kPieces = 2048;

struct TopSmem {
  Key room[kRoom];            // candidates
  Key best[kMaxTop];          // the slice's list
  uint32_t pieces[kPieces];   // order of the largest logit of each piece
  int counts[2][kWarps];
  int n;
};

// Pieces of a slice: what a warp reads as two vectors a lane in one round (the
// first or the second two of its four), in so many rounds that they fit.
struct Pieces {
  int rounds;  // of the slice
  int bits;    // a piece is of 2^bits rounds
  __device__ __forceinline__ Pieces(const Slice& sl) {
    rounds = (sl.i1 - sl.i0 + kThreads * U - 1) / (kThreads * U);
    bits = 0;
    while ((((rounds - 1) >> bits) + 1) * 2 * kWarps > kPieces) ++bits;
  }
  __device__ __forceinline__ int count() const { return rounds > 0 ? (((rounds - 1) >> bits) + 1) * 2 * kWarps : 0; }
  __device__ __forceinline__ int at(int round, int warp, int pair) const { return ((round >> bits) * kWarps + warp) * 2 + pair; }
};

// The k largest of room[0 .. n) to best[], sorted, 0 past the last one.
__device__ void select(TopSmem& sm, int n, int k) {
  const int tid = threadIdx.x;
  if (n <= kThreads) {
    for (int j = tid; j < k; j += kThreads)
      if (j >= n) sm.best[j] = 0;
    if (tid < n) {
      const Key mine = sm.room[tid];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += sm.room[j] > mine;
      if (rank < k) sm.best[rank] = mine;
    }
  } else {
    // The k-th largest, bit by bit (keys differ), then the k entries that reach it.
    constexpr int N = kRoom / kThreads;
    Key held[N];
#pragma unroll
    for (int q = 0; q < N; ++q) held[q] = q * kThreads + tid < n ? sm.room[q * kThreads + tid] : 0;
    Key bound = 0;
    for (int bit = 63, turn = 0; bit >= 0; --bit, turn ^= 1) {
      const Key next = bound | (Key)1 << bit;
      int c = 0;
#pragma unroll
      for (int q = 0; q < N; ++q) c += held[q] >= next;
      c = __reduce_add_sync(0xffffffffu, c);
      if (tid % 32 == 0) sm.counts[turn][tid / 32] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) c += sm.counts[turn][w];
      if (c >= k) bound = next;
      if (c == k) break;
    }
    if (tid == 0) sm.n = 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (held[q] >= bound) sm.room[atomicAdd(&sm.n, 1)] = held[q];
    __syncthreads();
    if (tid < k) {
      const Key mine = sm.room[tid];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < k; ++j) rank += sm.room[j] > mine;
      sm.best[rank] = mine;
    }
  }
  __syncthreads();
}

// The slice's k largest logits.  `top`: the thread's largest one among its
// vectors; sm.pieces holds the pieces', n 0.
template <typename T>
__device__ void top_of_slice(TopSmem& sm, const T* x, int vocab, const Slice& sl, const Pieces& pieces, float top, int k) {
  constexpr int E = 16 / sizeof(T);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  // A bound that k threads' maxima reach, from its first bit down.
  const uint32_t mine = order(top);
  uint32_t bound = 0;
  for (int bit = 31; bit >= 8; --bit) {
    const uint32_t next = bound | 1u << bit;
    const int reach = __syncthreads_count(mine >= next);  // (also: the pieces are written)
    if (reach >= k) bound = next;
    if (reach == k) break;
  }
  auto offer = [&](float f, int v) {
    const uint32_t o = order(f);
    if (o >= bound && o > kMasked && f == f) {
      const int n = atomicAdd(&sm.n, 1);
      if (n < kRoom) sm.room[n] = key_of(o, v);
    }
  };
  // (the row's ragged ends are in no thread's maximum)
  if (tid < E) {
    if (sl.e0 + tid < sl.head) offer(at(x, tid), tid);
    if (sl.e1 > sl.tail && sl.tail + tid < vocab) offer(at(x, sl.tail + tid), sl.tail + tid);
  }
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  const int count = pieces.count();
  for (int p0 = warp; p0 < count; p0 += kThreads) {  // (a warp's pieces are the CTA's warps apart)
    const uint32_t o = p0 + kWarps * lane < count ? sm.pieces[p0 + kWarps * lane] : 0u;
    uint32_t hot = __ballot_sync(0xffffffffu, o >= bound && o > kMasked);
    while (hot) {
      const int p = p0 + kWarps * (__ffs(hot) - 1);
      hot &= hot - 1;
      const int r0 = p / (2 * kWarps) << pieces.bits, of = p / 2 % kWarps, r1 = min(pieces.rounds, r0 + (1 << pieces.bits));
      for (int r = r0; r < r1; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = sl.i0 + (r * U + 2 * (p % 2) + u) * kThreads + 32 * of + lane;
          if (i >= sl.i1) continue;
          const uint4 raw = __ldg(xv + i);
          T e[E];
          memcpy(e, &raw, 16);
#pragma unroll
          for (int q = 0; q < E; ++q) offer(to_f32(e[q]), sl.head + i * E + q);
        }
    }
  }
  __syncthreads();
  const int n = sm.n;
  if (n <= kRoom) {
    select(sm, n, k);
    return;
  }
  // In order, a few logits per thread at a time; what beats the list so far is
  // a candidate for the next one.
  constexpr int kStep = 4 * kThreads;
  Key least = 0;
  int held = 0;
  __syncthreads();
  for (int v0 = sl.e0; v0 < sl.e1; v0 += kStep) {
    if (tid == 0) sm.n = held;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int v = v0 + q * kThreads + tid;
      if (v >= sl.e1) continue;
      const float f = at(x, v);
      const Key key = key_of(order(f), v);
      if (f > -CUDART_INF_F && key > least) sm.room[atomicAdd(&sm.n, 1)] = key;  // (at most kRoom: held is half of it)
    }
    __syncthreads();
    held = sm.n;
    if (held > kRoom - kStep || v0 + kStep >= sl.e1) {
      select(sm, held, k);
      held = min(held, k);
      if (tid < held) sm.room[tid] = sm.best[tid];
      if (held == k) least = sm.best[k - 1];
      __syncthreads();
    }
  }
}

template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kThreads, 4) score_kernel(const AiScoreArgs a, const int splits) {
  constexpr int E = 16 / sizeof(T);
  __shared__ Part s_part[kWarps];
  __shared__ Part s_slices[kMaxSplit];  // of the cluster, in its first CTA
  __shared__ float s_row[2];
  extern __shared__ __align__(16) uint8_t smem[];
  TopSmem& top = *reinterpret_cast<TopSmem*>(smem);
  Key* lists = reinterpret_cast<Key*>(smem + sizeof(TopSmem));  // the cluster's, in its first CTA
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t row = blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const int64_t b = row / a.seq_len, t = row - b * a.seq_len;
  const int k = kTop ? a.top_k : 0;
  const long long token = a.tokens[row];
  const T* x = static_cast<const T*>(a.logits) + b * a.stride_b + t * a.stride_t;
  const Slice sl = slice_of(x, a.vocab, split, splits, kWidth);
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  const uint4 none = make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
  // (the next round's loads are in flight while this one's are summed)
  uint4 next[U];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = i + u * kThreads < sl.i1 ? __ldg(xv + i + u * kThreads) : none;
  };
  if (splits > 1) load(sl.i0 + tid);  // (few rows: they do not wait for the token)
  if (token < 0 || token >= a.vocab) {
    if (split > 0) return;
    if (tid == 0) {
      if (token >= a.vocab) report(a.status, AI_ERR_DEV_BOUNDS);
      a.logprobs[row] = 0.f;
      if constexpr (kEntropy) a.entropy[row] = 0.f;
    }
    if (tid < k) {
      a.top_logprobs[row * k + tid] = -CUDART_INF_F;
      a.top_tokens[row * k + tid] = -1;
    }
    return;
  }
  // (a CTA of the cluster must run before its shared memory is written to)
  if (splits > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");
  const float tau = row_tau(a.temperature, b, split == 0 && tid == 0 ? a.status : nullptr);
  const float c = slope(tau), inv = inverse(tau);
  const float given = split == 0 && tid == 0 ? at(x, token) : 0.f;
  Part p{-CUDART_INF_F, 0.f, 0.f};
  if (splits == 1) load(sl.i0 + tid);
  const Pieces pieces(sl);
  if (kTop && tid == 0) top.n = 0;
  // (whole rounds of the CTA, for the pieces' sake)
  for (int i0 = sl.i0, r = 0; i0 < sl.i1; i0 += kThreads * U, ++r) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    load(i0 + tid + kThreads * U);
    if constexpr (kTop) {
      const float a0 = largest<T, U>(raw, 0, 2), a1 = largest<T, U>(raw, 2, 4);
      const uint32_t o0 = __reduce_max_sync(0xffffffffu, order(a0)), o1 = __reduce_max_sync(0xffffffffu, order(a1));
      if (lane < 2) {
        uint32_t& to = top.pieces[pieces.at(r, warp, lane)];
        const uint32_t o = lane ? o1 : o0;
        to = (r & ((1 << pieces.bits) - 1)) == 0 || o > to ? o : to;
      }
      accumulate<T, U, kEntropy>(p, raw, c, fmaxf(a0, a1));
    } else {
      accumulate<T, U, kEntropy>(p, raw, c);
    }
  }
  const float mine = p.m;
  if (tid < E) {
    auto one = [&](int v) {
      const float f = at(x, v);
      p = merge(p, Part{f, f == -CUDART_INF_F ? 0.f : f - f + 1.f, 0.f}, c);  // (NaN for +inf and NaN)
    };
    if (sl.e0 + tid < sl.head) one(tid);
    if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) one(sl.tail + tid);
  }
  p = merge_lanes(p, c);
  if (lane == 0) s_part[warp] = p;
  if constexpr (kTop) {
    top_of_slice(top, x, a.vocab, sl, pieces, mine, k);
  } else {
    __syncthreads();
  }
  if (tid == 0)
    for (int w = 1; w < kWarps; ++w) p = merge(p, s_part[w], c);
  if (splits > 1) {
    const cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (tid == 0) cluster.map_shared_rank(s_slices, 0)[split] = p;
    if (tid < k) cluster.map_shared_rank(lists, 0)[split * k + tid] = top.best[tid];
    cluster.sync();
    if (split > 0) return;
    if (tid == 0)
#pragma unroll 4
      for (int r = 1; r < splits; ++r) p = merge(p, s_slices[r], c);
    if constexpr (kTop) {
      // An entry below some slice's k-th one, or below the (k / splits)-th ones of all
      // slices, is in no list of k.
      const int share = (k - 1) / splits;
      Key least = 0, all = ~(Key)0;
#pragma unroll 4
      for (int r = 0; r < splits; ++r) {
        least = max(least, lists[r * k + k - 1]);
        all = min(all, lists[r * k + share]);
      }
      least = max(least, all);
      if (tid == 0) top.n = 0;
      __syncthreads();
      for (int j = tid; j < splits * k; j += kThreads) {
        const Key key = lists[j];
        if (key != 0 && key >= least) top.room[atomicAdd(&top.n, 1)] = key;
      }
      __syncthreads();
      select(top, top.n, k);
    }
  }
  if (tid == 0) {
    const bool empty = p.s == 0.f;
    const float l2 = log2f(p.s), h = empty ? 0.f : (l2 - p.t / p.s) * kLn2;
    a.logprobs[row] = empty ? -CUDART_INF_F : scaled(given - p.m, inv) - l2 * kLn2;
    if constexpr (kEntropy) a.entropy[row] = h;
    if (a.row_stats) reinterpret_cast<float4*>(a.row_stats)[row] = make_float4(p.m, l2, h, empty ? 1.f : 0.f);
    s_row[0] = p.m, s_row[1] = l2;
  }
  if constexpr (kTop) {
    __syncthreads();
    if (tid < k) {
      const float m = s_row[0], l2 = s_row[1];
      const Key key = l2 == l2 ? top.best[tid] : 0;  // (a row with a NaN has no order)
      a.top_logprobs[row * k + tid] = l2 != l2 ? l2 : key ? scaled(key_value(key) - m, inv) - l2 * kLn2 : -CUDART_INF_F;
      a.top_tokens[row * k + tid] = key ? key_index(key) : -1;
    }
  }
}

// A CTA per (row, slice): the dense part of the gradient, then the few words
// that the row's entries name, each whole (an entry may repeat another's word).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) score_bwd_kernel(const AiScoreBwdArgs g, const int splits) {
  constexpr int E = 16 / sizeof(T);
  const AiScoreArgs& a = g.fwd;
  __shared__ float s_up[kMaxTop + 1];
  __shared__ int s_word[kMaxTop + 1];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - row * splits);
  const int64_t b = row / a.seq_len, t = row - b * a.seq_len;
  const int k = g.g_top ? a.top_k : 0;
  const T* x = static_cast<const T*>(a.logits) + b * a.stride_b + t * a.stride_t;
  T* d = static_cast<T*>(g.dlogits) + b * g.dstride_b + t * g.dstride_t;
  const long long token = a.tokens[row];
  bool live = token >= 0 && token < a.vocab;
  if (tid <= k) {
    float up = 0.f;
    long long word = -1;
    if (live) {
      word = tid == 0 ? token : a.top_tokens[row * k + tid - 1];
      up = tid == 0 ? (g.g_logprobs ? g.g_logprobs[row] : 0.f) : g.g_top[row * k + tid - 1];
      if (word < 0 || word >= a.vocab) word = -1, up = 0.f;  // (past the list's end)
    }
    s_up[tid] = up;
    s_word[tid] = (int)word;
  }
  const float gh = live && g.g_entropy ? g.g_entropy[row] : 0.f;
  float4 st = make_float4(0.f, 0.f, 0.f, 1.f);
  if (live) st = __ldg(reinterpret_cast<const float4*>(a.row_stats) + row);
  __syncthreads();
  float up = 0.f;
  bool any = gh != 0.f;
  for (int j = 0; j <= k; ++j) {
    up += s_up[j];
    any |= s_up[j] != 0.f;
  }
  live = live && any && st.w == 0.f;
  const float m = st.x, l2 = st.y;
  // The row and its gradient may lie differently on 16-byte boundaries.
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const Slice sl = slice_of(live && !alike ? x : d, a.vocab, split, splits, kThreads);
  uint4* dv = reinterpret_cast<uint4*>(d + sl.head);
  if (!live) {
    for (int i = sl.i0 + tid; i < sl.i1; i += kThreads) __stcs(dv + i, make_uint4(0u, 0u, 0u, 0u));
    if (tid < E) {
      if (sl.e0 + tid < sl.head) d[tid] = from_f32<T>(0.f);
      if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) d[sl.tail + tid] = from_f32<T>(0.f);
    }
    return;
  }
  const float tau = row_tau(a.temperature, b, nullptr), c = slope(tau), inv = inverse(tau);
  const float ca = over_tau(-(up + gh * st.z), inv), cb = over_tau(-gh * kLn2, inv);
  auto dense = [&](float xv) {
    const float y = (xv - m) * c - l2;
    return ptx::ex2(y) * fmaf(cb, fmaxf(y, kNoWeight), ca);
  };
  const float2 nm = make_float2(-m, -m), nl = make_float2(-l2, -l2), cc = make_float2(c, c);
  const float2 aa = make_float2(ca, ca), bb = make_float2(cb, cb);
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  uint4 next[U];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kThreads < sl.i1) next[u] = __ldcs(xv + i + u * kThreads);
  };
  load(sl.i0 + tid);
  for (int i = sl.i0 + tid; i < sl.i1; i += kThreads * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = next[u];
    load(i + kThreads * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kThreads >= sl.i1) break;
      float2 f[E / 2];
      Vec<T>::get(raw[u], f);
#pragma unroll
      for (int q = 0; q < E / 2; ++q) {
        const float2 y = __ffma2_rn(__fadd2_rn(f[q], nm), cc, nl);
        const float2 w = __ffma2_rn(bb, make_float2(fmaxf(y.x, kNoWeight), fmaxf(y.y, kNoWeight)), aa);
        f[q] = __fmul2_rn(make_float2(ptx::ex2(y.x), ptx::ex2(y.y)), w);
      }
      const uint4 out = Vec<T>::put(f);
      if (alike) {
        __stcs(dv + i + u * kThreads, out);
      } else {
        T e[E];
        memcpy(e, &out, 16);
#pragma unroll
        for (int q = 0; q < E; ++q) d[sl.head + (i + u * kThreads) * E + q] = e[q];
      }
    }
  }
  if (tid < E) {
    if (sl.e0 + tid < sl.head) d[tid] = from_f32<T>(dense(at(x, tid)));
    if (sl.e1 > sl.tail && sl.tail + tid < a.vocab) d[sl.tail + tid] = from_f32<T>(dense(at(x, sl.tail + tid)));
  }
  __syncthreads();
  if (tid <= k) {
    const int word = s_word[tid];
    bool first = word >= sl.e0 && word < sl.e1;
    float sum = 0.f;
    for (int j = 0; j <= k; ++j)
      if (s_word[j] == word) {
        if (j < tid) first = false;
        sum += s_up[j];
      }
    if (first) d[word] = from_f32<T>(over_tau(sum, inv) + dense(at(x, word)));
  }
}

int check(const AiScoreArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->vocab <= 0 || a->vocab > 0x40000000 || a->top_k < 0 || a->top_k > kMaxTop)
    return AI_ERR_SHAPE;
  if ((int64_t)a->batch * a->seq_len > 0x7fffffff / kMaxSplit) return AI_ERR_SHAPE;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  if (!a->logits || !a->tokens) return AI_ERR_NULL;
  if (a->stride_b < 0 || a->stride_t < 0) return AI_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(a->row_stats) & 15) return AI_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(a->logits) & (a->dtype == AI_DTYPE_F32 ? 3 : 1)) return AI_ERR_ALIGN;
  return AI_OK;
}

// Slices of a row: CTAs for four per SM, at least kLeast logits each.
int slices(const AiScoreArgs& a, int most) {
  const int64_t rows = (int64_t)a.batch * a.seq_len;
  const int least = a.dtype == AI_DTYPE_F32 ? kLeast / 2 : kLeast;
  int64_t n = 4 * (int64_t)sm_count() / rows;
  if (n > (a.vocab + least - 1) / least) n = (a.vocab + least - 1) / least;
  int s = 1;
  while (2 * s <= n && 2 * s <= most) s *= 2;
  return s;
}

template <typename T, bool kEntropy, bool kTop>
int launch(const AiScoreArgs& a, cudaStream_t st) {
  const auto kernel = score_kernel<T, kEntropy, kTop>;
  const int splits = slices(a, kMaxSplit);
  if (splits > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return AI_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.batch * a.seq_len * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kTop ? sizeof(TopSmem) + (splits > 1 ? splits * a.top_k * sizeof(Key) : 0) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  ProfScope ps(AI_PROF_SCORE, st);
  if (cudaLaunchKernelEx(&cfg, kernel, a, splits) != cudaSuccess) return AI_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int dispatch(const AiScoreArgs& a, cudaStream_t st) {
  if (a.entropy) return a.top_k ? launch<T, true, true>(a, st) : launch<T, true, false>(a, st);
  return a.top_k ? launch<T, false, true>(a, st) : launch<T, false, false>(a, st);
}

template <typename T>
int launch_bwd(const AiScoreBwdArgs& g, cudaStream_t st) {
  const int splits = slices(g.fwd, kMaxSplit);
  ProfScope ps(AI_PROF_SCORE, st);
  score_bwd_kernel<T><<<(unsigned)((int64_t)g.fwd.batch * g.fwd.seq_len * splits), kThreads, 0, st>>>(g, splits);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace score
}  // namespace ai

extern "C" int ai_token_logprobs(const AiScoreArgs* args, void* stream) {
  const int rc = ai::score::check(args);
  if (rc != AI_OK) return rc;
  if (!args->logprobs || (args->top_k > 0 && (!args->top_logprobs || !args->top_tokens))) return AI_ERR_NULL;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::score::dispatch<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::score::dispatch<__half>(*args, st);
  return ai::score::dispatch<float>(*args, st);
}

extern "C" int ai_token_logprobs_bwd(const AiScoreBwdArgs* args, void* stream) {
  if (!args) return AI_ERR_NULL;
  const AiScoreArgs& a = args->fwd;
  const int rc = ai::score::check(&a);
  if (rc != AI_OK) return rc;
  if (!args->dlogits || !a.row_stats || (args->g_top && a.top_k > 0 && !a.top_tokens)) return AI_ERR_NULL;
  if (args->dstride_b < 0 || args->dstride_t < 0) return AI_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(args->dlogits) & (a.dtype == AI_DTYPE_F32 ? 3 : 1)) return AI_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == AI_DTYPE_BF16) return ai::score::launch_bwd<__nv_bfloat16>(*args, st);
  if (a.dtype == AI_DTYPE_F16) return ai::score::launch_bwd<__half>(*args, st);
  return ai::score::launch_bwd<float>(*args, st);
}
