// Per-head RMS norms of queries and keys with the position rotation in the
// same pass, forward and backward (declared in include/ai_attn.h).
//
//   r = (mean(x^2) + eps)^-1/2, n = x r, y = n w, out = R(pos) y
//   g = R(pos)^T dout, dw = sum over rows of g n, u = g w,
//   dx = r (u - n mean(u n))
//
// A row of D elements sits in D / 16 lanes (ai_head_row.cuh).  Nothing but x
// is read again by the backward: r is one row sum away.  HBM-bound: the
// forward moves each row in and out once, the backward x and dout in and dx
// out.  A warp takes one token's heads, so that the token's cos / sin row and
// the weights stay in registers over them, kUnroll row groups at a time in
// flight.  The backward's warps keep the weight gradient of their dims in
// registers over all their rows; each CTA leaves one fp32 row and a second
// launch adds them in CTA order, so equal inputs give equal bits.
//
// Measured on 4 x 4096 tokens, 32 + 8 heads, D 128, bf16: forward 60 us,
// backward 90 us, both 5.6 TB/s; 2 x 1021 tokens, 16 + 2 heads, D 64, fp32:
// 6.3 + 10.2 us; 8 tokens: 2.5 us (a launch).

#include <cuda_runtime.h>

#include <cstring>

#include "ai_head_row.cuh"
#include "ai_kernels.h"

namespace ai {
namespace headnorm {

using namespace headrow;

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
// Row groups that a warp has in flight (backward: of x and dout each).  On 4 x
// 4096 tokens, 32 + 8 heads, D 128, bf16: forward 70 / 60 / 69 us with 1 / 2 /
// 4, backward 108 / 90 with 1 / 2.  A group of fp32 rows has the bytes of two.
template <typename T> constexpr int kUnrollOf = sizeof(T) == 4 ? 1 : 2;
// CTAs per SM of the backward (same case: 127 / 90 / 140 us with 1 / 2 / 3, the
// third by spilled registers).
constexpr int kCtasPerSm = 2;
// What a token costs beside its row groups, in row groups (101 / 90 / 92 us with
// 0 / 1 / 2).
constexpr int kStart = 1;

// How one tensor's rows are cut: `chunks` items per token, `per` heads each.
struct Cut {
  int heads, per, chunks;
};

struct Item {
  uint32_t b, t, chunk;
};

// (the launch keeps the item count within 32 bits: a 64-bit division costs
// more than a row)
__device__ __forceinline__ Item item_of(uint32_t it, const Cut& c, int seq_len) {
  const uint32_t tok = it / (uint32_t)c.chunks, b = tok / (uint32_t)seq_len;
  return {b, tok - b * (uint32_t)seq_len, it - tok * (uint32_t)c.chunks};
}

template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads, 3) fwd_kernel(const AiHeadNormArgs a, const Cut cq, const Cut ck,
                                                       const uint32_t items_q, const uint32_t items) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kUnroll = kUnrollOf<T>;
  const int lane = threadIdx.x % 32, sub = lane / kLanes, l = lane % kLanes;
  uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  const bool is_k = it >= items_q;
  if (is_k) it -= items_q;
  const Cut c = is_k ? ck : cq;
  const AiTensor4 src = is_k ? a.k : a.q, dst = is_k ? a.k_out : a.q_out;
  const void* weight = is_k ? a.k_weight : a.q_weight;
  const Item i0 = item_of(it, c, a.seq_len);
  const int64_t b = i0.b, t = i0.t;
  const int h0 = i0.chunk * c.per, h1 = min(c.heads, h0 + c.per);
  const T* x = static_cast<const T*>(src.ptr) + b * src.stride_b + t * src.stride_t + 8 * l;
  T* y = static_cast<T*>(dst.ptr) + b * dst.stride_b + t * dst.stride_t + 8 * l;
  F8 wlo, whi, cs, sn;
  int64_t row = 0;
  if (a.rope_cos) row = table_row(a.pos, b, t, a.n_pos, a.status);
  load_angles(a.rope_cos, a.rope_sin, row, D / 2, l, cs, sn);
  load_weight<T>(weight, a.weight_dtype == AI_DTYPE_F32, D, l, wlo, whi);
  for (int h = h0; h < h1; h += kUnroll * kRows) {
    Raw8<T> lo[kUnroll], hi[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      // (a row past the last head repeats the last one, so that every lane
      // takes part in the shuffles; it is not stored)
      const T* p = x + (int64_t)min(h + u * kRows + sub, h1 - 1) * src.stride_h;
      lo[u] = load8<T, kVec>(p);
      hi[u] = load8<T, kVec>(p + D / 2);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      F8 flo = unpack(lo[u]), fhi = unpack(hi[u]);
      norm_rotate<D>(flo, fhi, weight != nullptr, wlo, whi, cs, sn, a.eps);
      const int hh = h + u * kRows + sub;
      if (hh < h1) {
        T* p = y + (int64_t)hh * dst.stride_h;
        store8<T, kVec>(p, pack<T>(flo));
        store8<T, kVec>(p + D / 2, pack<T>(fhi));
      }
    }
  }
}

// CTAs [0, blocks_q) walk q's items, the others k's, so that a warp has one
// weight and one gradient of it.
template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) bwd_kernel(const AiHeadNormBwdArgs g, const Cut cq, const Cut ck,
                                                       const int blocks_q, const uint32_t tokens,
                                                       float* __restrict__ part) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kUnroll = kUnrollOf<T>;
  const AiHeadNormArgs& a = g.fwd;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, sub = lane / kLanes, l = lane % kLanes;
  const bool is_k = (int)blockIdx.x >= blocks_q;
  const uint32_t block = is_k ? blockIdx.x - blocks_q : blockIdx.x;
  const uint32_t n_warps = (is_k ? gridDim.x - blocks_q : blocks_q) * kWarps;
  const Cut c = is_k ? ck : cq;
  const AiTensor4 xt = is_k ? a.k : a.q, gt = is_k ? g.dk_out : g.dq_out, dt = is_k ? g.dk : g.dq;
  const void* weight = is_k ? a.k_weight : a.q_weight;
  F8 wlo, whi, dwlo = fill8(0.f), dwhi = fill8(0.f);
  load_weight<T>(weight, a.weight_dtype == AI_DTYPE_F32, D, l, wlo, whi);

  for (uint32_t it = block * kWarps + warp; it < tokens * (uint32_t)c.chunks; it += n_warps) {
    const Item i0 = item_of(it, c, a.seq_len);
    const int64_t b = i0.b, t = i0.t;
    const int h0 = i0.chunk * c.per, h1 = min(c.heads, h0 + c.per);
    const T* x = static_cast<const T*>(xt.ptr) + b * xt.stride_b + t * xt.stride_t + 8 * l;
    const T* go = static_cast<const T*>(gt.ptr) + b * gt.stride_b + t * gt.stride_t + 8 * l;
    T* dx = static_cast<T*>(dt.ptr) + b * dt.stride_b + t * dt.stride_t + 8 * l;
    F8 cs, sn;
    int64_t row = 0;
    if (a.rope_cos) row = table_row(a.pos, b, t, a.n_pos, a.status);
    load_angles(a.rope_cos, a.rope_sin, row, D / 2, l, cs, sn);
    for (int h = h0; h < h1; h += kUnroll * kRows) {
      Raw8<T> xlo[kUnroll], xhi[kUnroll], glo[kUnroll], ghi[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t hh = min(h + u * kRows + sub, h1 - 1);
        glo[u] = load8<T, kVec>(go + hh * gt.stride_h);
        ghi[u] = load8<T, kVec>(go + hh * gt.stride_h + D / 2);
        if (weight) {
          xlo[u] = load8<T, kVec>(x + hh * xt.stride_h);
          xhi[u] = load8<T, kVec>(x + hh * xt.stride_h + D / 2);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int hh = h + u * kRows + sub;
        F8 flo = unpack(glo[u]), fhi = unpack(ghi[u]);
        rotate<true>(flo, fhi, cs, sn);
        if (weight) {
          // With F = r R^T dout and U = F w: dw += F x, mean(u n) = sum(U x) / D
          // and dx = U - x r^2 mean(u n).
          const F8 x0 = unpack(xlo[u]), x1 = unpack(xhi[u]);
          const float r = inv_rms<D>(x0, x1, a.eps);
          scale8(flo, r);
          scale8(fhi, r);
          if (hh < h1) {  // a repeated row adds nothing to dw
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              dwlo.v[i] = __ffma2_rn(flo.v[i], x0.v[i], dwlo.v[i]);
              dwhi.v[i] = __ffma2_rn(fhi.v[i], x1.v[i], dwhi.v[i]);
            }
          }
          mul8(flo, wlo);
          mul8(fhi, whi);
          const float m = -r * r * (row_sum<kLanes>(dot8(flo, x0, fhi, x1)) * (1.f / D));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            flo.v[i] = __ffma2_rn(x0.v[i], make_float2(m, m), flo.v[i]);
            fhi.v[i] = __ffma2_rn(x1.v[i], make_float2(m, m), fhi.v[i]);
          }
        }
        if (hh < h1) {
          T* p = dx + (int64_t)hh * dt.stride_h;
          store8<T, kVec>(p, pack<T>(flo));
          store8<T, kVec>(p + D / 2, pack<T>(fhi));
        }
      }
    }
  }

  // The CTA's row of dw: lanes of equal dims, then the warps in order.
  __shared__ __align__(8) float s_dw[kWarps][D];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) {
      dwlo.v[i].x += __shfl_xor_sync(0xffffffffu, dwlo.v[i].x, o), dwlo.v[i].y += __shfl_xor_sync(0xffffffffu, dwlo.v[i].y, o);
      dwhi.v[i].x += __shfl_xor_sync(0xffffffffu, dwhi.v[i].x, o), dwhi.v[i].y += __shfl_xor_sync(0xffffffffu, dwhi.v[i].y, o);
    }
    if (sub == 0) {
      *reinterpret_cast<float2*>(&s_dw[warp][8 * l + 2 * i]) = dwlo.v[i];
      *reinterpret_cast<float2*>(&s_dw[warp][D / 2 + 8 * l + 2 * i]) = dwhi.v[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += s_dw[w][threadIdx.x];
    part[(int64_t)blockIdx.x * D + threadIdx.x] = s;
  }
}

// One CTA of 32 x 32 threads per (tensor, 32 dims): sums the CTAs' rows.
template <typename T>
__global__ void __launch_bounds__(1024) dw_kernel(const AiHeadNormBwdArgs g, const float* __restrict__ part,
                                                  const int blocks_q, const int blocks, const int D) {
  const bool is_k = blockIdx.y != 0;
  void* out = is_k ? g.dk_weight : g.dq_weight;
  if (!out) return;
  const int d = blockIdx.x * 32 + threadIdx.x;
  const int lo = is_k ? blocks_q : 0, hi = is_k ? blocks : blocks_q;
  float s = 0.f;
  for (int i = lo + (int)threadIdx.y; i < hi; i += 32) s += part[(int64_t)i * D + d];
  __shared__ float sm[32][33];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) s += sm[w][threadIdx.x];
  if (g.fwd.weight_dtype == AI_DTYPE_F32)
    static_cast<float*>(out)[d] = s;
  else
    static_cast<T*>(out)[d] = from_f32<T>(s);
}

int check(const AiHeadNormArgs* a, bool outs) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->num_q_heads <= 0 || a->num_kv_heads < 0) return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  if (a->weight_dtype != a->dtype && a->weight_dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  const AiTensor4* ts[4] = {&a->q, &a->q_out, &a->k, &a->k_out};
  for (int i = 0; i < (a->num_kv_heads > 0 ? 4 : 2); ++i) {
    if (!outs && (i & 1)) continue;
    if (!ts[i]->ptr) return AI_ERR_NULL;
    if (ts[i]->stride_b < 0 || ts[i]->stride_h < 0 || ts[i]->stride_t < 0) return AI_ERR_STRIDE;
  }
  if ((a->rope_cos != nullptr) != (a->rope_sin != nullptr)) return AI_ERR_NULL;
  if (a->rope_cos) {
    if (!a->pos.ptr) return AI_ERR_NULL;
    if (a->n_pos <= 0) return AI_ERR_SHAPE;
    if (a->pos.stride_b < 0) return AI_ERR_STRIDE;
    if ((reinterpret_cast<uintptr_t>(a->rope_cos) | reinterpret_cast<uintptr_t>(a->rope_sin)) & 15)
      return AI_ERR_ALIGN;
  }
  return AI_OK;
}

int check_bwd(const AiHeadNormBwdArgs* g) {
  if (!g) return AI_ERR_NULL;
  const int rc = check(&g->fwd, false);
  if (rc != AI_OK) return rc;
  const AiTensor4* ts[4] = {&g->dq_out, &g->dq, &g->dk_out, &g->dk};
  for (int i = 0; i < (g->fwd.num_kv_heads > 0 ? 4 : 2); ++i) {
    if (!ts[i]->ptr) return AI_ERR_NULL;
    if (ts[i]->stride_b < 0 || ts[i]->stride_h < 0 || ts[i]->stride_t < 0) return AI_ERR_STRIDE;
  }
  if ((g->fwd.q_weight && !g->dq_weight) || (g->fwd.num_kv_heads > 0 && g->fwd.k_weight && !g->dk_weight))
    return AI_ERR_NULL;
  return AI_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// A token's heads are cut into items of whole unrolled row groups once there
// are too few tokens for every SM to have a few warps of them; a long
// sequence keeps a token's heads together (its angles are then read once).
Cut cut(int heads, int64_t tokens, int head_dim, int unroll) {
  Cut c{heads, heads, 1};
  const int rows = 32 / (head_dim / 16);
  const int groups = (heads + rows - 1) / rows;
  if (tokens < (int64_t)sm_count() * 2 * kWarps) {
    const int per_item = tokens * groups <= (int64_t)sm_count() * kWarps ? 1 : unroll;
    c.per = per_item * rows < heads ? per_item * rows : heads;
    c.chunks = (heads + c.per - 1) / c.per;
  }
  return c;
}

struct BwdPlan {
  Cut q, k;
  int blocks_q, blocks;
};

// CTAs in proportion to what a token's heads cost, all resident at once.
BwdPlan plan_bwd(const AiHeadNormArgs& a) {
  BwdPlan p;
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  const int unroll = a.dtype == AI_DTYPE_F32 ? kUnrollOf<float> : kUnrollOf<__half>;
  p.q = cut(a.num_q_heads, tokens, a.head_dim, unroll);
  p.k = cut(a.num_kv_heads > 0 ? a.num_kv_heads : 1, tokens, a.head_dim, unroll);
  const int64_t most = kCtasPerSm * (int64_t)sm_count();
  const int rows = 32 / (a.head_dim / 16);
  auto cost = [&](const Cut& c) { return (c.heads + rows - 1) / rows + kStart * c.chunks; };  // of a token
  const int64_t cq = cost(p.q), ck = a.num_kv_heads > 0 ? cost(p.k) : 0;
  auto blocks = [&](const Cut& c, int64_t share) {
    const int64_t need = (tokens * c.chunks + kWarps - 1) / kWarps;
    if (share < 1) share = 1;
    return (int)(need < share ? need : share);
  };
  int64_t share_k = (most * ck + (cq + ck) / 2) / (cq + ck);
  p.blocks_q = blocks(p.q, most - share_k);
  p.blocks = p.blocks_q + (ck > 0 ? blocks(p.k, share_k) : 0);
  return p;
}

template <typename T, int D>
int launch_fwd(const AiHeadNormArgs& a, cudaStream_t st) {
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  const Cut cq = cut(a.num_q_heads, tokens, D, kUnrollOf<T>);
  const Cut ck = cut(a.num_kv_heads > 0 ? a.num_kv_heads : 1, tokens, D, kUnrollOf<T>);
  const int64_t items_q = tokens * cq.chunks, items = items_q + (a.num_kv_heads > 0 ? tokens * ck.chunks : 0);
  const int64_t blocks = (items + kWarps - 1) / kWarps;
  if (items > 0x7fffffff) return AI_ERR_SHAPE;
  bool vec = rows_aligned(a.q, a.dtype) && rows_aligned(a.q_out, a.dtype);
  if (a.num_kv_heads > 0) vec = vec && rows_aligned(a.k, a.dtype) && rows_aligned(a.k_out, a.dtype);
  ProfScope ps(AI_PROF_HEAD_NORM, st);
  if (vec)
    fwd_kernel<T, D, true><<<(unsigned)blocks, kThreads, 0, st>>>(a, cq, ck, (uint32_t)items_q, (uint32_t)items);
  else
    fwd_kernel<T, D, false><<<(unsigned)blocks, kThreads, 0, st>>>(a, cq, ck, (uint32_t)items_q, (uint32_t)items);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T, int D>
int launch_bwd(const AiHeadNormBwdArgs& g, cudaStream_t st) {
  const AiHeadNormArgs& a = g.fwd;
  const BwdPlan p = plan_bwd(a);
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  // (a warp's next item may lie one round past the last)
  if ((tokens * p.q.chunks > tokens * p.k.chunks ? tokens * p.q.chunks : tokens * p.k.chunks) > 0x7fffffff) return AI_ERR_SHAPE;
  float* part = static_cast<float*>(g.workspace);
  bool vec = rows_aligned(a.q, a.dtype) && rows_aligned(g.dq_out, a.dtype) && rows_aligned(g.dq, a.dtype);
  if (a.num_kv_heads > 0)
    vec = vec && rows_aligned(a.k, a.dtype) && rows_aligned(g.dk_out, a.dtype) && rows_aligned(g.dk, a.dtype);
  {
    ProfScope ps(AI_PROF_HEAD_NORM, st);
    if (vec)
      bwd_kernel<T, D, true><<<p.blocks, kThreads, 0, st>>>(g, p.q, p.k, p.blocks_q, (uint32_t)tokens, part);
    else
      bwd_kernel<T, D, false><<<p.blocks, kThreads, 0, st>>>(g, p.q, p.k, p.blocks_q, (uint32_t)tokens, part);
    if (cudaGetLastError() != cudaSuccess) return AI_ERR_LAUNCH;
  }
  if (a.q_weight || (a.num_kv_heads > 0 && a.k_weight)) {
    ProfScope ps(AI_PROF_HEAD_NORM, st);
    AiHeadNormBwdArgs gw = g;  // only the weights that exist have a gradient
    if (!a.q_weight) gw.dq_weight = nullptr;
    if (!a.k_weight) gw.dk_weight = nullptr;
    dw_kernel<T><<<dim3(D / 32, a.num_kv_heads > 0 ? 2 : 1), dim3(32, 32), 0, st>>>(gw, part, p.blocks_q, p.blocks, D);
    if (cudaGetLastError() != cudaSuccess) return AI_ERR_LAUNCH;
  }
  return AI_OK;
}

template <typename T>
int dispatch_fwd(const AiHeadNormArgs& a, cudaStream_t st) {
  if (a.head_dim == 128) return launch_fwd<T, 128>(a, st);
  if (a.head_dim == 64) return launch_fwd<T, 64>(a, st);
  return launch_fwd<T, 32>(a, st);
}

template <typename T>
int dispatch_bwd(const AiHeadNormBwdArgs& g, cudaStream_t st) {
  if (g.fwd.head_dim == 128) return launch_bwd<T, 128>(g, st);
  if (g.fwd.head_dim == 64) return launch_bwd<T, 64>(g, st);
  return launch_bwd<T, 32>(g, st);
}

}  // namespace headnorm
}  // namespace ai

extern "C" int ai_head_norm_fwd(const AiHeadNormArgs* args, void* stream) {
  const int rc = ai::headnorm::check(args, true);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::headnorm::dispatch_fwd<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::headnorm::dispatch_fwd<__half>(*args, st);
  return ai::headnorm::dispatch_fwd<float>(*args, st);
}

extern "C" int ai_head_norm_bwd_workspace(const AiHeadNormBwdArgs* args, size_t* bytes) {
  const int rc = ai::headnorm::check_bwd(args);
  if (rc != AI_OK) return rc;
  if (!bytes) return AI_ERR_NULL;
  *bytes = (size_t)ai::headnorm::plan_bwd(args->fwd).blocks * args->fwd.head_dim * sizeof(float);
  return AI_OK;
}

extern "C" int ai_head_norm_bwd(const AiHeadNormBwdArgs* args, void* stream) {
  size_t need = 0;
  const int rc = ai_head_norm_bwd_workspace(args, &need);
  if (rc != AI_OK) return rc;
  if (!args->workspace || args->workspace_bytes < need) return AI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(args->workspace) & 15) return AI_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->fwd.dtype == AI_DTYPE_BF16) return ai::headnorm::dispatch_bwd<__nv_bfloat16>(*args, st);
  if (args->fwd.dtype == AI_DTYPE_F16) return ai::headnorm::dispatch_bwd<__half>(*args, st);
  return ai::headnorm::dispatch_bwd<float>(*args, st);
}
