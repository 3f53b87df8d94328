// New keys and values into the paged cache (declared in include/ai_attn.h):
// keys normalised and rotated on the way, values copied, straight from the
// projections' layout to each token's slot.
//
// A row of D elements sits in D / 16 lanes (ai_head_row.cuh); a warp takes a
// few heads of one token, K rows and V rows alike, so the token's page and
// its angles are looked up once per item; the rows are loaded beside that
// lookup.  HBM-bound (each row moves in and out once); with one token per
// sequence it is a launch latency.  Measured: 8 sequences of up to 2047 fp16
// tokens, 8 heads, D 128: 17.7 us = 4.5 TB/s, a ramp of a few us included
// (18.2 with the rows loaded after the page; 17.8 at eight CTAs per SM, 19.6
// at ten); one token of 64 sequences: 2.9 us.

#include <cuda_runtime.h>

#include <cstring>

#include "ai_head_row.cuh"
#include "ai_kernels.h"

namespace ai {
namespace append {

using namespace headrow;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kThreads, 6) append_kernel(const AiPagedAppendArgs a, const int per, const int chunks,
                                                          const uint32_t items) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  const int lane = threadIdx.x % 32, sub = lane / kLanes, l = lane % kLanes;
  const uint32_t it = blockIdx.x * kWarps + threadIdx.x / 32;
  if (it >= items) return;
  // (32-bit divisions: the launch keeps the item count within them)
  const uint32_t tok = it / (uint32_t)chunks, seq = tok / (uint32_t)a.seq_len;
  const int64_t b = seq;
  const int t = (int)(tok - seq * (uint32_t)a.seq_len);
  const int n_new = a.new_lens ? __ldg(a.new_lens + b) : a.seq_len;
  if (n_new < 0 || n_new > a.seq_len) report(a.status, AI_ERR_DEV_BOUNDS);  // (taken as the nearest in range)
  if (t >= n_new) return;
  const int64_t n = (int64_t)__ldg(a.lens + b) + t;
  // (the rows' loads below wait for neither the page nor its check)
  const int col = n >= 0 && n <= 0x7fffffff ? (int)n / a.page_size : -1;
  const bool listed = col >= 0 && col < a.max_pages;
  const int page = listed ? __ldg(a.page_table + b * a.page_table_stride + col) : -1;
  const int64_t slot = (int)n - col * a.page_size;
  const int h0 = (int)(it - tok * (uint32_t)chunks) * per, h1 = min(a.num_kv_heads, h0 + per);
  const T* k = static_cast<const T*>(a.k.ptr) + b * a.k.stride_b + t * a.k.stride_t + 8 * l;
  const T* v = static_cast<const T*>(a.v.ptr) + b * a.v.stride_b + t * a.v.stride_t + 8 * l;
  T* ko = static_cast<T*>(a.k_pages.ptr) + page * a.k_pages.stride_b + slot * a.k_pages.stride_t + 8 * l;
  T* vo = static_cast<T*>(a.v_pages.ptr) + page * a.v_pages.stride_b + slot * a.v_pages.stride_t + 8 * l;
  F8 wlo, whi, cs, sn;
  int64_t row = 0;
  if (a.rope_cos) row = table_row(a.pos, b, t, a.n_pos, a.status);
  load_angles(a.rope_cos, a.rope_sin, row, D / 2, l, cs, sn);
  load_weight<T>(a.k_weight, a.weight_dtype == AI_DTYPE_F32, D, l, wlo, whi);
  const bool held = page >= 0 && page < a.n_pages;
  for (int hb = h0; hb < h1; hb += kRows) {
    const int64_t h = min(hb + sub, h1 - 1);  // (rows past the last head repeat it, unstored)
    const Raw8<T> klo = load8<T, kVec>(k + h * a.k.stride_h), khi = load8<T, kVec>(k + h * a.k.stride_h + D / 2);
    const Raw8<T> vlo = load8<T, kVec>(v + h * a.v.stride_h), vhi = load8<T, kVec>(v + h * a.v.stride_h + D / 2);
    F8 flo = unpack(klo), fhi = unpack(khi);
    norm_rotate<D>(flo, fhi, a.k_weight != nullptr, wlo, whi, cs, sn, a.eps);
    if (held && hb + sub < h1) {
      store8<T, kVec>(ko + h * a.k_pages.stride_h, pack<T>(flo));
      store8<T, kVec>(ko + h * a.k_pages.stride_h + D / 2, pack<T>(fhi));
      store8<T, kVec>(vo + h * a.v_pages.stride_h, vlo);
      store8<T, kVec>(vo + h * a.v_pages.stride_h + D / 2, vhi);
    }
  }
  if (!held) report(a.status, AI_ERR_DEV_BOUNDS);
}

int check(const AiPagedAppendArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->num_kv_heads <= 0 || a->n_pages <= 0 || a->page_size <= 0 ||
      a->max_pages <= 0)
    return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  if (a->weight_dtype != a->dtype && a->weight_dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  for (const AiTensor4* t : {&a->k, &a->v, &a->k_pages, &a->v_pages}) {
    if (!t->ptr) return AI_ERR_NULL;
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < 0) return AI_ERR_STRIDE;
  }
  if (!a->page_table || !a->lens) return AI_ERR_NULL;
  if (a->page_table_stride < 0) return AI_ERR_STRIDE;
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

template <typename T, int D>
int launch(const AiPagedAppendArgs& a, cudaStream_t st) {
  // One row group per item while that gives every SM at most a few warps;
  // then a token's heads stay together (16,376 tokens: 17.8 us, cut 20.0).
  constexpr int kRows = 32 / (D / 16);
  const int64_t tokens = (int64_t)a.batch * a.seq_len;
  const int per = tokens <= 4096 ? (kRows < a.num_kv_heads ? kRows : a.num_kv_heads) : a.num_kv_heads;
  const int chunks = (a.num_kv_heads + per - 1) / per;
  const int64_t items = tokens * chunks, blocks = (items + kWarps - 1) / kWarps;
  if (items > 0x7fffffff) return AI_ERR_SHAPE;
  const bool vec = rows_aligned(a.k, a.dtype) && rows_aligned(a.v, a.dtype) && rows_aligned(a.k_pages, a.dtype) &&
                   rows_aligned(a.v_pages, a.dtype);
  ProfScope ps(AI_PROF_APPEND, st);
  if (vec)
    append_kernel<T, D, true><<<(unsigned)blocks, kThreads, 0, st>>>(a, per, chunks, (uint32_t)items);
  else
    append_kernel<T, D, false><<<(unsigned)blocks, kThreads, 0, st>>>(a, per, chunks, (uint32_t)items);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int dispatch(const AiPagedAppendArgs& a, cudaStream_t st) {
  if (a.head_dim == 128) return launch<T, 128>(a, st);
  if (a.head_dim == 64) return launch<T, 64>(a, st);
  return launch<T, 32>(a, st);
}

}  // namespace append
}  // namespace ai

extern "C" int ai_paged_append(const AiPagedAppendArgs* args, void* stream) {
  const int rc = ai::append::check(args);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::append::dispatch<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::append::dispatch<__half>(*args, st);
  return ai::append::dispatch<float>(*args, st);
}
