// The paged cache in 4 bits: a row's codes and scales (include/ai_attn.h,
// AiPool4), lengths and pages.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "../../include/ai_attn.h"
#include "ai_common.cuh"

namespace ai {
namespace kv4 {

constexpr int kGroup = 32;  // dims that share a scale

// Tokens [.., n) of a sequence that a call is about: its count, clamped to what
// was given.
__device__ __forceinline__ int new_tokens(const int32_t* n, int64_t b, int given, int32_t* status) {
  const int x = n ? __ldg(n + b) : given;
  if (x < 0 || x > given) report(status, AI_ERR_DEV_BOUNDS);
  return max(0, min(x, given));
}

// Page and slot of token `at` of sequence b; page -1 where there is none.
struct Place {
  int page;
  int slot;
};

__device__ __forceinline__ Place place(const AiPool4& p, int64_t b, int64_t at) {
  Place r{-1, 0};
  const int64_t col = at / p.page_size;
  if (at < 0 || col >= p.max_pages) return r;
  r.slot = (int)(at - col * p.page_size);
  const int page = __ldg(p.page_table + b * p.page_table_stride + col);
  if (page >= 0 && page < p.n_pages) r.page = page;
  return r;
}

inline int check_pool(const AiPool4& p, int head_dim) {
  // (a slot's bytes from its page's start are counted in 31 bits)
  if (p.n_pages <= 0 || p.page_size < 16 || p.page_size > AI_POOL4_MAX_PAGE || (p.page_size & (p.page_size - 1)) || p.max_pages <= 0)
    return AI_ERR_SHAPE;
  if (!p.page_table) return AI_ERR_NULL;
  if (p.page_table_stride < 0) return AI_ERR_STRIDE;
  for (int i = 0; i < 4; ++i) {
    const AiTensor4& t = i == 0 ? p.k_codes : i == 1 ? p.v_codes : i == 2 ? p.k_scales : p.v_scales;
    if (!t.ptr) return AI_ERR_NULL;
    if (t.stride_b < 0 || t.stride_h < 0 || t.stride_t < 0) return AI_ERR_STRIDE;
    // (the slots of a page and head follow one another, from a 16-byte boundary)
    if (t.stride_t != (i < 2 ? head_dim / 2 : head_dim / kGroup)) return AI_ERR_STRIDE;
    if ((t.stride_b | t.stride_h) % (i < 2 ? 16 : 8)) return AI_ERR_STRIDE;
    if (t.stride_b / (i < 2 ? 16 : 8) > 0xffffffffLL) return AI_ERR_STRIDE;  // (kernels count 16-byte units in 32 bits)
    if (reinterpret_cast<uintptr_t>(t.ptr) & 15) return AI_ERR_ALIGN;
  }
  return AI_OK;
}

}  // namespace kv4
}  // namespace ai
