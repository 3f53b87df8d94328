// Shared by the kernels of the shared-prefix attention.
#pragma once

#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "../../include/ai_attn.h"
#include "ai_common.cuh"

namespace ai {
namespace prefix {

// The tensor-core kernels (ai_prefix_attn_sm100.cu): whether they take the
// call, the scratch they need, and the launch.
bool sm100_fits(const AiPrefixAttnArgs& a);
size_t sm100_workspace(const AiPrefixAttnArgs& a);
int sm100_launch(const AiPrefixAttnArgs& a, cudaStream_t st);

// Own keys of a sequence (clamped to what its page table can hold) and its
// real query tokens.
struct Lens {
  int keys, n;
};

__device__ __forceinline__ Lens seq_lens(const AiPrefixAttnArgs& a, int64_t b) {
  Lens r;
  r.keys = __ldg(a.lens + b);
  r.n = a.query_lens ? __ldg(a.query_lens + b) : a.seq_len;
  if (r.keys < 0 || r.keys > a.max_pages * a.page_size || r.n < 0 || r.n > a.seq_len) {
    report(a.status, AI_ERR_DEV_BOUNDS);
    r.keys = max(0, min(r.keys, a.max_pages * a.page_size));
    r.n = max(0, min(r.n, a.seq_len));
  }
  return r;
}

// Page i of a table; a page outside the pool is reported and read as page 0.
__device__ __forceinline__ int page_of(const AiPrefixAttnArgs& a, const int32_t* table, int64_t i) {
  const int p = __ldg(table + i);
  if (p < 0 || p >= a.n_pages) {
    report(a.status, AI_ERR_DEV_BOUNDS);
    return 0;
  }
  return p;
}

// The log-sum `lse` of a partial result with exponentials' sum l: -inf without
// keys, +inf where l is NaN (a NaN among the row's scores), which makes the
// joined row NaN.
__device__ __forceinline__ float part_lse(float l, float lse) {
  return l > 0.f ? lse : l == 0.f ? -CUDART_INF_F : CUDART_INF_F;
}

}  // namespace prefix
}  // namespace ai
