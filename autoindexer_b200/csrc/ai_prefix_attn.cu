// Attention over a paged cache of a batch whose sequences share a prefix
// (declared in include/ai_attn.h): argument checks, the kernels for the types
// and layouts the tensor-core kernels do not take (fp32; head_dim 32; page
// sizes other than powers of two from 16; rows off 16-byte boundaries; a
// scale of 0 or less; more sequences than their scans hold), and dispatch.
//
// rows kernel: a CTA per (16 query rows of a KV head that share a key list,
// chunk of the list).  32 keys at a time go to shared memory as fp32; a lane
// per key forms four rows' scores, the rows' running maximum and sum stay in
// the warp, and a lane per D / 32 dims adds four rows' weighted values, so a
// value from shared memory meets four rows.  The chunks' partial results (O / l
// and the log-sum, fp32) are joined by a second launch.  Bound by the chain of
// a step (page, K and V rows, shared memory) at four CTAs per SM, then by
// shared memory: eight 128-byte wavefronts per 16 warp multiply-adds.
// Measured on 16 sequences x 32 heads (8 KV heads, D 128), one token each, on
// a prefix of 4096 keys and up to 512 own: 104 us in fp32, 100 us in bf16 with
// 48-slot pages (a CTA per query row: 1453 and 1526 us).

#include <cuda_runtime.h>
#include <math_constants.h>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_prefix_attn.h"

namespace ai {
namespace prefix {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kRows = 16, kWarpRows = kRows / kWarps;  // query rows of a CTA, of a warp
constexpr int kKeys = 32;                              // keys of a step
constexpr int kLeastChunk = 4 * kKeys;                 // a partial result costs about as much as a few steps
constexpr int kCtasPerSm = 8;                          // CTAs to aim at: two rounds of the four that fit

struct Plan {
  int group, rows_seq;               // G, T G
  int groups_prefix, groups_own;     // groups of kRows rows, per KV head / per KV head and sequence
  int splits_prefix, splits_own;     // chunks of a list (own: of what the table can hold)
  int chunk_prefix, chunk_own;       // keys of a chunk
  int items_prefix, items;           // CTAs
  bool vec_q, vec;                   // Q rows, K and V rows start on 16-byte boundaries
  float *part_o, *part_lse;          // [B Hq T][splits_prefix + splits_own] rows
};

template <typename T>
__device__ __forceinline__ float4 load4(const T* p, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      return __ldg(reinterpret_cast<const float4*>(p));
    } else {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
      const T* e = reinterpret_cast<const T*>(&r);
      return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
    }
  }
  return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
}

// E floats from shared memory.
template <int E>
__device__ __forceinline__ void read(const float* p, float (&v)[E]) {
  if constexpr (E == 4)
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
  else if constexpr (E == 2)
    *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p);
  else
    v[0] = p[0];
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rows_kernel(const AiPrefixAttnArgs a, const Plan p) {
  constexpr int E = D / 32, C = D / 4;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  __shared__ __align__(16) float s_q[kRows][D], s_k[kKeys][D + 4], s_v[kKeys][D], s_p[kRows][kKeys];
  __shared__ int64_t s_at[2][kKeys];  // offsets of the keys' K and V rows
  __shared__ int64_t s_row[kRows];    // partial-result row, -1: none
  __shared__ int64_t s_src[kRows];    // offset of its query
  __shared__ int s_limit[kRows];      // keys of the list that the row sees

  // The chunk and its rows.
  const bool pre = (int)blockIdx.x < p.items_prefix;
  int x = pre ? blockIdx.x : blockIdx.x - p.items_prefix;
  const int splits = pre ? p.splits_prefix : p.splits_own, groups = pre ? p.groups_prefix : p.groups_own;
  const int split = x % splits;
  x /= splits;
  const int hk = x % a.num_kv_heads;
  x /= a.num_kv_heads;
  const int row0 = (x % groups) * kRows;
  const int64_t b = x / groups;  // (own keys)
  const int keys = pre ? a.prefix_len : seq_lens(a, b).keys, chunk = pre ? p.chunk_prefix : p.chunk_own;
  const int64_t k_begin = (int64_t)split * chunk;
  const int k_end = (int)min((int64_t)keys, k_begin + chunk);
  if (k_begin >= k_end) return;
  const int32_t* table = pre ? a.prefix_pages : a.page_table + b * a.page_table_stride;

  // Offset of key k's row in K (threads below kKeys) or V.
  const AiTensor4& pool = tid < kKeys ? a.k_pages : a.v_pages;
  auto key_at = [&](int k) -> int64_t {
    if (tid >= 2 * kKeys || k >= k_end) return -1;
    const int page = k / a.page_size;
    return page_of(a, table, page) * pool.stride_b + hk * pool.stride_h + (k - page * a.page_size) * pool.stride_t;
  };
  int64_t next_at = key_at((int)k_begin + tid % kKeys);
  if (tid < kRows) {
    int64_t part = -1, src = -1;
    int limit = 0;
    if (row0 + tid < (pre ? a.batch * p.rows_seq : p.rows_seq)) {
      const int n = row0 + tid, rb = pre ? n / p.rows_seq : (int)b, rem = pre ? n - rb * p.rows_seq : n;
      const int t = rem / p.group, h = hk * p.group + rem - t * p.group;
      const Lens len = seq_lens(a, rb);
      if (t < len.n) {
        src = rb * a.q.stride_b + h * a.q.stride_h + t * a.q.stride_t;
        limit = pre ? keys : max(0, keys - len.n + t + 1);
        part = (((int64_t)rb * a.num_q_heads + h) * a.seq_len + t) * (p.splits_prefix + p.splits_own) +
               (pre ? split : p.splits_prefix + split);
      }
    }
    s_row[tid] = part, s_limit[tid] = limit, s_src[tid] = src;
  }
  __syncthreads();
#pragma unroll
  for (int i = tid; i < kRows * C; i += kThreads) {
    const int r = i / C, c = i % C;
    const int64_t src = s_src[r];
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
    if (src >= 0) q = load4(static_cast<const T*>(a.q.ptr) + src + 4 * c, p.vec_q);
    q.x *= a.scale, q.y *= a.scale, q.z *= a.scale, q.w *= a.scale;
    *reinterpret_cast<float4*>(&s_q[r][4 * c]) = q;
  }
  int limit[kWarpRows], least = 0x7fffffff;
  float m[kWarpRows], l[kWarpRows], acc[kWarpRows][E];
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    const int row = kWarpRows * warp + r;
    limit[r] = s_limit[row];
    if (s_row[row] >= 0) least = min(least, limit[r]);
    m[r] = -CUDART_INF_F, l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[r][e] = 0.f;
  }
  for (int k0 = (int)k_begin; k0 < k_end; k0 += kKeys) {
    if (tid < 2 * kKeys) s_at[tid / kKeys][tid % kKeys] = next_at;
    __syncthreads();
    next_at = key_at(k0 + kKeys + tid % kKeys);
    // (past the list: the step's first key's row, as zeros)
    constexpr int kLoads = kKeys * C / kThreads;
    float4 kv[kLoads], vv[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int x = tid + i * kThreads, k = k0 + x / C < k_end ? x / C : 0;
      kv[i] = load4(static_cast<const T*>(a.k_pages.ptr) + s_at[0][k] + 4 * (x % C), p.vec);
      vv[i] = load4(static_cast<const T*>(a.v_pages.ptr) + s_at[1][k] + 4 * (x % C), p.vec);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int x = tid + i * kThreads;
      const bool in = k0 + x / C < k_end;
      const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
      *reinterpret_cast<float4*>(&s_k[x / C][4 * (x % C)]) = in ? kv[i] : zero;
      *reinterpret_cast<float4*>(&s_v[x / C][4 * (x % C)]) = in ? vv[i] : zero;
    }
    __syncthreads();
    // Scores of key `lane` with the warp's rows.
    float s[kWarpRows];
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) s[r] = 0.f;
#pragma unroll 8
    for (int c = 0; c < C; ++c) {
      const float4 k = *reinterpret_cast<const float4*>(&s_k[lane][4 * c]);
#pragma unroll
      for (int r = 0; r < kWarpRows; ++r) {
        const float4 q = *reinterpret_cast<const float4*>(&s_q[kWarpRows * warp + r][4 * c]);
        s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
      }
    }
    const int key = k0 + lane;
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) {
      if (key >= min(limit[r], k_end)) s[r] = -CUDART_INF_F;
      float top = s[r];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float m_new = fmaxf(m[r], top), base = m_new == -CUDART_INF_F ? 0.f : m_new;
      const float w = expf(s[r] - base), alpha = expf(m[r] - base);  // 0 while m is -inf
      float sum = w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[r] = l[r] * alpha + sum;
      m[r] = m_new;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[r][e] *= alpha;
      s_p[kWarpRows * warp + r][lane] = w;
    }
    __syncwarp();
    const bool ragged = k0 + kKeys > min(least, k_end);
    for (int k = 0; k < kKeys; k += 4) {
      float v[4][E];
#pragma unroll
      for (int i = 0; i < 4; ++i) read<E>(&s_v[k + i][E * lane], v[i]);
#pragma unroll
      for (int r = 0; r < kWarpRows; ++r) {
        float w[4];
        read<4>(&s_p[kWarpRows * warp + r][k], w);
        // (a row takes nothing from a key it does not see, whatever it holds)
        if (ragged) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (k0 + k + i < limit[r]) acc[r][e] = fmaf(w[i], v[i][e], acc[r][e]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] = fmaf(w[i], v[i][e], acc[r][e]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    const int64_t row = s_row[kWarpRows * warp + r];
    if (row < 0) continue;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
    for (int e = 0; e < E; ++e) p.part_o[row * D + E * lane + e] = acc[r][e] * inv;
    if (lane == 0) p.part_lse[row] = part_lse(l[r], m[r] + logf(l[r]));
  }
}

// A warp per (sequence, query head, query token) joins its chunks.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) join_kernel(const AiPrefixAttnArgs a, const Plan p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x % 32;
  const int64_t row = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (row >= (int64_t)a.batch * a.num_q_heads * a.seq_len) return;
  const int64_t b = row / ((int64_t)a.num_q_heads * a.seq_len);
  const int h = (int)(row / a.seq_len % a.num_q_heads), t = (int)(row % a.seq_len);
  const Lens len = seq_lens(a, b);
  float m = -CUDART_INF_F, l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (t < len.n) {
    const int pre = p.splits_prefix, all = pre + p.splits_own;
    const int n = pre + (len.keys > 0 ? (len.keys - 1) / p.chunk_own + 1 : 0);
    const float* lse = p.part_lse + row * all;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, lse[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m != -CUDART_INF_F) {
      for (int i0 = 0; i0 < n; i0 += 32) {
        const float mine = i0 + lane < n ? expf(lse[i0 + lane] - m) : 0.f;
        const int cnt = min(32, n - i0);
#pragma unroll 4
        for (int k = 0; k < cnt; ++k) {
          const float w = __shfl_sync(0xffffffffu, mine, k);
          float o[E];
          read<E>(p.part_o + (row * all + i0 + k) * D + E * lane, o);
          l += w;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(w, o[e], acc[e]);
        }
      }
    }
  }
  T* o = static_cast<T*>(a.out.ptr) + b * a.out.stride_b + h * a.out.stride_h + t * a.out.stride_t + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f32<T>(l == 0.f ? 0.f : acc[e] / l);
  if (lane == 0 && a.lse) a.lse[row] = l == 0.f ? -CUDART_INF_F : m + logf(l);
}

int check(const AiPrefixAttnArgs* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->seq_len <= 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads != 0 || a->n_pages <= 0 || a->page_size <= 0 || a->max_pages < 0 ||
      a->prefix_len < 0)
    return AI_ERR_SHAPE;
  if (a->batch > 65535 || (int64_t)a->seq_len * a->num_q_heads > 0x7fffffff ||
      (int64_t)a->max_pages * a->page_size > 0x7fffffff)
    return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16 && a->dtype != AI_DTYPE_F32) return AI_ERR_DTYPE;
  for (const AiTensor4* t : {&a->q, &a->out, &a->k_pages, &a->v_pages}) {
    if (!t->ptr) return AI_ERR_NULL;
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < 0) return AI_ERR_STRIDE;
  }
  if (!a->lens || (a->max_pages > 0 && !a->page_table) || (a->prefix_len > 0 && !a->prefix_pages)) return AI_ERR_NULL;
  if (a->page_table_stride < 0) return AI_ERR_STRIDE;
  return AI_OK;
}

// The launch's shape and the workspace's layout; false when the sizes do not fit.
bool make_plan(const AiPrefixAttnArgs& a, Plan* p, size_t* bytes) {
  const int64_t G = a.num_q_heads / a.num_kv_heads, rows = G * a.seq_len, all = rows * a.batch, H = a.num_kv_heads;
  const int64_t capacity = (int64_t)a.max_pages * a.page_size;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t aim = (int64_t)kCtasPerSm * sms;
  p->group = (int)G;
  p->rows_seq = (int)rows;
  // As many chunks as there is room for, none shorter than kLeastChunk keys.
  auto cut = [&](int64_t keys, int64_t units, int& splits, int& chunk) {
    const int64_t most = (keys + kLeastChunk - 1) / kLeastChunk, room = units < aim ? aim / units : 1;
    const int64_t n = most < room ? most : room;
    const int64_t size = n > 0 ? ((keys + n - 1) / n + kKeys - 1) / kKeys * kKeys : kKeys;
    chunk = (int)(size < 0x7fffffff ? size : 0x7fffffff);
    splits = (int)((keys + chunk - 1) / chunk);
  };
  const int64_t groups_prefix = (all + kRows - 1) / kRows, groups_own = (rows + kRows - 1) / kRows;
  const int64_t units_prefix = groups_prefix * H, units_own = groups_own * H * a.batch;
  cut(a.prefix_len, units_prefix, p->splits_prefix, p->chunk_prefix);
  cut(capacity, units_own, p->splits_own, p->chunk_own);
  const int64_t items_prefix = units_prefix * p->splits_prefix, items = items_prefix + units_own * p->splits_own;
  if (all > 0x7fffffff || items > 0x7fffffff) return false;
  p->groups_prefix = (int)groups_prefix;
  p->groups_own = (int)groups_own;
  p->items_prefix = (int)items_prefix;
  p->items = (int)items;
  const int64_t es = a.dtype == AI_DTYPE_F32 ? 4 : 2;
  auto aligned = [&](const AiTensor4& t) {
    return ((reinterpret_cast<uintptr_t>(t.ptr) | (t.stride_b * es) | (t.stride_h * es) | (t.stride_t * es)) & 15) == 0;
  };
  p->vec_q = aligned(a.q);
  p->vec = aligned(a.k_pages) && aligned(a.v_pages);
  const size_t slots = (size_t)all * H * (p->splits_prefix + p->splits_own);
  const size_t o_bytes = (slots * a.head_dim * 4 + 255) & ~size_t(255);
  p->part_o = static_cast<float*>(a.workspace);
  p->part_lse = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + o_bytes);
  *bytes = o_bytes + ((slots * 4 + 255) & ~size_t(255));
  return true;
}

template <typename T, int D>
int rows_launch_d(const AiPrefixAttnArgs& a, const Plan& p, cudaStream_t st) {
  ProfScope ps(AI_PROF_PREFIX, st);
  if (p.items > 0) rows_kernel<T, D><<<p.items, kThreads, 0, st>>>(a, p);
  const int64_t rows = (int64_t)a.batch * a.num_q_heads * a.seq_len;
  join_kernel<T, D><<<(unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, st>>>(a, p);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int rows_launch(const AiPrefixAttnArgs& a, cudaStream_t st) {
  Plan p;
  size_t bytes;
  if (!make_plan(a, &p, &bytes)) return AI_ERR_SHAPE;
  if ((bytes > 0 && !a.workspace) || a.workspace_bytes < bytes) return AI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) & 255) return AI_ERR_ALIGN;
  if (a.head_dim == 128) return rows_launch_d<T, 128>(a, p, st);
  return a.head_dim == 64 ? rows_launch_d<T, 64>(a, p, st) : rows_launch_d<T, 32>(a, p, st);
}

}  // namespace prefix
}  // namespace ai

extern "C" int ai_prefix_attn_workspace(const AiPrefixAttnArgs* args, size_t* bytes) {
  const int rc = ai::prefix::check(args);
  if (rc != AI_OK) return rc;
  if (!bytes) return AI_ERR_NULL;
  if (ai::prefix::sm100_fits(*args)) {
    *bytes = ai::prefix::sm100_workspace(*args);
    return AI_OK;
  }
  ai::prefix::Plan p;
  return ai::prefix::make_plan(*args, &p, bytes) ? AI_OK : AI_ERR_SHAPE;
}

extern "C" int ai_prefix_attn(const AiPrefixAttnArgs* args, void* stream) {
  const int rc = ai::prefix::check(args);
  if (rc != AI_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (ai::prefix::sm100_fits(*args)) return ai::prefix::sm100_launch(*args, st);
  if (args->dtype == AI_DTYPE_BF16) return ai::prefix::rows_launch<__nv_bfloat16>(*args, st);
  if (args->dtype == AI_DTYPE_F16) return ai::prefix::rows_launch<__half>(*args, st);
  return ai::prefix::rows_launch<float>(*args, st);
}
