// Shared-prefix attention on the tensor cores: bf16 / fp16, head_dim 64 or
// 128, page sizes that are powers of two from 16.
//
// Work is key tiles of 64 keys.  A unit is 128 query rows of one KV head with
// one key list: either 128 of the B T G rows that share the prefix (G query
// heads per KV head), or the rows of one sequence with its own keys.  The
// tiles of all units stand in one line, the prefix's units first, and every
// CTA takes an equal stretch of it, whatever the lengths are (they are read on
// the device); a stretch crosses units, and the rows of a unit cut by a
// stretch's end leave partial results (O / l in fp32 and the log2-sum) that
// the combine launch joins with the other key list's.
//
// Per CTA (192 threads, two CTAs per SM, whose phases fill each other's
// gaps): four softmax warps (a thread per row), a TMA warp streaming K and V
// pages into a ring of tiles, an MMA warp.
//   S = Q K^T    tcgen05, M = 128 rows, N = 64 keys, two S buffers in TMEM
//   P = 2^(S - m) written over S as the 16-bit A operand of O += P V
//   O             fp32 in TMEM, rescaled only when a row's maximum grows by
//                 more than 2^8 (P then stays below 2^8 and sums in fp32)
// The MMA warp issues S of tile g + 1 before P V of tile g, so the scores of
// the next tile are ready when the softmax returns.
//
// Few rows per KV head: HBM-bound, each K / V byte is read once and most of
// the 128 rows are empty (their warps skip the softmax).  Many rows:
// tensor-bound, 4 D 128 64 FLOP per 32 KB (D = 128) tile pair.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_prefix_attn.h"
#include "sm100_ptx.cuh"
#include "sm100_tile.cuh"

namespace ai {
namespace prefix {
namespace tc {

constexpr int BM = 128, BN = 64;
constexpr int kThreads = 192;
constexpr int kMaxBatch = 2048;  // the tile scan of the sequences sits in shared memory
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t C_S = 0;    // two S buffers of 64 columns (P over their first 32)
constexpr uint32_t C_O = 128;  // D columns
constexpr long long kWait = 1000000000LL;

template <int D>
struct Smem {
  static constexpr uint32_t kTile = BN * D * 2;    // one K or V tile: D / 64 column blocks of 64 rows x 128 bytes
  static constexpr uint32_t kQBlock = BM * 128;    // one column block of Q
  static constexpr int kSlots = D == 128 ? 4 : 8;  // ring of tiles, K and V alternating (64 KB)
  static constexpr uint32_t Q = 0;
  static constexpr uint32_t RING = Q + BM * D * 2;
  static constexpr uint32_t BARS = RING + kSlots * kTile;
  static constexpr int FULL = 0, EMPTY = kSlots, S_FULL = 2 * kSlots, P_READY = S_FULL + 2, O_DONE = P_READY + 2,
                       Q_READY = O_DONE + 2, FINAL = Q_READY + 1, N_BARS = FINAL + 1;
  static constexpr uint32_t TMEM_SLOT = BARS + 8 * N_BARS;
  static constexpr uint32_t ABORT = TMEM_SLOT + 4;
  static constexpr uint32_t SCAN = ABORT + 4;  // int [B + 1]
  static size_t bytes(int batch) { return SCAN + 4 * ((size_t)batch + 1) + 1024; }
};
static_assert(2 * (Smem<128>::SCAN + 4 * (kMaxBatch + 1) + 1024 + 1024) <= 228 * 1024, "two CTAs per SM");

// What the host knows of the work.
struct Plan {
  int group;        // G: query heads per KV head
  int rows_seq;     // T G
  int rows_all;     // B T G
  int tiles_prefix; // key tiles of the prefix
  int rt, tt;       // row tiles of all rows / of one sequence
  int units_prefix; // Hkv rt (0 without a prefix)
  int part_rows;    // rows kept of a sequence's unit: min(128, T G)
  float* part_o;    // prefix slots [units_prefix + ctas][128][D], then own slots [B tt Hkv + ctas][part_rows][D]
  float* part_lse;  // the same rows
  int* scan;        // [B + 1] own tiles before each sequence
  int64_t own_base; // rows of the prefix slots
};

// A CTA's stretch within one unit.
struct Seg {
  int unit;        // prefix unit, or unit of the sequences (b tt + row tile) Hkv + hk
  int b;           // -1: the prefix
  int hk, row0, rows;
  int j0, n;       // key tiles [j0, j0 + n)
  int keys;        // keys of the list
};

__device__ __forceinline__ Seg locate(const AiPrefixAttnArgs& a, const Plan& p, const int* scan, int w, int w1) {
  Seg s;
  const int before = p.units_prefix * p.tiles_prefix;
  if (w < before) {
    s.unit = w / p.tiles_prefix;
    s.b = -1;
    s.hk = s.unit / p.rt;
    s.row0 = (s.unit % p.rt) * BM;
    s.rows = min(BM, p.rows_all - s.row0);
    s.j0 = w % p.tiles_prefix;
    s.n = min(p.tiles_prefix - s.j0, w1 - w);
    s.keys = a.prefix_len;
    return s;
  }
  const int per = p.tt * a.num_kv_heads, x = w - before;
  int lo = 0, hi = a.batch - 1;  // the last sequence with scan * per <= x that has tiles
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (scan[mid] * per <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int tiles = scan[lo + 1] - scan[lo], rem = x - scan[lo] * per, v = rem / tiles;
  s.b = lo;
  s.unit = lo * per + v;
  s.hk = v % a.num_kv_heads;
  s.row0 = (v / a.num_kv_heads) * BM;
  s.rows = min(BM, p.rows_seq - s.row0);
  s.j0 = rem % tiles;
  s.n = min(tiles - s.j0, w1 - w);
  s.keys = seq_lens(a, lo).keys;
  return s;
}

// First tile of CTA `cta` of the `ctas` that have work (at most one per tile,
// so that no stretch is empty).
__device__ __forceinline__ int stretch(int64_t total, int cta, int ctas) { return (int)(total * cta / ctas); }

// The CTA whose stretch holds tile w.
__device__ __forceinline__ int cta_of(int64_t w, int64_t total, int ctas) { return (int)(((w + 1) * ctas - 1) / total); }

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Pair<__half> {
  static constexpr uint32_t kFmt = 0;
  __device__ static uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// kind::f16 instruction descriptor with fp32 accumulation (fields as in sm100_ptx.cuh).
__host__ __device__ constexpr uint32_t idesc(uint32_t fmt, int M, int N, bool b_mn) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    split_kernel(const AiPrefixAttnArgs a, const Plan p, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const bool q_vec) {
  using L = Smem<D>;
  constexpr int CB = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = tile::align1024(smem_raw);
  const uint32_t sbase = ptx::smem_u32(sm);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  volatile int* s_abort = reinterpret_cast<volatile int*>(sm + L::ABORT);
  int* scan = reinterpret_cast<int*>(sm + L::SCAN);
  auto bar = [&](int i) { return sbase + L::BARS + 8u * (uint32_t)i; };

  if (tid == 0) {
    for (int i = 0; i < L::N_BARS; ++i) {
      const bool wide = i == L::P_READY || i == L::P_READY + 1 || i == L::Q_READY;
      ptx::mbar_init(bar(i), wide ? 128 : 1);
    }
    *s_abort = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 5) {
    ptx::tmem_alloc(sbase + L::TMEM_SLOT, kTmemCols);
    ptx::tmem_relinquish();
  }
  // Own key tiles before each sequence (warp 0, 32 sequences at a time).
  if (warp == 0) {
    int base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      int v = b < a.batch ? (seq_lens(a, b).keys + BN - 1) / BN : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b < a.batch) scan[b + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) scan[0] = 0;
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + L::TMEM_SLOT);
  const int64_t total = (int64_t)p.units_prefix * p.tiles_prefix + (int64_t)scan[a.batch] * p.tt * a.num_kv_heads;
  const int ctas = (int)min((int64_t)gridDim.x, total);
  const bool busy = (int)blockIdx.x < ctas;
  const int w0 = busy ? stretch(total, blockIdx.x, ctas) : 0, w1 = busy ? stretch(total, blockIdx.x + 1, ctas) : 0;
  if (blockIdx.x == 0)
    for (int b = tid; b <= a.batch; b += kThreads) p.scan[b] = scan[b];

  // Bounded wait of a whole warp: true in every lane or false in every lane
  // (a warp leaves its loops together).
  auto wait = [&](int i, uint32_t parity) -> bool {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar(i), parity))) return true;
    bool ok = !*s_abort;
    if (ok && !ptx::mbar_wait(bar(i), parity, kWait)) {
      report(a.status, AI_ERR_DEV_TIMEOUT);
      *s_abort = 1;
      ok = false;
    }
    return __all_sync(0xffffffffu, ok);
  };

  if (warp < 4) {
    // ------------------------------------------------------------ softmax
    const int r = tid;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const float sl2 = a.scale * kLog2e;
    int g = 0;
    bool ok = true;
    for (int w = w0; w < w1 && ok;) {
      const Seg s = locate(a, p, scan, w, w1);
      w += s.n;
      // Q rows (the last S of the segment before has been waited for, so no
      // MMA reads Q any more): 16-byte chunks, neighbouring threads along a row.
      for (int x = tid; x < BM * (D / 8); x += 128) {
        const int row = x / (D / 8), c = x % (D / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < s.rows) {
          const int all = s.row0 + row, b = s.b < 0 ? all / p.rows_seq : s.b;
          const int rem = s.b < 0 ? all % p.rows_seq : all, t = rem / p.group, h = s.hk * p.group + rem % p.group;
          const T* q = static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + h * a.q.stride_h + t * a.q.stride_t + 8 * c;
          if (q_vec) {
            v = __ldg(reinterpret_cast<const uint4*>(q));
          } else {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = q[i];
            memcpy(&v, e, 16);
          }
        }
        *reinterpret_cast<uint4*>(sm + L::Q + tile::chunk_off<BM>(row, c)) = v;
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar(L::Q_READY));
      // The row's visible keys of this list.  Rows without a query are not
      // masked and not stored (their TMEM lanes reach no other row).
      int limit = 0x7fffffff;
      bool valid = false;
      if (r < s.rows) {
        const int all = s.row0 + r, b = s.b < 0 ? all / p.rows_seq : s.b;
        const int t = (s.b < 0 ? all % p.rows_seq : all) / p.group;
        const Lens len = seq_lens(a, b);
        valid = t < len.n;
        if (valid) limit = s.b < 0 ? s.keys : max(0, s.keys - len.n + t + 1);
      }
      const bool active = __any_sync(0xffffffffu, valid);
      int least = limit;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));

      float m = -CUDART_INF_F, l = 0.f;
      for (int j = 0; j < s.n; ++j, ++g) {
        const int k0 = (s.j0 + j) * BN, x = g & 1;
        const uint32_t c_s = tmem + lane_base + C_S + 64u * (uint32_t)x;
        if (!(ok = wait(L::S_FULL + x, (g >> 1) & 1))) break;
        ptx::tc_fence_after();
        if (active) {
          uint32_t s0[32], s1[32];
          ptx::tmem_ld32(c_s, s0);
          ptx::tmem_ld32(c_s + 32, s1);
          ptx::tmem_wait_ld();
          if (k0 + BN > least) {
            const int lim = limit - k0;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (i >= lim) s0[i] = 0xff800000u;  // -inf
              if (i + 32 >= lim) s1[i] = 0xff800000u;
            }
          }
          float ma = -CUDART_INF_F, mb = -CUDART_INF_F;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            ma = ptx::fmax3(ma, __uint_as_float(s0[i]), __uint_as_float(s0[i + 1]));
            mb = ptx::fmax3(mb, __uint_as_float(s1[i]), __uint_as_float(s1[i + 1]));
          }
          const float m_new = fmaxf(m, fmaxf(ma, mb) * sl2);
          float alpha = 1.f;
          bool rescale = false;
          if (m_new > m + 8.f) {
            if (l > 0.f) {
              alpha = ptx::ex2(m - m_new);
              rescale = true;
            }
            m = m_new;
          }
          if (__any_sync(0xffffffffu, rescale)) {
            // O holds the tiles before this one once their last P V is done.
            if (!(ok = wait(L::O_DONE + (x ^ 1), ((g - 1) >> 1) & 1))) break;
            ptx::tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              ptx::tmem_ld16(tmem + lane_base + C_O + 16 * c, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              ptx::tmem_st16(tmem + lane_base + C_O + 16 * c, o);
            }
            l *= alpha;
          }
          const float base = m == -CUDART_INF_F ? 0.f : m;
          const float2 nm = make_float2(-base, -base), sc = make_float2(sl2, sl2);
          float2 suma = make_float2(0.f, 0.f), sumb = make_float2(0.f, 0.f);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 e = __ffma2_rn(make_float2(__uint_as_float(s0[2 * i]), __uint_as_float(s0[2 * i + 1])), sc, nm);
            const float2 pr = make_float2(ptx::ex2(e.x), ptx::ex2(e.y));
            suma = __fadd2_rn(suma, pr);
            pk[i] = Pair<T>::pack(pr.x, pr.y);
          }
          ptx::tmem_st16(c_s, pk);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 e = __ffma2_rn(make_float2(__uint_as_float(s1[2 * i]), __uint_as_float(s1[2 * i + 1])), sc, nm);
            const float2 pr = make_float2(ptx::ex2(e.x), ptx::ex2(e.y));
            sumb = __fadd2_rn(sumb, pr);
            pk[i] = Pair<T>::pack(pr.x, pr.y);
          }
          ptx::tmem_st16(c_s + 16, pk);
          l += (suma.x + suma.y) + (sumb.x + sumb.y);
          ptx::tmem_wait_st();
        }
        ptx::tc_fence_before();
        if (k0 + BN > s.keys) {
          // Slots past the list hold anything, NaN included, and meet P = 0:
          // clear their V rows.
          const int item = 2 * g + 1;
          if (!(ok = wait(L::FULL + item % L::kSlots, (item / L::kSlots) & 1))) break;
          uint8_t* v = sm + L::RING + (item % L::kSlots) * L::kTile;
          const int first = s.keys - k0;
          for (int i = tid; i < (BN - first) * CB * 8; i += 128) {
            const int row = first + i / (CB * 8), c = i % (CB * 8);
            *reinterpret_cast<uint4*>(v + (c / 8) * (BN * 128) + row * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          ptx::fence_proxy_async_smem();
        }
        ptx::mbar_arrive(bar(L::P_READY + x));
      }
      if (!ok) break;
      // The rows' partial results.
      if (!(ok = wait(L::O_DONE + ((g - 1) & 1), ((g - 1) >> 1) & 1))) break;
      ptx::tc_fence_after();
      if (active) {
        const int64_t row = s.b < 0 ? (int64_t)(s.unit + (int)blockIdx.x) * BM + r
                                    : p.own_base + (int64_t)(s.unit + (int)blockIdx.x) * p.part_rows + r;
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          ptx::tmem_ld32(tmem + lane_base + C_O + 32 * c, o);
          ptx::tmem_wait_ld();
          if (valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t v8[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v8[e] = l > 0.f ? __float_as_uint(__uint_as_float(o[i + e]) * inv) : 0u;
              ptx::st_global_v8(p.part_o + row * D + 32 * c + i, v8);
            }
          }
        }
        if (valid) p.part_lse[row] = l > 0.f ? m + log2f(l) : -CUDART_INF_F;
      }
      ptx::tc_fence_before();
    }
  } else if (warp == 4) {
    // ------------------------------------------------------------ TMA
    if (lane == 0) {
      ptx::prefetch_tmap(&tm_k);
      ptx::prefetch_tmap(&tm_v);
    }
    const int box = min(a.page_size, BN);  // keys per load
    const int piece = lane / CB, cb = lane % CB;
    int item = 0;
    bool ok = true;
    for (int w = w0; w < w1 && ok;) {
      const Seg s = locate(a, p, scan, w, w1);
      w += s.n;
      const int32_t* table = s.b < 0 ? a.prefix_pages : a.page_table + s.b * a.page_table_stride;
      for (int j = 0; j < s.n && ok; ++j) {
        const int k0 = (s.j0 + j) * BN;
        const int pieces = (min(BN, s.keys - k0) + box - 1) / box;  // pages past the list are not read
        const bool mine = piece < pieces;
        const int key = k0 + piece * box;
        const int page = mine ? page_of(a, table, key / a.page_size) : 0, at = key % a.page_size;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++item) {
          const int slot = item % L::kSlots;
          if (item >= L::kSlots) {
            if (!(ok = wait(L::EMPTY + slot, (item / L::kSlots - 1) & 1))) break;
          }
          if (lane == 0) ptx::mbar_arrive_expect_tx(bar(L::FULL + slot), (uint32_t)(pieces * box * 128 * CB));
          __syncwarp();
          if (mine)
            ptx::tma_load_4d(sbase + L::RING + slot * L::kTile + cb * (BN * 128) + piece * box * 128,
                             kv ? &tm_v : &tm_k, bar(L::FULL + slot), 64 * cb, at, s.hk, page);
        }
      }
    }
    // After a wait that gave up: the loads in flight land before the CTA ends.
    if (!ok || *s_abort)
      for (int i = max(0, item - L::kSlots); i < item; ++i)
        ptx::mbar_wait(bar(L::FULL + i % L::kSlots), (i / L::kSlots) & 1, kWait);
  } else {
    // ------------------------------------------------------------ MMA
    constexpr uint32_t i_qk = idesc(Pair<T>::kFmt, BM, BN, false), i_pv = idesc(Pair<T>::kFmt, BM, D, true);
    const uint64_t d_q = ptx::sdesc_sw128(sbase + L::Q, 16, 1024);
    const uint64_t d_k = ptx::sdesc_sw128(sbase + L::RING, 16, 1024);
    const uint64_t d_v = ptx::sdesc_sw128(sbase + L::RING, BN * 128, 1024);
    constexpr uint64_t kT = L::kTile >> 4;
    auto issue_s = [&](int g) -> bool {
      const int item = 2 * g, slot = item % L::kSlots;
      if (!wait(L::FULL + slot, (item / L::kSlots) & 1)) return false;
      ptx::tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        ptx::mma_ss_w(tmem + C_S + 64u * (uint32_t)(g & 1),
                      d_q + (uint64_t)(((kk >> 2) * L::kQBlock + (kk & 3) * 32) >> 4),
                      d_k + kT * (uint64_t)slot + (uint64_t)(((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4), i_qk, kk > 0);
      ptx::mma_commit_w(bar(L::S_FULL + (g & 1)));
      ptx::mma_commit_w(bar(L::EMPTY + slot));
      return true;
    };
    int g = 0, seg = 0;
    bool ok = true;
    for (int w = w0; w < w1 && ok; ++seg) {
      const Seg s = locate(a, p, scan, w, w1);
      w += s.n;
      if (!wait(L::Q_READY, seg & 1)) break;
      ptx::tc_fence_after();
      ok = issue_s(g) && (s.n < 2 || issue_s(g + 1));
      for (int j = 0; j < s.n && ok; ++j) {
        const int gj = g + j, item = 2 * gj + 1, slot = item % L::kSlots;
        ok = wait(L::P_READY + (gj & 1), (gj >> 1) & 1) && wait(L::FULL + slot, (item / L::kSlots) & 1);
        if (!ok) break;
        ptx::tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          ptx::mma_ts_w(tmem + C_O, tmem + C_S + 64u * (uint32_t)(gj & 1) + 8u * (uint32_t)kk,
                        d_v + kT * (uint64_t)slot + (uint64_t)((kk * 2048) >> 4), i_pv, (j > 0 || kk > 0) ? 1u : 0u);
        ptx::mma_commit_w(bar(L::O_DONE + (gj & 1)));
        ptx::mma_commit_w(bar(L::EMPTY + slot));
        if (j + 2 < s.n) ok = issue_s(gj + 2);
      }
      g += s.n;
    }
    // Every MMA issued has completed before TMEM is released.
    ptx::mma_commit_w(bar(L::FINAL));
    ptx::mbar_wait(bar(L::FINAL), 0, kWait);
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
}

// A warp per (sequence, query token, query head): joins the partial results
// of the row's prefix and own stretches, in stretch order.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(const AiPrefixAttnArgs a, const Plan p, const int grid) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int E = D / 32;
  const int b = blockIdx.y, lane = threadIdx.x % 32, item = blockIdx.x * 8 + threadIdx.x / 32;
  if (item >= a.seq_len * a.num_q_heads) return;
  const int t = item / a.num_q_heads, h = item % a.num_q_heads, hk = h / p.group;
  const int rem = t * p.group + h % p.group;
  float M = -CUDART_INF_F, sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (t < seq_lens(a, b).n) {
    const int64_t before = (int64_t)p.units_prefix * p.tiles_prefix;
    const int per = p.tt * a.num_kv_heads, s0 = p.scan[b], tiles = p.scan[b + 1] - s0;
    const int64_t total = before + (int64_t)p.scan[a.batch] * per;
    const int ctas = (int)min((int64_t)grid, total);
    const int all = b * p.rows_seq + rem, up = hk * p.rt + all / BM;
    const int own = (rem / BM) * a.num_kv_heads + hk;
    int64_t row[2] = {0, 0}, step[2] = {BM, p.part_rows};
    int n[2] = {0, 0};
    if (p.units_prefix > 0) {
      const int64_t w = (int64_t)up * p.tiles_prefix;
      const int c = cta_of(w, total, ctas);
      n[0] = cta_of(w + p.tiles_prefix - 1, total, ctas) - c + 1;
      row[0] = (int64_t)(up + c) * BM + all % BM;
    }
    if (tiles > 0) {
      const int64_t w = before + (int64_t)s0 * per + (int64_t)own * tiles;
      const int c = cta_of(w, total, ctas);
      n[1] = cta_of(w + tiles - 1, total, ctas) - c + 1;
      row[1] = p.own_base + (int64_t)(b * per + own + c) * p.part_rows + rem % BM;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      for (int i = 0; i < n[k]; ++i) M = fmaxf(M, p.part_lse[row[k] + i * step[k]]);
    if (M != -CUDART_INF_F) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll 4
        for (int i = 0; i < n[k]; ++i) {
          const int64_t rr = row[k] + i * step[k];
          const float wgt = exp2f(p.part_lse[rr] - M);
          float o[E];
          if constexpr (E == 4)
            *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(p.part_o + rr * D + E * lane);
          else
            *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(p.part_o + rr * D + E * lane);
          sum += wgt;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(wgt, o[e], acc[e]);
        }
    }
  }
  T* o = static_cast<T*>(a.out.ptr) + b * a.out.stride_b + h * a.out.stride_h + t * a.out.stride_t + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f32<T>(sum > 0.f ? acc[e] / sum : 0.f);
  if (lane == 0 && a.lse)
    a.lse[((int64_t)b * a.num_q_heads + h) * a.seq_len + t] =
        sum > 0.f ? (M + log2f(sum)) * kLn2 : -CUDART_INF_F;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// The launch's shape and the workspace's layout; false when the sizes do not fit.
bool make_plan(const AiPrefixAttnArgs& a, Plan* p, int* ctas, size_t* bytes) {
  const int64_t G = a.num_q_heads / a.num_kv_heads, rows = G * a.seq_len, all = rows * a.batch;
  const int64_t tiles = ((int64_t)a.prefix_len + BN - 1) / BN, rt = (all + BM - 1) / BM, tt = (rows + BM - 1) / BM;
  const int64_t most_own = ((int64_t)a.max_pages * a.page_size + BN - 1) / BN;
  const int64_t units = tiles > 0 ? rt * a.num_kv_heads : 0, units_own = a.batch * tt * a.num_kv_heads;
  const int64_t most = units * tiles + units_own * most_own;
  if (all > 0x7fffffff || most > 0x7fffffff || units_own > 0x7fffffff) return false;
  const int64_t slots = 2 * (int64_t)sm_count();
  *ctas = (int)(most < 1 ? 1 : most < slots ? most : slots);
  p->group = (int)G;
  p->rows_seq = (int)rows;
  p->rows_all = (int)all;
  p->tiles_prefix = (int)tiles;
  p->rt = (int)rt;
  p->tt = (int)tt;
  p->units_prefix = (int)units;
  p->part_rows = (int)(rows < BM ? rows : BM);
  p->own_base = units > 0 ? (units + *ctas) * BM : 0;
  const int64_t n = p->own_base + (units_own + *ctas) * p->part_rows;
  char* ws = static_cast<char*>(a.workspace);
  size_t at = 0;
  auto take = [&](size_t want) {
    char* q = ws + at;
    at += (want + 255) & ~size_t(255);
    return q;
  };
  p->part_o = reinterpret_cast<float*>(take((size_t)n * a.head_dim * 4));
  p->part_lse = reinterpret_cast<float*>(take((size_t)n * 4));
  p->scan = reinterpret_cast<int*>(take(((size_t)a.batch + 1) * 4));
  *bytes = at;
  return true;
}

template <typename T, int D>
int launch_t(const AiPrefixAttnArgs& a, const Plan& p, int ctas, const CUtensorMap& tk, const CUtensorMap& tv,
             cudaStream_t st) {
  const size_t smem = Smem<D>::bytes(a.batch);
  if (cudaFuncSetAttribute(split_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return AI_ERR_LAUNCH;
  const bool q_vec = (reinterpret_cast<uintptr_t>(a.q.ptr) & 15) == 0 &&
                     ((a.q.stride_b | a.q.stride_h | a.q.stride_t) & 7) == 0;
  ProfScope ps(AI_PROF_PREFIX, st);
  split_kernel<T, D><<<ctas, kThreads, smem, st>>>(a, p, tk, tv, q_vec);
  if (cudaGetLastError() != cudaSuccess) return AI_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.seq_len * a.num_q_heads + 7) / 8), a.batch);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  if (cudaLaunchKernelEx(&cfg, combine_kernel<T, D>, a, p, ctas) != cudaSuccess) return AI_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace tc

bool sm100_fits(const AiPrefixAttnArgs& a) {
  if (a.dtype != AI_DTYPE_BF16 && a.dtype != AI_DTYPE_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  if (a.page_size < 16 || (a.page_size & (a.page_size - 1)) || a.batch > tc::kMaxBatch) return false;
  if (!(a.scale > 0.f)) return false;  // the row maximum is taken before the scale
  for (const AiTensor4* t : {&a.k_pages, &a.v_pages}) {
    // what a tensor map asks for
    if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) || ((t->stride_b | t->stride_h | t->stride_t) & 7)) return false;
    if (t->stride_b <= 0 || t->stride_h <= 0 || t->stride_t <= 0) return false;
  }
  tc::Plan p;
  int ctas;
  size_t bytes;
  return tc::make_plan(a, &p, &ctas, &bytes);
}

size_t sm100_workspace(const AiPrefixAttnArgs& a) {
  tc::Plan p;
  int ctas;
  size_t bytes = 0;
  tc::make_plan(a, &p, &ctas, &bytes);
  return bytes;
}

int sm100_launch(const AiPrefixAttnArgs& a, cudaStream_t st) {
  tc::Plan p;
  int ctas;
  size_t bytes;
  if (!tc::make_plan(a, &p, &ctas, &bytes)) return AI_ERR_SHAPE;
  if (!a.workspace || a.workspace_bytes < bytes) return AI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) & 255) return AI_ERR_ALIGN;
  const int box = a.page_size < tc::BN ? a.page_size : tc::BN;
  CUtensorMap tk, tv;
  if (!sm100_make_map_of(&tk, a.k_pages, a.n_pages, a.num_kv_heads, a.page_size, box, a.head_dim, a.dtype) ||
      !sm100_make_map_of(&tv, a.v_pages, a.n_pages, a.num_kv_heads, a.page_size, box, a.head_dim, a.dtype))
    return AI_ERR_TMA;
  if (a.dtype == AI_DTYPE_BF16)
    return a.head_dim == 128 ? tc::launch_t<__nv_bfloat16, 128>(a, p, ctas, tk, tv, st)
                             : tc::launch_t<__nv_bfloat16, 64>(a, p, ctas, tk, tv, st);
  return a.head_dim == 128 ? tc::launch_t<__half, 128>(a, p, ctas, tk, tv, st)
                           : tc::launch_t<__half, 64>(a, p, ctas, tk, tv, st);
}

}  // namespace prefix
}  // namespace ai
