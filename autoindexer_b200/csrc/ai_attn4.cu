// Attention over the paged cache in 4 bits (declared in include/ai_attn.h; the
// format at AiPool4).
//
// A unit is a (sequence, KV head, group of up to 24 query rows); its keys are
// cut into tiles of 32, the tiles of all units stand in one line, and each worker,
// a warp, takes an equal stretch of the line, whatever the lengths are (they
// are read on the device).  The rows of a unit that a worker touched leave
// partial results (O / l in fp32 and the log2-sum), which a second launch joins.
//
// A warp's tile, on 16 x 8 x 16 fp16 matrix instructions with fp32 sums:
//   S^T = K Q^T   the sums of a group of 32 dims, less 8 sum(q), meet the group's
//                 scale in fp32;
//   O^T += V^T P  P takes each key's V scale, per group of 32 dims: weights, held 2^7
//                 above 1 at the running maximum, times scales, divided by a power of two
//                 of the group's own (two to four times the largest |scale| met so far), in
//                 fp32 and rounded to fp16 once.  A product of 2^-19 of the largest weight's
//                 with the group's largest scale begins to lose digits, one of 2^-30 does
//                 not count.  (Scales divided, and bf16 queries' weights rounded, in fp16
//                 before that: 73 us for 76 on the first case below, but scales of 2^-14 of
//                 the group's largest lose digits whatever their weight.)
// The codes are fp16's subnormal numbers as they lie, 2^-24 c: one logical operation
// a pair.  (Their 8 comes off K's as the sums start, off V's before the product.)
// Both products have the tile's keys on the instruction's long side, so up to 8
// query rows of a KV head cost one column block.
//
// HBM-bound when few rows meet each key: 144 bytes per token and KV head at D 128.
// Measured (32 query heads, 8 KV heads of 128): 64 sequences of up to 8192 tokens, one
// query token each, 76 us (4.0 TB/s); 32 of up to 32,768 130 us (4.5 TB/s).  Neither the
// memory nor the issue slots are full (706 instructions a tile of 32 keys, issued in 67%
// of the cycles): what is left are the waits within a warp's tile, scores, maximum, weights
// and sums one after the other, which the 16 warps that the registers allow do not hide
// from one another.  With up to five query tokens (20 rows to a KV head, three column
// blocks) 153 us: eight warps an SM, as their sums take 255 registers, and 1070
// instructions a tile, issued in 46%.  4 sequences of 322 tokens 13.5 us: one tile's
// latency, a launch, and the second one's joining.

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cfloat>
#include <cstring>

#include "ai_common.cuh"
#include "ai_kernels.h"
#include "ai_kv4.cuh"
#include "sm100_ptx.cuh"

namespace ai {
namespace attn4 {

using namespace kv4;

constexpr int kMaxBatch = 1024;  // a scan of the sequences sits in shared memory
constexpr int kKeys = 32;      // keys of a tile
constexpr int kStart = 4;      // what starting a unit costs, in tiles
constexpr int kLeast = 4;      // positions a worker takes, at least
constexpr int kMaxBlocks = 3;  // column blocks (of 8 query rows) of a unit, at most (four do not fit the registers)
constexpr float kLift = 7.f;   // a weight of 1 is held as 2^7
constexpr float kSlack = 8.f;  // the running maximum moves when a score passes it by 2^8
constexpr int kLeastExp = -14;  // V scales below 2^-14 are divided by no less
// Before the first score: below any (of a row scaled to fp16's top, 2^-9 a dim and
// step of a code, with |scale| <= 2^16: 2^17 at most), near enough for a difference.
constexpr float kNoRef = -0x1p20f;

// Warps of a CTA (one per SM), by column blocks.
__host__ __device__ constexpr int warps_of(int blocks) { return blocks == 1 ? 16 : 8; }
constexpr int kStages = 2;     // tiles of a warp's ring: one is loaded while one is multiplied

// A tile in shared memory: codes of K and V, scales of K and V, as they lie in
// the pools.  Row i of a product's 16 keys is key place(i): the rows that a
// quarter of a warp reads together are then neighbours (K's even and odd ones,
// V's four of a pair's first or second key).
template <int D>
struct Tile {
  static constexpr int C = D / kGroup, kRow = D / 2, kCodes = kKeys * kRow, kScales = kKeys * C * 2;
  static constexpr int K = 0, V = kCodes, KS = 2 * kCodes, VS = KS + kScales, kBytes = VS + kScales;
  __device__ static int place(int i) { return (i & 8) | (i & 1 ? 4 + (i >> 1 & 3 ^ 1) : i >> 1 & 3); }
};

// A CTA's shared memory: rings, the query fragments of its warps with the
// groups' offsets, the sequences' places on the line and lengths.
template <int D, int NT>
struct Smem {
  static constexpr int W = warps_of(NT), C = D / kGroup;
  static constexpr int kQ = NT * C * 512, kOff = NT * C * 512;
  static constexpr int RING = 0, Q = W * kStages * Tile<D>::kBytes, OFF = Q + W * kQ, SCAN = OFF + W * kOff;
  static constexpr size_t bytes(int batch) { return SCAN + (3 * (size_t)batch + 1) * sizeof(int); }
};
static_assert(Smem<128, 1>::bytes(kMaxBatch) <= 227 * 1024 && Smem<128, 2>::bytes(kMaxBatch) <= 227 * 1024 &&
                  Smem<128, 3>::bytes(kMaxBatch) <= 227 * 1024,
              "a CTA's shared memory");

struct Plan {
  int group;       // G: query heads per KV head
  int rows;        // T G
  int groups;      // groups of query rows per (sequence, KV head)
  int unit_rows;   // rows of a unit (the last group may have fewer)
  int blocks;      // column blocks of a unit
  int workers;
  float* part_o;   // [units + workers][unit_rows][D]
  float* part_lse;
};

struct Lens {
  int keys, n;
};

// Keys of a sequence (clamped to what its page table can hold) and its real
// query tokens.
__device__ __forceinline__ Lens seq_lens(const AiPagedAttn4Args& a, int64_t b) {
  Lens r;
  r.keys = __ldg(a.lens + b);
  r.n = new_tokens(a.query_lens, b, a.seq_len, a.status);
  const int64_t most = min((int64_t)a.pool.max_pages * a.pool.page_size, (int64_t)0x7fffffff);
  if (r.keys < 0 || r.keys > most) report(a.status, AI_ERR_DEV_BOUNDS);
  r.keys = max(0, (int)min((int64_t)r.keys, most));
  return r;
}

// Positions of a sequence's unit: its tiles behind `kStart` idle positions; none
// without a key or a query.
__device__ __forceinline__ int unit_size(const Lens& l) { return l.keys > 0 && l.n > 0 ? kStart + (l.keys - 1) / kKeys + 1 : 0; }

// The line's stretches: n workers, none less than kLeast positions unless the
// line is shorter; the first `more` take one position more.
struct Split {
  int n, len, more;
  __device__ __forceinline__ int begin(int w) const { return w * len + min(w, more); }
  __device__ __forceinline__ int worker(int x) const {
    const int head = more * (len + 1);
    return x < head ? x / (len + 1) : more + (x - head) / len;
  }
};

__device__ __forceinline__ Split split_line(int workers, int total) {
  Split s{0, 1, 0};
  if (total > 0) {
    s.n = min(workers, (total + kLeast - 1) / kLeast);
    s.len = total / s.n;
    s.more = total - s.len * s.n;
  }
  return s;
}

// A worker's stretch within one unit: tiles [tile, end) of it.
struct Seg {
  int unit, b, hk, grp;
  int tile, end;
  int keys, n;
};

// The next stretch with tiles from position w on; false: there is none.  `scan`
// is followed by the sequences' keys and query tokens.
__device__ __forceinline__ bool next_seg(const AiPagedAttn4Args& a, const Plan& p, const int* scan, int& w, int w1, Seg& s) {
  const int per = a.num_kv_heads * p.groups;
  while (w < w1) {
    int lo = 0, hi = a.batch - 1;  // the last sequence that starts by w (it has positions)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (scan[mid] * per <= w)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int size = scan[lo + 1] - scan[lo], rem = w - scan[lo] * per, sub = rem / size, at = rem - sub * size;
    const int end = min(size, at + (w1 - w));
    w += end - at;
    s.tile = max(0, at - kStart);
    s.end = end - kStart;
    if (s.tile >= s.end) continue;
    s.b = lo;
    s.hk = sub / p.groups;
    s.grp = sub - s.hk * p.groups;
    s.unit = lo * per + sub;
    s.keys = scan[a.batch + 1 + lo];
    s.n = scan[2 * a.batch + 1 + lo];
    return true;
  }
  return false;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                    float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}

// An 8 x 8 matrix of 16-bit elements, a row of pairs per four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Lower (or upper) halves of two words, side by side.
__device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b, bool upper) { return __byte_perm(a, b, upper ? 0x7632 : 0x5410); }

// Words of a lane's codes by N bytes from shared memory.
template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[(N + 3) / 4], const uint8_t* p) {
  if constexpr (N == 16) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
  } else if constexpr (N == 8) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    w[0] = r.x, w[1] = r.y;
  } else if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
}

// Four pairs of codes (at bits 4 j and 16 + 4 j of x) as fp16's subnormal numbers
// 2^-24 c and, for odd j, 2^-20 c: the bits as they lie.
__device__ __forceinline__ void numbers(uint32_t x, uint32_t (&f)[4]) {
  const uint32_t y = x >> 8;
  f[0] = x & 0x000f000fu;
  f[1] = x & 0x00f000f0u;
  f[2] = y & 0x000f000fu;
  f[3] = y & 0x00f000f0u;
}
// Less 8 in either measure, exactly.  (A second product with a constant -8, and the
// sums' rounding of it, costs more: 85 us for 82 on 64 sequences of up to 8192 tokens.)
__device__ __forceinline__ uint32_t less8(uint32_t x, uint32_t off) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight elements of a query row, any strides of the rows; and one of them.
template <typename T>
__device__ __forceinline__ uint4 load_q(const T* p) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) return __ldg(reinterpret_cast<const uint4*>(p));
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = p[i];
  uint4 r;
  memcpy(&r, e, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ float element(const uint4& r, int i) {
  const uint32_t w = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
  const uint16_t h = (uint16_t)(i % 2 ? w >> 16 : w);
  T x;
  memcpy(&x, &h, 2);
  return to_f32(x);
}

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
// A half in both halves.
__device__ __forceinline__ uint32_t twice(uint32_t h) { return h | h << 16; }
__device__ __forceinline__ float half_of(uint32_t w, int i) {
  return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w)));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * warps_of(NT), 1) split_kernel(const AiPagedAttn4Args a, const Plan p) {
  using L = Tile<D>;
  using M = Smem<D, NT>;
  constexpr int C = L::C, H = (C + 1) / 2, S = kStages;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t smem[];
  int* scan = reinterpret_cast<int*>(smem + M::SCAN);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  if (warp == 0) {
    int base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      int v = 0;
      if (b < a.batch) {
        const Lens l = seq_lens(a, b);
        v = unit_size(l);
        scan[a.batch + 1 + b] = l.keys;
        scan[2 * a.batch + 1 + b] = l.n;
      }
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
  __syncthreads();
  const Split line = split_line(p.workers, scan[a.batch] * a.num_kv_heads * p.groups);
  const int worker = warp * gridDim.x + blockIdx.x;  // (few workers: on as many SMs)
  if (worker >= line.n) return;
  const int w0 = line.begin(worker), w1 = line.begin(worker + 1);
  const uint8_t* ring = smem + warp * S * L::kBytes;
  const uint32_t ring_at = ptx::smem_u32(ring);

  // ---- loads, S - 1 tiles ahead of the products: a half of a tile, 16 keys, lies
  // in one page, its pieces in one stretch each.  (Bulk copies of the pieces, eight
  // a tile, take more instructions: they are issued one by one.)
  const int page_bits = 31 - __clz(a.pool.page_size), page_mask = a.pool.page_size - 1;
  constexpr int kHalfCodes = 16 * L::kRow, kHalfScales = 16 * 2 * C, kPer = kHalfScales / 16;
  const int s_half = lane / kPer & 1;               // of the scales this lane copies, if any
  const bool s_has = lane < 4 * kPer, s_v = lane >= 2 * kPer;
  const AiTensor4 &kc = a.pool.k_codes, &vc = a.pool.v_codes;
  const uint32_t s_step = (uint32_t)((s_v ? a.pool.v_scales.stride_b : a.pool.k_scales.stride_b) >> 3);  // (16-byte units)
  const uint32_t k_step = (uint32_t)(kc.stride_b >> 4), v_step = (uint32_t)(vc.stride_b >> 4);
  const int s_at = (s_v ? L::VS : L::KS) + s_half * kHalfScales + lane % kPer * 16;
  Seg ld;
  int wl = w0, at_stage = 0, page[2] = {0, 0};
  const uint8_t *k_from = nullptr, *v_from = nullptr, *s_from = nullptr;  // the head's, in page 0
  auto look_up = [&]() {  // pages of the tile's halves
    const int key = ld.tile * kKeys;
    const int32_t* table = a.pool.page_table + ld.b * a.pool.page_table_stride + (key >> page_bits);
    page[0] = __ldg(table);
    page[1] = page[0];
    if (page_bits == 4) page[1] = ld.keys - key > 16 ? __ldg(table + 1) : 0;
  };
  auto enter = [&]() -> bool {  // the next stretch to load
    if (!next_seg(a, p, scan, wl, w1, ld)) return false;
    k_from = static_cast<const uint8_t*>(kc.ptr) + ld.hk * kc.stride_h + 16 * lane;
    v_from = static_cast<const uint8_t*>(vc.ptr) + ld.hk * vc.stride_h + 16 * lane;
    s_from = s_v ? static_cast<const uint8_t*>(a.pool.v_scales.ptr) + 2 * ld.hk * a.pool.v_scales.stride_h
                 : static_cast<const uint8_t*>(a.pool.k_scales.ptr) + 2 * ld.hk * a.pool.k_scales.stride_h;
    s_from += lane % kPer * 16;
    // (its queries on their way to L2 meanwhile)
    const int i = ld.grp * p.unit_rows + lane, tok = i / p.group;
    if (lane < p.unit_rows && i < p.rows)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const T*>(a.q.ptr) + ld.b * a.q.stride_b +
                                                    (ld.hk * p.group + i - tok * p.group) * a.q.stride_h + tok * a.q.stride_t));
    return true;
  };
  bool loads = enter();
  if (loads) look_up();
  auto issue = [&]() {
    if (loads) {
      const int key = ld.tile * kKeys;
      const bool both = ld.keys - key > 16;
      const uint32_t to = ring_at + at_stage * L::kBytes;
      // (here, not at the look-up: the ids have had a tile's time to arrive)
      if ((uint32_t)page[0] >= (uint32_t)a.pool.n_pages) report(a.status, AI_ERR_DEV_BOUNDS), page[0] = 0;
      const int slot = key & page_mask;
      const uint8_t* k = k_from + ((uint64_t)page[0] * k_step << 4) + slot * L::kRow;
      const uint8_t* v = v_from + ((uint64_t)page[0] * v_step << 4) + slot * L::kRow;
      const uint8_t* c = s_from + ((uint64_t)page[0] * s_step << 4) + slot * 2 * C;
      const uint32_t dst = to + 16 * lane;
      if (page_bits > 4 && both) {  // (a whole tile in one page)
#pragma unroll
        for (int i = 0; i < 2 * kHalfCodes; i += 512)
          if (i + 16 * lane < 2 * kHalfCodes) {
            copy16(dst + L::K + i, k + i);
            copy16(dst + L::V + i, v + i);
          }
        if (s_has) copy16(to + s_at, c + s_half * kHalfScales);
      } else {
        if ((uint32_t)page[1] >= (uint32_t)a.pool.n_pages) report(a.status, AI_ERR_DEV_BOUNDS), page[1] = 0;
        const int slot1 = (key + 16) & page_mask;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1) {
            k = k_from + ((uint64_t)page[1] * k_step << 4) + slot1 * L::kRow;
            v = v_from + ((uint64_t)page[1] * v_step << 4) + slot1 * L::kRow;
          }
          if ((h == 0 || both) && 16 * lane < kHalfCodes) {
#pragma unroll
            for (int i = 0; i < kHalfCodes; i += 512) {
              copy16(dst + L::K + h * kHalfCodes + i, k + i);
              copy16(dst + L::V + h * kHalfCodes + i, v + i);
            }
          }
        }
        if (s_half) c = s_from + ((uint64_t)page[1] * s_step << 4) + slot1 * 2 * C;
        if (s_has && (s_half == 0 || both)) copy16(to + s_at, c);
      }
      at_stage = at_stage + 1 == S ? 0 : at_stage + 1;
      if (++ld.tile == ld.end) loads = enter();
      if (loads) look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int st = 0;
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue();

  // ---- products
  int wc = w0;
  Seg s;
  const int row_g = L::place(g);  // the lane's key of a product's first eight, as they lie
  // (a lane reads its own fragments alone)
  uint4* q_smem = reinterpret_cast<uint4*>(smem + M::Q + warp * M::kQ) + lane;
  float4* off_smem = reinterpret_cast<float4*>(smem + M::OFF + warp * M::kOff) + lane;
  while (next_seg(a, p, scan, wc, w1, s)) {
    const int row0 = s.grp * p.unit_rows, n_rows = min(p.rows - row0, p.unit_rows);
    // Query fragments: lane (g, t) has dims 32 c + 8 t + {0 .. 7} of row 8 nt + g,
    // scaled by the power of two that brings the row's largest element to the top of
    // fp16's range (and odd dims by 2^-4, for their codes).  Rows without a query
    // are zeros, whatever the padding holds.
    // Keys that row 8 nt + 2 t + e sees; -1: no query.  (Looked up where it is
    // wanted when registers are short.)
    auto count = [&](int nt, int e) -> int {
      const int i = 8 * nt + 2 * t + e, tok = (row0 + i) / p.group;
      return i < n_rows && tok < s.n ? max(0, s.keys - s.n + tok + 1) : -1;
    };
    const int first[2] = {count(0, 0), count(0, 1)};
    auto seen = [&](int nt, int e) -> int { return NT == 1 ? first[e] : count(nt, e); };
    int least = s.keys;               // tiles that end by it are seen whole
    float2 slope[NT];                 // of rows 2 t and 2 t + 1's scores, in units of log 2, above zero (its sign is the fragments')
    {
      const float sign = a.scale < 0.f ? -1.f : 1.f;
      uint4 raw[NT][C];  // (all of them in flight at once)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int i = 8 * nt + g, r = i < n_rows ? row0 + i : row0, tok = r / p.group, head = s.hk * p.group + r - tok * p.group;
        const T* src = static_cast<const T*>(a.q.ptr) + s.b * a.q.stride_b + head * a.q.stride_h + tok * a.q.stride_t + 8 * t;
        const bool real = i < n_rows && tok < s.n;
#pragma unroll
        for (int c = 0; c < C; ++c) raw[nt][c] = real ? load_q(src + kGroup * c) : make_uint4(0u, 0u, 0u, 0u);
      }
      __syncwarp();  // (the last unit's fragments have been read)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = fabsf(element<T>(raw[nt][c], e));
            if (f < CUDART_INF_F) top = fmaxf(top, f);
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int up = top > 0.f ? 14 - ilogbf(top) : 0;
        // (in two factors: up reaches 163)
        const float up1 = sign * ldexpf(1.f, up / 2), up2 = ldexpf(1.f, up - up / 2);
        // (above 0, so that a masked score stays -inf, and finite)
        const float mine = fminf(fmaxf(ldexpf(fabsf(a.scale) * kLog2e, 24 - up), FLT_MIN), FLT_MAX);
        slope[nt] = make_float2(__shfl_sync(0xffffffffu, mine, 8 * t), __shfl_sync(0xffffffffu, mine, 8 * t + 4));
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t h[4];
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // (dims 8 t + e and 8 t + 4 + e are a pair)
            const float odd = e % 2 ? 0x1p-4f : 1.f;
            h[e] = pack2(element<T>(raw[nt][c], e) * up1 * up2 * odd, element<T>(raw[nt][c], 4 + e) * up1 * up2 * odd);
            sum += (half_of(h[e], 0) + half_of(h[e], 1)) * (e % 2 ? 0x1p-20f : 0x1p-24f);
          }
          q_smem[(nt * C + c) * 32] = make_uint4(h[0], h[1], h[2], h[3]);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          const float2 off = make_float2(-8.f * __shfl_sync(0xffffffffu, sum, 8 * t), -8.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4));
          off_smem[(nt * C + c) * 32] = make_float4(off.x, off.y, off.x, off.y);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = seen(nt, e);
          if (n >= 0) least = min(least, n);
        }
      }
      least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
      least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
    }

    float o[NT][2 * C][4];             // (odd rows of a block, of odd dims, are 2^4 times the even ones)
    float ref[NT][2];                  // what the scores are taken less: their running maximum
    float2 l[NT], l_before[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2 * C; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      ref[nt][0] = ref[nt][1] = kNoRef;
      l[nt] = l_before[nt] = make_float2(0.f, 0.f);
    }
    // Per group of dims: |V scales| so far are at most a power of two (v_lim, two
    // groups a word), and v_unit divides by it.
    float2 v_unit[H];
    uint32_t v_lim[H];
#pragma unroll
    for (int i = 0; i < H; ++i) v_unit[i] = make_float2(0x1p14f, 0x1p14f), v_lim[i] = twice(0x0400u);
    static_assert(kLeastExp == -14, "v_unit and v_lim");

    for (int tile = s.tile; tile < s.end; ++tile) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
      __syncwarp();
      issue();  // (into the stage of the tile before: every lane has read it)
      const uint8_t* sm = ring + st * L::kBytes;
      st = st + 1 == S ? 0 : st + 1;
      const int k0 = tile * kKeys;

      // Scores: keys place(g) (e = 0, 1) and 8 behind (2, 3) of half mt, rows 2 t + e % 2.
      float2 sc[2][NT][2];
      uint32_t vs[2][2][H];
      // (both halves at once share their query fragments; with more column blocks
      // the registers are the blocks')
      constexpr int kAtOnce = NT == 1 ? 2 : 1;
#pragma unroll
      for (int m0 = 0; m0 < 2; m0 += kAtOnce) {
        uint32_t kw[kAtOnce][2][C], ks[kAtOnce][2][H];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = 16 * (m0 + i) + 8 * h + row_g;
            lds<4 * C>(kw[i][h], sm + L::K + key * L::kRow + 4 * C * t);
            lds<2 * C>(ks[i][h], sm + L::KS + key * 2 * C);
            lds<2 * C>(vs[m0 + i][h], sm + L::VS + key * 2 * C);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[m0 + i][nt][h] = make_float2(0.f, 0.f);
          }
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t f[kAtOnce][2][4];
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) numbers(C == 1 ? kw[i][h][0] : halves(kw[i][h][c / 2], kw[i][h][(C + c) / 2], c % 2), f[i][h]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 q = q_smem[(nt * C + c) * 32];
            const float4 off = off_smem[(nt * C + c) * 32];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
              float acc[4];
              mma(acc, f[i][0][0], f[i][1][0], f[i][0][1], f[i][1][1], q.x, q.y, off.x, off.y, off.z, off.w);
              mma(acc, f[i][0][2], f[i][1][2], f[i][0][3], f[i][1][3], q.z, q.w);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float d = half_of(ks[i][h][c / 2], c % 2);
                sc[m0 + i][nt][h] = __ffma2_rn(make_float2(d, d), make_float2(acc[2 * h], acc[2 * h + 1]), sc[m0 + i][nt][h]);
              }
            }
          }
        }
      }
      // The running maximum of each row, and of the V scales, lazily; masks where a
      // row does not see the whole tile.
      const bool ragged = least - k0 < kKeys;  // (lists end by 2^31: differences)
      float top[NT][2];
      auto tops = [&]() -> bool {
        bool move = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          top[nt][0] = fmaxf(ptx::fmax3(sc[0][nt][0].x, sc[0][nt][1].x, sc[1][nt][0].x), sc[1][nt][1].x);
          top[nt][1] = fmaxf(ptx::fmax3(sc[0][nt][0].y, sc[0][nt][1].y, sc[1][nt][0].y), sc[1][nt][1].y);
          move |= (top[nt][0] - ref[nt][0]) * slope[nt].x > kSlack || (top[nt][1] - ref[nt][1]) * slope[nt].y > kSlack;
        }
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const __half2 big = __hmax2(__hmax2(__habs2(as_half2(vs[0][0][i])), __habs2(as_half2(vs[0][1][i]))),
                                      __hmax2(__habs2(as_half2(vs[1][0][i])), __habs2(as_half2(vs[1][1][i]))));
          move |= !__hble2(big, as_half2(v_lim[i]));
        }
        return move;
      };
      bool guard = false;  // some row must not meet an infinite or NaN scale that another sees
      if (__any_sync(0xffffffffu, tops() || ragged)) {
        if (ragged) {
          bool odd = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int s0 = seen(nt, 0) - k0 - row_g, s1 = seen(nt, 1) - k0 - row_g;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (16 * mt + 8 * h >= s0) sc[mt][nt][h].x = -CUDART_INF_F;
                if (16 * mt + 8 * h >= s1) sc[mt][nt][h].y = -CUDART_INF_F;
              }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int i = 0; i < H; ++i) {
                if (16 * mt + 8 * h + row_g >= s.keys - k0) vs[mt][h][i] = 0;  // (a slot that no one wrote)
                odd |= !__hble2(__habs2(as_half2(vs[mt][h][i])), as_half2(0x7bff7bffu));
              }
            }
          guard = __any_sync(0xffffffffu, odd);
        }
        if (__any_sync(0xffffffffu, tops())) {
          // (an infinite scale makes what it meets infinite; it has no part in the bound)
          float down[2 * H];
#pragma unroll
          for (int c = 0; c < 2 * H; ++c) {
            float size = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float d = fabsf(half_of(vs[mt][h][c / 2], c % 2));
                if (d < CUDART_INF_F) size = fmaxf(size, d);
              }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, d));
            float& unit = c % 2 ? v_unit[c / 2].y : v_unit[c / 2].x;
            down[c] = 1.f;
            if (size * unit > 1.f) {
              const int e = min(ilogbf(size) + 2, 16);  // (room for twice as much: few lists then meet a larger one)
              const float to = ptx::ex2((float)-e);
              down[c] = to / unit;
              unit = to;
              const uint32_t lim = e > 15 ? 0x7bffu : (uint32_t)(15 + e) << 10;  // 2^e
              v_lim[c / 2] = c % 2 ? (v_lim[c / 2] & 0xffffu) | lim << 16 : (v_lim[c / 2] & 0xffff0000u) | lim;
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float alpha[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = top[nt][e], to = ref[nt][e];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              const float per = e ? slope[nt].y : slope[nt].x;
              if ((x - to) * per > kSlack) to = x;
              alpha[e] = ptx::ex2((ref[nt][e] - to) * per);
              ref[nt][e] = to;
#pragma unroll
              for (int i = 0; i < 2 * C; ++i) o[nt][i][e] *= alpha[e] * down[i / 2], o[nt][i][2 + e] *= alpha[e] * down[i / 2];
            }
            l[nt] = __fmul2_rn(l[nt], make_float2(alpha[0], alpha[1]));
            l_before[nt] = __fmul2_rn(l_before[nt], make_float2(alpha[0], alpha[1]));
          }
        }
      }
      // Weights, and per group of dims the weights times the V scales as the
      // second product takes them.
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t pv[NT][C][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // (the difference first: scores of any size then have the largest one's weight exact)
            const float2 y = __ffma2_rn(__fadd2_rn(sc[mt][nt][h], make_float2(-ref[nt][0], -ref[nt][1])), slope[nt], make_float2(kLift, kLift));
            const float2 w = make_float2(ptx::ex2(y.x), ptx::ex2(y.y));
            l[nt] = __fadd2_rn(l[nt], w);
#pragma unroll
            for (int i = 0; i < H; ++i) {
              const float2 d = __fmul2_rn(__half22float2(as_half2(vs[mt][h][i])), v_unit[i]);
              pv[nt][2 * i][h] = pack2(w.x * d.x, w.y * d.x);
              if (2 * i + 1 < C) pv[nt][2 * i + 1][h] = pack2(w.x * d.y, w.y * d.y);
            }
            if (guard) {
              const uint32_t keep = (sc[mt][nt][h].x == -CUDART_INF_F ? 0u : 0xffffu) | (sc[mt][nt][h].y == -CUDART_INF_F ? 0u : 0xffff0000u);
#pragma unroll
              for (int c = 0; c < C; ++c) pv[nt][c][h] &= keep;
            }
#pragma unroll
            for (int c = 0; c < C; ++c) pv[nt][c][h] = transpose8(pv[nt][c][h]);
          }
        uint32_t vw[4][H];  // the keys of rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int i = 0; i < 4; ++i) lds<2 * C>(vw[i], sm + L::V + (16 * mt + L::place(8 * (i / 2) + 2 * t + i % 2)) * L::kRow + 2 * C * g);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t f[2][4];
          numbers(halves(vw[0][c / 2], vw[1][c / 2], c % 2), f[0]);
          numbers(halves(vw[2][c / 2], vw[3][c / 2], c % 2), f[1]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) f[h][j] = less8(f[h][j], j % 2 ? 0x00800080u : 0x00080008u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              mma(o[nt][2 * c + i], f[0][2 * i], f[0][2 * i + 1], f[1][2 * i], f[1][2 * i + 1], pv[nt][c][0], pv[nt][c][1]);
        }
      }
      // (a sum of sums: one running sum of a long list would round its small weights away)
      if (tile % 16 == 15) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) l_before[nt] = __fadd2_rn(l_before[nt], l[nt]), l[nt] = make_float2(0.f, 0.f);
      }
    }
    // Partial rows: dims 32 c + 4 g + {0 .. 3} of rows 2 t and 2 t + 1.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = e ? l_before[nt].y + l[nt].y : l_before[nt].x + l[nt].x;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (seen(nt, e) <= 0) continue;
        const int64_t row = (int64_t)(s.unit + worker) * p.unit_rows + 8 * nt + 2 * t + e;
        const float all = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float inv = all / (c % 2 ? v_unit[c / 2].y : v_unit[c / 2].x);  // (a power of two)
          *reinterpret_cast<float4*>(p.part_o + row * D + kGroup * c + 4 * g) =
              make_float4(o[nt][2 * c][e] * 0x1p24f * inv, o[nt][2 * c][2 + e] * 0x1p20f * inv, o[nt][2 * c + 1][e] * 0x1p24f * inv,
                          o[nt][2 * c + 1][2 + e] * 0x1p20f * inv);
        }
        // (NaN among the scores: +inf, which makes the joined row NaN)
        if (g == 0) p.part_lse[row] = sum > 0.f ? fmaf(ref[nt][e], e ? slope[nt].y : slope[nt].x, log2f(sum) - kLift) : sum == 0.f ? -CUDART_INF_F : CUDART_INF_F;
      }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// `wide` warps per (sequence, query token, query head) join the row's partial
// results: each takes every wide-th of them, the first adds up the warps' in order.
// Where they lie follows from the lengths alone, which are the caller's: all of it
// is worked out before the first launch has ended.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(const AiPagedAttn4Args a, const Plan p, const int wide) {
  constexpr int E = D / 32, kAhead = 4;
  __shared__ int s_sum[2][8];
  __shared__ float s_acc[8][D + 2];
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid % 32, warp = tid / 32, part = warp % wide;
  // Positions before sequence b, and all.
  int before = 0, all = 0;
  for (int i = tid; i < a.batch; i += 256) {
    const int v = unit_size(seq_lens(a, i));
    all += v;
    if (i < b) before += v;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  all = __reduce_add_sync(0xffffffffu, all);
  if (lane == 0) s_sum[0][warp] = before, s_sum[1][warp] = all;
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < 8; ++w) before += s_sum[0][w], all += s_sum[1][w];
  const Lens len = seq_lens(a, b);
  const int item = blockIdx.x * (8 / wide) + warp / wide;
  const bool has = item < a.seq_len * a.num_q_heads;
  const int t = has ? item / a.num_q_heads : 0, h = has ? item - t * a.num_q_heads : 0, hk = h / p.group;
  const int seen = has && t < len.n ? len.keys - len.n + t + 1 : 0;
  int n = 0;
  int64_t row = 0;
  if (seen > 0) {
    const int per = a.num_kv_heads * p.groups, size = unit_size(len);
    const Split line = split_line(p.workers, all * per);
    const int i = t * p.group + h - hk * p.group, grp = i / p.unit_rows, sub = hk * p.groups + grp;
    const int x = before * per + sub * size + kStart, tiles = (seen - 1) / kKeys + 1;
    const int first = line.worker(x);
    n = line.worker(x + tiles - 1) - first + 1;
    row = (int64_t)(b * per + sub + first) * p.unit_rows + i - grp * p.unit_rows;
  }
  auto row_at = [&](int k) { return row + (int64_t)k * p.unit_rows; };
  auto load = [&](int k, float (&o)[E]) {
    const float* src = p.part_o + row_at(k) * D + E * lane;
    if constexpr (E == 4)
      *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(src);
    else if constexpr (E == 2)
      *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(src);
    else
      o[0] = *src;
  };
  float M = -CUDART_INF_F, sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (the first rows are on their way beside the sums' logarithms)
  float ahead[kAhead][E];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (part + k * wide < n) load(part + k * wide, ahead[k]);
  for (int k = lane; k < n; k += 32) M = fmaxf(M, p.part_lse[row_at(k)]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  if (M != -CUDART_INF_F) {
    for (int k0 = part; k0 < n; k0 += 32 * wide) {
      const int mine = k0 + lane * wide;
      const float my_w = mine < n ? exp2f(p.part_lse[row_at(mine)] - M) : 0.f;
      const int cnt = min(32, (n - k0 + wide - 1) / wide);
      auto add = [&](int k, const float (&o)[E]) {
        const float w = __shfl_sync(0xffffffffu, my_w, k);
        sum += w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, o[e], acc[e]);
      };
      int k = 0;
      if (k0 == part) {
#pragma unroll
        for (; k < kAhead; ++k)
          if (k < cnt) add(k, ahead[k]);
      }
#pragma unroll 4
      for (; k < cnt; ++k) {
        float o[E];
        load(k0 + k * wide, o);
        add(k, o);
      }
    }
  }
  if (wide > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_acc[warp][E * lane + e] = acc[e];
    if (lane == 0) s_acc[warp][D] = sum;
    __syncthreads();
    if (part > 0) return;
    for (int w = 1; w < wide; ++w) {
      sum += s_acc[warp + w][D];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += s_acc[warp + w][E * lane + e];
    }
  }
  if (!has) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* out = static_cast<T*>(const_cast<void*>(a.out.ptr)) + b * a.out.stride_b + h * a.out.stride_h + t * a.out.stride_t + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_f32<T>(acc[e] * inv);
  if (a.lse && lane == 0)
    a.lse[((int64_t)b * a.num_q_heads + h) * a.seq_len + t] = sum == 0.f ? -CUDART_INF_F : (M + log2f(sum)) * kLn2;
}

int check(const AiPagedAttn4Args* a) {
  if (!a) return AI_ERR_NULL;
  if (a->batch <= 0 || a->batch > kMaxBatch || a->seq_len <= 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads)
    return AI_ERR_SHAPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return AI_ERR_HEAD_DIM;
  if (a->dtype != AI_DTYPE_BF16 && a->dtype != AI_DTYPE_F16) return AI_ERR_DTYPE;
  for (const AiTensor4* t : {&a->q, &a->out}) {
    if (!t->ptr) return AI_ERR_NULL;
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < 0) return AI_ERR_STRIDE;
  }
  if (!a->lens) return AI_ERR_NULL;
  const int rc = check_pool(a->pool, a->head_dim);
  if (rc != AI_OK) return rc;
  // The line's positions and the combine launch's grid fit in 31 bits.
  const int64_t rows = (int64_t)a->num_q_heads * a->seq_len, groups = rows / a->num_kv_heads / (8 * kMaxBlocks) + 1;
  const int64_t tiles = (int64_t)a->pool.max_pages * a->pool.page_size / kKeys + kStart + 1;
  if (rows > 0x7ffffff0 || tiles > 0x7fffffff || a->batch * a->num_kv_heads * groups > 0x7fffffff / tiles) return AI_ERR_SHAPE;
  return AI_OK;
}

size_t layout(const AiPagedAttn4Args& a, Plan* p) {
  p->group = a.num_q_heads / a.num_kv_heads;
  p->rows = p->group * a.seq_len;
  p->groups = (p->rows + 8 * kMaxBlocks - 1) / (8 * kMaxBlocks);
  p->unit_rows = (p->rows + p->groups - 1) / p->groups;
  p->blocks = (p->unit_rows + 7) / 8;
  p->workers = sm_count() * warps_of(p->blocks);
  const size_t rows = ((size_t)a.batch * a.num_kv_heads * p->groups + p->workers) * p->unit_rows;
  const size_t o = (rows * a.head_dim * sizeof(float) + 255) & ~size_t(255), l = (rows * sizeof(float) + 255) & ~size_t(255);
  char* w = static_cast<char*>(a.workspace);
  p->part_o = reinterpret_cast<float*>(w);
  p->part_lse = reinterpret_cast<float*>(w + o);
  return o + l;
}

template <typename T, int D, int NT>
int launch(const AiPagedAttn4Args& a, const Plan& p, cudaStream_t st) {
  const size_t smem = Smem<D, NT>::bytes(a.batch);
  // (the limit is the kernel's, not the call's: always the same, so that calls of other
  // threads never find it lower than they need)
  if (cudaFuncSetAttribute(split_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)Smem<D, NT>::bytes(kMaxBatch)) != cudaSuccess)
    return AI_ERR_LAUNCH;
  split_kernel<T, D, NT><<<p.workers / warps_of(NT), 32 * warps_of(NT), smem, st>>>(a, p);
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T, int D>
int run(const AiPagedAttn4Args& a, const Plan& p, cudaStream_t st) {
  ProfScope ps(AI_PROF_ATTN4, st);
  const int rc = p.blocks == 1   ? launch<T, D, 1>(a, p, st)
                 : p.blocks == 2 ? launch<T, D, 2>(a, p, st)
                                 : launch<T, D, 3>(a, p, st);
  if (rc != AI_OK) return rc;
  // Warps that join a row: by the partial results it has, where the lists are alike.
  const int64_t parts = p.workers / ((int64_t)a.batch * a.num_kv_heads * p.groups);
  const int wide = parts >= 32 ? 8 : parts >= 16 ? 4 : parts >= 8 ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.seq_len * (int64_t)a.num_q_heads * wide + 7) / 8), a.batch);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, combine_kernel<T, D>, a, p, wide) != cudaSuccess) return AI_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

template <typename T>
int dispatch(const AiPagedAttn4Args& a, const Plan& p, cudaStream_t st) {
  if (a.head_dim == 128) return run<T, 128>(a, p, st);
  if (a.head_dim == 64) return run<T, 64>(a, p, st);
  return run<T, 32>(a, p, st);
}

}  // namespace attn4
}  // namespace ai

extern "C" int ai_paged_attn_4bit_workspace(const AiPagedAttn4Args* args, size_t* bytes) {
  const int rc = ai::attn4::check(args);
  if (rc != AI_OK) return rc;
  if (!bytes) return AI_ERR_NULL;
  ai::attn4::Plan p;
  *bytes = ai::attn4::layout(*args, &p);
  return AI_OK;
}

extern "C" int ai_paged_attn_4bit(const AiPagedAttn4Args* args, void* stream) {
  const int rc = ai::attn4::check(args);
  if (rc != AI_OK) return rc;
  ai::attn4::Plan p;
  const size_t need = ai::attn4::layout(*args, &p);
  if (!args->workspace || args->workspace_bytes < need) return AI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(args->workspace) & 255) return AI_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AI_DTYPE_BF16) return ai::attn4::dispatch<__nv_bfloat16>(*args, p, st);
  return ai::attn4::dispatch<__half>(*args, p, st);
}
