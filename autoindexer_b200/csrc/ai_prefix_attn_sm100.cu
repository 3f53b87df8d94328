// Shared-prefix attention on the tensor cores: bf16 / fp16, head_dim 64 or
// 128, page sizes that are powers of two from 16.
//
// Every query row attends over two key lists, the prefix's and its own
// sequence's.  The rows that share a list (of one KV head) are a unit: the
// B T G rows over the batch for the prefix (G query heads per KV head), the
// T G rows of a sequence for its own keys.  A unit's keys are cut into tiles;
// the tiles of all units stand in one line, and every worker takes an equal
// stretch of it, whatever the lengths are (they are read on the device).  A
// stretch crosses units, and the rows of a unit that a worker touched leave
// partial results (O / l in fp32 and the log2-sum), which the combine launch
// joins with the other list's.
//
// Two kernels, by the rows that meet each key:
//   tile kernel   many rows, long lists: 128 rows x 64 keys or 256 rows x
//                 128 keys a step on tcgen05 (worker: a CTA);
//   warp kernel   few rows, short lists: 16 rows x 32 keys a step on
//                 mma.sync, K and V by TMA (worker: one to four warps).
//                 HBM-bound with few rows; a worker has no barrier of the CTA
//                 in its loop and a short list costs a few loads, where the
//                 tile kernel pays a chain of TMA, MMA and TMEM latencies per
//                 unit (4.8 us per unit of one 64-key tile).  Own lists of 64
//                 sequences of up to 2048 keys: 48 us, 5.6 TB/s.
// P is rounded to the values' type for its product (the MMAs take one type), the
// sums take it unrounded: about the error of the output's own rounding (1.3 to
// 1.4 times a single-rounded result's in either type; none for up to 8 rows a
// warp).  fp16 holds small weights to 2^-32 of the largest (see Pair), bf16 to
// its 8 bits at any size.  The MMAs cut a product 25 bits below its accumulator,
// so n weights of under 2^-25 of what a stretch has gathered may add n 2^-25 to
// the relative error, in either type.
// The second is launched by programmatic dependent launch: it fills the SMs the
// first leaves, or takes its share of them from the start (make_plan).
//
// Measured (bf16, 32 + 8 heads, D 128, up to 2048 own keys): 64 sequences of
// one token on a prefix of 32,768 keys 95 us, of up to five tokens 183 us (217
// at the power limit); 16 on 4096 + 512 keys 24 us; four on 257 + 65 keys 14 us (two launches' latency).

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

constexpr int BM = 128;
constexpr int kMaxBatch = 1024;  // two scans of the sequences sit in shared memory
constexpr long long kWait = 1000000000LL;

// One kernel's line of tiles.  Starting a unit costs about as much as `start`
// tiles (its rows in, its partial results out), so `start` idle positions
// stand before its tiles.
struct Line {
  int workers;
  int least;          // positions a worker takes at least
  int start;
  int units_prefix;   // prefix units on this line, each of tiles_prefix tiles: (KV head, group of rows)
  int groups;         // groups of rows a KV head has
  int rows_prefix;    // rows of a prefix unit
  int slot_prefix;    // rows of its slots (the most a unit can have)
  int tiles_prefix;
  int per_seq;        // units per sequence on this line (0: own keys are not on it)
  int rows_own;       // rows of a sequence's unit
  int64_t base_prefix, base_own;  // first row of each region; slot (unit + worker) follows
};

// Threads of a tile-kernel CTA with NT row tiles: a softmax warpgroup each, a
// TMA and an MMA warp.
// (NT = 2: whole warpgroups, for the register split.)
__host__ __device__ constexpr int tile_threads(int NT) { return NT == 1 ? 192 : 384; }
// Keys of its tiles.
__host__ __device__ constexpr int tile_keys(int NT) { return NT == 1 ? 64 : 128; }
// NT = 2: launched at 168 registers a thread; a row's 128 scores stay in the
// softmax warpgroups', the third warpgroup (TMA and MMA warps) gives its up.
constexpr uint32_t kRegLaunch = 168, kRegSoftmax = 208, kRegOther = 88;
static_assert(256 * kRegSoftmax + 128 * kRegOther <= 384 * kRegLaunch, "register split");

template <int D, int NT>
struct Smem {
  static constexpr int BN = tile_keys(NT), kBufs = 128 / BN;  // S buffers of a row tile
  static constexpr uint32_t kTile = BN * D * 2;    // one K or V tile: D / 64 column blocks of BN rows x 128 bytes
  static constexpr uint32_t kQBlock = BM * 128;    // one column block of a Q tile
  static constexpr uint32_t kQ = BM * D * 2;
  static constexpr int kSlots = D == 128 ? 4 : 8;  // ring of tiles, K and V alternating (64 KB per row tile)
  static constexpr uint32_t Q = 0;
  static constexpr uint32_t RING = Q + NT * kQ;
  static constexpr uint32_t BARS = RING + kSlots * kTile;
  // (kBufs of each per row tile; P_HALF: the first half of P, with one S buffer)
  static constexpr int FULL = 0, EMPTY = kSlots, S_FULL = 2 * kSlots, P_READY = S_FULL + kBufs * NT,
                       O_DONE = P_READY + kBufs * NT, Q_READY = O_DONE + kBufs * NT, P_HALF = Q_READY + NT,
                       FINAL = P_HALF + NT, N_BARS = FINAL + 1;
  static constexpr uint32_t LINE = BARS + 8 * N_BARS;  // the line with the rows that there are
  static constexpr uint32_t TMEM_SLOT = LINE + sizeof(Line);
  static constexpr uint32_t ABORT = TMEM_SLOT + 4;
  static constexpr uint32_t SCAN = ABORT + 4;  // int [2][B + 1]
  static size_t bytes(int batch) { return SCAN + 8 * ((size_t)batch + 1) + 1024; }
  // TMEM: 128 columns per row tile for its S buffers (P over a buffer's first half), then O of D columns each.
  static constexpr uint32_t kTmemCols = 256 * NT;
  static constexpr uint32_t C_S = 0, C_O = 128 * NT;
};
static_assert(2 * (Smem<128, 1>::SCAN + 8 * (kMaxBatch + 1) + 1024 + 1024) <= 228 * 1024, "two CTAs per SM");
static_assert(Smem<128, 2>::SCAN + 8 * (kMaxBatch + 1) + 1024 <= 227 * 1024, "one CTA per SM");

constexpr int kWarpRows = 64;   // most rows of a sequence on the warp kernel
constexpr int kWarpKeys = 32;   // keys of its tile
// Cuts, with both sides measured (bf16, 32 + 8 heads, D 128, one token; us;
// "64 on 2048 + 256": 64 sequences, prefix, most own keys).  kShortPrefix:
// positions of a prefix per worker of the warp kernel, at most (3 / 6 / 12: 36 /
// 24 / 23 on 64 on 1024 + 64; 45 / 44 / 34 on 64 on 2048 + 256, but 29 / 29 / 34
// on 16 on 8192 + 512).  kFewOwn: positions of own keys per worker of the tile
// kernel, at most (0 / 6 / 12: 34 / 29 / 27 on 16 on 8192 + 512, 47 / 39 / 39 on
// 4 on 32,768 + 1; larger cuts send lists there that the warp kernel streams).
constexpr int kShortPrefix = 6, kFewOwn = 6;
// What starting a unit costs, in tiles of its kernel (kStartTile 2 / 4 / 8: 112 /
// 108 / 107 on 64 on 32,768 + 2048, 27 / 28 / 36 on 16 on 8192 + 512; kStartWarp
// 1 / 2 / 4: 68 / 59 / 57 on 64 on 64 + 2048, 24 / 24 / 25 on 64 on 1024 + 64).
constexpr int kStartTile = 4, kStartWarp = 2;

namespace warpk {
__host__ __device__ constexpr int workers(int split) { return split == 4 ? 2 : split == 2 ? 5 : 6; }  // per CTA (one per SM)
}

// What the host knows of the work.
struct Plan {
  int group;        // G: query heads per KV head
  int rows_seq;     // T G
  int nt;           // row tiles of a tile-kernel CTA
  int split;        // warps of a warp-kernel worker
  bool prefix_warp, own_warp;  // which kernel has the list
  int tile_cost;    // of a position of the tile kernel, in positions of the warp kernel
  int share;        // SMs that the two kernels divide between them; 0: each has all
  Line tile, warp;
  float* part_o;    // [rows][D]
  float* part_lse;  // [rows]
  int* scan;        // [B + 1] positions before each sequence's own units, per unit
  int* tokens;      // [B + 1] real query tokens before each sequence, then the tile kernel's SMs
};

// The line with the rows that there are: the prefix's units have the real
// query tokens' rows, evenly over as few groups as hold them (the host knows
// only that slot_prefix is the most a unit can have).
__device__ __forceinline__ Line live_line(const AiPrefixAttnArgs& a, const Line& l, int rows) {
  Line r = l;
  if (l.units_prefix > 0) {
    r.groups = (rows + l.slot_prefix - 1) / l.slot_prefix;
    r.units_prefix = r.groups * a.num_kv_heads;
    r.rows_prefix = r.groups > 0 ? (rows + r.groups - 1) / r.groups : 0;
  }
  return r;
}

// Positions of a line whose sequences have `own` positions per unit (the host
// has checked that they fit in an int).
__device__ __forceinline__ int line_total(const Line& l, int own) {
  return l.units_prefix * (l.start + l.tiles_prefix) + own * l.per_seq;
}

// SMs of the tile kernel where the two run side by side: in proportion to what
// the lines cost (own: positions per unit of the sequences' own lists).
__device__ __forceinline__ int tile_sms(const AiPrefixAttnArgs& a, const Plan& p, int rows, int own) {
  if (p.share == 0) return 0;
  const int64_t tile = (int64_t)line_total(live_line(a, p.tile, rows), 0) * p.tile_cost, warp = line_total(p.warp, own);
  if (warp == 0) return p.share;
  const int64_t x = (p.share * tile + tile + warp - 1) / (tile + warp);
  return (int)(x < 1 ? 1 : x > p.share - 1 ? p.share - 1 : x);
}

// The tile kernel's line (or the warp kernel's) with the rows and the workers
// that there are, x SMs being the tile kernel's.
__device__ __forceinline__ Line active_line(const AiPrefixAttnArgs& a, const Plan& p, bool tile, int rows, int x) {
  Line l = live_line(a, tile ? p.tile : p.warp, rows);
  if (p.share > 0) l.workers = min(l.workers, tile ? x : (p.share - x) * warpk::workers(p.split));
  return l;
}

// The line's stretches: n workers have work, none less than `least` positions
// unless the line is shorter; the first `more` take one position more.
struct Split {
  int n, len, more;
  __device__ __forceinline__ int begin(int w) const { return w * len + min(w, more); }
  __device__ __forceinline__ int worker(int x) const {
    const int head = more * (len + 1);
    return x < head ? x / (len + 1) : more + (x - head) / len;
  }
};

__device__ __forceinline__ Split split_line(const Line& l, int total) {
  Split s{0, 1, 0};
  if (total > 0) {
    s.n = min(l.workers, (total + l.least - 1) / l.least);
    s.len = total / s.n;
    s.more = total - s.len * s.n;
  }
  return s;
}

// scan[b] = positions before sequence b on the line of its own keys, for one
// unit per sequence (zeros if the line has none); tokens[b] = real query
// tokens before it.  One warp; tiles of `keys` keys.
__device__ __forceinline__ void scan_seqs(const AiPrefixAttnArgs& a, const Line& l, int keys, int* scan, int* tokens) {
  const int lane = threadIdx.x % 32;
  int base = 0, base_t = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    int v = 0, n = 0;
    if (b < a.batch) {
      const Lens len = seq_lens(a, b);
      n = len.n;
      if (l.per_seq > 0 && len.keys > 0) v = l.start + (len.keys + keys - 1) / keys;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o), x = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) v += u, n += x;
    }
    if (b < a.batch) scan[b + 1] = base + v, tokens[b + 1] = base_t + n;
    base += __shfl_sync(0xffffffffu, v, 31);
    base_t += __shfl_sync(0xffffffffu, n, 31);
  }
  if (lane == 0) scan[0] = tokens[0] = 0;
}

// The last sequence b with scan[b] * per <= x.
__device__ __forceinline__ int find_seq(const int* scan, int batch, int per, int x) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (scan[mid] * per <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A worker's stretch within one unit.
struct Seg {
  int unit;        // of its region
  int b;           // sequence, -1: the prefix
  int sub;         // unit within the sequence, or within the prefix
  int j0, n;       // tiles [j0, j0 + n) of the unit
  int keys;        // keys of the list
};

// The stretch [w, w1) within the unit at position w; `w` moves to its end.
// (n may be 0: idle positions only.)
__device__ __forceinline__ Seg locate(const AiPrefixAttnArgs& a, const Line& l, const int* scan, int& w, int w1) {
  Seg s;
  const int per = l.start + l.tiles_prefix, before = l.units_prefix * per;
  int at, size;  // position within the unit, and its positions
  if (w < before) {
    s.unit = s.sub = w / per;
    s.b = -1;
    at = w - s.unit * per;
    size = per;
    s.keys = a.prefix_len;
  } else {
    const int x = w - before;
    const int lo = find_seq(scan, a.batch, l.per_seq, x);  // (it has tiles)
    size = scan[lo + 1] - scan[lo];
    const int rem = x - scan[lo] * l.per_seq;
    s.b = lo;
    s.sub = rem / size;
    s.unit = lo * l.per_seq + s.sub;
    at = rem - s.sub * size;
    s.keys = seq_lens(a, lo).keys;
  }
  const int end = min(size, at + (w1 - w));
  s.j0 = max(0, at - l.start);
  s.n = max(0, end - l.start - s.j0);
  w += end - at;
  return s;
}

// The next stretch with tiles from position w on (n = 0: there is none).
__device__ __forceinline__ Seg next_seg(const AiPrefixAttnArgs& a, const Line& l, const int* scan, int& w, int w1) {
  Seg s{};
  while (w < w1 && s.n == 0) s = locate(a, l, scan, w, w1);
  return s;
}

// Query row `i` of a list's rows: i counts (t, query head of the group) of a
// sequence, and the real tokens of the sequences before it for the prefix.
struct Row {
  int b, t, g;
};

__device__ __forceinline__ Row row_of(const AiPrefixAttnArgs& a, const Plan& p, const int* tokens, int b, int i) {
  Row r;
  r.t = i / p.group;
  r.g = i - r.t * p.group;
  r.b = b;
  if (b < 0) {
    r.b = r.t / a.seq_len;  // right where every sequence has all its tokens
    if (tokens[r.b] > r.t || tokens[r.b + 1] <= r.t) r.b = find_seq(tokens, a.batch, 1, r.t);
    r.t -= tokens[r.b];
  }
  return r;
}

// Keys of the list that row r sees; -1 for a padding token.
__device__ __forceinline__ int visible(const AiPrefixAttnArgs& a, const Row& r, bool prefix, int keys) {
  const Lens len = seq_lens(a, r.b);
  if (r.t >= len.n) return -1;
  return prefix ? keys : max(0, keys - len.n + r.t + 1);
}

// Two values of a type.  top: a maximum as the softmax takes it, for fp16 lower
// by 7, so that P = 2^(s - m) and the sums are 2^7 times the weights (m plus the
// sum's logarithm stays what it is).  The lazy maximum lets P reach 2^8; fp16
// has room for 2^15, and each bit used above is one kept below, where weights
// under 2^-25 of the maximum were lost and those under 2^-14 lost bits.  limit:
// the maximum moves when a score's top passes it.  In fp16 the one is rounded up
// and the other down, so that P stays at 2^15 however large the scores are (a
// maximum of 2^26 is a multiple of 8).
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;
  __device__ static float top(float score, float sl2) { return score * sl2; }
  __device__ static float limit(float m) { return m + 8.f; }
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float2 unpack(uint32_t p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p)); }
};
template <> struct Pair<__half> {
  static constexpr uint32_t kFmt = 0;
  __device__ static float top(float score, float sl2) { return __fmaf_ru(score, sl2, -7.f); }
  __device__ static float limit(float m) { return __fadd_rd(m, 8.f); }
  __device__ static uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float2 unpack(uint32_t p) { return __half22float2(*reinterpret_cast<const __half2*>(&p)); }
};

// kind::f16 instruction descriptor with fp32 accumulation (fields as in sm100_ptx.cuh).
__host__ __device__ constexpr uint32_t idesc(uint32_t fmt, int M, int N, bool b_mn) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// NT = 1: up to 128 rows a unit, two CTAs per SM whose phases fill each
// other's gaps, 64 keys a tile and two S buffers (S of the tile after next
// runs during a tile's softmax).  NT = 2: up to 256 rows, halved over two row
// tiles that share every K and V tile (each is read from L2 once, not twice),
// one CTA per SM; one row tile's MMAs run during the other's softmax, so one S
// buffer each is enough and a tile has 128 keys: an S MMA of 64 keys reads as
// much of Q from shared memory for half the work (172 us with 64-key tiles,
// 158 us so, 64 sequences x 5 tokens x 32 heads on 32,768 keys, bf16, D 128).
// P goes out in two halves, so that only half of P V and the next S stand
// between a row tile's last exponential and its next scores (with own keys of
// up to 2048: 196 us whole, 192 so).
// Bound by the softmax: a row is one thread's, its exponentials a chain of
// multiply-add, ex2, pack and store of about 600 instructions a tile (tensor
// pipe and ex2 unit are each busy half of the time).
template <typename T, int D, int NT>
__global__ void __launch_bounds__(tile_threads(NT), NT == 1 ? 2 : 1)
    tile_kernel(const AiPrefixAttnArgs a, const Plan p, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v) {
  using L = Smem<D, NT>;
  constexpr int CB = D / 64, kTma = 4 * NT, kMma = kTma + 1;
  constexpr int BN = L::BN, kBufs = L::kBufs;
  constexpr uint32_t C_S = L::C_S, C_O = L::C_O;
  // (the warp kernel reads nothing this one writes)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = tile::align1024(smem_raw);
  const uint32_t sbase = ptx::smem_u32(sm);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  volatile int* s_abort = reinterpret_cast<volatile int*>(sm + L::ABORT);
  int* scan = reinterpret_cast<int*>(sm + L::SCAN);
  int* tokens = scan + a.batch + 1;
  auto bar = [&](int i) { return sbase + L::BARS + 8u * (uint32_t)i; };

  if (tid == 0) {
    for (int i = 0; i < L::N_BARS; ++i) {
      const bool wide = (i >= L::P_READY && i < L::O_DONE) || (i >= L::Q_READY && i < L::FINAL);
      ptx::mbar_init(bar(i), wide ? 128 : 1);
    }
    *s_abort = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMma) {
    ptx::tmem_alloc(sbase + L::TMEM_SLOT, L::kTmemCols);
    ptx::tmem_relinquish();
  }
  if (warp == 0) {
    // (side by side with the warp kernel: that one's scan, this line has no own lists)
    scan_seqs(a, p.share > 0 ? p.warp : p.tile, p.share > 0 ? kWarpKeys : BN, scan, tokens);
    __syncwarp();
    if (lane == 0) {
      const int rows = tokens[a.batch] * p.group, x = tile_sms(a, p, rows, scan[a.batch]);
      *reinterpret_cast<Line*>(sm + L::LINE) = active_line(a, p, true, rows, x);
      if (blockIdx.x == 0) p.tokens[a.batch + 1] = x;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + L::TMEM_SLOT);
  const int all_rows = tokens[a.batch] * p.group;
  const Line& ln = *reinterpret_cast<const Line*>(sm + L::LINE);
  const Split line = split_line(ln, line_total(ln, scan[a.batch]));
  const bool busy = (int)blockIdx.x < line.n;
  const int w0 = busy ? line.begin(blockIdx.x) : 0, w1 = busy ? line.begin(blockIdx.x + 1) : 0;
  if (blockIdx.x == 0)
    for (int b = tid; b <= a.batch; b += tile_threads(NT)) {
      if (ln.per_seq > 0) p.scan[b] = scan[b];
      p.tokens[b] = tokens[b];
    }
  auto head = [&](const Seg& s) { return s.b < 0 ? s.sub / ln.groups : s.sub % a.num_kv_heads; };

  if constexpr (NT == 2) {
    if (warp < kTma)
      ptx::setmaxnreg_inc<kRegSoftmax>();
    else
      ptx::setmaxnreg_dec<kRegOther>();
  }

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

  if (warp < kTma) {
    // ------------------------------------------------------------ softmax
    const int wg = warp / 4, r = tid % 128;  // row tile, row of it
    const uint32_t lane_base = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t c_o = tmem + lane_base + C_O + (uint32_t)(wg * D);
    const int S_FULL = L::S_FULL + kBufs * wg, P_READY = L::P_READY + kBufs * wg, O_DONE = L::O_DONE + kBufs * wg;
    const float sl2 = a.scale * kLog2e;
    // The rows of a segment: the thread's visible keys of its list, and Q into
    // shared memory (once no MMA reads the Q before it).  A thread finds its
    // row; a warp then loads its 32 rows, D / 8 lanes a row, eight loads in
    // flight.  Rows without a query are neither loaded, masked nor stored:
    // their TMEM lanes reach no other row.
    int limit = 0, least = 0;
    bool valid = false, active = false;
    int in_unit = 0;  // the thread's row of the unit
    auto load_rows = [&](const Seg& s) {
      constexpr int kLanes = D / 8, kPer = 32 / kLanes, kFly = 8;  // lanes a row, rows a load, loads in flight
      const bool pre = s.b < 0;
      // (a row tile's rows in whole warps: a warp without rows does nothing)
      const int per = pre ? ln.rows_prefix : ln.rows_own, half = NT == 1 ? per : (per + 63) / 64 * 32, hk = head(s);
      const int row0 = (pre ? s.sub % ln.groups : s.sub / a.num_kv_heads) * per + wg * half;
      const int n_rows = min(min(half, per - wg * half), (pre ? all_rows : p.rows_seq) - row0);
      int seen = -1;
      unsigned long long src = 0;
      if (r < n_rows) {
        const Row x = row_of(a, p, tokens, s.b, row0 + r);
        src = reinterpret_cast<unsigned long long>(static_cast<const T*>(a.q.ptr) + x.b * a.q.stride_b +
                                                   (hk * p.group + x.g) * a.q.stride_h + x.t * a.q.stride_t);
        seen = visible(a, x, pre, s.keys);
      }
      uint8_t* q_sm = sm + L::Q + wg * L::kQ;
      const int base = (warp % 4) * 32;
#pragma unroll
      for (int i0 = 0; i0 < 32; i0 += kPer * kFly) {
        if (base + i0 >= n_rows) break;
        uint4 v[kFly];
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
          const unsigned long long at = __shfl_sync(0xffffffffu, src, i0 + i * kPer + lane / kLanes);
          if (at) v[i] = __ldg(reinterpret_cast<const uint4*>(at) + lane % kLanes);
        }
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
          const int row = base + i0 + i * kPer + lane / kLanes;
          if (row < n_rows) *reinterpret_cast<uint4*>(q_sm + tile::chunk_off<BM>(row, lane % kLanes)) = v[i];
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar(L::Q_READY + wg));
      valid = seen >= 0;
      limit = valid ? seen : 0x7fffffff;
      active = __any_sync(0xffffffffu, valid);
      least = limit;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      in_unit = wg * half + r;
    };
    int g = 0, seg = 0;
    bool ok = true;
    int w = w0;
    Seg s = next_seg(a, ln, scan, w, w1);
    if (s.n > 0) load_rows(s);
    while (s.n > 0) {
      float m = -CUDART_INF_F, l = 0.f;
      for (int j = 0; j < s.n; ++j, ++g) {
        const int k0 = (s.j0 + j) * BN, x = g % kBufs;
        const uint32_t c_s = tmem + lane_base + C_S + (uint32_t)(wg * 128 + x * BN);
        if (!(ok = wait(S_FULL + x, (g / kBufs) & 1))) break;
        ptx::tc_fence_after();
        if (wg == 0 && k0 + BN > s.keys) {
          // Slots past the list hold anything, NaN included, and meet P = 0:
          // clear their V rows (before the first row tile's P V, which the
          // second's follows).
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
        if (active) {
          uint32_t sc[BN / 32][32];
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) ptx::tmem_ld32(c_s + 32 * c, sc[c]);
          ptx::tmem_wait_ld();
          if (k0 + BN > least) {
            const int lim = limit - k0;
#pragma unroll
            for (int c = 0; c < BN / 32; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i + 32 * c >= lim) sc[c][i] = 0xff800000u;  // -inf
          }
          float mx[BN / 32];
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) mx[c] = fmaxf(__uint_as_float(sc[c][0]), __uint_as_float(sc[c][1]));
#pragma unroll
          for (int i = 2; i < 32; i += 2)
#pragma unroll
            for (int c = 0; c < BN / 32; ++c)
              mx[c] = ptx::fmax3(mx[c], __uint_as_float(sc[c][i]), __uint_as_float(sc[c][i + 1]));
#pragma unroll
          for (int c = 1; c < BN / 32; ++c) mx[0] = fmaxf(mx[0], mx[c]);
          const float m_new = fmaxf(m, Pair<T>::top(mx[0], sl2));
          float alpha = 1.f;
          bool rescale = false;
          if (m_new > Pair<T>::limit(m)) {
            if (l > 0.f) {
              alpha = ptx::ex2(m - m_new);
              rescale = true;
            }
            m = m_new;
          }
          if (__any_sync(0xffffffffu, rescale)) {
            // O holds the tiles before this one once their last P V is done
            // (with one S buffer, this tile's S came after it).
            if (kBufs > 1 && !(ok = wait(O_DONE + (x ^ 1), ((g - 1) / kBufs) & 1))) break;
            ptx::tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              ptx::tmem_ld16(c_o + 16 * c, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              ptx::tmem_st16(c_o + 16 * c, o);
            }
            l *= alpha;
          }
          const float base = m == -CUDART_INF_F ? 0.f : m;
          const float2 nm = make_float2(-base, -base), sc2 = make_float2(sl2, sl2);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 e = __ffma2_rn(make_float2(__uint_as_float(sc[c][2 * i]), __uint_as_float(sc[c][2 * i + 1])), sc2, nm);
              const float2 pr = make_float2(ptx::ex2(e.x), ptx::ex2(e.y));
              sum[c % 2] = __fadd2_rn(sum[c % 2], pr);
              pk[i] = Pair<T>::pack(pr.x, pr.y);
            }
            ptx::tmem_st16(c_s + 16 * c, pk);
            if (kBufs == 1 && c == BN / 64 - 1) {
              ptx::tmem_wait_st();
              ptx::tc_fence_before();
              ptx::mbar_arrive(bar(L::P_HALF + wg));
            }
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          ptx::tmem_wait_st();
        } else if (kBufs == 1) {
          ptx::mbar_arrive(bar(L::P_HALF + wg));
        }
        ptx::tc_fence_before();
        ptx::mbar_arrive(bar(P_READY + x));
      }
      if (!ok) break;
      // The last S of this segment is done: the next segment's rows come in
      // while its last P V runs.
      const Seg cur = s;
      const bool cur_valid = valid, cur_active = active;
      const int cur_row = in_unit;
      s = next_seg(a, ln, scan, w, w1);
      if (s.n > 0) load_rows(s);
      // The rows' partial results.
      if (!(ok = kBufs > 1 ? wait(O_DONE + (g - 1) % kBufs, ((g - 1) / kBufs) & 1) : wait(O_DONE, seg & 1))) break;
      ++seg;
      ptx::tc_fence_after();
      if (cur_active) {
        const int64_t slot = cur.unit + (int)blockIdx.x;
        const int64_t row = (cur.b < 0 ? ln.base_prefix + slot * ln.slot_prefix
                                       : ln.base_own + slot * ln.rows_own) + cur_row;
        const float inv = 1.f / l;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          ptx::tmem_ld32(c_o + 32 * c, o);
          ptx::tmem_wait_ld();
          if (cur_valid) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t v8[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v8[e] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i + e]) * inv);
              ptx::st_global_v8(p.part_o + row * D + 32 * c + i, v8);
            }
          }
        }
        if (cur_valid) p.part_lse[row] = part_lse(l, m + log2f(l));
      }
      ptx::tc_fence_before();
    }
  } else if (warp == kTma) {
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
      const Seg s = next_seg(a, ln, scan, w, w1);
      const int32_t* table = s.b < 0 ? a.prefix_pages : a.page_table + s.b * a.page_table_stride;
      const int hk = head(s);
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
                             kv ? &tm_v : &tm_k, bar(L::FULL + slot), 64 * cb, at, hk, page);
        }
      }
    }
    // After a wait that gave up: the loads in flight land before the CTA ends.
    if (!ok || *s_abort)
      for (int i = max(0, item - L::kSlots); i < item; ++i)
        ptx::mbar_wait(bar(L::FULL + i % L::kSlots), (i / L::kSlots) & 1, kWait);
  } else if (warp == kMma) {
    // ------------------------------------------------------------ MMA
    constexpr uint32_t i_qk = idesc(Pair<T>::kFmt, BM, BN, false), i_pv = idesc(Pair<T>::kFmt, BM, D, true);
    const uint64_t d_q = ptx::sdesc_sw128(sbase + L::Q, 16, 1024);
    const uint64_t d_k = ptx::sdesc_sw128(sbase + L::RING, 16, 1024);
    const uint64_t d_v = ptx::sdesc_sw128(sbase + L::RING, BN * 128, 1024);
    constexpr uint64_t kT = L::kTile >> 4;
    auto wait_k = [&](int g) -> bool {
      const int item = 2 * g;
      if (!wait(L::FULL + item % L::kSlots, (item / L::kSlots) & 1)) return false;
      ptx::tc_fence_after();
      return true;
    };
    // S of row tile t and tile g (after the last one its K slot is free).
    auto issue_s = [&](int t, int g) {
      const int slot = (2 * g) % L::kSlots;
#pragma unroll
      for (int c = 0; c < CB; ++c)
        ptx::mma_ss4_w(tmem + C_S + (uint32_t)(t * 128 + (g % kBufs) * BN),
                       d_q + (uint64_t)((t * L::kQ + c * L::kQBlock) >> 4),
                       d_k + kT * (uint64_t)slot + (uint64_t)((c * (BN * 128)) >> 4), i_qk, c > 0);
      ptx::mma_commit_w(bar(L::S_FULL + kBufs * t + g % kBufs));
      if (t == NT - 1) ptx::mma_commit_w(bar(L::EMPTY + slot));
    };
    int g = 0, seg = 0;
    bool ok = true;
    for (int w = w0; w < w1 && ok; ++seg) {
      const Seg s = next_seg(a, ln, scan, w, w1);
      if (s.n == 0) break;
      for (int t = 0; t < NT && ok; ++t) ok = wait(L::Q_READY + t, seg & 1);
      for (int j = 0; j < kBufs && j < s.n && ok; ++j) {
        if (!(ok = wait_k(g + j))) break;
#pragma unroll
        for (int t = 0; t < NT; ++t) issue_s(t, g + j);
      }
      for (int j = 0; j < s.n && ok; ++j) {
        const int gj = g + j, item = 2 * gj + 1, slot = item % L::kSlots;
        const bool more = j + kBufs < s.n;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (t == 0 && !(ok = wait(L::FULL + slot, (item / L::kSlots) & 1))) break;
          // P V of k-steps [k0, k1)
          auto pv = [&](int k0, int k1) {
            ptx::tc_fence_after();
#pragma unroll
            for (int kk = k0; kk < k1; kk += 4)
              ptx::mma_ts4_w(tmem + C_O + (uint32_t)(t * D), tmem + C_S + (uint32_t)(t * 128 + (gj % kBufs) * BN + 8 * kk),
                             d_v + kT * (uint64_t)slot + (uint64_t)((kk * 2048) >> 4), i_pv, (j > 0 || kk > 0) ? 1u : 0u);
          };
          if constexpr (kBufs == 1) {
            if (!(ok = wait(L::P_HALF + t, gj & 1))) break;
            pv(0, BN / 32);
            if (t == 0 && more && !(ok = wait_k(gj + 1))) break;
          }
          if (!(ok = wait(L::P_READY + kBufs * t + gj % kBufs, (gj / kBufs) & 1))) break;
          pv(kBufs == 1 ? BN / 32 : 0, BN / 16);
          // (one S buffer: nobody waits for another than a segment's last)
          if (kBufs > 1 || j + 1 == s.n) ptx::mma_commit_w(bar(L::O_DONE + kBufs * t + gj % kBufs));
          if (t == NT - 1) ptx::mma_commit_w(bar(L::EMPTY + slot));
          if (more) {
            if (kBufs > 1 && t == 0 && !(ok = wait_k(gj + kBufs))) break;
            issue_s(t, gj + kBufs);
          }
        }
      }
      g += s.n;
    }
    // Every MMA issued has completed before TMEM is released.
    ptx::mma_commit_w(bar(L::FINAL));
    ptx::mbar_wait(bar(L::FINAL), 0, kWait);
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, L::kTmemCols);
  }
}

// ---------------------------------------------------------------- warp kernel
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Pair<T>::kFmt == 1)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8 x 8 matrices of 16-bit elements, a row address from each lane.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// A worker is `split` warps, each with 16 of the unit's rows, that share a
// ring of tiles (K and V of 32 keys, 128-byte swizzle).  The CTA's last warp
// fills the rings by TMA, a lane per worker, running ahead across units; no
// barrier of the CTA is in the loop.  A warp's step: S = Q K^T and O += P V as
// 16 x 8 x 16 MMAs, Q's fragments and O in registers, K and V by ldmatrix.
// With a few warps per scheduler the step is bound by its own chain of
// instructions, so loads and look-ups are kept out of it.
namespace warpk {
// The largest CTA, five workers of two warps and the loading one.  (With a bound of
// 384 the fp16 kernel spills: 61 us for 58 on own lists of 64 sequences of up to
// 2048 keys.  bf16: 56 either way, 16 sequences on 4096 + 512 keys 24.8 with 384
// and 25.0 so.)
constexpr int kMaxThreads = 352;
template <int D>
struct Ring {
  static constexpr uint32_t kHalf = kWarpKeys * 128;  // 64 dims of a tile's keys
  static constexpr uint32_t kTile = (D / 64) * kHalf;
  // 192 KB in flight per SM, shared by its workers.
  __host__ __device__ static constexpr int stages(int split) { return 192 * 1024 / (workers(split) * 2 * (int)kTile); }
  static size_t bytes(int split, int batch) {
    return workers(split) * stages(split) * (2 * kTile + 16) + sizeof(Line) + 8 + 8 * ((size_t)batch + 1) + 1024;
  }
};
}  // namespace warpk

template <typename T, int D>
__global__ void __launch_bounds__(warpk::kMaxThreads, 1)
    warp_kernel(const AiPrefixAttnArgs a, const Plan p, const int split, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v) {
  using R = warpk::Ring<D>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int KS = D / 16, NB = D / 8;  // k steps of Q K^T, 8-dim blocks of O
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = tile::align1024(smem_raw);
  const uint32_t sbase = ptx::smem_u32(sm);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, r = lane / 4, c = lane % 4;
  const int n_local = warpk::workers(split), n_warps = n_local * split;
  // (lane i of the loading warp serves the CTA's worker i)
  const int local = warp < n_warps ? warp / split : min(lane, n_local - 1);
  const int stages = R::stages(split);
  const uint32_t bars = sbase + n_local * stages * 2 * R::kTile;
  Line* s_line = reinterpret_cast<Line*>(sm + n_local * stages * (2 * R::kTile + 16));
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_line + 1);
  int* scan = const_cast<int*>(s_abort) + 2;
  int* tokens = scan + a.batch + 1;
  auto full = [&](int st) { return bars + 16u * (uint32_t)(local * stages + st); };
  auto empty = [&](int st) { return full(st) + 8; };
  if (tid == 0) {
    for (int i = 0; i < n_local * stages; ++i) {
      ptx::mbar_init(bars + 16u * i, 1);
      ptx::mbar_init(bars + 16u * i + 8, split);
    }
    *s_abort = 0;
    s_abort[1] = p.share == 0 || blockIdx.x == 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tm_k);
    ptx::prefetch_tmap(&tm_v);
  }
  if (warp == 0) {
    scan_seqs(a, p.warp, kWarpKeys, scan, tokens);
    __syncwarp();
    if (lane == 0) *s_line = active_line(a, p, false, tokens[a.batch] * p.group, tile_sms(a, p, tokens[a.batch] * p.group, scan[a.batch]));
  }
  __syncthreads();
  const int all_rows = tokens[a.batch] * p.group;
  const Line& ln = *s_line;
  if (blockIdx.x == 0)
    for (int b = tid; b <= a.batch; b += blockDim.x) {
      p.scan[b] = scan[b];
      if (ln.units_prefix > 0) p.tokens[b] = tokens[b];
    }
  const Split line = split_line(ln, line_total(ln, scan[a.batch]));
  const int worker = blockIdx.x * n_local + local;
  const bool busy = worker < line.n;
  const int w0 = busy ? line.begin(worker) : 0, w1 = busy ? line.begin(worker + 1) : 0;
  const float sl2 = a.scale * kLog2e;
  const uint32_t ring = sbase + local * stages * 2 * R::kTile;

  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
    bool ok = !*s_abort;
    if (ok && !ptx::mbar_wait(bar, parity, kWait)) {
      report(a.status, AI_ERR_DEV_TIMEOUT);
      *s_abort = 1;
      ok = false;
    }
    return __all_sync(0xffffffffu, ok);
  };

  // The combine launch waits for this one, which must not end before the tile
  // kernel (one CTA sees to that, the others make room).
  auto finish = [&]() {
    if (s_abort[1]) asm volatile("griddepcontrol.wait;" ::: "memory");
  };

  if (warp == n_warps) {
    // ------------------------------------------------------------ loads
    // Every lane walks its worker's stretch; a stage that is still in use is
    // looked at again in the next round, after the other lanes' turns.
    constexpr int CB = D / 64;
    const int box = min(a.page_size, kWarpKeys), page_bits = 31 - __clz(a.page_size);
    int w = w0, st = 0, turn = 0, j = 0;
    Seg s{};
    const int32_t* table = nullptr;
    int hk = 0;
    bool live = lane < n_local;
    auto advance = [&]() {
      s = next_seg(a, ln, scan, w, w1);
      j = 0;
      live = s.n > 0;
      table = s.b < 0 ? a.prefix_pages : a.page_table + s.b * a.page_table_stride;
      hk = s.b < 0 ? s.sub / ln.groups : s.sub;
    };
    if (live) advance();
    long long last = clock64();
    while (__any_sync(0xffffffffu, live)) {
      bool moved = false;
      if (live && (turn == 0 || ptx::mbar_test_wait(empty(st), (turn - 1) & 1))) {
        const int k0 = (s.j0 + j) * kWarpKeys;
        // (pages past the list are not read)
        const int pieces = box == kWarpKeys ? 1 : (min(kWarpKeys, s.keys - k0) + box - 1) / box;
        const uint32_t dst = ring + st * 2 * R::kTile;
        ptx::mbar_arrive_expect_tx(full(st), (uint32_t)(pieces * box * D * 4));
        for (int piece = 0; piece < pieces; ++piece) {
          const int key = k0 + piece * box, at = key & (a.page_size - 1);
          const int page = page_of(a, table, key >> page_bits);
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            const uint32_t to = dst + cb * R::kHalf + piece * box * 128;
            ptx::tma_load_4d(to, &tm_k, full(st), 64 * cb, at, hk, page);
            ptx::tma_load_4d(to + R::kTile, &tm_v, full(st), 64 * cb, at, hk, page);
          }
        }
        moved = true;
        if (++st == stages) st = 0, ++turn;
        if (++j == s.n) advance();
      }
      if (__any_sync(0xffffffffu, moved)) {
        last = clock64();
      } else if (__any_sync(0xffffffffu, *s_abort || clock64() - last > kWait)) {
        if (!*s_abort) report(a.status, AI_ERR_DEV_TIMEOUT);
        *s_abort = 1;
        break;
      }
    }
    // After a wait that gave up: the loads in flight land before the CTA ends.
    if (*s_abort && lane < n_local)
      for (int i = 0; i < stages; ++i) {
        const int turns = turn + (i < st);  // loads of stage i
        if (turns > 0) ptx::mbar_wait(full(i), (turns - 1) & 1, kWait);
      }
    finish();
    return;
  }

  // Lane's place in an 8 x 8 matrix set (K by rows, V transposed): row and
  // swizzled chunk offsets, for every second chunk of a 128-byte row.
  const int mat = lane / 8, in = lane % 8;
  const uint32_t k_row = ((mat >> 1) * 8 + in) * 128, v_row = ((mat & 1) * 8 + in) * 128;
  uint32_t k_off[4], v_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k_off[i] = k_row + (((2 * i + (mat & 1)) ^ in) << 4);
    v_off[i] = v_row + (((2 * i + (mat >> 1)) ^ in) << 4);
  }
  int st = 0;
  uint32_t turn = 0;  // parity of the stage's current load
  bool ok = true;
  for (int w = w0; w < w1 && ok;) {
    const Seg s = next_seg(a, ln, scan, w, w1);
    if (s.n == 0) break;
    const bool pre = s.b < 0;
    const int hk = pre ? s.sub / ln.groups : s.sub, in_unit = (warp % split) * 16;
    const int unit0 = pre ? (s.sub - hk * ln.groups) * ln.rows_prefix : 0, row0 = unit0 + in_unit;
    const int n_rows = min((pre ? all_rows : p.rows_seq) - unit0, pre ? ln.rows_prefix : p.rows_seq) - in_unit;  // of this warp, when positive
    const bool any = n_rows > 0;
    // Q's fragments of rows r and r + 8 (zero past the unit's rows), and the
    // keys that those rows see.
    uint32_t q[KS][4];
    int seen[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = r + 8 * h;
      const bool has = i < n_rows;
      const Row x = row_of(a, p, tokens, s.b, has ? row0 + i : 0);
      const T* src = static_cast<const T*>(a.q.ptr) + x.b * a.q.stride_b + (hk * p.group + x.g) * a.q.stride_h +
                     x.t * a.q.stride_t + 2 * c;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(src + 16 * ks + 8 * e));
          q[ks][h + 2 * e] = has ? v : 0u;
        }
      seen[h] = has ? visible(a, x, s.b < 0, s.keys) : -1;
    }
    // Tiles that end by `least` are seen whole (rows without a query see
    // whatever there is and are not stored).
    int least = min(seen[0] < 0 ? 0x7fffffff : seen[0], seen[1] < 0 ? 0x7fffffff : seen[1]);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, d));
    float o[NB][4];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
    // l takes the exponentials of one turn of the ring, l_before the turns'
    // sums: one running sum of a long list would round away its small weights
    // beside a large one (the fp32 sum's error then goes by keys / (32 stages)
    // additions, not by keys / 8).
    float l_before[2] = {0.f, 0.f};

    for (int j = s.j0; j < s.j0 + s.n; ++j) {
      const int k0 = j * kWarpKeys;
      const uint32_t kt = ring + st * 2 * R::kTile, vt = kt + R::kTile;
      if (!(ok = wait(full(st), turn))) break;
      if (any) {
        float sc[4][4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t k4[4];  // keys 16 half + 0..7 and 8..15, dims 16 ks + 0..7 and 8..15
            ldsm4(k4, kt + k_off[ks & 3] + (ks >> 2) * R::kHalf + half * 2048);
            mma16816<T>(sc[2 * half], q[ks], k4[0], k4[1]);
            mma16816<T>(sc[2 * half + 1], q[ks], k4[2], k4[3]);
          }
        // Softmax of rows r (h = 0) and r + 8 (h = 1): the lane's keys are
        // 8 nt + 2 c + {0, 1}.
        float base[2], alpha[2] = {1.f, 1.f};
        bool rescale = false;
        if (k0 + kWarpKeys > least) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int lim = seen[h] - k0 - 2 * c;
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (8 * nt + e >= lim) sc[nt][2 * h + e] = -CUDART_INF_F;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(sc[0][2 * h], sc[0][2 * h + 1]);
#pragma unroll
          for (int nt = 1; nt < 4; ++nt) mx = ptx::fmax3(mx, sc[nt][2 * h], sc[nt][2 * h + 1]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = Pair<T>::top(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)), sl2);
          // (O is rescaled only when the maximum grows by more than 2^8)
          if (mx > Pair<T>::limit(m[h])) {
            if (m[h] != -CUDART_INF_F) {
              alpha[h] = ptx::ex2(m[h] - mx);
              rescale = true;
            }
            m[h] = mx;
          }
          base[h] = m[h] == -CUDART_INF_F ? 0.f : m[h];
        }
        // Without a query among rows 8 to 15 these take what rounding P leaves of
        // rows 0 to 7, so the output is rounded once, at no cost (a second MMA
        // for it took 3 % to 6 % where rows 8 to 15 are in use).
        const bool few = !__any_sync(0xffffffffu, seen[1] >= 0);
        if (few) alpha[1] = alpha[0];
        if (__any_sync(0xffffffffu, rescale)) {
          l[0] *= alpha[0], l[1] *= alpha[1];
          l_before[0] *= alpha[0], l_before[1] *= alpha[1];
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            o[i][0] *= alpha[0], o[i][1] *= alpha[0];
            o[i][2] *= alpha[1], o[i][3] *= alpha[1];
          }
        }
        // P's fragments of keys 0..15 and 16..31, rounded to the values' type.
        uint32_t pa[2][4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          uint32_t* frag = &pa[nt >> 1][(nt & 1) * 2];
          float p0 = ptx::ex2(fmaf(sc[nt][0], sl2, -base[0])), p1 = ptx::ex2(fmaf(sc[nt][1], sl2, -base[0]));
          l[0] += p0 + p1;
          frag[0] = Pair<T>::pack(p0, p1);
          if (few) {
            const float2 rounded = Pair<T>::unpack(frag[0]);
            p0 -= rounded.x, p1 -= rounded.y;
          } else {
            p0 = ptx::ex2(fmaf(sc[nt][2], sl2, -base[1])), p1 = ptx::ex2(fmaf(sc[nt][3], sl2, -base[1]));
            l[1] += p0 + p1;
          }
          frag[1] = Pair<T>::pack(p0, p1);
        }
        const bool ragged = k0 + kWarpKeys > s.keys;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          // Slots past the list hold anything, NaN included, and meet P = 0:
          // their values are cleared.
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (ragged) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int left = s.keys - (k0 + 16 * kk + 8 * e + 2 * c);
              keep[e] = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
            }
          }
#pragma unroll
          for (int i = 0; i < NB; i += 2) {
            uint32_t v4[4];  // keys 16 kk + 0..7 and 8..15 of dims 8 i + 0..7, then of 8 (i + 1) + 0..7
            ldsm4_t(v4, vt + v_off[(i >> 1) & 3] + (i >> 3) * R::kHalf + kk * 2048);
            if (ragged) v4[0] &= keep[0], v4[1] &= keep[1], v4[2] &= keep[0], v4[3] &= keep[1];
            mma16816<T>(o[i], pa[kk], v4[0], v4[1]);
            mma16816<T>(o[i + 1], pa[kk], v4[2], v4[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(empty(st));
      if (++st == stages) {
        st = 0, turn ^= 1;
        l_before[0] += l[0], l_before[1] += l[1];
        l[0] = l[1] = 0.f;
      }
    }
    if (!ok) break;
    if (!__any_sync(0xffffffffu, seen[1] >= 0)) {
#pragma unroll
      for (int i = 0; i < NB; ++i) o[i][0] += o[i][2], o[i][1] += o[i][3];
    }
    // Partial rows: the lane's dims 8 i + 2 c + {0, 1} of rows r and r + 8.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = l_before[h] + l[h];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (seen[h] < 0) continue;
      const int64_t slot = s.unit + worker;
      const int64_t row = (s.b < 0 ? ln.base_prefix + slot * ln.slot_prefix
                                   : ln.base_own + slot * ln.rows_own) + in_unit + r + 8 * h;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int i = 0; i < NB; ++i)
        *reinterpret_cast<float2*>(p.part_o + row * D + 8 * i + 2 * c) = make_float2(o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
      if (c == 0) p.part_lse[row] = part_lse(sum, m[h] + log2f(sum));
    }
  }
  finish();
}

// ---------------------------------------------------------------- combine
// `wide` warps per (sequence, query token, query head) join the partial
// results of the row's prefix and own stretches: each takes every wide-th of
// them, and the first adds up the warps' sums in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(const AiPrefixAttnArgs a, const Plan p, const int wide) {
  constexpr int E = D / 32;
  __shared__ float s_acc[8][D + 2];
  const int b = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32, part = warp % wide;
  const int item = blockIdx.x * (8 / wide) + warp / wide;
  const bool has = item < a.seq_len * a.num_q_heads;
  const int t = has ? item / a.num_q_heads : 0, h = has ? item % a.num_q_heads : 0, hk = h / p.group;
  const int rem = t * p.group + h % p.group;
  const bool real = has && t < seq_lens(a, b).n;  // (the caller's lengths: read before the wait)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float M = -CUDART_INF_F, sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (real) {
    // (without room for own keys neither kernel has written the scan)
    const bool own = a.max_pages > 0, pre = a.prefix_len > 0;
    const int s0 = own ? p.scan[b] : 0, size = own ? p.scan[b + 1] - s0 : 0, own_all = own ? p.scan[a.batch] : 0;
    const int all_rows = pre ? p.tokens[a.batch] * p.group : 0, sms = p.share > 0 ? p.tokens[a.batch + 1] : 0;
    int64_t row[2] = {0, 0}, step[2] = {0, 0};
    int n[2] = {0, 0};
    if (pre) {
      const Line l = active_line(a, p, !p.prefix_warp, all_rows, sms);
      const int all = p.tokens[b] * p.group + rem, grp = all / l.rows_prefix, unit = hk * l.groups + grp;
      const Split line = split_line(l, line_total(l, own_all));
      const int x = unit * (l.start + l.tiles_prefix) + l.start, first = line.worker(x);
      n[0] = line.worker(x + l.tiles_prefix - 1) - first + 1;
      step[0] = l.slot_prefix;
      row[0] = l.base_prefix + (unit + first) * step[0] + all - grp * l.rows_prefix;
    }
    if (size > 0) {
      const Line l = active_line(a, p, !p.own_warp, all_rows, sms);
      const int grp = rem / l.rows_own, sub = grp * a.num_kv_heads + hk, unit = b * l.per_seq + sub;
      const Split line = split_line(l, line_total(l, own_all));
      const int x = l.units_prefix * (l.start + l.tiles_prefix) + s0 * l.per_seq + sub * size + l.start;
      const int first = line.worker(x);
      n[1] = line.worker(x + size - l.start - 1) - first + 1;
      step[1] = l.rows_own;
      row[1] = l.base_own + (unit + first) * step[1] + rem - grp * l.rows_own;
    }
    const int all_n = n[0] + n[1];
    auto row_at = [&](int i) { return i < n[0] ? row[0] + i * step[0] : row[1] + (i - n[0]) * step[1]; };
    for (int i = lane; i < all_n; i += 32) M = fmaxf(M, p.part_lse[row_at(i)]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    if (M != -CUDART_INF_F) {
      for (int i0 = part; i0 < all_n; i0 += 32 * wide) {
        const int mine = i0 + lane * wide;
        const float my_wgt = mine < all_n ? exp2f(p.part_lse[row_at(mine)] - M) : 0.f;
        const int cnt = min(32, (all_n - i0 + wide - 1) / wide);
#pragma unroll 4
        for (int k = 0; k < cnt; ++k) {
          const float wgt = __shfl_sync(0xffffffffu, my_wgt, k);
          const float* src = p.part_o + row_at(i0 + k * wide) * D + E * lane;
          float o[E];
          if constexpr (E == 4)
            *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(src);
          else
            *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(src);
          sum += wgt;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(wgt, o[e], acc[e]);
        }
      }
    }
  }
  if (wide > 1) {
    if (part > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) s_acc[warp][E * lane + e] = acc[e];
      if (lane == 0) s_acc[warp][D] = sum;
    }
    __syncthreads();
    if (part > 0) return;
    for (int k = 1; k < wide; ++k) {
      sum += s_acc[warp + k][D];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += s_acc[warp + k][E * lane + e];
    }
  }
  if (!has) return;
  T* o = static_cast<T*>(a.out.ptr) + b * a.out.stride_b + h * a.out.stride_h + t * a.out.stride_t + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f32<T>(sum == 0.f ? 0.f : acc[e] / sum);
  if (lane == 0 && a.lse)
    a.lse[((int64_t)b * a.num_q_heads + h) * a.seq_len + t] =
        sum == 0.f ? -CUDART_INF_F : (M + log2f(sum)) * kLn2;
}

// ---------------------------------------------------------------- host
// Warps of a warp-kernel worker for units of `rows` rows.
int warp_split(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// The launches' shape and the workspace's layout; false when the sizes do not fit.
bool make_plan(const AiPrefixAttnArgs& a, Plan* p, size_t* bytes) {
  *p = Plan{};
  const int64_t G = a.num_q_heads / a.num_kv_heads, rows = G * a.seq_len, all = rows * a.batch, H = a.num_kv_heads;
  const int64_t capacity = (int64_t)a.max_pages * a.page_size;
  if (all > 0x7fffffff || a.batch * rows * H > 0x7fffffff) return false;
  p->group = (int)G;
  p->rows_seq = (int)rows;
  p->own_warp = rows <= kWarpRows;
  p->split = warp_split(rows);
  const int sms = sm_count(), workers = sms * warpk::workers(p->split);
  // A prefix goes with the sequences' own keys to the warp kernel, in groups
  // of rows that read it again each, while that gives a worker few positions
  // (a launch of the tile kernel costs as much).
  const int64_t group_rows = 16 * p->split, groups = (all + group_rows - 1) / group_rows;
  p->prefix_warp = p->own_warp && groups * H * (kStartWarp + (a.prefix_len + kWarpKeys - 1) / kWarpKeys) <=
                                      (int64_t)kShortPrefix * workers;
  int64_t at = 0;  // rows of the partial results so far
  // (most: rows of a prefix unit at most; own: rows and units of a sequence)
  auto line = [&](Line& l, bool prefix, bool own, int keys, int64_t most_unit, int64_t per_seq, int64_t rows_own,
                  int64_t workers, int start, int least) {
    const int64_t tiles = ((int64_t)a.prefix_len + keys - 1) / keys;
    l.tiles_prefix = (int)tiles;
    l.slot_prefix = (int)(all < most_unit ? all : most_unit);
    l.units_prefix = prefix && tiles > 0 ? (int)((all + most_unit - 1) / most_unit * H) : 0;
    l.per_seq = own ? (int)per_seq : 0;
    const int64_t most_own = (capacity + keys - 1) / keys;
    const int64_t most = l.units_prefix * (start + tiles) +
                         a.batch * (int64_t)l.per_seq * (most_own > 0 ? start + most_own : 0);
    if (most > 0x7fffffff) return false;
    const int64_t want = (most + least - 1) / least;
    l.workers = (int)(want < workers ? want : workers);
    l.least = least;
    l.start = start;
    l.rows_own = (int)rows_own;
    if (l.units_prefix > 0) {
      l.base_prefix = at;
      at += (int64_t)(l.units_prefix + l.workers) * l.slot_prefix;
    }
    if (l.per_seq > 0) {
      l.base_own = at;
      at += (a.batch * (int64_t)l.per_seq + l.workers) * rows_own;
    }
    return true;
  };
  p->nt = (a.prefix_len > 0 ? all : rows) > BM ? 2 : 1;
  const int64_t most_unit = BM * p->nt, tt = (rows + most_unit - 1) / most_unit;
  // Own keys join the tile kernel's line when there is room for few of them
  // and the kernel runs anyway: a launch less.
  const int BN = tile_keys(p->nt);
  if (!p->prefix_warp && a.batch * H * tt * (kStartTile + (capacity + BN - 1) / BN) <=
                             (int64_t)kFewOwn * (p->nt == 1 ? 2 * sms : sms))
    p->own_warp = false;
  // (256 rows x 128 keys outweigh a start, so a short line spreads over all
  // SMs: 39 us with one position a CTA at least, 44 with five, 64 sequences on
  // 2048 + 256 keys.  64-key tiles: no difference beyond 1 us.)
  if (!line(p->tile, !p->prefix_warp, !p->own_warp, BN, most_unit, tt * H, (rows + tt - 1) / tt,
            p->nt == 1 ? 2 * sms : sms, kStartTile, p->nt == 1 ? kStartTile + 1 : 1))
    return false;
  if (!line(p->warp, p->prefix_warp, p->own_warp, kWarpKeys, group_rows, H, rows, workers, kStartWarp, 2)) return false;
  // A 256-row tile CTA fills its SM and leaves HBM idle; the warp kernel streams
  // as fast from three quarters of the SMs as from all.  So they run side by
  // side (one after the other / so, bf16, 64 sequences of one token: 110 / 95 us
  // on 32,768 + 2048 keys, 38 / 32 on 2048 + 256; five tokens: 193 / 183 and
  // 51 / 48 on 4096 + 5).  A tile position costs about 8 positions of the warp
  // kernel, 11 with head_dim 64 (its CTA is bound by exponentials, theirs by
  // bytes), fewer where a warp kernel position has several warps' rows (at 6 /
  // 8 / 11: 109 / 96 / 100 us and 184 / 213 / 262 on the two largest above;
  // head_dim 64 at 8 / 11 / 14: 73 / 66 / 72 us on 32,768 + 2048, 153 / 146 / 158
  // with five tokens, 26.0 / 25.5 / 25.9 on 2048 + 256, but three tokens on 30,000
  // + 300 99 / 101 / 128).
  if (p->nt == 2 && p->tile.workers > 0 && p->tile.per_seq == 0 && p->warp.workers > 0) {
    p->share = sms;
    p->tile_cost = (a.head_dim == 128 ? 8 : 11) * (p->split == 1 ? 4 : 3) / 4;
  }
  char* ws = static_cast<char*>(a.workspace);
  size_t off = 0;
  auto take = [&](size_t want) {
    char* q = ws + off;
    off += (want + 255) & ~size_t(255);
    return q;
  };
  p->part_o = reinterpret_cast<float*>(take((size_t)at * a.head_dim * 4));
  p->part_lse = reinterpret_cast<float*>(take((size_t)at * 4));
  p->scan = reinterpret_cast<int*>(take(((size_t)a.batch + 1) * 4));
  p->tokens = reinterpret_cast<int*>(take(((size_t)a.batch + 2) * 4));
  *bytes = off;
  return true;
}

template <typename T, int D>
int launch_t(const AiPrefixAttnArgs& a, const Plan& p, cudaStream_t st) {
  ProfScope ps(AI_PROF_PREFIX, st);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 0;  // the first launch follows whatever ran before in full
  CUtensorMap tk, tv;
  auto maps = [&](int keys) {
    const int box = a.page_size < keys ? a.page_size : keys;
    return sm100_make_map_of(&tk, a.k_pages, a.n_pages, a.num_kv_heads, a.page_size, box, D, a.dtype) &&
           sm100_make_map_of(&tv, a.v_pages, a.n_pages, a.num_kv_heads, a.page_size, box, D, a.dtype);
  };
  // (the limit is the kernel's, not the call's: always all that there is, so that calls of
  // other threads never find it lower than they need)
  auto smem_of = [&](auto kernel, size_t bytes) {
    cfg.dynamicSmemBytes = bytes;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) == cudaSuccess;
  };
  if (p.tile.workers > 0) {
    if (!maps(tile_keys(p.nt))) return AI_ERR_TMA;
    cfg.gridDim = dim3(p.tile.workers);
    cfg.blockDim = dim3(tile_threads(p.nt));
    const bool ok = p.nt == 1 ? smem_of(tile_kernel<T, D, 1>, Smem<D, 1>::bytes(a.batch)) &&
                                    cudaLaunchKernelEx(&cfg, tile_kernel<T, D, 1>, a, p, tk, tv) == cudaSuccess
                              : smem_of(tile_kernel<T, D, 2>, Smem<D, 2>::bytes(a.batch)) &&
                                    cudaLaunchKernelEx(&cfg, tile_kernel<T, D, 2>, a, p, tk, tv) == cudaSuccess;
    if (!ok) return AI_ERR_LAUNCH;
    cfg.numAttrs = 1;
  }
  if (p.warp.workers > 0) {
    const int split = p.split, per = warpk::workers(split);
    if (!maps(kWarpKeys)) return AI_ERR_TMA;
    if (!smem_of(warp_kernel<T, D>, warpk::Ring<D>::bytes(split, a.batch))) return AI_ERR_LAUNCH;
    cfg.gridDim = dim3((p.warp.workers + per - 1) / per);
    cfg.blockDim = dim3(32 * (split * per + 1));
    if (cudaLaunchKernelEx(&cfg, warp_kernel<T, D>, a, p, split, tk, tv) != cudaSuccess) return AI_ERR_LAUNCH;
    cfg.numAttrs = 1;
  }
  // Warps per row: one for every four partial results, while the rows leave
  // the GPU's warps idle.
  const Line& lp = p.prefix_warp ? p.warp : p.tile;
  const int64_t rows = (int64_t)a.batch * a.seq_len * a.num_q_heads;
  const int parts = lp.units_prefix > 0 ? lp.workers / lp.units_prefix : 1;
  int wide = 1;
  while (wide < 8 && 4 * wide < parts && 2 * wide * rows <= 32 * (int64_t)sm_count()) wide *= 2;
  const int per = 8 / wide;
  cfg.gridDim = dim3((unsigned)((a.seq_len * a.num_q_heads + per - 1) / per), a.batch);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, combine_kernel<T, D>, a, p, wide) != cudaSuccess) return AI_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? AI_OK : AI_ERR_LAUNCH;
}

}  // namespace tc

bool sm100_fits(const AiPrefixAttnArgs& a) {
  if (a.dtype != AI_DTYPE_BF16 && a.dtype != AI_DTYPE_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  if (a.page_size < 16 || (a.page_size & (a.page_size - 1)) || a.batch > tc::kMaxBatch) return false;
  if (!(a.scale > 0.f)) return false;  // the row maximum is taken before the scale
  for (const AiTensor4* t : {&a.q, &a.k_pages, &a.v_pages}) {
    // 16-byte rows: what a tensor map and the loads of Q ask for
    if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) || ((t->stride_b | t->stride_h | t->stride_t) & 7)) return false;
    if (t == &a.q) continue;
    if (t->stride_b <= 0 || t->stride_h <= 0 || t->stride_t <= 0) return false;
  }
  tc::Plan p;
  size_t bytes;
  return tc::make_plan(a, &p, &bytes);
}

size_t sm100_workspace(const AiPrefixAttnArgs& a) {
  tc::Plan p;
  size_t bytes = 0;
  tc::make_plan(a, &p, &bytes);
  return bytes;
}

int sm100_launch(const AiPrefixAttnArgs& a, cudaStream_t st) {
  tc::Plan p;
  size_t bytes;
  if (!tc::make_plan(a, &p, &bytes)) return AI_ERR_SHAPE;
  if (!a.workspace || a.workspace_bytes < bytes) return AI_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) & 255) return AI_ERR_ALIGN;
  if (a.dtype == AI_DTYPE_BF16)
    return a.head_dim == 128 ? tc::launch_t<__nv_bfloat16, 128>(a, p, st) : tc::launch_t<__nv_bfloat16, 64>(a, p, st);
  return a.head_dim == 128 ? tc::launch_t<__half, 128>(a, p, st) : tc::launch_t<__half, 64>(a, p, st);
}

}  // namespace prefix
}  // namespace ai
