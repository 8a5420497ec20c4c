// Attention of drafted-token trees on the 5th-generation tensor cores
// (tcgen05 + TMA), sm_100a: head dim 64 or 128, pages of a multiple of 8.
//
// The rows of one request share its context, and the query heads of one KV
// head share its keys, so the M dimension of both products is (row, head of
// the group): R = 128 / group rows make one tile of 128, against tiles of 128
// tokens:
//   S[128 x 128] = Q K^T        (A, B from shared memory, D in TMEM)
//   P = exp2(scale log2e (S - m)),  running maximum m and sum l in registers
//   O[128 x d] += P V           (A from TMEM, B from shared memory, D in TMEM)
// Two softmax warpgroups work on S tiles of their own while the tensor core
// runs the other's products.  DUAL (more rows than one tile holds): each has
// rows of its own and both read the same key and value tiles.  Otherwise both
// have the same rows and take alternate token tiles, joined at the end; with
// heads of 64, up to 64 rows lie in the lower half of the first warpgroup's S and the upper
// half of the second's, so that the two compute on different schedulers (61
// single rows of heads of 64: 107 -> 99 us).
//
// Roles: warp 0 loads query, key and value tiles page by page with TMA into a
// ring; one lane of warp 1 issues all tensor-core work; warps 2-5 and 6-9
// are the softmax warpgroups, one thread per row of S (a TMEM lane).
//  * The maximum that p is taken against moves only when a tile's p add up to
//    more than 2^8 (rescaling O costs a round trip through TMEM), which also
//    bounds each of them, and no tile but a piece's first needs its maximum
//    taken.  p keeps its relative precision in bf16.  fp16 has no such range:
//    there p, and with it l and O, is taken 2^7 times as large (at most 2^15),
//    so that its last bit is 2^-31 of the maximum, and what 2^20 tokens lose
//    below it at most half an output's rounding.
//  * P overwrites its S tile, two values to a column.
//  * Tiles that lie wholly before the drafted tokens on mapped pages carry no
//    mask.  In the others each row forms its 128 mask bits, values of tokens
//    that may not be read are zeroed in shared memory (0 * NaN is NaN), and
//    infinite or NaN values of drafted tokens are zeroed and remembered: the
//    rows that see them add them at the end.
//
// Work split.  All (request, KV head, row tile) units, each of its number of
// token tiles, form one line that is cut into equal ranges; a unit cut between
// ranges leaves partial results that a second kernel joins in a fixed order.
// When a request has several row tiles, `cohort` CTAs take the same range of
// tokens with a row tile each, so that the keys and values one brings from
// memory the others find in L2.
//
// Measured on a B200, in long runs (the power limit then holds the clocks near
// 1.5 GHz).  64 requests of 8k-32k tokens, trees of 16, 32 query heads over 4
// KV heads of 128 (memory-bound): 507 us, 5.3 TB/s of keys and values, 82% of
// a copy's rate; without the softmax arithmetic 485 us.  8 requests of 131072
// tokens, trees of 64 (twice 128 rows a KV head and CTA pair): 1110 us, 0.97
// PFLOP/s; without the softmax arithmetic 916.  There a CTA's two row tiles
// spend 3400 cycles on a tile of tokens: 2048 of the tensor core, 2400 of the
// two softmax passes (2048 of it the special-function unit), which overlap in
// part, as a row tile's next scores wait for its P V: TMEM holds two S and two
// O tiles and no more.  Taking every tile's maximum beside its exponentials
// cost 1147 and 522 us; exponentials by a polynomial on the multiply-add pipe,
// a quarter of them, gained nothing (issue slots run out first).
//
// Every wait is bounded; on expiry the error word is set, the CTA stops
// issuing work, waits (bounded) for its own copies and products, frees its
// TMEM and returns.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace qsa {
namespace {

// 10 warps, at most three to a scheduler: 168 registers a thread, which the
// softmax threads fill.  Held whole, a row's 128 scores spilled in the tile
// loop, and a spill goes to L2, as shared memory leaves hardly any L1: 1520 us
// then, 490 since.  36 to 44 bytes a thread are spilled still.
constexpr int kTreeThreads = 320;
constexpr int kTile = 128;          // tokens per tile, and rows per row tile
constexpr int kMetaRing = 8;
constexpr int kTmemCols = 512;      // S0 S1 O0 O1
constexpr float kMostSum = 256.0f;  // of a tile's p against a maximum that stays
template <bool F16> constexpr float kLift = F16 ? 7.0f : 0.0f;  // log2 of the factor on p
constexpr int64_t kMinTiles = 2;    // token tiles that a CTA takes at least

// What the merge kernel learns of a range that begins inside a unit.
struct PieceInfo {
  int64_t total;  // tiles of all units
  int64_t base;   // first tile of the unit
  int tiles;      // tiles of the unit
  int row0, count;  // the request's packed rows
  int h, grp;
  int ranges;       // ranges in use
  int valid;
};

struct TreeGeometry {
  int rows_per_tile;  // R: packed rows of one row tile
  FastDiv group_div;
  int cohort, cohorts;
  int box_rows;       // token rows of one TMA box (divides the page and the tile)
  PieceInfo* info;    // [cohorts * cohort]
  float* part_o;      // [cohorts * cohort][2][rows][dim]
  float* part_lse;    // [cohorts * cohort][2][rows], log2
};

template <int D, bool DUAL>
struct TreeCfg {
  static constexpr int kSub = D / 64;                 // 128-byte columns of a row
  static constexpr int kSubBytes = kTile * 128;       // 16 KB
  static constexpr int kTileBytes = kSub * kSubBytes;
  static constexpr int kStreams = DUAL ? 2 : 1;       // row tiles
  // Up to 64 rows of a single row tile, shifted apart: room for the second
  // warpgroup's O.  Not for head dim 128, where it would cost a sixth of the
  // ring (475 -> 550 us for the first shape above, in short runs).
  static constexpr bool kApart = !DUAL && D == 64;
  static constexpr int kXchgBytes = kApart ? 64 * D * 4 : 16;
  static constexpr int kFit =
      (224 * 1024 - kStreams * kTileBytes - (kApart ? kXchgBytes : 0)) / kTileBytes;
  static constexpr int S = kFit > 10 ? 10 : kFit;
  // Values follow their keys by kLag tiles through the ring.  With alternate
  // tiles the product with the values of tile j comes between the scores of
  // tiles j + 1 and j + 2; loaded beside their keys they would hold their
  // places, and those of the keys behind them, for two tiles (487 us instead
  // of 475 for the first shape above, in short runs; two tiles later they are no better).
  static constexpr int kLag = DUAL ? 0 : 1;
  static __device__ __forceinline__ int key_pos(int n) { return n < kLag ? n : 2 * n - kLag; }
  static __device__ __forceinline__ int value_pos(int n) { return 2 * n + kLag + 1; }
  static constexpr int kRows = kStreams * kTile;
};

// A unit's part inside a CTA's range, handed by the producer to the others.
struct TreePiece {
  TreeRequest r;
  int b, h;
  int first;   // the CTA's first row of the request
  int region;  // tokens from here on are not seen by all of its rows
  int t0, t1;  // token tiles
  int tiles;   // of the whole unit
  int shift;   // the second warpgroup's first row of S (single row tile)
  int end;     // no more pieces
};
// A piece's slot is written again four pieces later, when the products of the
// piece three later have been issued and its softmax is two pieces past it.
constexpr int kPieceRing = 4;

template <int D, bool DUAL>
struct TreeSmem {
  using C = TreeCfg<D, DUAL>;
  alignas(1024) uint8_t ring[C::S][C::kTileBytes];    // key and value tiles, 128B-swizzled
  alignas(1024) uint8_t q[C::kStreams][C::kTileBytes];
  uint64_t full[C::S], empty[C::S], q_full, q_empty, s_full[2], p_ready[2], o_full[2];
  uint64_t vsync, xchg[2], drain, piece_full[kPieceRing];
  TreePiece piece[kPieceRing];
  alignas(16) uint32_t meta[kMetaRing][4];  // tokens of the tile that exist on mapped pages
  float2 ml[kTile];              // (m, l) of the second softmax warpgroup
  float xo[C::kXchgBytes / 4];   // [column][row]: its O, when its rows are shifted
  int64_t scan[kTreeThreads / 32];
  int64_t first_base;
  TreeRequest first_r;           // of the range's first tile
  int first_b;
  int bad[2];                    // number of the piece that met infinite or NaN values
  uint32_t tmem_base;
  int abort_flag;
};

// ---------------------------------------------------------------- the work
// The packed rows, group of units and token tiles that a CTA is at.
struct TreeUnit {
  int b, h, grp, groups, tiles;
  int64_t base;
  TreeRequest r;
};

__device__ __forceinline__ int unit_tiles(const TreeParams& p, const TreeRequest& r, int grp,
                                          int span) {
  int end = r.tokens;
  if (p.mask == nullptr) end = min(end, r.prefix + min(r.count, (grp + 1) * span));
  return max(1, (end + kTile - 1) / kTile);
}

__device__ __forceinline__ int64_t head_tiles(const TreeParams& p, const TreeRequest& r, int span) {
  const int groups = (r.count + span - 1) / span;
  if (groups == 0) return 0;
  if (p.mask != nullptr) return static_cast<int64_t>(groups) * unit_tiles(p, r, 0, span);
  int64_t n = 0;
  for (int g = 0; g < groups; ++g) n += unit_tiles(p, r, g, span);
  return n;
}

__device__ __forceinline__ void unit_first(const TreeParams& p, TreeUnit& u, int span) {
  u.h = u.grp = 0;
  u.groups = (u.r.count + span - 1) / span;
  u.tiles = unit_tiles(p, u.r, 0, span);
}

// Enters request b (or the next with rows); false past the last.
__device__ __forceinline__ bool unit_enter(const TreeParams& p, TreeUnit& u, int span) {
  for (; u.b < p.requests; ++u.b) {
    u.r = tree_request_info(p, u.b);
    if (u.r.count == 0) continue;
    unit_first(p, u, span);
    return true;
  }
  return false;
}

__device__ __forceinline__ bool unit_next(const TreeParams& p, TreeUnit& u, int span) {
  u.base += u.tiles;
  if (++u.grp == u.groups) {
    u.grp = 0;
    if (++u.h == p.kv_heads) {
      ++u.b;
      return unit_enter(p, u, span);
    }
  }
  u.tiles = unit_tiles(p, u.r, u.grp, span);
  return true;
}

// The unit that holds tile `begin`, from the request that holds it.
__device__ __forceinline__ bool unit_seek(const TreeParams& p, TreeUnit& u, const TreeRequest& r,
                                          int b, int64_t base, int64_t begin, int span) {
  u.r = r;
  u.b = b;
  u.base = base;
  unit_first(p, u, span);
  const int64_t per_head = head_tiles(p, u.r, span);
  u.h = static_cast<int>((begin - base) / per_head);
  u.base += u.h * per_head;
  while (u.base + u.tiles <= begin)
    if (!unit_next(p, u, span)) return false;
  return true;
}

// ------------------------------------------------------------- tensor cores
template <bool F16, int N, bool B_MN>
constexpr uint32_t tree_idesc() {
  const uint32_t fmt = F16 ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((B_MN ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

// Descriptor of a value tile as the B operand of P V: tokens (K) are rows of
// 128 bytes, so the operand is MN-major in the 128-byte swizzle: 8-token atoms
// 1024 B apart (stride), 64-column chunks one sub-tile apart (leading).
__device__ __forceinline__ uint64_t value_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((kTile * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// A place in the ring of key and value tiles, which alternate.
struct RingPos {
  int slot;
  uint32_t phase;
  template <int S>
  __device__ __forceinline__ void step(int n) {
    slot += n;
    if (slot >= S) {
      slot -= S;
      phase ^= 1;
    }
  }
};

// D += A(TMEM) * B(shared memory).
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                        uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1 : 0)
      : "memory");
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    return pack_bf16x2(lo, hi);
  }
}
template <bool F16>
__device__ __forceinline__ float unpack(uint16_t x) {
  if constexpr (F16) return __half2float(__ushort_as_half(x));
  else return __uint_as_float(static_cast<uint32_t>(x) << 16);
}

// ------------------------------------------------------------------ softmax
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A row's highest score.
__device__ __forceinline__ float row_max(uint32_t ts) {
  float high = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t s[32];
    tmem_ld32(ts + k * 32, s);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; e += 2)
      high = max3(high, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
  }
  return high;
}

// The exponentials of a row's 128 scores against m, times 2^kLift, as 16-bit
// pairs in pk; returns their sum in 32 bits.  The special-function unit takes 8 cycles for
// a warp's exponential, 1024 for the row; the rest is issued beside it.
template <bool F16>
__device__ __forceinline__ float score_pass(uint32_t ts, float c, float m, uint32_t* pk) {
  const float shift = m == -INFINITY ? 0.0f : fmaf(-m, c, kLift<F16>);
  const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift);
  float2 sum = make_float2(0.0f, 0.0f);
  uint32_t s[2][32];
  tmem_ld32(ts, s[0]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    tmem_wait_ld();
    if (k < 3) tmem_ld32(ts + (k + 1) * 32, s[(k + 1) & 1]);
    uint32_t* v = s[k & 1];
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float2 x = fma2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), c2, shift2);
      x.x = fast_exp2(x.x);
      x.y = fast_exp2(x.y);
      sum = add2(sum, x);
      pk[k * 16 + e / 2] = pack2<F16>(x.x, x.y);
    }
  }
  return sum.x + sum.y;
}

// Clears the bits of tile t's columns that row i0 + local of the request does
// not see.  Collective over the warp.
__device__ __forceinline__ void row_mask(uint32_t (&w)[4], const TreeParams& p,
                                         const TreeRequest& r, int t, int i0, int local, int R,
                                         int lane) {
  const int node0 = t * kTile - r.prefix;  // drafted token of column 0
  if (p.mask == nullptr) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int see = i0 + local - node0 - k * 32 + 1;  // columns of this word that are seen
      w[k] &= see >= 32 ? 0xffffffffu : see <= 0 ? 0u : (1u << see) - 1;
    }
    return;
  }
  // the distinct rows of this warp, one after another: 128 mask bytes read
  // side by side, turned into bits by ballots
  const int lo = __shfl_sync(0xffffffffu, local, 0);
  const int hi = min(__shfl_sync(0xffffffffu, local, 31), R - 1);
  uint32_t sees[4] = {0u, 0u, 0u, 0u};
  for (int k = lo; k <= hi; ++k) {
    if (i0 + k >= r.count) break;
    const uint8_t* bytes = p.mask + (r.row0 + i0 + k) * p.mask_stride;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int node = node0 + q * 32 + lane;
      const bool see = node < 0 || (node < p.mask_width && bytes[node] != 0);
      const uint32_t bits = __ballot_sync(0xffffffffu, see);
      if (k == local) sees[q] = bits;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] &= sees[k];
}

// --------------------------------------------------------------- the kernel
template <int D, bool DUAL, bool F16>
__global__ void __launch_bounds__(kTreeThreads, 1)
tree_attention_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ TreeGeometry g,
                      const __grid_constant__ CUtensorMap qmap,
                      const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap) {
  using C = TreeCfg<D, DUAL>;
  extern __shared__ uint8_t smem_raw[];
  TreeSmem<D, DUAL>& sm = *reinterpret_cast<TreeSmem<D, DUAL>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cohort_id = blockIdx.x / g.cohort, member = blockIdx.x - cohort_id * g.cohort;
  const int R = g.rows_per_tile;
  const int span = R * C::kStreams * g.cohort;  // packed rows of one group of units

  if (tid == 0) {
    for (int s = 0; s < C::S; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.p_ready[s], 4);
      mbar_init(&sm.o_full[s], 1);
      mbar_init(&sm.xchg[s], kTile);
      sm.bad[s] = -1;
    }
    for (int s = 0; s < kPieceRing; ++s) mbar_init(&sm.piece_full[s], 1);
    mbar_init(&sm.vsync, 2 * kTile);
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    sm.first_b = -1;
    fence_mbar_init();
  }
  if (tid == 32) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  pdl_wait();
  pdl_trigger();

  // This cohort's range of the line of tiles: each thread adds up a run of
  // requests, the block scans the runs, and the thread whose run holds the
  // range's first tile names its request.
  const int per = (p.requests + kTreeThreads - 1) / kTreeThreads;
  int64_t mine = 0;
  TreeRequest info_r{};  // of the run's last request: of all of it, for up to 320 requests
  for (int k = 0; k < per; ++k) {
    const int b = tid * per + k;
    if (b >= p.requests) break;
    info_r = tree_request_info(p, b);
    mine += p.kv_heads * head_tiles(p, info_r, span);
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sm.scan[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kTreeThreads / 32; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  before += incl - mine;
  const int64_t most = (total + kMinTiles - 1) / kMinTiles;
  const int ranges = static_cast<int>(most < g.cohorts ? most : g.cohorts);
  const bool idle = cohort_id >= ranges;
  const int64_t begin = idle ? 0 : total * cohort_id / ranges;
  const int64_t end = idle ? 0 : total * (cohort_id + 1) / ranges;
  if (idle) {  // the whole block
    if (tid == 0) g.info[blockIdx.x].valid = 0;
    return;
  }
  if (before <= begin && begin < before + mine) {
    int64_t at = before;
    for (int k = 0; k < per; ++k) {
      const int b = tid * per + k;
      if (per > 1 && b < p.requests) info_r = tree_request_info(p, b);
      const int64_t n =
          per == 1 ? mine : b < p.requests ? p.kv_heads * head_tiles(p, info_r, span) : 0;
      if (begin < at + n) {
        sm.first_b = b;
        sm.first_base = at;
        sm.first_r = info_r;
        break;
      }
      at += n;
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sm.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const uint32_t tmem_s[2] = {tmem, tmem + 128}, tmem_o[2] = {tmem + 256, tmem + 384};

  bool ok = true;
  auto give_up = [&]() {
    record_error(p.err, kDeviceErrWaitTimeout);
    *reinterpret_cast<volatile int*>(&sm.abort_flag) = 1;
  };
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&sm.abort_flag)) return false;
    return mbar_wait(bar, parity);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int n = 0, piece = 0;  // tiles and pieces so far
    const int boxes = kTile / g.box_rows;
    const uint32_t box_bytes = g.box_rows * 128;
    TreeUnit u;
    bool more = unit_seek(p, u, sm.first_r, sm.first_b, sm.first_base, begin, span);
    if (lane == 0) {
      PieceInfo info = {total, u.base, u.tiles, u.r.row0, u.r.count, u.h, u.grp, ranges,
                        begin > u.base};
      g.info[blockIdx.x] = info;
    }
    struct Place {  // this lane's box of a tile
      int page, at, h;
    };
    Place past[C::kLag > 0 ? C::kLag : 1] = {};  // of the tiles whose values are to come
    auto load = [&](const CUtensorMap* map, int pos, const Place& x) {
      const int slot = pos % C::S;
      ok = __all_sync(0xffffffffu, wait(&sm.empty[slot], ((pos / C::S) & 1) ^ 1));
      if (!ok) return;
      if (lane == 0) mbar_arrive_expect(&sm.full[slot], C::kTileBytes);
      __syncwarp();
      if (lane < boxes) {
        uint8_t* dst = sm.ring[slot] + lane * box_bytes;
#pragma unroll
        for (int c = 0; c < C::kSub; ++c)
          tma_load_4d(dst + c * C::kSubBytes, map, c * 64, x.h, x.at,
                      x.page >= 0 ? x.page : p.num_blocks, &sm.full[slot]);
      }
    };
    for (;; ++piece) {
      more = more && u.base < end;
      const int t0 = static_cast<int>(max(begin - u.base, static_cast<int64_t>(0)));
      const int t1 = static_cast<int>(min(end - u.base, static_cast<int64_t>(u.tiles)));
      const int first = (u.grp * g.cohort + member) * C::kStreams * R;
      const int32_t* table = p.table + (more ? u.b : 0) * p.table_stride;
      auto page_of = [&](int tile, int& at) {
        const int t = tile * kTile + lane * g.box_rows;
        int q;
        p.page_div.divmod(t, q, at);
        return lane < boxes && t < u.r.tokens ? ld_once(table + q) : -1;
      };
      // the queries, once those of the piece before have been used: behind the
      // first keys, as the last values of that piece come with them
      bool handed = false;
      auto hand_over = [&]() {
        handed = true;
        ok = __all_sync(0xffffffffu, wait(&sm.q_empty, (piece & 1) ^ 1));
        if (!ok) return;
        if (lane == 0) {
          const int region =
              max(p.mask != nullptr ? u.r.prefix : u.r.prefix + first + 1, 0);
          sm.piece[piece % kPieceRing] =
              TreePiece{u.r, u.b, u.h, first, region, t0, t1, u.tiles,
                        C::kApart && min(u.r.count - first, R) * p.group <= 64 ? 64 : 0, !more};
          mbar_arrive(&sm.piece_full[piece % kPieceRing]);
          if (more) {
            const int rows = R * p.group;
            mbar_arrive_expect(&sm.q_full, C::kStreams * C::kSub * rows * 128);
            for (int s = 0; s < C::kStreams; ++s)
              for (int c = 0; c < C::kSub; ++c)
                tma_load_4d(sm.q[s] + c * C::kSubBytes, &qmap, c * 64, 0, u.h,
                            u.r.row0 + first + s * R, &sm.q_full);
          }
        }
        __syncwarp();
      };
      if (!more) {  // the last values, then the end
        for (int k = C::kLag; k > 0 && ok; --k) {
          if (n >= k) load(&vmap, C::value_pos(n - k), past[0]);
          for (int x = 0; x + 1 < C::kLag; ++x) past[x] = past[x + 1];
        }
        if (ok) hand_over();
        break;
      }
      int at_next, page_next = page_of(t0, at_next);
      for (int t = t0; t < t1; ++t, ++n) {
        if (t - t0 == (piece > 0 ? C::kLag : 0)) hand_over();
        if (!ok) break;
        const Place place = {page_next >= 0 && page_next < p.num_blocks ? page_next : -1, at_next,
                             u.h};
        if (t + 1 < t1) page_next = page_of(t + 1, at_next);
        const uint32_t mapped = __ballot_sync(0xffffffffu, place.page >= 0);
        const int slot = C::key_pos(n) % C::S;
        ok = __all_sync(0xffffffffu,
                        wait(&sm.empty[slot], ((C::key_pos(n) / C::S) & 1) ^ 1));
        if (!ok) break;
        if (lane < 4) {
          uint32_t word;
          if (g.box_rows >= 32) {
            word = (mapped >> (lane * 32 / g.box_rows)) & 1 ? 0xffffffffu : 0u;
          } else {
            const int in_word = 32 / g.box_rows;
            word = 0;
            for (int k = 0; k < in_word; ++k)
              if ((mapped >> (lane * in_word + k)) & 1)
                word |= ((1u << g.box_rows) - 1) << (k * g.box_rows);
          }
          const int left = u.r.tokens - t * kTile - lane * 32;
          if (left < 32) word &= left <= 0 ? 0u : (1u << left) - 1;
          sm.meta[n % kMetaRing][lane] = word;
        }
        __syncwarp();
        load(&kmap, C::key_pos(n), place);
        if constexpr (C::kLag == 0) {
          if (ok) load(&vmap, C::value_pos(n), place);
        } else {
          if (ok && n >= C::kLag) load(&vmap, C::value_pos(n - C::kLag), past[0]);
#pragma unroll
          for (int x = 0; x + 1 < C::kLag; ++x) past[x] = past[x + 1];
          past[C::kLag - 1] = place;
        }
      }
      if (ok && !handed) hand_over();
      if (!ok) break;
      more = unit_next(p, u, span);
    }
    if (!ok && lane == 0) give_up();
    // copies in flight end before the block may
    if (!ok) mbar_wait(&sm.q_full, piece & 1);
    for (int k = 0; !ok && k < C::S; ++k) {
      const int pos = C::key_pos(n) + 1 - k;
      if (pos >= 0) mbar_wait(&sm.full[pos % C::S], (pos / C::S) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------------- tensor cores
    // The whole warp keeps the loop (descriptors then stay in uniform
    // registers); one elected lane issues.
    constexpr uint32_t kQk = tree_idesc<F16, kTile, false>();
    constexpr uint32_t kPv = tree_idesc<F16, D, true>();
    const bool leader = elect_lane();
    const uint64_t q_desc = sw128_desc(smem_u32(sm.q[0]));
    const uint64_t k_desc = sw128_desc(smem_u32(sm.ring[0]));
    const uint64_t v_desc = value_desc(smem_u32(sm.ring[0]));
    int piece = 0, shift = 0;
    uint32_t given[2] = {0, 0};  // P tiles taken of each softmax warpgroup
    RingPos kp{0, 0}, vp{C::kLag + 1, 0};
    int keys = 0;  // key tiles met
    auto qk = [&](int s) {
      if (leader) {
        // shifted rows: the tile begins 64 rows before the queries, with
        // whatever lies there (the rows of S do not meet)
        const uint64_t a = DUAL ? q_desc + s * (C::kTileBytes >> 4)
                                : q_desc - (s ? static_cast<uint32_t>(shift) * 128 >> 4 : 0);
        const uint64_t b = k_desc + static_cast<uint32_t>(kp.slot) * (C::kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k / 4) * C::kSubBytes + (k % 4) * 32) >> 4;
          umma_bf16(tmem_s[s], a + off, b + off, kQk, k > 0);
        }
        umma_commit(&sm.s_full[s]);
      }
    };
    auto pv = [&](int s, bool accumulate) {
      if (leader) {
        const uint64_t b = v_desc + static_cast<uint32_t>(vp.slot) * (C::kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          umma_ts(tmem_o[s], tmem_s[s] + k * 8, b + ((k * 2048) >> 4), kPv, accumulate || k > 0);
      }
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
    };
    auto arrived = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
    };
    auto k_in = [&]() { return arrived(&sm.full[kp.slot], kp.phase); };
    auto v_in = [&]() { return arrived(&sm.full[vp.slot], vp.phase); };
    auto p_in = [&](int s) { return arrived(&sm.p_ready[s], given[s]++ & 1); };
    for (;; ++piece) {
      const TreePiece& pc = sm.piece[piece % kPieceRing];
      ok = arrived(&sm.piece_full[piece % kPieceRing], piece / kPieceRing & 1);
      if (!ok || pc.end) break;
      const int m = pc.t1 - pc.t0;
      shift = pc.shift;
      ok = arrived(&sm.q_full, piece & 1);
      if (!ok) break;
      if constexpr (DUAL) {
        for (int j = 0; j <= m && ok; ++j) {  // product j - 1, then scores j
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (j > 0) {
              ok = ok && (s || (v_in() && (j == m || k_in()))) && p_in(s);
              if (!ok) break;
              tc_fence_after();
              pv(s, j > 1);
            }
            if (j < m) {
              if (j == 0) ok = ok && (s || k_in());
              if (!ok) break;
              tc_fence_after();
              qk(s);
            } else {
              commit(&sm.o_full[s]);
            }
          }
          if (!ok) break;
          if (j > 0) {
            commit(&sm.empty[vp.slot]);
            vp.template step<C::S>(2);
          }
          if (j < m) {
            commit(&sm.empty[kp.slot]);
            kp.template step<C::S>(2);
          }
          if (j == m - 1) commit(&sm.q_empty);
        }
      } else {
        for (int j = 0; j < m + 2 && ok; ++j) {  // product j - 2, then scores j
          const int s = j & 1;
          if (j >= 2) {
            ok = v_in() && (j >= m || k_in()) && p_in(s);
            if (!ok) break;
            tc_fence_after();
            pv(s, j >= 4);
            commit(&sm.empty[vp.slot]);
            vp.template step<C::S>(2);
          }
          if (j < m) {
            if (j < 2) ok = k_in();
            if (!ok) break;
            tc_fence_after();
            qk(s);
            commit(&sm.empty[kp.slot]);
            kp.template step<C::S>(keys++ < C::kLag ? 1 : 2);
            if (j == m - 1) commit(&sm.q_empty);
          }
        }
        if (!ok) break;
        commit(&sm.o_full[0]);
        commit(&sm.o_full[1]);
      }
      if (!ok) break;
    }
    if (!ok) {
      if (lane == 0) give_up();
      commit(&sm.drain);  // products in flight end before the block may
      mbar_wait(&sm.drain, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------- softmax
    const int st = warp >= 6 ? 1 : 0;
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t ts = tmem_s[st] + lane_off, to = tmem_o[st] + lane_off;
    const float c = p.scale_log2;
    int n = 0, piece = 0;
    uint32_t tiles_done = 0, vsyncs = 0;
    for (;; ++piece) {
      // what a piece is stays in shared memory, so as not to take registers
      // through the tile loop
      const TreePiece& pc = sm.piece[piece % kPieceRing];
      ok = __all_sync(0xffffffffu,
                      wait(&sm.piece_full[piece % kPieceRing], piece / kPieceRing & 1));
      if (!ok || pc.end) break;
      const int t0 = pc.t0, t1 = pc.t1;
      const int region = pc.region;
      // this thread's row of the row tile, and whether its warp has any
      const int vrow = row - (st ? pc.shift : 0);
      const int rows = min(pc.r.count - pc.first - (DUAL ? st * R : 0), R) * p.group;
      const bool busy = vrow - lane < rows && vrow - lane >= 0;
      float m = -INFINITY, l = 0.0f;
      const int step = DUAL ? 1 : 2;
      bool fresh = true;
      for (int t = t0 + (DUAL ? 0 : st); t < t1; t += step) {
        const int seq = n + (t - t0);
        ok = __all_sync(0xffffffffu, wait(&sm.s_full[st], tiles_done & 1));
        if (!ok) break;
        ++tiles_done;
        tc_fence_after();
        const uint4 words = *reinterpret_cast<const uint4*>(sm.meta[seq % kMetaRing]);
        const bool masked = (t + 1) * kTile > region ||
                            (words.x & words.y & words.z & words.w) != 0xffffffffu;
        if (masked && busy) {
          uint32_t w[4] = {words.x, words.y, words.z, words.w};
          row_mask(w, p, pc.r, t, pc.first + (DUAL ? st * R : 0), g.group_div.div(vrow), R, lane);
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // hidden scores become -inf in place
            uint32_t s[32];
            tmem_ld32(ts + k * 32, s);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((w[k] >> e) & 1)) s[e] = 0xff800000u;
            tmem_st32(ts + k * 32, s);
          }
          tmem_wait_st();
        }
        if (masked) {
          // Values of tokens that may not be read become 0; infinite or NaN
          // elements of drafted tokens too, and the piece remembers them.
          const int vseq = C::value_pos(seq);
          ok = __all_sync(0xffffffffu, wait(&sm.full[vseq % C::S], (vseq / C::S) & 1));
          if (!ok) break;
          constexpr int kParts = DUAL ? 2 : 1;   // threads of one token
          const int token = DUAL ? st * 64 + row / 2 : row;
          const int part = DUAL ? row & 1 : 0;
          const uint32_t word = sm.meta[seq % kMetaRing][token / 32];
          const bool exists = (word >> (token % 32)) & 1;
          uint4* v = reinterpret_cast<uint4*>(sm.ring[vseq % C::S]);
          constexpr int kChunks = C::kSub * 8 / kParts;  // 16-byte chunks of this thread
          if (!exists || t * kTile + token >= region) {
#pragma unroll 1
            for (int k = 0; k < kChunks; ++k) {
              const int at = part * kChunks + k;
              uint4* x = v + (at / 8) * (C::kSubBytes / 16) + token * 8 + at % 8;
              uint32_t e[4] = {0u, 0u, 0u, 0u};
              if (exists) {
                const uint4 was = *x;
                e[0] = was.x, e[1] = was.y, e[2] = was.z, e[3] = was.w;
                constexpr uint32_t kExp = F16 ? 0x7c00u : 0x7f80u;
                uint32_t found = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  if ((e[q] & kExp) == kExp) e[q] &= 0xffff0000u, found = 1;
                  if (((e[q] >> 16) & kExp) == kExp) e[q] &= 0x0000ffffu, found = 1;
                }
                if (!found) continue;
                sm.bad[piece & 1] = piece;
              }
              *x = make_uint4(e[0], e[1], e[2], e[3]);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if constexpr (DUAL) {  // both warpgroups clean half of a tile that both use
            mbar_arrive(&sm.vsync);
            ok = __all_sync(0xffffffffu, wait(&sm.vsync, vsyncs & 1));
            if (!ok) break;
            ++vsyncs;
          }
        }
        if (!busy) {  // P of rows that are none may be anything
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_ready[st]);
          continue;
        }
        // A piece's first tile gives the maximum that exponentials are taken
        // against.  Later tiles take theirs against it at once: only where
        // their sum passes kMostSum (no exponential can, then), or the row has
        // seen nothing so far, is the tile's own maximum looked up, and the
        // pass made again against that: S is still whole, as P is only
        // written behind it.
        if (fresh) m = row_max(ts);
        uint32_t pk[kTile / 2];
        float sum = score_pass<F16>(ts, c, m, pk);
        if (!fresh) {
          constexpr float kMost = kMostSum * (F16 ? 128.0f : 1.0f);  // 2^kLift
          const bool move = m == -INFINITY || sum > kMost;
          if (__any_sync(0xffffffffu, move)) {
            const float top = row_max(ts);  // of the whole warp's rows, as loads go
            const float high = move ? fmaxf(top, m) : m;
            // the products so far are done: this S was issued behind them
            const float f = !move || high == m ? 1.0f
                            : m == -INFINITY   ? 0.0f
                                               : fast_exp2((m - high) * c);
            l *= f;
#pragma unroll
            for (int k = 0; k < D; k += 16) {
              uint32_t o[16];
              tmem_ld16(to + k, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(to + k, o);
            }
            m = high;
            sum = score_pass<F16>(ts, c, m, pk);
          }
        }
        fresh = false;
        tmem_st32(ts, pk);
        tmem_st32(ts + 32, pk + 32);
        l += sum;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_ready[st]);
      }
      if (!ok) break;
      // ---- the piece's end: sums, outputs or partials
      const int tiles = t1 - t0;
      ok = __all_sync(0xffffffffu, wait(&sm.o_full[st], piece & 1));
      if (!ok) break;
      float f0 = 1.0f, f1 = 0.0f;  // factors of this and the other warpgroup's O
      const bool apart = C::kApart && pc.shift;  // the warpgroups' rows lie in other lanes
      if constexpr (!DUAL) {
        if (st == 1) {
          if (vrow >= 0) sm.ml[vrow] = make_float2(m, l);
          if (apart && busy && tiles > 1) {
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D; k += 32) {
              uint32_t o[32];
              tmem_ld32(to + k, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) sm.xo[(k + e) * 64 + vrow] = __uint_as_float(o[e]);
            }
            tc_fence_before();
          }
          mbar_arrive(&sm.xchg[0]);
          ok = __all_sync(0xffffffffu, wait(&sm.xchg[1], piece & 1));
          if (!ok) break;
        } else {
          ok = __all_sync(0xffffffffu, wait(&sm.o_full[1], piece & 1) &&
                                           wait(&sm.xchg[0], piece & 1));
          if (!ok) break;
          const float2 other = sm.ml[row];
          const float both = fmaxf(m, other.x);
          const float base = both == -INFINITY ? 0.0f : both;
          f0 = fast_exp2((m - base) * c);
          f1 = fast_exp2((other.x - base) * c);
          l = l * f0 + other.y * f1;
          m = both;
        }
      }
      if (DUAL || st == 0) {
        tc_fence_after();
        const TreeRequest r = pc.r;
        int local, head;
        g.group_div.divmod(max(vrow, 0), local, head);
        const int i = pc.first + (DUAL ? st * R : 0) + local;  // this thread's row of the request
        const bool live = busy && local < R && i < r.count;
        const bool whole = tiles == pc.tiles;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const float lse2 = l == 0.0f ? -INFINITY : m * c + (log2f(l) - kLift<F16>);
        const int64_t packed = r.row0 + i;
        const int q_head = pc.h * p.group + head;
        const int64_t part_row =
            (static_cast<int64_t>(blockIdx.x) * 2 + (t0 > 0 ? 0 : 1)) * C::kRows +
            (DUAL ? st * kTile : 0) + row;
        const bool bad = sm.bad[piece & 1] == piece;
#pragma unroll
        for (int k = 0; k < D; k += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o[DUAL ? st : 0] + lane_off + k, o);
          if constexpr (!DUAL) {
            if (tiles > 1) {
              uint32_t o1[32];
              if (apart) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  o1[e] = __float_as_uint(sm.xo[(k + e) * 64 + (row & 63)]);
              } else {
                tmem_ld32(tmem_o[1] + lane_off + k, o1);
              }
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * (f0 * inv) +
                                       __uint_as_float(o1[e]) * (f1 * inv));
            }
          }
          tmem_wait_ld();
          if (DUAL || tiles <= 1) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * (f0 * inv));
          }
          if (bad && live) {
            const int last = min(r.tokens, t1 * kTile);
#pragma unroll 1
            for (int t = max(region, t0 * kTile); t < last; ++t) {
              if (!tree_sees(p, r, i, t)) continue;
              int q, at;
              p.page_div.divmod(t, q, at);
              const int page = p.table[pc.b * p.table_stride + q];
              if (page < 0 || page >= p.num_blocks) continue;
              const uint16_t* v = static_cast<const uint16_t*>(p.v_cache) +
                                  page * p.v_block_stride + at * p.v_token_stride +
                                  pc.h * p.v_head_stride + k;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float x = unpack<F16>(v[e]);
                if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
              }
            }
          }
          if (!live) continue;
          if (whole) {
            uint16_t* out = static_cast<uint16_t*>(p.out) + packed * p.out_row_stride +
                            q_head * p.out_head_stride + k;
            uint32_t h[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              h[e] = pack2<F16>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
            if (p.out_vec) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<uint4*>(out)[e] =
                    make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                out[2 * e] = static_cast<uint16_t>(h[e]);
                out[2 * e + 1] = static_cast<uint16_t>(h[e] >> 16);
              }
            }
          } else {
            // whole 32-byte sectors: rows are 4 D bytes apart from lane to lane
            float* out = g.part_o + part_row * D + k;
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + e),
                           "r"(o[e]), "r"(o[e + 1]), "r"(o[e + 2]), "r"(o[e + 3]), "r"(o[e + 4]),
                           "r"(o[e + 5]), "r"(o[e + 6]), "r"(o[e + 7])
                           : "memory");
          }
        }
        if (live) {
          if (!whole) g.part_lse[part_row] = lse2;
          else if (p.lse != nullptr)
            p.lse[packed * p.lse_row_stride + q_head] = lse2 * 0.69314718055994531f;
        }
        tc_fence_before();
        if (!DUAL) mbar_arrive(&sm.xchg[1]);  // O of both is free
      }
      n += tiles;
    }
    if (!ok && lane == 0) give_up();
    __syncwarp();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
}

// Joins the pieces of the units that the ranges cut, one warp per row: the
// block of a range that is the first to begin inside its unit takes the unit,
// whose pieces are the end of the range before (slot 1) and the beginnings
// (slot 0) of this range and of those that follow inside it.
template <int D, bool F16>
__global__ void __launch_bounds__(256)
tree_merge_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ TreeGeometry g,
                  int rows, int streams) {
  pdl_wait();
  pdl_trigger();
  const PieceInfo info = g.info[blockIdx.x];
  if (!info.valid) return;
  const int first = blockIdx.x / g.cohort, member = blockIdx.x - first * g.cohort;
  if (info.total * (first - 1) / info.ranges > info.base) return;  // taken by an earlier range
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int R = g.rows_per_tile;
  int local, head;
  g.group_div.divmod(row & (kTile - 1), local, head);
  const int i = ((info.grp * g.cohort + member) * streams + row / kTile) * R + local;
  if (local >= R || i >= info.count) return;
  int last = first;  // one past the last range of the unit
  while (last < info.ranges && info.total * last / info.ranges < info.base + info.tiles) ++last;
  auto slot = [&](int k) {  // k-th piece, from the range before on
    return (static_cast<int64_t>((first - 1 + k) * g.cohort + member) * 2 + (k == 0)) * rows + row;
  };
  const int pieces = last - first + 1;
  float high = -INFINITY;
  for (int k = lane; k < pieces; k += 32) high = fmaxf(high, g.part_lse[slot(k)]);
#pragma unroll
  for (int o = 16; o; o >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  const float base = high == -INFINITY ? 0.0f : high;
  constexpr int kPer = D / 32;
  float acc[kPer], total = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
#pragma unroll 4
  for (int k = 0; k < pieces; ++k) {
    const int64_t at = slot(k);
    const float w = fast_exp2(g.part_lse[at] - base);
    total += w;
    const float* o = g.part_o + at * D + lane * kPer;
    if constexpr (kPer == 4) {
      const float4 x = *reinterpret_cast<const float4*>(o);
      acc[0] = fmaf(w, x.x, acc[0]);
      acc[1] = fmaf(w, x.y, acc[1]);
      acc[2] = fmaf(w, x.z, acc[2]);
      acc[3] = fmaf(w, x.w, acc[3]);
    } else {
      const float2 x = *reinterpret_cast<const float2*>(o);
      acc[0] = fmaf(w, x.x, acc[0]);
      acc[1] = fmaf(w, x.y, acc[1]);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t packed = info.row0 + i;
  const int q_head = info.h * p.group + head;
  uint16_t* out = static_cast<uint16_t*>(p.out) + packed * p.out_row_stride +
                  q_head * p.out_head_stride + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) {
    const uint32_t two = pack2<F16>(acc[e] * inv, acc[e + 1] * inv);
    if (p.out_vec) {
      *reinterpret_cast<uint32_t*>(out + e) = two;
    } else {
      out[e] = static_cast<uint16_t>(two);
      out[e + 1] = static_cast<uint16_t>(two >> 16);
    }
  }
  if (lane == 0 && p.lse != nullptr)
    p.lse[packed * p.lse_row_stride + q_head] =
        total == 0.0f ? -INFINITY : (base + log2f(total)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------- host side
// Row tiles of a CTA and CTAs of a cohort, from the longest request's rows.
void tree_shape(int group, int max_query_len, bool* dual, int* cohort) {
  const int R = kTile / group;
  *dual = max_query_len > R;
  const int units = (max_query_len + (*dual ? 2 : 1) * R - 1) / ((*dual ? 2 : 1) * R);
  *cohort = std::min(units, 4);
}

template <int D, bool DUAL, bool F16>
cudaError_t launch_tree_typed(const TreeParams& p, TreeGeometry& g, const CUtensorMap& qmap,
                              const CUtensorMap& kmap, const CUtensorMap& vmap,
                              cudaStream_t stream) {
  using C = TreeCfg<D, DUAL>;
  const size_t smem = sizeof(TreeSmem<D, DUAL>) + 1024;
  auto fn = tree_attention_kernel<D, DUAL, F16>;
  cudaError_t e = set_attr_once(reinterpret_cast<const void*>(fn),
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  const int ctas = g.cohorts * g.cohort;
  e = count_launches(launch_kernel(fn, dim3(ctas), dim3(kTreeThreads), smem, stream, 1, p, g, qmap,
                                   kmap, vmap));
  if (e != cudaSuccess) return e;
  return count_launches(launch_kernel(tree_merge_kernel<D, F16>, dim3(ctas, C::kRows / 8),
                                      dim3(256), 0, stream, 1, p, g, C::kRows, C::kStreams));
}

template <int D, bool F16>
cudaError_t launch_tree_rows(bool dual, const TreeParams& p, TreeGeometry& g,
                             const CUtensorMap& qmap, const CUtensorMap& kmap,
                             const CUtensorMap& vmap, cudaStream_t stream) {
  return dual ? launch_tree_typed<D, true, F16>(p, g, qmap, kmap, vmap, stream)
              : launch_tree_typed<D, false, F16>(p, g, qmap, kmap, vmap, stream);
}

}  // namespace

bool encode_rows(CUtensorMap* map, bool f16, const void* base, const cuuint64_t (&dims)[4],
                 const int64_t (&strides)[3], const cuuint32_t (&box)[4]) {
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  cuuint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of size 1 is never used, but is checked
    bytes[i] = static_cast<cuuint64_t>(dims[i + 1] == 1 ? 64 : strides[i]) * 2;
    if (dims[i + 1] > 1 && (strides[i] <= 0 || bytes[i] % 16 != 0)) return false;
  }
  return tensor_map_encoder()(map,
                              f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                              4, const_cast<void*>(base), dims, bytes, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t tree_attention_tc_workspace(int group, int dim, int max_query_len) {
  if ((dim != 64 && dim != 128) || group > kTile) return 0;
  bool dual;
  int cohort;
  tree_shape(group, max_query_len, &dual, &cohort);
  const size_t ctas = static_cast<size_t>(num_sms() / cohort * cohort);
  const size_t rows = dual ? 2 * kTile : kTile;
  return ctas * 64 + 2 * ctas * rows * (dim + 1) * sizeof(float);
}

bool tree_attention_tc_eligible(const TreeParams& p) {
  return (p.dim == 64 || p.dim == 128) && p.group <= kTile && p.page_size % 8 == 0 &&
         p.num_blocks > 0 && p.table_width > 0 && tensor_map_encoder() != nullptr;
}

cudaError_t launch_tree_attention_tc(const TreeParams& p, cudaStream_t stream) {
  static_assert(sizeof(PieceInfo) <= 64, "workspace layout");
  TreeGeometry g = {};
  bool dual;
  tree_shape(p.group, p.max_query_len, &dual, &g.cohort);
  g.cohorts = num_sms() / g.cohort;
  g.rows_per_tile = kTile / p.group;
  g.group_div = FastDiv(static_cast<uint32_t>(p.group));
  g.box_rows = gcd_int(p.page_size, kTile);
  const size_t ctas = static_cast<size_t>(g.cohorts) * g.cohort;
  char* ws = static_cast<char*>(p.workspace);
  g.info = reinterpret_cast<PieceInfo*>(ws);
  g.part_o = reinterpret_cast<float*>(ws + ctas * 64);
  g.part_lse = g.part_o + 2 * ctas * (dual ? 2 * kTile : kTile) * p.dim;
  const bool f16 = p.dtype == kDtypeF16;
  CUtensorMap qmap, kmap, vmap;
  const cuuint64_t d = static_cast<cuuint64_t>(p.dim), kvh = static_cast<cuuint64_t>(p.kv_heads);
  const cuuint64_t page = static_cast<cuuint64_t>(p.page_size);
  const cuuint64_t blocks = static_cast<cuuint64_t>(p.num_blocks);
  const cuuint32_t box = static_cast<cuuint32_t>(g.box_rows);
  if (!encode_rows(&qmap, f16, p.q,
                   {d, static_cast<cuuint64_t>(p.group), kvh, static_cast<cuuint64_t>(p.rows)},
                   {p.q_head_stride, p.q_head_stride * p.group, p.q_row_stride},
                   {64, static_cast<cuuint32_t>(p.group), 1,
                    static_cast<cuuint32_t>(g.rows_per_tile)}) ||
      !encode_rows(&kmap, f16, p.k_cache, {d, kvh, page, blocks},
                   {p.k_head_stride, p.k_token_stride, p.k_block_stride}, {64, 1, box, 1}) ||
      !encode_rows(&vmap, f16, p.v_cache, {d, kvh, page, blocks},
                   {p.v_head_stride, p.v_token_stride, p.v_block_stride}, {64, 1, box, 1}))
    return cudaErrorNotSupported;
  if (p.dim == 64)
    return f16 ? launch_tree_rows<64, true>(dual, p, g, qmap, kmap, vmap, stream)
               : launch_tree_rows<64, false>(dual, p, g, qmap, kmap, vmap, stream);
  return f16 ? launch_tree_rows<128, true>(dual, p, g, qmap, kmap, vmap, stream)
             : launch_tree_rows<128, false>(dual, p, g, qmap, kmap, vmap, stream);
}

}  // namespace qsa
