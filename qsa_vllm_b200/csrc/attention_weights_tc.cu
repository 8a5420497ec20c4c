// Attention weight received by cached tokens on the 5th-generation tensor
// cores (tcgen05 + TMA), sm_100a: head dim 64 or 128, pages of a multiple of 8.
//
//   w[b,kv,t] += sum_i f_i sum_{h of kv} exp2(scale log2e q_ih.k_t - lse2_ih)
//
// The log-sum-exps are known, so there is no running maximum and every token
// stands alone: keys are the M side (128 tokens, a TMEM lane each), the (row,
// head) pairs of the request the N side, up to 256 at a time, and each
// thread of the epilogue adds up the columns of its own token:
//   S[128 x N] = K Q^T     (A, B from shared memory, D in TMEM, two in turn)
// Only rows that count (factor not 0, some head's log-sum-exp not -inf) are
// gathered into the N side.  Requests with more pairs than 256 take several
// passes over the tile range, one after another (all epilogue warps meet
// between them).
//
// Bound by the keys' way from memory: a tile is 32 KB (head dim 128), its
// products N/2 cycles of the tensor core's 8192 flops, its exponentials
// 8 N cycles of a scheduler's special-function unit.
//
// Measured on a B200: 64 requests of 8k-32k tokens, 16 rows of which 40%
// count, 32 query heads over 4 KV heads of 128: 284 us in long runs, 267 in
// short ones, of which 226 remain without the epilogue's arithmetic; the floor
// at a copy's rate is 213 us.
// What mattered: columns without branches between them (373 -> 355 us), four
// score buffers, mask bits per row and factors folded into the exponents
// (-> 307), weights prefetched into L2 well ahead (-> 267): with 128 KB of
// keys in flight per SM a load from memory waits behind them for longer than
// two tiles take.
//
// Roles: warp 0 loads key tiles page by page with TMA into a ring; one lane of
// warp 1 issues the products; warps 2-5 and 6-9 gather the pairs of a piece,
// and take alternate tiles.  Work split: the (request, KV head) units, each of
// its number of tiles, form one line cut into equal ranges, one per CTA.
//
// Every wait is bounded, as in the attention kernel.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace qsa {
namespace {

constexpr int kWThreads = 320;
constexpr int kTile = 128;     // tokens per tile
constexpr int kPairs = 256;    // (row, head) pairs of one pass
constexpr int kPieceRing = 4;
constexpr int kWTmemCols = 512;
constexpr int kBuffers = 4;    // of 128 columns; passes of more pairs take two at a time

template <int D>
struct WeightsCfg {
  static constexpr int kSub = D / 64;
  static constexpr int kSubBytes = kTile * 128;
  static constexpr int kTileBytes = kSub * kSubBytes;
  static constexpr int kQSubBytes = kPairs * 128;
  static constexpr int kFit = (216 * 1024 - kSub * kQSubBytes) / kTileBytes;
  static constexpr int S = kFit > 8 ? 8 : kFit;
};

struct WeightsPiece {
  TreeRequest r;
  int b, h, t0, t1, end;
};

template <int D>
struct WeightsSmem {
  using C = WeightsCfg<D>;
  alignas(1024) uint8_t ring[C::S][C::kTileBytes];
  alignas(1024) uint8_t q[C::kSub][C::kQSubBytes];
  float shift[kPairs];      // of a pair: -lse2 (+ log2 of a factor above 0)
  float factor[kPairs];     // what is left of the factor
  int list[kPairs];         // rows that count, of this pass
  uint64_t full[C::S], empty[C::S], s_full[kBuffers], s_empty[kBuffers], q_ready, drain;
  uint64_t piece_full[kPieceRing], piece_empty[kPieceRing], sync, taken;
  WeightsPiece piece[kPieceRing];
  int64_t scan[kWThreads / 32], first_base;
  int first_b;
  int pairs;        // of this pass
  uint32_t bits[kPairs][4];  // first 128 drafted tokens that a listed row sees
  int folded[8];    // per epilogue warp: its factors all went into the shifts
  int next_row;     // where the next pass goes on; r.count when there is none
  uint32_t tmem_base;
  int abort_flag;
};

struct WeightsGeometry {
  FastDiv group_div;
  int box_rows;
  int ranges;
};

__device__ __forceinline__ int weight_tokens(const TreeParams& p, const TreeRequest& r) {
  return min(r.tokens, p.capacity);
}
__device__ __forceinline__ int weight_tiles(const TreeParams& p, int b) {
  return (weight_tokens(p, tree_request_info(p, b)) + kTile - 1) / kTile;
}

// TMEM buffer of the j-th tile of a pass.
__device__ __forceinline__ int weights_buffer(int j, int pairs) {
  return pairs <= 128 ? j & 3 : (j & 1) * 2;
}

// Whether a packed row counts: a factor other than 0, and a log-sum-exp of KV
// head h other than -inf (its first, almost always).
__device__ __forceinline__ bool weights_row_counts(const TreeParams& p, int64_t row, int h) {
  if (p.row_factors != nullptr && p.row_factors[row * p.factor_stride] == 0.0f) return false;
  const float* lse = p.lse + row * p.lse_row_stride + h * p.group;
  for (int g = 0; g < p.group; ++g)
    if (lse[g] != -INFINITY) return true;
  return false;
}

template <int D, bool F16>
__global__ void __launch_bounds__(kWThreads, 1)
attention_weights_kernel(const __grid_constant__ TreeParams p,
                         const __grid_constant__ WeightsGeometry g,
                         const __grid_constant__ CUtensorMap kmap) {
  using C = WeightsCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  WeightsSmem<D>& sm = *reinterpret_cast<WeightsSmem<D>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < C::S; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int s = 0; s < kBuffers; ++s) {
      mbar_init(&sm.s_full[s], 1);
      mbar_init(&sm.s_empty[s], 4);
    }
    for (int s = 0; s < kPieceRing; ++s) {
      mbar_init(&sm.piece_full[s], 1);
      mbar_init(&sm.piece_empty[s], 9);
    }
    mbar_init(&sm.q_ready, 8);
    mbar_init(&sm.taken, 1);
    mbar_init(&sm.sync, 8);
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    sm.first_b = -1;
    fence_mbar_init();
  }
  if (tid == 32) prefetch_tensormap(&kmap);
  pdl_wait();
  pdl_trigger();

  // this CTA's range of the line of tiles, as in the attention kernel
  const int per = (p.requests + kWThreads - 1) / kWThreads;
  int64_t mine = 0;
  for (int k = 0; k < per; ++k) {
    const int b = tid * per + k;
    if (b < p.requests) mine += static_cast<int64_t>(p.kv_heads) * weight_tiles(p, b);
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
  for (int w = 0; w < kWThreads / 32; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  before += incl - mine;
  const int ranges = static_cast<int>(total < g.ranges ? total : g.ranges);
  if (static_cast<int>(blockIdx.x) >= ranges) return;  // the whole block
  const int64_t begin = total * blockIdx.x / ranges, end = total * (blockIdx.x + 1) / ranges;
  if (before <= begin && begin < before + mine) {
    int64_t at = before;
    for (int k = 0; k < per; ++k) {
      const int b = tid * per + k;
      const int64_t n = b < p.requests ? static_cast<int64_t>(p.kv_heads) * weight_tiles(p, b) : 0;
      if (begin < at + n) {
        sm.first_b = b;
        sm.first_base = at;
        break;
      }
      at += n;
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sm.tmem_base)),
                 "r"(kWTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  bool ok = true;
  auto give_up = [&]() {
    record_error(p.err, kDeviceErrWaitTimeout);
    *reinterpret_cast<volatile int*>(&sm.abort_flag) = 1;
  };
  auto arrived = [&](uint64_t* bar, uint32_t parity) -> bool {
    bool yes = mbar_try_wait(bar, parity);
    if (!yes && !*reinterpret_cast<volatile int*>(&sm.abort_flag)) yes = mbar_wait(bar, parity);
    return __all_sync(0xffffffffu, yes) != 0;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const int boxes = kTile / g.box_rows;
    const uint32_t box_bytes = g.box_rows * 128;
    int seq = 0;
    int b = sm.first_b, h = 0, t0 = 0;
    int64_t base = sm.first_base;
    {
      const int tiles = weight_tiles(p, b);
      h = static_cast<int>((begin - base) / tiles);
      base += static_cast<int64_t>(h) * tiles;
      t0 = static_cast<int>(begin - base);
    }
    for (int piece = 0;; ++piece) {
      TreeRequest r = tree_request_info(p, b < p.requests ? b : 0);
      const int tiles = (weight_tokens(p, r) + kTile - 1) / kTile;
      const bool more = base < end && b < p.requests;
      const int t1 = static_cast<int>(min(end - base, static_cast<int64_t>(tiles)));
      ok = arrived(&sm.piece_empty[piece % kPieceRing], (piece / kPieceRing & 1) ^ 1);
      if (!ok) break;
      if (lane == 0) {
        sm.piece[piece % kPieceRing] = WeightsPiece{r, b, h, t0, t1, !more};
        mbar_arrive(&sm.piece_full[piece % kPieceRing]);
      }
      __syncwarp();
      if (!more) break;
      const int32_t* table = p.table + b * p.table_stride;
      auto page_of = [&](int tile, int& at) {
        const int t = tile * kTile + lane * g.box_rows;
        int q;
        p.page_div.divmod(t, q, at);
        const int page = lane < boxes && t < r.tokens ? ld_once(table + q) : -1;
        return page >= 0 && page < p.num_blocks ? page : -1;
      };
      // passes of this piece: the consumers count the rows, which takes the
      // same loads; the number of rows alone bounds the passes, and a pass
      // without rows that count is not made, so count here too
      int counted = 0;
      for (int i0 = 0; i0 < r.count; i0 += 32) {
        const int i = i0 + lane;
        const bool in = i < r.count && weights_row_counts(p, r.row0 + i, h);
        counted += __popc(__ballot_sync(0xffffffffu, in));
      }
      const int rows_per_pass = kPairs / p.group;
      const int passes = (counted + rows_per_pass - 1) / rows_per_pass;
      for (int pass = 0; pass < passes && ok; ++pass) {
        int at_next, page_next = page_of(t0, at_next);
        for (int t = t0; t < t1; ++t, ++seq) {
          const int page = page_next, at = at_next;
          if (t + 1 < t1) page_next = page_of(t + 1, at_next);
          const int slot = seq % C::S;
          ok = arrived(&sm.empty[slot], ((seq / C::S) & 1) ^ 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect(&sm.full[slot], C::kTileBytes);
          __syncwarp();
          if (lane < boxes) {
            uint8_t* dst = sm.ring[slot] + lane * box_bytes;
#pragma unroll
            for (int c = 0; c < C::kSub; ++c)
              tma_load_4d(dst + c * C::kSubBytes, &kmap, c * 64, h, at,
                          page >= 0 ? page : p.num_blocks, &sm.full[slot]);
          }
        }
      }
      if (!ok) break;
      base += tiles;
      t0 = 0;
      if (++h == p.kv_heads) {
        h = 0;
        do ++b;
        while (b < p.requests && weight_tiles(p, b) == 0);
      }
    }
    if (!ok && lane == 0) give_up();
    // copies in flight end before the block may
    for (int k = 0; !ok && k < C::S; ++k) {
      const int s = seq - k;
      if (s >= 0) mbar_wait(&sm.full[s % C::S], (s / C::S) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------------- tensor cores
    const bool leader = elect_lane();
    const uint64_t q_desc = sw128_desc(smem_u32(sm.q[0]));
    const uint64_t k_desc = sw128_desc(smem_u32(sm.ring[0]));
    int seq = 0, passes = 0;
    uint32_t freed = 0;  // phase of each buffer's s_empty
    for (int piece = 0;; ++piece) {
      const WeightsPiece& pc = sm.piece[piece % kPieceRing];
      ok = arrived(&sm.piece_full[piece % kPieceRing], piece / kPieceRing & 1);
      if (!ok || pc.end) break;
      const int m = pc.t1 - pc.t0;
      for (bool last = false; !last && ok;) {
        ok = arrived(&sm.q_ready, passes++ & 1);
        if (!ok) break;
        tc_fence_after();
        const int pairs = sm.pairs;
        last = sm.next_row >= pc.r.count;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.taken);  // both may be written again
        if (pairs == 0) continue;
        const uint32_t n16 = static_cast<uint32_t>((pairs + 15) / 16);
        const uint32_t fmt = F16 ? 0u : 1u;
        const uint32_t idesc =
            (1u << 4) | (fmt << 7) | (fmt << 10) | ((n16 * 2) << 17) | ((kTile >> 4) << 24);
        for (int j = 0; j < m; ++j, ++seq) {
          const int slot = seq % C::S, a = weights_buffer(j, pairs);
          ok = arrived(&sm.full[slot], (seq / C::S) & 1) &&
               arrived(&sm.s_empty[a], ((freed >> a) & 1) ^ 1);
          if (!ok) break;
          freed ^= 1u << a;
          tc_fence_after();
          if (leader) {
            const uint64_t ka = k_desc + static_cast<uint32_t>(slot) * (C::kTileBytes >> 4);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_bf16(tmem + a * 128, ka + (((k / 4) * C::kSubBytes + (k % 4) * 32) >> 4),
                        q_desc + (((k / 4) * C::kQSubBytes + (k % 4) * 32) >> 4), idesc, k > 0);
            umma_commit(&sm.empty[slot]);
            umma_commit(&sm.s_full[a]);
          }
        }
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.piece_empty[piece % kPieceRing]);
    }
    if (!ok) {
      if (lane == 0) give_up();
      if (leader) umma_commit(&sm.drain);  // products in flight end before the block may
      mbar_wait(&sm.drain, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int et = tid - 64;                 // 0..255
    const int st = warp >= 6 ? 1 : 0;
    const int quad = warp & 3, token = quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const float c = p.scale_log2;
    const float2 c2 = make_float2(c, c);
    const int rows_per_pass = kPairs / p.group;
    int syncs = 0, passes = 0;
    uint32_t filled = 0;  // phase of each buffer's s_full
    // all eight warps meet
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.sync);
      return arrived(&sm.sync, syncs++ & 1);
    };
    for (int piece = 0;; ++piece) {
      const WeightsPiece& pc = sm.piece[piece % kPieceRing];
      ok = arrived(&sm.piece_full[piece % kPieceRing], piece / kPieceRing & 1);
      if (!ok || pc.end) break;
      const TreeRequest r = pc.r;
      const int t0 = pc.t0, m = pc.t1 - pc.t0;
      const int tokens = weight_tokens(p, r);
      const float* w_in = p.weights + pc.b * p.w_req_stride + pc.h * p.w_head_stride;
      float* w_out = p.weights_out + pc.b * p.wo_req_stride + pc.h * p.wo_head_stride;
      const int32_t* table = p.table + pc.b * p.table_stride;
      int from = 0;
      for (bool first = true; ok && (first || from < r.count); first = false) {
        // The rows of this pass: the first warp lists those that count, from
        // row `from` on, until the pass is full.
        if (warp == 2) {
          int got = 0, i0 = from, next = r.count;
          for (; i0 < r.count; i0 += 32) {
            const int i = i0 + lane;
            const bool in = i < r.count && weights_row_counts(p, r.row0 + i, pc.h);
            const uint32_t bits = __ballot_sync(0xffffffffu, in);
            const int at = got + __popc(bits & ((1u << lane) - 1));
            if (in && at < rows_per_pass) sm.list[at] = i;
            const bool over = in && at >= rows_per_pass;
            const uint32_t rest = __ballot_sync(0xffffffffu, over);
            got += __popc(bits);
            if (rest != 0) {
              next = i0 + __ffs(rest) - 1;
              break;
            }
          }
          got = min(got, rows_per_pass);
          if (lane == 0) {
            sm.pairs = got * p.group;
            sm.next_row = next;
          }
        }
        ok = meet();
        if (!ok) break;
        const int pairs = sm.pairs;
        from = sm.next_row;
        // their queries into shared memory, 128-byte swizzled, zeros up to the
        // next 16 pairs; log-sum-exps and factors beside them
        const int padded = (pairs + 15) / 16 * 16;
        for (int x = et; x < padded * (D / 8); x += 256) {
          const int n = x / (D / 8), ch = x - n * (D / 8);
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (n < pairs) {
            int j, head;
            g.group_div.divmod(n, j, head);
            v = *reinterpret_cast<const uint4*>(
                static_cast<const uint16_t*>(p.q) +
                static_cast<int64_t>(r.row0 + sm.list[j]) * p.q_row_stride +
                static_cast<int64_t>(pc.h * p.group + head) * p.q_head_stride + ch * 8);
          }
          *reinterpret_cast<uint4*>(sm.q[ch / 8] + n * 128 + (((ch % 8) ^ (n % 8)) * 16)) = v;
        }
        if (p.mask != nullptr && pc.t1 * kTile > r.prefix) {
          const int listed = g.group_div.div(pairs);
          for (int x = warp - 2; x < listed; x += 8) {
            const uint8_t* bytes = p.mask + (r.row0 + sm.list[x]) * p.mask_stride;
            uint8_t byte[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              byte[k] = k * 32 + lane < p.mask_width ? bytes[k * 32 + lane] : 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t word = __ballot_sync(0xffffffffu, byte[k] != 0);
              if (lane == 0) sm.bits[x][k] = word;
            }
          }
        }
        bool fold = true;
        {
          float l = 0.0f, f = 0.0f;
          int i = -1;
          if (et < pairs) {
            const int j = et / p.group, head = et - j * p.group;
            i = sm.list[j];
            const int64_t row = r.row0 + i;
            l = p.lse[row * p.lse_row_stride + pc.h * p.group + head] * -1.4426950408889634f;
            f = p.row_factors == nullptr ? 1.0f : p.row_factors[row * p.factor_stride];
            if (l == INFINITY) f = 0.0f;  // a head that saw nothing, in a row that counts
            fold = f > 0.0f && f < INFINITY && l == l;
            if (fold) {
              l += log2f(f);
              f = 1.0f;
            }
          } else {
            l = -INFINITY;  // columns of no pair add nothing
          }
          sm.shift[et] = l;
          sm.factor[et] = f;
        }
        fold = __all_sync(0xffffffffu, fold);
        if (lane == 0) sm.folded[warp - 2] = fold;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_ready);
        // sums of a pass read what all warps wrote
        ok = meet();
        if (!ok) break;
        int folds = 1;
#pragma unroll
        for (int k = 0; k < 8; ++k) folds &= sm.folded[k];  // also no NaN among the log-sum-exps
        // The weight so far and the page of this thread's token in a tile are
        // fetched a tile ahead, the weight into L2 kAhead tiles before that:
        // behind the key tiles in flight memory takes longer than two tiles.
        constexpr int kAhead = 4;
        auto prefetch = [&](int j) {
          const int tok = (t0 + j) * kTile + token;
          if (j < m && tok < tokens && (lane & 7) == 0)
            asm volatile("prefetch.global.L2 [%0];" ::"l"((first ? w_in : w_out) + tok));
        };
        auto fetch = [&](int j, float& was, int& page) {
          const int tok = (t0 + j) * kTile + token;
          was = 0.0f;
          page = -1;
          prefetch(j + kAhead);
          if (j >= m || tok >= tokens) return;
          was = first ? w_in[tok] : w_out[tok];
          int q, at;
          p.page_div.divmod(tok, q, at);
          page = ld_once(table + q);
        };
        for (int j = st; j < st + kAhead; j += 2) prefetch(j);
        float was_next;
        int page_next;
        fetch(st, was_next, page_next);
        for (int j = 0; j < m; ++j) {
          const int t = t0 + j, tok = t * kTile + token;
          const int a = weights_buffer(j, pairs);
          const uint32_t phase = (filled >> a) & 1;
          if (pairs > 0) filled ^= 1u << a;  // the other warpgroup's buffers too
          if ((j & 1) != st) continue;
          const bool here = tok < tokens;
          const float was = was_next;
          const int page = page_next;
          float got = 0.0f;
          fetch(j + 2, was_next, page_next);
          if (pairs > 0) {
            ok = arrived(&sm.s_full[a], phase);
            if (!ok) break;
            tc_fence_after();
            const bool drafted = (t + 1) * kTile > r.prefix;  // some tokens not seen by all
            const uint32_t ts = tmem + a * 128 + lane_off;
            float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll 1
            for (int k = 0; k < pairs; k += 32) {
              uint32_t v[32];
              tmem_ld32(ts + k, v);
              uint32_t sees = pairs - k >= 32 ? 0xffffffffu : (1u << (pairs - k)) - 1;
              if (drafted) {
                // each row's bit once, then spread over its heads' columns
                uint32_t rows = 0, cols = 0;
                const int j0 = k / p.group, j1 = (min(k + 32, pairs) - 1) / p.group;
#pragma unroll 4
                for (int x = j0; x <= j1; ++x) {
                  const int node = tok - r.prefix;
                  bool see;
                  if (p.mask == nullptr || node >= kTile) see = tree_sees(p, r, sm.list[x], tok);
                  else see = node < 0 || ((sm.bits[x][node >> 5] >> (node & 31)) & 1);
                  rows |= static_cast<uint32_t>(here && see) << (x - j0);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  cols |= ((rows >> ((g.group_div.div(k + e) - j0) & 31)) & 1) << e;
                sees &= cols;
              }
              tmem_wait_ld();
              if (folds) {
                // a hidden score becomes -inf, and its exponential 0
                if (sees != 0xffffffffu) {
#pragma unroll
                  for (int e = 0; e < 32; ++e)
                    if (!((sees >> e) & 1)) v[e] = 0xff800000u;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const float4 sh = *reinterpret_cast<const float4*>(&sm.shift[k + e]);
                  float2 x = fma2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), c2,
                                  make_float2(sh.x, sh.y));
                  float2 y = fma2(make_float2(__uint_as_float(v[e + 2]),
                                              __uint_as_float(v[e + 3])), c2,
                                  make_float2(sh.z, sh.w));
                  x.x = fast_exp2(x.x);
                  x.y = fast_exp2(x.y);
                  y.x = fast_exp2(y.x);
                  y.y = fast_exp2(y.y);
                  acc[0] = add2(acc[0], x);
                  acc[1] = add2(acc[1], y);
                }
              } else {
                // a factor below 0, infinite or NaN, a NaN log-sum-exp, or a
                // head that saw nothing (factor 0)
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float f = sm.factor[k + e];
                  const float x = f * fast_exp2(fmaf(__uint_as_float(v[e]), c, sm.shift[k + e]));
                  acc[e & 1].x += (sees >> e) & 1 && f != 0.0f ? x : 0.0f;
                }
              }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.s_empty[a]);
            acc[0] = add2(acc[0], acc[1]);
            if (page >= 0 && page < p.num_blocks) got = acc[0].x + acc[0].y;
          }
          if (here) w_out[tok] = was + got;
        }
        if (!ok) break;
        // the next pass writes the queries over: every product of this one is
        // behind its scores, which both warpgroups have read
        ok = arrived(&sm.taken, passes++ & 1) && meet();
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.piece_empty[piece % kPieceRing]);
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
                 "r"(kWTmemCols)
                 : "memory");
  }
}

template <int D, bool F16>
cudaError_t launch_weights_typed(const TreeParams& p, const WeightsGeometry& g,
                                 const CUtensorMap& kmap, cudaStream_t stream) {
  const size_t smem = sizeof(WeightsSmem<D>) + 1024;
  auto fn = attention_weights_kernel<D, F16>;
  const cudaError_t e = set_attr_once(reinterpret_cast<const void*>(fn),
                                      cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  return count_launches(launch_kernel(fn, dim3(g.ranges), dim3(kWThreads), smem, stream, 1, p, g,
                                      kmap));
}

}  // namespace

bool attention_weights_tc_eligible(const TreeParams& p) {
  return (p.dim == 64 || p.dim == 128) && p.group <= kPairs && p.page_size % 8 == 0 &&
         p.num_blocks > 0 && p.table_width > 0 && tensor_map_encoder() != nullptr;
}

cudaError_t launch_attention_weights_tc(const TreeParams& p, cudaStream_t stream) {
  WeightsGeometry g = {};
  g.box_rows = gcd_int(p.page_size, kTile);
  g.ranges = num_sms();
  g.group_div = FastDiv(static_cast<uint32_t>(p.group));
  const bool f16 = p.dtype == kDtypeF16;
  CUtensorMap kmap;
  if (!encode_rows(&kmap, f16, p.k_cache,
                   {static_cast<cuuint64_t>(p.dim), static_cast<cuuint64_t>(p.kv_heads),
                    static_cast<cuuint64_t>(p.page_size), static_cast<cuuint64_t>(p.num_blocks)},
                   {p.k_head_stride, p.k_token_stride, p.k_block_stride},
                   {64, 1, static_cast<cuuint32_t>(g.box_rows), 1}))
    return cudaErrorNotSupported;
  if (p.dim == 64)
    return f16 ? launch_weights_typed<64, true>(p, g, kmap, stream)
               : launch_weights_typed<64, false>(p, g, kmap, stream);
  return f16 ? launch_weights_typed<128, true>(p, g, kmap, stream)
             : launch_weights_typed<128, false>(p, g, kmap, stream);
}

}  // namespace qsa
