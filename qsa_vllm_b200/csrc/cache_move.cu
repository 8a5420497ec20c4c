// Moves of cached tokens between places of the paged cache, and the eviction
// that decides them (sm_100a).
//
// Compaction: for every request b, KV head h and j < count, the key and value
// rows of token indices[b, h, j] go to token starts[b] + j, of the same pages
// or of another table's.  Eviction: the same with a list made from `sinks`
// first tokens, the top-k of the accumulated weights between, and `recent`
// last tokens, all ascending; the weights move along.
//
// In place a row's destination may be another row's source.  With ascending
// sources and source >= destination, every destination of the j-th group of
// moves lies below the sources of all later groups, so writing group j after
// groups 0..j have been read is enough: the CTAs of one (request, head) form
// a cluster that takes one round of groups after another, reads it into
// registers, meets at the cluster barrier, and writes.  To other pages
// nothing overlaps and every group is a CTA of its own.
//
// Bound by memory: each moved row is read and written once.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace qsa {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveBatch = 8;        // chunks in flight per thread
constexpr int kMoveCluster = 8;      // CTAs of one (request, head), in place

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}

template <int BYTES> struct Unit;
template <> struct Unit<16> { using type = uint4; };
template <> struct Unit<4> { using type = uint32_t; };
template <> struct Unit<2> { using type = uint16_t; };

// Token the j-th entry of (request b, head h) comes from, -1 for none.
__device__ __forceinline__ int move_source(const MoveParams& p, int b, int h, int j, int seq,
                                           int kept) {
  if (!p.evict) return p.indices[b * p.idx_req_stride + h * p.idx_head_stride + j];
  if (j >= kept) return -1;
  if (seq <= p.budget || j < p.sinks) return j;
  if (j >= p.budget - p.recent) return seq - p.budget + j;
  return p.sinks + p.chosen[static_cast<int64_t>(b * p.list_heads + h) * p.chosen_width + j -
                            p.sinks];
}

// Row of token `t` in a table's pages: page number and offset; false if unmapped.
__device__ __forceinline__ bool locate(const MoveParams& p, const int32_t* table, int64_t stride,
                                       int width, int b, int t, int64_t& page, int& at) {
  int q;
  p.page_div.divmod(t, q, at);
  if (q >= width) return false;
  page = table[b * stride + q];
  return page >= 0 && page < p.num_blocks;
}

template <typename U, bool IN_PLACE>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(MoveParams p) {
  pdl_wait();
  // no early trigger: a later kernel may read the list's lengths before its own wait
  const int pair = blockIdx.y;
  int b, h;
  p.head_div.divmod(pair, b, h);
  const int lh = p.list_heads == 1 ? 0 : h;
  const int seq = p.evict ? min(max(p.seq_lens[b], 0), p.capacity) : 0;
  const int kept = p.evict ? min(seq, p.budget) : 0;
  const int start = p.starts != nullptr ? p.starts[b] : 0;
  const int units = p.row_units;            // copy units of one row (key or value)
  const int group = p.group;                // tokens of one group of moves
  const int lanes = 2 * units;              // units of one token: key row, then value row
  const int items = group * lanes;
  U val[kMoveBatch];
  const U* src[kMoveBatch];
  U* dst[kMoveBatch];
  // Items of group g: this thread's units, loaded.
  auto read = [&](int g) {
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u) {
      const int n = threadIdx.x + u * kMoveThreads;
      src[u] = nullptr;
      if (n >= items) continue;
      int r, c;
      p.lane_div.divmod(n, r, c);
      const int j = g * group + r;
      if (j >= p.count) continue;
      const int from = move_source(p, b, lh, j, seq, kept);
      if (p.evict && p.kept != nullptr && c == 0 && h < p.list_heads)
        p.kept[static_cast<int64_t>(b * p.list_heads + h) * p.count + j] = from;
      if (from < 0) continue;
      const int to = start + j;
      if (IN_PLACE && from == to) continue;
      int64_t pa, pb;
      int ta, tb;
      if (to < 0 || (IN_PLACE && from < to) ||
          !locate(p, p.table, p.table_stride, p.table_width, b, from, pa, ta) ||
          !locate(p, p.out_table, p.out_table_stride, p.out_table_width, b, to, pb, tb)) {
        if (c == 0) record_error(p.err, kDeviceErrOutOfRange);
        continue;
      }
      if (c < units) {
        char* base = static_cast<char*>(p.k_cache) + h * p.k_head + c * sizeof(U);
        src[u] = reinterpret_cast<const U*>(base + pa * p.k_block + ta * p.k_token);
        dst[u] = reinterpret_cast<U*>(base + pb * p.k_block + tb * p.k_token);
      } else {
        char* base = static_cast<char*>(p.v_cache) + h * p.v_head + (c - units) * sizeof(U);
        src[u] = reinterpret_cast<const U*>(base + pa * p.v_block + ta * p.v_token);
        dst[u] = reinterpret_cast<U*>(base + pb * p.v_block + tb * p.v_token);
      }
    }
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u)
      if (src[u] != nullptr) val[u] = *src[u];
  };
  const int groups = (p.count + group - 1) / group;
  for (int g0 = 0; g0 < groups; g0 += gridDim.x) {  // uniform over the cluster
    const int g = g0 + blockIdx.x;
    read(g);
    if constexpr (IN_PLACE) cluster_barrier();
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u)
      if (src[u] != nullptr) *dst[u] = val[u];
  }
}

// Weights of the kept tokens to the front, zeros behind them up to the old
// length.  One CTA per (request, list head): sources ascend and never lie
// below their destination, so a batch is written once it has been read whole.
__global__ void __launch_bounds__(kMoveThreads) move_weights_kernel(MoveParams p) {
  pdl_wait();
  int b, h;
  p.list_div.divmod(static_cast<int>(blockIdx.x), b, h);
  const int seq = min(max(p.seq_lens[b], 0), p.capacity);
  const int kept = min(seq, p.budget);
  const float* in = p.weights + b * p.w_req_stride + h * p.w_head_stride;
  float* out = p.weights_out + b * p.wo_req_stride + h * p.wo_head_stride;
  if (in == out && seq <= p.budget) return;
  constexpr int kU = 8;
  for (int j0 = 0; j0 < kept; j0 += kU * kMoveThreads) {
    float v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int j = j0 + u * kMoveThreads + threadIdx.x;
      if (j < kept) v[u] = in[move_source(p, b, h, j, seq, kept)];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int j = j0 + u * kMoveThreads + threadIdx.x;
      if (j < kept) out[j] = v[u];
    }
  }
  __syncthreads();
  for (int j = kept + threadIdx.x; j < seq; j += kMoveThreads) out[j] = 0.0f;
}

// New lengths, and the number of tokens each list head chooses from (0 where
// nothing is evicted).  Written before the next kernel may start: the top-k
// reads its rows' lengths before its own wait.
__global__ void evict_lengths_kernel(MoveParams p, int32_t* lengths_out, int32_t* middle) {
  pdl_wait();
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n < p.requests * p.list_heads) {
    int b, h;
    p.list_div.divmod(n, b, h);
    const int seq = min(max(p.seq_lens[b], 0), p.capacity);
    middle[n] = seq > p.budget ? seq - p.sinks - p.recent : 0;
    if (h == 0) lengths_out[b] = min(seq, p.budget);
  }
  __threadfence();
  pdl_trigger();
}

template <typename U>
cudaError_t launch_move_typed(const MoveParams& p, cudaStream_t stream) {
  const int groups = (p.count + p.group - 1) / p.group;
  const int pairs = p.requests * p.kv_heads;
  if (groups == 0 || pairs == 0) return cudaSuccess;
  if (!p.in_place)
    return count_launches(launch_kernel(move_kernel<U, false>, dim3(groups, pairs),
                                        dim3(kMoveThreads), 0, stream, 1, p));
  int cluster = 1;
  while (cluster < kMoveCluster && 2 * cluster <= groups && pairs * cluster < 4 * num_sms())
    cluster *= 2;
  return count_launches(launch_kernel(move_kernel<U, true>, dim3(cluster, pairs),
                                      dim3(kMoveThreads), 0, stream,
                                      static_cast<unsigned>(cluster), p));
}

cudaError_t launch_move_rows(MoveParams p, cudaStream_t stream) {
  p.row_units = p.row_bytes / p.unit;
  const int lanes = 2 * p.row_units;
  p.group = std::max(1, kMoveThreads * kMoveBatch / lanes);
  p.lane_div = FastDiv(static_cast<uint32_t>(lanes));
  return p.unit == 16  ? launch_move_typed<uint4>(p, stream)
         : p.unit == 4 ? launch_move_typed<uint32_t>(p, stream)
                       : launch_move_typed<uint16_t>(p, stream);
}

}  // namespace

int move_max_row_units() { return kMoveThreads * kMoveBatch / 2; }

cudaError_t launch_cache_compact(const MoveParams& p, cudaStream_t stream) {
  return launch_move_rows(p, stream);
}

cudaError_t launch_cache_evict(const MoveParams& p, int32_t* lengths_out, int32_t* middle,
                               int32_t* chosen, cudaStream_t stream) {
  const int lists = p.requests * p.list_heads;
  cudaError_t e = count_launches(launch_kernel(
      evict_lengths_kernel, dim3((lists + 255) / 256), dim3(256), 0, stream, 1, p, lengths_out,
      middle));
  if (e != cudaSuccess) return e;
  if (p.chosen_width > 0 && p.capacity > p.budget) {
    TopkParams t = {};
    t.scores = p.weights + p.sinks;
    t.score_row_stride = p.list_heads == 1 ? p.w_req_stride : p.w_head_stride;
    t.rows = lists;
    t.width = p.capacity - p.sinks - p.recent;
    t.lengths = middle;
    t.output = chosen;
    t.out_row_stride = p.chosen_width;
    t.out_col_stride = 1;
    t.out_width = p.chosen_width;
    t.ratio = 1;
    t.page_size = 1;
    t.topk = p.chosen_width;
    t.vec4 = reinterpret_cast<uintptr_t>(t.scores) % 16 == 0 && t.score_row_stride % 4 == 0;
    e = launch_topk(t, stream, nullptr);
    if (e != cudaSuccess) return e;
  }
  e = count_launches(launch_kernel(move_weights_kernel, dim3(lists), dim3(kMoveThreads), 0, stream,
                                   1, p));
  if (e != cudaSuccess) return e;
  return launch_move_rows(p, stream);
}

}  // namespace qsa
