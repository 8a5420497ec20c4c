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
// Bound by memory: each moved row is read and written once.  One thread per
// token of a group finds its source and destination and leaves their offsets
// in shared memory, where the threads that copy 16 bytes at a time pick them
// up: found by every copying thread for itself they cost more instructions
// than the memory leaves time for (464 instead of 180 us for 1.07 GB of rows
// to other pages, whose floor at a copy's rate is 164).  In place a round at a
// time is in flight, and the number of CTAs in a cluster decides (us for 1 / 2
// / 4 / 8: 32 lists that keep 8192 of 33k to 131k tokens 452 / 373 / 211 / 128,
// 64 lists of 8191 rows 336 / 232 / 150 / 103, floor 82), as long as the lists
// alone do not fill the GPU (512 lists of 2048 tokens 120 / 132 / 132 / 132,
// the rule's choice being 2).
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace qsa {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveBatch = 8;        // copy units in flight per thread
constexpr int kMoveCluster = 8;      // CTAs of one (request, head), in place
constexpr int kMoveTokens = 256;     // most tokens of a group: one per thread

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}

// Token the j-th entry of (request b, list lh) comes from, -1 for none.
__device__ __forceinline__ int move_source(const MoveParams& p, int b, int lh, int j, int seq,
                                           int kept) {
  if (!p.evict) return p.indices[b * p.idx_req_stride + lh * p.idx_head_stride + j];
  if (j >= kept) return -1;
  if (seq <= p.budget || j < p.sinks) return j;
  if (j >= p.budget - p.recent) return seq - p.budget + j;
  return p.sinks + p.chosen[static_cast<int64_t>(b * p.list_heads + lh) * p.chosen_width + j -
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

struct MoveRow {
  const char *k_src, *v_src;  // k_src null: nothing to move
  char *k_dst, *v_dst;
};

// ORDERED: in place (cache or weights), round by round over the cluster.
template <typename U, bool ORDERED>
__global__ void __launch_bounds__(kMoveThreads, 4) move_kernel(MoveParams p) {
  __shared__ MoveRow rows[kMoveTokens];
  pdl_wait();
  // no early trigger: a later kernel may read the lengths before its own wait
  const int pair = blockIdx.y, tid = threadIdx.x;
  int b, h;
  p.head_div.divmod(pair, b, h);
  const int lh = p.list_heads == 1 ? 0 : h;
  const int seq = p.evict ? min(max(p.seq_lens[b], 0), p.capacity) : 0;
  const int kept = p.evict ? min(seq, p.budget) : 0;
  const int start = p.starts != nullptr ? p.starts[b] : 0;
  const int units = p.row_units;            // copy units of one row (key or value)
  const int group = p.group;                // tokens of one group of moves
  const int items = group * 2 * units;      // of a token: key row, then value row
  const bool lists = p.evict && h < p.list_heads;  // this pair writes the list and the weights
  const float* w_in = lists ? p.weights + b * p.w_req_stride + h * p.w_head_stride : nullptr;
  float* w_out = lists ? p.weights_out + b * p.wo_req_stride + h * p.wo_head_stride : nullptr;
  const int groups = (p.count + group - 1) / group;
  for (int g0 = 0; g0 < groups; g0 += gridDim.x) {  // uniform over the cluster
    const int j = (g0 + static_cast<int>(blockIdx.x)) * group + tid;
    const bool mine = tid < group && j < p.count;
    int from = -1;
    float weight = 0.0f;
    if (tid < group) {
      MoveRow row = {nullptr, nullptr, nullptr, nullptr};
      if (mine) {
        from = move_source(p, b, lh, j, seq, kept);
        if (lists) {
          p.kept[static_cast<int64_t>(b * p.list_heads + h) * p.count + j] = from;
          if (from >= 0) weight = w_in[from];
        }
        const int to = start + j;
        if (from >= 0 && !(p.in_place && from == to)) {
          int64_t pa, pb;
          int ta, tb;
          if (to >= 0 && !(p.in_place && from < to) &&
              locate(p, p.table, p.table_stride, p.table_width, b, from, pa, ta) &&
              locate(p, p.out_table, p.out_table_stride, p.out_table_width, b, to, pb, tb)) {
            char* k = static_cast<char*>(p.k_cache) + h * p.k_head;
            char* v = static_cast<char*>(p.v_cache) + h * p.v_head;
            row = MoveRow{k + pa * p.k_block + ta * p.k_token, v + pa * p.v_block + ta * p.v_token,
                          k + pb * p.k_block + tb * p.k_token, v + pb * p.v_block + tb * p.v_token};
          } else {
            record_error(p.err, kDeviceErrOutOfRange);
          }
        }
      }
      rows[tid] = row;
    }
    __syncthreads();
    U val[kMoveBatch];
    U* dst[kMoveBatch];
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u) {
      const int n = tid + u * kMoveThreads;
      dst[u] = nullptr;
      if (n >= items) continue;
      int r, c;
      p.lane_div.divmod(n, r, c);
      const MoveRow& row = rows[r];
      if (row.k_src == nullptr) continue;
      const bool key = c < units;
      if (!key) c -= units;
      val[u] = reinterpret_cast<const U*>(key ? row.k_src : row.v_src)[c];
      dst[u] = reinterpret_cast<U*>(key ? row.k_dst : row.v_dst) + c;
    }
    if constexpr (ORDERED) cluster_barrier();
    else if (g0 + gridDim.x < groups) __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u)
      if (dst[u] != nullptr) *dst[u] = val[u];
    if (mine && lists && from >= 0) w_out[j] = weight;
  }
  // zeros behind the kept weights: in place every source has been read by now
  if (lists && (w_in != w_out || seq > p.budget)) {
    for (int j = kept + static_cast<int>(blockIdx.x) * kMoveThreads + tid; j < seq;
         j += gridDim.x * kMoveThreads)
      w_out[j] = 0.0f;
  }
}

// New lengths, and the number of tokens each list head chooses from (0 where
// nothing is evicted), which the top-k reads behind its wait for this kernel.
__global__ void evict_lengths_kernel(MoveParams p, int32_t* lengths_out, int32_t* middle) {
  pdl_wait();
  pdl_trigger();
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n < p.requests * p.list_heads) {
    int b, h;
    p.list_div.divmod(n, b, h);
    const int seq = min(max(p.seq_lens[b], 0), p.capacity);
    middle[n] = seq > p.budget ? seq - p.sinks - p.recent : 0;
    if (h == 0) lengths_out[b] = min(seq, p.budget);
  }
}

template <typename U>
cudaError_t launch_move_typed(const MoveParams& p, cudaStream_t stream) {
  // an eviction to a budget of nothing still writes the weights' zeros
  const int groups = std::max((p.count + p.group - 1) / p.group, p.evict ? 1 : 0);
  const int pairs = p.requests * p.kv_heads;
  if (groups == 0 || pairs == 0) return cudaSuccess;
  if (!p.in_place && (!p.evict || p.weights != p.weights_out))
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
  p.group = std::min(std::max(1, kMoveThreads * kMoveBatch / lanes), kMoveTokens);
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
    t.lengths_behind_wait = 1;
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
  return launch_move_rows(p, stream);
}

}  // namespace qsa
