// Attention of drafted-token trees over a paged cache, and the weights that
// cached tokens receive: the forms for every layout (any page size, head dims
// up to 256 that are a multiple of 8).
//
//   out[i,h] = sum_t p_iht v_t,   p_iht = exp(scale q_ih.k_t) / sum_t' exp(scale q_ih.k_t')
//   lse[i,h] = log sum_t exp(scale q_ih.k_t)          over the tokens row i sees
//   w[b,kv,t] += sum_i f_i sum_{h of kv} exp(scale q_ih.k_t - lse[i,h])
//
// 32-bit arithmetic throughout, one rounding of each output.  These kernels
// take the layouts that the tensor-core kernels do not (see their files);
// they re-read a request's keys and values for each of its rows, and are bound
// by their fp32 products: 64 requests of 8k-32k tokens, 16 rows, 32 heads of
// 128: 9.35 ms for the weights (267 us there).
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace qsa {
namespace {

constexpr int kGenThreads = 128;  // one thread per token of a tile
constexpr int kGenHeads = 8;      // query heads at a time
constexpr int kGenDim = 256;

__device__ __forceinline__ float half_to_f(uint16_t x, int dtype) {
  return dtype == kDtypeBF16 ? __uint_as_float(static_cast<uint32_t>(x) << 16)
                             : __half2float(__ushort_as_half(x));
}
__device__ __forceinline__ uint16_t f_to_half(float x, int dtype) {
  return dtype == kDtypeBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x))
                             : __half_as_ushort(__float2half_rn(x));
}

// Start of a token's row of KV head h in one cache; nullptr when unmapped.
__device__ __forceinline__ const uint16_t* tree_row(const TreeParams& p, const void* cache,
                                                    int64_t block, int64_t token, int64_t head,
                                                    int b, int h, int t) {
  int q, at;
  p.page_div.divmod(t, q, at);
  const int page = p.table[b * p.table_stride + q];
  if (page < 0 || page >= p.num_blocks) return nullptr;
  return static_cast<const uint16_t*>(cache) + page * block + at * token + h * head;
}

// Scores of one token against `n` query rows held as fp32 in shared memory.
template <int N>
__device__ __forceinline__ void dot_rows(const uint16_t* k, const float (*q)[kGenDim], int dim,
                                         int dtype, float (&s)[N]) {
#pragma unroll
  for (int r = 0; r < N; ++r) s[r] = 0.0f;
  for (int c = 0; c < dim; c += 8) {
    const uint4 raw = *reinterpret_cast<const uint4*>(k + c);
    const uint16_t* e = reinterpret_cast<const uint16_t*>(&raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = half_to_f(e[j], dtype);
#pragma unroll
      for (int r = 0; r < N; ++r) s[r] = fmaf(x, q[r][c + j], s[r]);
    }
  }
}

__global__ void __launch_bounds__(kGenThreads) tree_attention_general(TreeParams p) {
  __shared__ float q[kGenHeads][kGenDim];
  __shared__ float w[kGenHeads][kGenThreads];
  __shared__ float factor[kGenHeads], total[kGenHeads];
  __shared__ const uint16_t* vrow[kGenThreads];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31;
  const int b = tree_request(p, row);
  if (b < 0) return;
  const TreeRequest r = tree_request_info(p, b);
  const int i = row - r.row0;
  if (i < 0 || i >= r.count) return;
  for (int g0 = 0; g0 < p.group; g0 += kGenHeads) {
    const int n = min(kGenHeads, p.group - g0);
    const uint16_t* qrow = static_cast<const uint16_t*>(p.q) + row * p.q_row_stride +
                           (h * p.group + g0) * p.q_head_stride;
    for (int c = tid; c < kGenHeads * p.dim; c += kGenThreads) {
      const int g = c / p.dim, d = c - g * p.dim;
      q[g][d] = g < n ? half_to_f(qrow[g * p.q_head_stride + d], p.dtype) : 0.0f;
    }
    // warp w keeps the running maximum and sum of heads 2w, 2w + 1
    float high[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    float acc[kGenHeads][2];
#pragma unroll
    for (int g = 0; g < kGenHeads; ++g) acc[g][0] = acc[g][1] = 0.0f;
    __syncthreads();
    for (int t0 = 0; t0 < r.tokens; t0 += kGenThreads) {
      const int t = t0 + tid;
      float s[kGenHeads];
#pragma unroll
      for (int g = 0; g < kGenHeads; ++g) s[g] = -INFINITY;
      const uint16_t *krow = nullptr, *vr = nullptr;
      if (t < r.tokens && tree_sees(p, r, i, t)) {
        krow = tree_row(p, p.k_cache, p.k_block_stride, p.k_token_stride, p.k_head_stride, b, h, t);
        vr = tree_row(p, p.v_cache, p.v_block_stride, p.v_token_stride, p.v_head_stride, b, h, t);
      }
      if (krow != nullptr) dot_rows<kGenHeads>(krow, q, p.dim, p.dtype, s);
      vrow[tid] = vr;
#pragma unroll
      for (int g = 0; g < kGenHeads; ++g) w[g][tid] = s[g] * p.scale_log2;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int g = 2 * warp + u;
        float v[4], m = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = w[g][lane + 32 * j];
          m = fmaxf(m, v[j]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float next = fmaxf(high[u], m);
        const float base = next == -INFINITY ? 0.0f : next;
        const float f = exp2f(high[u] - base);  // 0 for the first tokens
        float add = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = exp2f(v[j] - base);
          add += v[j];
          w[g][lane + 32 * j] = v[j];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
        sum[u] = sum[u] * f + add;
        high[u] = next;
        if (lane == 0) factor[g] = f;
      }
      __syncthreads();
#pragma unroll
      for (int g = 0; g < kGenHeads; ++g) {
        acc[g][0] *= factor[g];
        acc[g][1] *= factor[g];
      }
      for (int j = 0; j < kGenThreads; ++j) {
        const uint16_t* v = vrow[j];
        if (v == nullptr) continue;  // an unseen value is not read
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int c = tid + half * kGenThreads;
          if (c >= p.dim) continue;
          const float x = half_to_f(v[c], p.dtype);
#pragma unroll
          for (int g = 0; g < kGenHeads; ++g) acc[g][half] = fmaf(w[g][j], x, acc[g][half]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int g = 2 * warp + u;
      if (lane == 0) {
        total[g] = sum[u];
        if (p.lse != nullptr && g < n)
          p.lse[row * p.lse_row_stride + h * p.group + g0 + g] =
              sum[u] > 0.0f || sum[u] != sum[u] ? (high[u] + log2f(sum[u])) * 0.69314718055994531f
                                                : -INFINITY;
      }
    }
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = tid + half * kGenThreads;
      if (c >= p.dim) continue;
#pragma unroll
      for (int g = 0; g < kGenHeads; ++g) {
        if (g >= n) continue;
        const float o = total[g] == 0.0f ? 0.0f : acc[g][half] / total[g];
        static_cast<uint16_t*>(p.out)[row * p.out_row_stride +
                                      (h * p.group + g0 + g) * p.out_head_stride + c] =
            f_to_half(o, p.dtype);
      }
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kGenThreads) attention_weights_general(TreeParams p) {
  __shared__ float q[kGenHeads][kGenDim];
  __shared__ float base[kGenHeads], factor[kGenHeads];
  __shared__ int row_of[kGenHeads];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.y / p.kv_heads, h = blockIdx.y - b * p.kv_heads, tid = threadIdx.x;
  const TreeRequest r = tree_request_info(p, b);
  const int tokens = min(r.tokens, p.capacity);
  const int t = blockIdx.x * kGenThreads + tid;
  if (blockIdx.x * kGenThreads >= tokens) return;
  const uint16_t* krow =
      t < tokens ? tree_row(p, p.k_cache, p.k_block_stride, p.k_token_stride, p.k_head_stride, b,
                            h, t)
                 : nullptr;
  float got = 0.0f;
  const int pairs = r.count * p.group;
  for (int n0 = 0; n0 < pairs; n0 += kGenHeads) {
    __syncthreads();
    for (int c = tid; c < kGenHeads * p.dim; c += kGenThreads) {
      const int n = c / p.dim, d = c - n * p.dim;
      const int i = (n0 + n) / p.group, g = (n0 + n) - i * p.group;
      q[n][d] = n0 + n < pairs
                    ? half_to_f(static_cast<const uint16_t*>(
                                    p.q)[(r.row0 + i) * p.q_row_stride +
                                         (h * p.group + g) * p.q_head_stride + d],
                                p.dtype)
                    : 0.0f;
    }
    if (tid < kGenHeads) {
      const int i = (n0 + tid) / p.group, g = (n0 + tid) - i * p.group;
      const bool in = n0 + tid < pairs;
      const int64_t row = r.row0 + i;
      row_of[tid] = in ? i : -1;
      const float l = in ? p.lse[row * p.lse_row_stride + h * p.group + g] : -INFINITY;
      const float f = !in ? 0.0f
                      : p.row_factors != nullptr ? p.row_factors[row * p.factor_stride] : 1.0f;
      // a row that saw nothing, or that counts for nothing, gives nothing
      if (l == -INFINITY || f == 0.0f) row_of[tid] = -1;
      base[tid] = l * 1.4426950408889634f;
      factor[tid] = f;
    }
    __syncthreads();
    if (krow == nullptr) continue;
    float s[kGenHeads];
    dot_rows<kGenHeads>(krow, q, p.dim, p.dtype, s);
#pragma unroll
    for (int n = 0; n < kGenHeads; ++n)
      if (row_of[n] >= 0 && tree_sees(p, r, row_of[n], t))
        got += factor[n] * exp2f(fmaf(s[n], p.scale_log2, -base[n]));
  }
  if (t < tokens)
    p.weights_out[b * p.wo_req_stride + h * p.wo_head_stride + t] =
        p.weights[b * p.w_req_stride + h * p.w_head_stride + t] + got;
}

}  // namespace

size_t tree_attention_workspace(int rows, int requests, int q_heads, int kv_heads, int dim,
                                int max_query_len) {
  return tree_attention_tc_workspace(q_heads / kv_heads, dim, std::min(max_query_len, rows));
}

cudaError_t launch_tree_attention(const TreeParams& p, cudaStream_t stream) {
  if (tree_attention_tc_eligible(p)) {
    const cudaError_t e = launch_tree_attention_tc(p, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  return count_launches(launch_kernel(tree_attention_general, dim3(p.rows, p.kv_heads),
                                      dim3(kGenThreads), 0, stream, 1, p));
}

cudaError_t launch_attention_weights(const TreeParams& p, cudaStream_t stream) {
  const int64_t reach = static_cast<int64_t>(p.table_width) * p.page_size;
  const int tokens = static_cast<int>(std::min<int64_t>(reach, p.capacity));
  const int tiles = (tokens + kGenThreads - 1) / kGenThreads;
  if (tiles == 0) return cudaSuccess;
  if (attention_weights_tc_eligible(p)) {
    const cudaError_t e = launch_attention_weights_tc(p, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  return count_launches(launch_kernel(attention_weights_general,
                                      dim3(tiles, p.requests * p.kv_heads), dim3(kGenThreads), 0,
                                      stream, 1, p));
}

}  // namespace qsa
