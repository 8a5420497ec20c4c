// Rotary positions of query and key heads, with the optional store of keys
// and values to the paged cache, one launch (sm_100a).
//
//   a_i = position * frequencies[i]                (i < rotary_dim / 2)
//   y1  = factor * (x1 cos a_i - x2 sin a_i)
//   y2  = factor * (x2 cos a_i + x1 sin a_i)       (sin negated for the inverse)
//
// on the pairs (x1, x2) = (x[i], x[i + rotary_dim/2]) of the half layout or
// (x[2i], x[2i+1]) of the interleaved one; dims from rotary_dim on are copied.
// The inverse with the same factor is the transposed matrix, so it also maps
// the gradient of y to the gradient of x.
//
// Angles: position * frequency / 2pi is formed and reduced to [-1/2, 1/2]
// turns in 64 bits (a position near 2^20 leaves 2^-33 of a turn; in 32 bits it
// would leave 2^-4), the sine and cosine of what is left are 32-bit, as are
// the products; each output is rounded once.
//
// Work split.  A block takes a few tokens: its threads compute the tokens'
// sines and cosines into shared memory, once for all heads, while their first
// loads of x are in flight, then walk the block's (token, head, chunk) items,
// 16 bytes of each half of the pairs per item.  The kernel is bound by memory:
// each value is read and written once.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace qsa {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotBatch = 4;  // items in flight per thread

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ float from_f(float x) { return x; }

template <typename T, int V> struct alignas(sizeof(T) * V) Chunk { T v[V]; };

// One item: a chunk of V pairs of one head, or V values to copy.
template <typename T, int V>
struct Item {
  const T* src;   // first chunk; nullptr: nothing to do
  T* dst;
  int second;     // element offset of the second chunk (half layout), 0 otherwise
  int angle;      // first pair's entry in the sine table, -1 to copy
};

// The block's item `n` (row-major token, section, head, chunk).
template <typename T, int V, bool INTER>
__device__ __forceinline__ Item<T, V> rotary_item(const RotaryParams& p, int token0, int n) {
  Item<T, V> it{nullptr, nullptr, 0, -1};
  int tok, i;
  p.item_div.divmod(n, tok, i);
  const int64_t token = token0 + tok;
  const T *src;
  T* dst;
  int c, copies;
  if (i < p.q_items) {
    int h;
    p.q_head_div.divmod(i, h, c);
    src = static_cast<const T*>(p.q) + token * p.q_row_stride + h * p.q_head_stride;
    dst = static_cast<T*>(p.q_out) + token * p.qo_row_stride + h * p.qo_head_stride;
    copies = 0;
  } else {
    i -= p.q_items;
    const bool key = i < p.k_items;
    int h;
    if (key) {
      p.k_head_div.divmod(i, h, c);
      src = static_cast<const T*>(p.k) + token * p.k_row_stride + h * p.k_head_stride;
    } else {
      p.v_head_div.divmod(i - p.k_items, h, c);
      src = static_cast<const T*>(p.v) + token * p.v_row_stride + h * p.v_head_stride;
    }
    if (p.slots == nullptr) {
      dst = static_cast<T*>(p.k_out) + token * p.ko_row_stride + h * p.ko_head_stride;
    } else {
      const int64_t slot = p.slots[token * p.slot_stride];
      if (slot < 0) return it;
      const int64_t block = slot < (int64_t{1} << 32)
                                ? static_cast<int64_t>(p.page_div.div(static_cast<uint32_t>(slot)))
                                : slot / p.page_size;
      const int64_t at = slot - block * p.page_size;
      if (block >= p.num_blocks) {
        record_error(p.err, kDeviceErrOutOfRange);
        return it;
      }
      dst = key ? static_cast<T*>(p.k_cache) + block * p.kc_block_stride +
                      at * p.kc_token_stride + h * p.kc_head_stride
                : static_cast<T*>(p.v_cache) + block * p.vc_block_stride +
                      at * p.vc_token_stride + h * p.vc_head_stride;
    }
    copies = key ? 0 : 1;
  }
  const int half = p.rotary_dim / 2;
  // chunks of a rotated head: first the pairs, then the rest of the head
  constexpr int kPairs = INTER && V > 1 ? V / 2 : V;  // pairs per chunk
  const int pair_chunks = half / kPairs;
  if (copies) {
    it.src = src + c * V;
    it.dst = dst + c * V;
  } else if (c < pair_chunks) {
    const int at = INTER ? c * kPairs * 2 : c * V;
    it.src = src + at;
    it.dst = dst + at;
    it.second = INTER ? (V > 1 ? 0 : 1) : half;
    it.angle = tok * half + c * kPairs;
  } else {
    const int at = p.rotary_dim + (c - pair_chunks) * V;
    it.src = src + at;
    it.dst = dst + at;
  }
  return it;
}

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRotThreads)
rotary_kernel(RotaryParams p, int tokens_per_block) {
  extern __shared__ float2 table[];  // [token of the block][pair] (cos, sin), times the factor
  pdl_wait();
  pdl_trigger();
  const int token0 = blockIdx.x * tokens_per_block;
  const int tokens = min(tokens_per_block, p.num_tokens - token0);
  const int items = tokens * static_cast<int>(p.item_div.d);
  const int half = p.rotary_dim / 2;
  using C = Chunk<T, V>;
  Item<T, V> it[kRotBatch];
  C a[kRotBatch], b[kRotBatch];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      const int n = base + u * kRotThreads;
      it[u].src = nullptr;
      if (n < items) it[u] = rotary_item<T, V, INTER>(p, token0, n);
      if (it[u].src != nullptr) {
        a[u] = *reinterpret_cast<const C*>(it[u].src);
        if (it[u].second) b[u] = *reinterpret_cast<const C*>(it[u].src + it[u].second);
      }
    }
  };
  int base = threadIdx.x;
  load(base);
  for (int n = threadIdx.x; n < tokens * half; n += kRotThreads) {
    const int tok = n / half, i = n - tok * half;
    double turns = static_cast<double>(p.positions[(token0 + tok) * p.positions_stride]) *
                   p.frequencies[i] * 0.15915494309189533577;  // 1 / 2pi
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    table[n] = make_float2(c * p.factor, (p.inverse ? -s : s) * p.factor);
  }
  __syncthreads();
  while (base < items) {
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      if (it[u].src == nullptr) continue;
      if (it[u].angle >= 0) {
        const float2* t = table + it[u].angle;
        if constexpr (INTER && V > 1) {
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float x = to_f(a[u].v[2 * j]), y = to_f(a[u].v[2 * j + 1]);
            a[u].v[2 * j] = from_f<T>(x * t[j].x - y * t[j].y);
            a[u].v[2 * j + 1] = from_f<T>(y * t[j].x + x * t[j].y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float x = to_f(a[u].v[j]), y = to_f(b[u].v[j]);
            a[u].v[j] = from_f<T>(x * t[j].x - y * t[j].y);
            b[u].v[j] = from_f<T>(y * t[j].x + x * t[j].y);
          }
          *reinterpret_cast<C*>(it[u].dst + it[u].second) = b[u];
        }
      }
      *reinterpret_cast<C*>(it[u].dst) = a[u];
    }
    base += kRotBatch * kRotThreads;
    if (base < items) load(base);
  }
}

template <typename T, int V>
cudaError_t launch_typed(const RotaryParams& p, int grid, int tokens, size_t smem,
                         cudaStream_t stream) {
  auto fn = p.interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
  return count_launches(launch_kernel(fn, dim3(grid), dim3(kRotThreads), smem, stream, 1, p,
                                      tokens), 1);
}

}  // namespace

cudaError_t launch_rotary(RotaryParams p, cudaStream_t stream) {
  const int size = p.dtype == kDtypeF32 ? 4 : 2;
  const int V = p.vec ? 16 / size : 1;
  const int half = p.rotary_dim / 2;
  const int pairs = p.interleaved && V > 1 ? V / 2 : V;
  // dims past the rotated ones are left alone when a head is turned in place
  const int rest = (p.head_dim - p.rotary_dim) / V;
  const int per_q = half / pairs + (p.q_in_place ? 0 : rest);
  const int per_k = half / pairs + (p.k_in_place ? 0 : rest);
  const int per_v = p.head_dim / V;
  p.q_items = p.q_heads * per_q;
  p.k_items = p.kv_heads * per_k;
  const int items = p.q_items + p.k_items + (p.slots != nullptr ? p.kv_heads * per_v : 0);
  p.item_div = FastDiv(static_cast<uint32_t>(items));
  p.q_head_div = FastDiv(static_cast<uint32_t>(per_q));
  p.k_head_div = FastDiv(static_cast<uint32_t>(per_k));
  p.v_head_div = FastDiv(static_cast<uint32_t>(per_v));
  // tokens per block: enough for one batch of items per thread, as long as the
  // blocks still fill the GPU twice; the sine table stays within 16 KB
  int tokens = std::max(1, kRotBatch * kRotThreads / items);
  while (tokens > 1 && (p.num_tokens + tokens - 1) / tokens < 2 * num_sms()) tokens /= 2;
  tokens = std::max(1, std::min(tokens, 2048 / half));
  const int grid = (p.num_tokens + tokens - 1) / tokens;
  const size_t smem = sizeof(float2) * tokens * half;
  switch (p.dtype) {
    case kDtypeBF16:
      return p.vec ? launch_typed<__nv_bfloat16, 8>(p, grid, tokens, smem, stream)
                   : launch_typed<__nv_bfloat16, 1>(p, grid, tokens, smem, stream);
    case kDtypeF16:
      return p.vec ? launch_typed<__half, 8>(p, grid, tokens, smem, stream)
                   : launch_typed<__half, 1>(p, grid, tokens, smem, stream);
    default:
      return p.vec ? launch_typed<float, 4>(p, grid, tokens, smem, stream)
                   : launch_typed<float, 1>(p, grid, tokens, smem, stream);
  }
}

}  // namespace qsa
