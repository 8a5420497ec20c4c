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
// Work split.  A warp takes a token, or `parts` warps share its heads when
// there are few tokens.  It computes the token's sines and cosines into shared
// memory once (while its first loads are in flight); each lane then keeps
// those of one chunk of pairs in registers and walks the heads with it, so
// that a head costs little more than its loads, products and stores: finding
// (token, head, chunk) anew for every 16 bytes was instruction-bound (39 us
// instead of 19.5 us for 8192 tokens of 20 heads).  What is only copied (dims
// past the rotated ones, values) follows.
//
// Each value is read and written once: 8192 tokens of 16 + 2 + 2 heads of 128,
// interleaved, would take 12.9 us at a copy's rate, and torch's elementwise
// kernel takes 14.5 us for as many bytes.  The interleaved 16-bit form, held to
// 64 registers for 8 blocks an SM, spills 24 bytes a thread, which is likely a
// part of what lies between that and its 19.5 us; the others do not spill.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace qsa {
namespace {

constexpr int kRotWarps = 4;   // of a block
constexpr int kRotBatch = 2;   // heads in flight per lane
constexpr int kRotAhead = 2;   // frequencies per lane that are loaded ahead

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ float from_f(float x) { return x; }
// Two neighbours rounded together.
__device__ __forceinline__ void store2(__nv_bfloat16* d, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(d) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void store2(__half* d, float a, float b) {
  *reinterpret_cast<__half2*>(d) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void store2(float* d, float a, float b) {
  d[0] = a;
  d[1] = b;
}

template <typename T, int V> struct alignas(sizeof(T) * V) Chunk { T v[V]; };

// A chunk of pairs turned: within it (the pairs side by side), or with its
// partner half a head on.
template <typename T, int V>
__device__ __forceinline__ void turn_within(Chunk<T, V>& a, const float2* t) {
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    const float x = to_f(a.v[2 * j]), y = to_f(a.v[2 * j + 1]);
    store2(&a.v[2 * j], x * t[j].x - y * t[j].y, y * t[j].x + x * t[j].y);
  }
}
template <typename T, int V>
__device__ __forceinline__ void turn_apart(Chunk<T, V>& a, Chunk<T, V>& b, const float2* t) {
  if constexpr (V == 1) {
    const float x = to_f(a.v[0]), y = to_f(b.v[0]);
    a.v[0] = from_f<T>(x * t[0].x - y * t[0].y);
    b.v[0] = from_f<T>(y * t[0].x + x * t[0].y);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float x0 = to_f(a.v[j]), y0 = to_f(b.v[j]);
      const float x1 = to_f(a.v[j + 1]), y1 = to_f(b.v[j + 1]);
      store2(&a.v[j], x0 * t[j].x - y0 * t[j].y, x1 * t[j + 1].x - y1 * t[j + 1].y);
      store2(&b.v[j], y0 * t[j].x + x0 * t[j].y, y1 * t[j + 1].x + x1 * t[j + 1].y);
    }
  }
}

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRotWarps * 32, INTER && V > 1 ? 8 : 5)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 tables[];  // [warp][pair] (cos, sin), times the factor
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.rotary_dim / 2;
  float2* table = tables + warp * half;
  int tok, part;
  p.part_div.divmod(static_cast<int>(blockIdx.x) * kRotWarps + warp, tok, part);
  if (tok >= p.num_tokens) return;
  const int64_t token = tok;
  // pairs whose halves lie in one chunk (interleaved), or chunks a half apart
  constexpr bool kWithin = INTER && V > 1;
  constexpr int kPairs = kWithin ? V / 2 : V;  // pairs of a chunk
  const int second = kWithin ? 0 : INTER ? 1 : half;
  using C = Chunk<T, V>;

  // What everything waits for is asked for first, and nothing but addresses
  // depends on it: position, slot, and the lane's first frequencies.
  const int64_t position = p.positions[token * p.positions_stride];
  const int64_t slot = p.slots != nullptr ? p.slots[token * p.slot_stride] : 0;
  double freq[kRotAhead];
#pragma unroll
  for (int n = 0; n < kRotAhead; ++n)
    freq[n] = n * 32 + lane < half ? p.frequencies[n * 32 + lane] : 0.0;

  // where the key and the value go
  T *k_out = static_cast<T*>(p.k_out) + token * p.ko_row_stride, *v_out = nullptr;
  int64_t k_head = p.ko_head_stride;
  bool stored = true;
  if (p.slots != nullptr) {
    const int64_t block = slot < (int64_t{1} << 32)
                              ? static_cast<int64_t>(p.page_div.div(static_cast<uint32_t>(slot)))
                              : slot / p.page_size;
    const int64_t at = slot - block * p.page_size;
    stored = slot >= 0 && block < p.num_blocks;
    if (slot >= 0 && !stored && lane == 0 && part == 0) record_error(p.err, kDeviceErrOutOfRange);
    k_out = static_cast<T*>(p.k_cache) + block * p.kc_block_stride + at * p.kc_token_stride;
    v_out = static_cast<T*>(p.v_cache) + block * p.vc_block_stride + at * p.vc_token_stride;
    k_head = p.kc_head_stride;
  }
  const T* q = static_cast<const T*>(p.q) + token * p.q_row_stride;
  const T* k = static_cast<const T*>(p.k) + token * p.k_row_stride;
  T* q_out = static_cast<T*>(p.q_out) + token * p.qo_row_stride;

  // the rotated part: lanes are (head of a group of heads, chunk)
  const int chunks = half / kPairs;
  const int step = p.heads_at_once * p.parts;  // heads that all warps of the token take at once
  const int mine = p.chunk_div.div(lane);      // this lane's head of the group
  bool ready = false;
  for (int c0 = 0; c0 < chunks; c0 += 32) {  // more than one turn only for chunks > 32
    const int c = c0 + lane - mine * chunks;
    const int at = c * (kWithin || !INTER ? V : 2);
    // a lane beyond the chunks, or beyond the group's heads, has no heads
    const int from = mine < p.heads_at_once && c < chunks ? part * p.heads_at_once + mine : 1 << 30;
    float2 t[kPairs];  // this lane's sines and cosines
    bool loaded = false;
    auto turn = [&](const T* src, int64_t src_step, T* out, int64_t out_step, int heads,
                    bool write) {
      src += from * src_step + at;
      out += from * out_step + at;
      for (int h0 = from; __any_sync(0xffffffffu, h0 < heads); h0 += step * kRotBatch) {
        C a[kRotBatch], b[kWithin ? 1 : kRotBatch];
#pragma unroll
        for (int u = 0; u < kRotBatch; ++u) {
          if (h0 + u * step >= heads) continue;
          const T* x = src + u * (step * src_step);
          a[u] = *reinterpret_cast<const C*>(x);
          if constexpr (!kWithin) b[u] = *reinterpret_cast<const C*>(x + second);
        }
        if (!ready) {
          ready = true;
          const double turn = static_cast<double>(position) * 0.15915494309189533577;  // / 2pi
          auto entry = [&](int n, double f) {
            double turns = turn * f;
            turns -= rint(turns);
            float si, co;
            sincospif(2.0f * static_cast<float>(turns), &si, &co);
            table[n] = make_float2(co * p.factor, (p.inverse ? -si : si) * p.factor);
          };
#pragma unroll
          for (int n = 0; n < kRotAhead; ++n)
            if (n * 32 + lane < half) entry(n * 32 + lane, freq[n]);
          for (int n = kRotAhead * 32 + lane; n < half; n += 32) entry(n, p.frequencies[n]);
          __syncwarp();
        }
        if (!loaded) {
          loaded = true;
#pragma unroll
          for (int j = 0; j < kPairs; ++j) t[j] = table[(c < chunks ? c : 0) * kPairs + j];
        }
#pragma unroll
        for (int u = 0; u < kRotBatch; ++u) {
          if (h0 + u * step >= heads || !write) continue;
          T* y = out + u * (step * out_step);
          if constexpr (kWithin) {
            turn_within<T, V>(a[u], t);
          } else {
            turn_apart<T, V>(a[u], b[u], t);
            *reinterpret_cast<C*>(y + second) = b[u];
          }
          *reinterpret_cast<C*>(y) = a[u];
        }
        src += kRotBatch * step * src_step;
        out += kRotBatch * step * out_step;
      }
    };
    turn(q, p.q_head_stride, q_out, p.qo_head_stride, p.q_heads, true);
    turn(k, p.k_head_stride, k_out, k_head, p.kv_heads, stored);
  }

  // what is copied: the rest of queries and keys, whole values
  const int rest = (p.head_dim - p.rotary_dim) / V;
  const int copies_q = p.q_in_place ? 0 : p.q_heads * rest;
  const int copies_k = p.k_in_place || !stored ? 0 : p.kv_heads * rest;
  const int copies_v = p.slots != nullptr && stored ? p.kv_heads * (p.head_dim / V) : 0;
  const int copies = copies_q + copies_k + copies_v;
  for (int n0 = part * 32 + lane; n0 < copies; n0 += p.parts * 32 * kRotBatch) {
    C a[kRotBatch];
    T* out[kRotBatch];
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u) {
      int n = n0 + u * p.parts * 32, h, c;
      if (n >= copies) continue;
      const T* src;
      if (n < copies_q + copies_k) {
        const bool key = n >= copies_q;
        p.rest_div.divmod(key ? n - copies_q : n, h, c);
        const int at = p.rotary_dim + c * V;
        src = (key ? k + h * p.k_head_stride : q + h * p.q_head_stride) + at;
        out[u] = (key ? k_out + h * k_head : q_out + h * p.qo_head_stride) + at;
      } else {
        p.value_div.divmod(n - copies_q - copies_k, h, c);
        src = static_cast<const T*>(p.v) + token * p.v_row_stride + h * p.v_head_stride + c * V;
        out[u] = v_out + h * p.vc_head_stride + c * V;
      }
      a[u] = *reinterpret_cast<const C*>(src);
    }
#pragma unroll
    for (int u = 0; u < kRotBatch; ++u)
      if (n0 + u * p.parts * 32 < copies) *reinterpret_cast<C*>(out[u]) = a[u];
  }
}

template <typename T, int V>
cudaError_t launch_typed(const RotaryParams& p, int grid, size_t smem, cudaStream_t stream) {
  auto fn = p.interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
  return count_launches(launch_kernel(fn, dim3(grid), dim3(kRotWarps * 32), smem, stream, 1, p), 1);
}

}  // namespace

cudaError_t launch_rotary(RotaryParams p, cudaStream_t stream) {
  const int size = p.dtype == kDtypeF32 ? 4 : 2;
  const int V = p.vec ? 16 / size : 1;
  const int half = p.rotary_dim / 2;
  const int chunks = half / (p.interleaved && V > 1 ? V / 2 : V);
  p.heads_at_once = std::max(1, 32 / chunks);
  p.chunk_div = FastDiv(static_cast<uint32_t>(std::min(chunks, 32)));
  p.rest_div = FastDiv(static_cast<uint32_t>(std::max(1, (p.head_dim - p.rotary_dim) / V)));
  p.value_div = FastDiv(static_cast<uint32_t>(std::max(1, p.head_dim / V)));
  // warps of a token: one batch of heads each while that still adds to what
  // the GPU has in flight (16 warps an SM)
  const int groups = (p.q_heads + p.kv_heads + p.heads_at_once - 1) / p.heads_at_once;
  int parts = 1;
  while (parts < groups && static_cast<int64_t>(p.num_tokens) * parts < 16 * num_sms()) parts *= 2;
  p.parts = parts;
  p.part_div = FastDiv(static_cast<uint32_t>(parts));
  const int64_t warps = static_cast<int64_t>(p.num_tokens) * parts;
  const int grid = static_cast<int>((warps + kRotWarps - 1) / kRotWarps);
  const size_t smem = sizeof(float2) * kRotWarps * half;
  switch (p.dtype) {
    case kDtypeBF16:
      return p.vec ? launch_typed<__nv_bfloat16, 8>(p, grid, smem, stream)
                   : launch_typed<__nv_bfloat16, 1>(p, grid, smem, stream);
    case kDtypeF16:
      return p.vec ? launch_typed<__half, 8>(p, grid, smem, stream)
                   : launch_typed<__half, 1>(p, grid, smem, stream);
    default:
      return p.vec ? launch_typed<float, 4>(p, grid, smem, stream)
                   : launch_typed<float, 1>(p, grid, smem, stream);
  }
}

}  // namespace qsa
