// C ABI of the QSA hot path (declared in include/qsa_b200.h): argument checks,
// error reporting and dispatch to the kernel launchers.  Nothing here
// allocates device memory or synchronises the host (except the explicit
// qsa_device_error_poll).
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <algorithm>
#include <cstring>
#include <atomic>
#include <mutex>
#include <set>
#include <tuple>

#include "../../include/qsa_b200.h"
#include "kernels.h"

namespace qsa {

namespace {
thread_local char g_last_error[512] = "";

int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

int cuda_fail(cudaError_t e, const char* what) {
  return fail(QSA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Device-side error word, one per device (a __device__ variable is
// instantiated per device context).
__device__ int g_device_error = 0;

constexpr int kMaxDevices = 64;
int* g_err_ptr[kMaxDevices] = {};
int g_sms[kMaxDevices] = {};
std::mutex g_mu;

int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}

int* device_error_word() {
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return nullptr;
  std::lock_guard<std::mutex> lk(g_mu);
  if (g_err_ptr[dev] == nullptr) {
    void* ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_device_error) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    g_err_ptr[dev] = static_cast<int*>(ptr);
  }
  return g_err_ptr[dev];
}
}  // namespace

int set_last_error(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

std::atomic<uint64_t> g_launches{0};
thread_local cudaEvent_t g_attention_events[2] = {nullptr, nullptr};

void record_attention_event(int which, cudaStream_t stream) {
  cudaEvent_t ev = g_attention_events[which];
  if (ev == nullptr) return;
  // under stream capture the record becomes an event node of the graph, so
  // graph replays time the kernel too
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaStreamIsCapturing(stream, &cap);
  cudaEventRecordWithFlags(ev, stream,
                           cap == cudaStreamCaptureStatusActive ? cudaEventRecordExternal
                                                                : cudaEventRecordDefault);
}

cudaError_t count_launches(cudaError_t e, int n) {
  if (e == cudaSuccess) g_launches.fetch_add(static_cast<uint64_t>(n), std::memory_order_relaxed);
  return e;
}

int num_sms() {
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices) return 148;
  std::lock_guard<std::mutex> lk(g_mu);
  if (g_sms[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    g_sms[dev] = n;
  }
  return g_sms[dev];
}

cudaError_t set_attr_once(const void* fn, cudaFuncAttribute attr, int value) {
  static std::mutex mu;
  static std::set<std::tuple<const void*, int, int, int>> done;
  const auto key = std::make_tuple(fn, static_cast<int>(attr), value, current_device());
  {
    std::lock_guard<std::mutex> lk(mu);
    if (done.count(key)) return cudaSuccess;
  }
  const cudaError_t e = cudaFuncSetAttribute(fn, attr, value);
  if (e == cudaSuccess) {
    std::lock_guard<std::mutex> lk(mu);
    done.insert(key);
  }
  return e;
}

}  // namespace qsa

using namespace qsa;

extern "C" {

const char* qsa_status_string(int status) {
  switch (status) {
    case QSA_OK: return "ok";
    case QSA_ERR_INVALID: return "invalid argument";
    case QSA_ERR_UNSUPPORTED: return "unsupported shape";
    case QSA_ERR_WORKSPACE: return "workspace too small";
    case QSA_ERR_CUDA: return "CUDA error";
    case QSA_ERR_DEVICE: return "not an sm_100 device";
    case QSA_ERR_TIMEOUT: return "device wait timed out";
  }
  return "unknown status";
}

const char* qsa_last_error(void) { return g_last_error; }

const char* qsa_version(void) { return "qsa_b200 0.1.0 (sm_100a)"; }

uint64_t qsa_kernel_launches(void) { return qsa::g_launches.load(std::memory_order_relaxed); }

int qsa_set_attention_timing_events(void* before, void* after) {
  qsa::g_attention_events[0] = static_cast<cudaEvent_t>(before);
  qsa::g_attention_events[1] = static_cast<cudaEvent_t>(after);
  return QSA_OK;
}

int qsa_device_check(void) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  int major = 0, minor = 0;
  cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
  if (major != 10 || minor != 0)
    return fail(QSA_ERR_DEVICE, "device %d is sm_%d%d; this library is built for sm_100a", dev,
                major, minor);
  return QSA_OK;
}

int qsa_device_error_poll(int32_t* error_bits) {
  int* w = device_error_word();
  if (w == nullptr) return fail(QSA_ERR_CUDA, "device error word unavailable");
  int v = 0;
  cudaError_t e = cudaMemcpy(&v, w, sizeof(int), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return cuda_fail(e, "reading device error word");
  if (v != 0) {
    const int zero = 0;
    e = cudaMemcpy(w, &zero, sizeof(int), cudaMemcpyHostToDevice);
    if (e != cudaSuccess) return cuda_fail(e, "clearing device error word");
  }
  if (error_bits) *error_bits = v;
  return QSA_OK;
}

int qsa_selftest_wait_timeout(void* stream) {
  int* w = device_error_word();
  if (w == nullptr) return fail(QSA_ERR_CUDA, "device error word unavailable");
  cudaError_t e = launch_wait_timeout_selftest(w, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "qsa_selftest_wait_timeout");
  return QSA_OK;
}

// ------------------------------------------------------------------ top-k
static int topk_common(TopkParams& p, void* stream, const char* who) {
  if (p.rows < 0 || p.width < 0) return fail(QSA_ERR_INVALID, "%s: negative rows/width", who);
  if (p.rows == 0) return QSA_OK;
  // lengths may be NULL only when the kernel can derive them (expansion)
  if (!p.scores || (!p.lengths && !p.expand) || !p.output)
    return fail(QSA_ERR_INVALID, "%s: null scores/lengths/output", who);
  if (p.score_row_stride < p.width)
    return fail(QSA_ERR_INVALID, "%s: score row stride %lld < width %d", who,
                (long long)p.score_row_stride, p.width);
  if (p.width > topk_max_width())
    return fail(QSA_ERR_UNSUPPORTED, "%s: score width %d exceeds %d", who, p.width,
                topk_max_width());
  if (p.topk > topk_max_blocks())
    return fail(QSA_ERR_UNSUPPORTED, "%s: top-k of %d blocks exceeds %d", who, p.topk,
                topk_max_blocks());
  p.vec4 = aligned(p.scores, 16) && (p.score_row_stride % 4 == 0);
  int cluster = 0;
  cudaError_t e = launch_topk(p, static_cast<cudaStream_t>(stream), &cluster);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

int qsa_topk_expand(const float* scores, int64_t score_row_stride, int32_t rows,
                    int32_t score_width, const int32_t* lengths, const int64_t* positions,
                    const int32_t* sequence_lengths, int32_t num_requests,
                    const int32_t* token_to_req, const int32_t* table,
                    int64_t table_row_stride, int32_t table_width, int32_t* output,
                    int64_t output_row_stride, int64_t output_col_stride,
                    int32_t output_width, int32_t* counts, int32_t ratio, int32_t page_size,
                    int32_t physical, void* stream) {
  if (ratio <= 0) return fail(QSA_ERR_INVALID, "qsa_topk_expand: ratio must be positive");
  if (physical && page_size <= 0)
    return fail(QSA_ERR_INVALID, "qsa_topk_expand: page_size must be positive");
  if (rows > 0 && (!positions || !sequence_lengths || !token_to_req))
    return fail(QSA_ERR_INVALID, "qsa_topk_expand: null metadata pointer");
  if (physical && rows > 0 && !table)
    return fail(QSA_ERR_INVALID, "qsa_topk_expand: physical output needs a table");
  if (output_width < 0 || num_requests < 0)
    return fail(QSA_ERR_INVALID, "qsa_topk_expand: negative output width / requests");
  TopkParams p = {};
  p.scores = scores;
  p.score_row_stride = score_row_stride;
  p.rows = rows;
  p.width = score_width;
  p.lengths = lengths;
  p.positions = positions;
  p.seq_lens = sequence_lengths;
  p.num_requests = num_requests;
  p.token_to_req = token_to_req;
  p.table = table;
  p.table_row_stride = table_row_stride;
  p.table_width = physical ? table_width : 0;
  p.output = output;
  p.out_row_stride = output_row_stride;
  p.out_col_stride = output_col_stride;
  p.out_width = output_width;
  p.counts = counts;
  p.ratio = ratio;
  p.page_size = physical ? page_size : 1;
  p.page_div = FastDiv(static_cast<uint32_t>(p.page_size));
  p.physical = physical ? 1 : 0;
  p.aligned_blocks = (physical && page_size % ratio == 0) ? 1 : 0;
  p.expand = 1;
  p.topk = output_width / ratio;
  return topk_common(p, stream, "qsa_topk_expand");
}

int qsa_topk(const float* scores, int64_t score_row_stride, int32_t rows, int32_t score_width,
             const int32_t* lengths, int32_t* output, int64_t output_row_stride, int32_t topk,
             void* stream) {
  if (topk < 0) return fail(QSA_ERR_INVALID, "qsa_topk: negative topk");
  TopkParams p = {};
  p.scores = scores;
  p.score_row_stride = score_row_stride;
  p.rows = rows;
  p.width = score_width;
  p.lengths = lengths;
  p.output = output;
  p.out_row_stride = output_row_stride;
  p.out_col_stride = 1;
  p.out_width = topk;
  p.ratio = 1;
  p.page_size = 1;
  p.expand = 0;
  p.topk = topk;
  return topk_common(p, stream, "qsa_topk");
}

// ---------------------------------------------------------------- indexer
int qsa_indexer_scores(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                       int32_t num_heads, int32_t head_dim, const void* k_cache,
                       int64_t cache_block_stride, int64_t cache_token_stride,
                       int32_t num_blocks, int32_t page_size, const int32_t* page_table,
                       int64_t table_row_stride, int32_t table_width, int32_t num_requests,
                       const int32_t* visible, const int64_t* positions,
                       const int32_t* sequence_lengths, int32_t num_sequences,
                       const int32_t* token_to_req, int32_t ratio,
                       const int32_t* query_start_loc, int32_t decode_query_len,
                       int32_t max_query_len, int32_t query_offset,
                       int32_t num_rows, const float* weights, int64_t weight_row_stride,
                       int64_t weight_head_stride, float scale, float* logits,
                       int64_t logits_row_stride, int32_t logits_width, void* stream) {
  const char* who = "qsa_indexer_scores";
  if (num_rows < 0 || logits_width < 0) return fail(QSA_ERR_INVALID, "%s: negative size", who);
  if (num_rows == 0) return QSA_OK;
  if (!q || !k_cache || !page_table || !logits)
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  if (!visible && (!positions || !sequence_lengths || !token_to_req || ratio <= 0 ||
                   num_sequences < 0))
    return fail(QSA_ERR_INVALID,
                "%s: without visible counts, positions / sequence_lengths / token_to_req and a "
                "positive ratio are needed", who);
  if (head_dim != 64 && head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", who, head_dim);
  const bool pow2 = num_heads > 0 && num_heads <= 8 && (num_heads & (num_heads - 1)) == 0;
  if (!(pow2 || (num_heads > 0 && num_heads % 8 == 0 && num_heads <= 128)))
    return fail(QSA_ERR_UNSUPPORTED, "%s: %d heads (supported: 1,2,4,8 or a multiple of 8)",
                who, num_heads);
  if (page_size <= 0 || table_width < 0 || num_blocks < 0)
    return fail(QSA_ERR_INVALID, "%s: bad page geometry", who);
  if (!aligned(q, 16) || q_row_stride % 8 || q_head_stride % 8 || !aligned(k_cache, 16) ||
      cache_block_stride % 8 || cache_token_stride % 8)
    return fail(QSA_ERR_INVALID, "%s: q / key cache need 16-byte aligned rows", who);
  if (query_start_loc == nullptr) {
    if (decode_query_len <= 0 || num_rows % decode_query_len)
      return fail(QSA_ERR_INVALID, "%s: %d decode rows not a multiple of query len %d", who,
                  num_rows, decode_query_len);
    if (decode_query_len * num_heads > 128)
      return fail(QSA_ERR_UNSUPPORTED, "%s: decode_query_len*heads > 128", who);
    if (query_offset != 0)
      return fail(QSA_ERR_INVALID, "%s: decode rows start at offset 0", who);
    if (num_rows / decode_query_len > num_requests)
      return fail(QSA_ERR_INVALID, "%s: %d decode requests but %d page-table rows", who,
                  num_rows / decode_query_len, num_requests);
  } else if (num_requests <= 0 || max_query_len <= 0) {
    return fail(QSA_ERR_INVALID, "%s: prefill needs requests and max_query_len", who);
  }
  IndexerParams p = {};
  p.q = q;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.heads = num_heads;
  p.dim = head_dim;
  p.k_cache = k_cache;
  p.block_stride = cache_block_stride;
  p.token_stride = cache_token_stride;
  p.num_blocks = num_blocks;
  p.page_size = page_size;
  p.page_div = FastDiv(static_cast<uint32_t>(page_size));
  p.table = page_table;
  p.table_row_stride = table_row_stride;
  p.table_width = table_width;
  p.num_requests = num_requests;
  p.visible = visible;
  p.positions = positions;
  p.seq_lens = sequence_lengths;
  p.num_sequences = num_sequences;
  p.token_to_req = token_to_req;
  p.ratio = ratio;
  p.query_start_loc = query_start_loc;
  p.decode_query_len = decode_query_len;
  p.max_query_len = max_query_len;
  p.query_offset = query_offset;
  p.num_rows = num_rows;
  p.weights = weights;
  p.w_row_stride = weight_row_stride;
  p.w_head_stride = weight_head_stride;
  p.scale = scale;
  p.logits = logits;
  p.logits_row_stride = logits_row_stride;
  p.logits_width = logits_width;
  p.err = device_error_word();
  cudaError_t e = launch_indexer(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

int qsa_select_decode(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                      int32_t num_heads, int32_t head_dim, const void* k_cache,
                      int64_t cache_block_stride, int64_t cache_token_stride, int32_t num_blocks,
                      int32_t page_size, const int32_t* page_table, int64_t table_row_stride,
                      int32_t table_width, int32_t num_requests, const int32_t* visible,
                      const int64_t* positions, const int32_t* sequence_lengths,
                      int32_t num_sequences, const int32_t* token_to_req, int32_t ratio,
                      int32_t decode_query_len, int32_t num_rows, const float* weights,
                      int64_t weight_row_stride, int64_t weight_head_stride, float scale,
                      int32_t score_width, const int32_t* main_table,
                      int64_t main_table_row_stride, int32_t main_table_width,
                      int32_t main_page_size, int32_t physical, int32_t* output,
                      int64_t output_row_stride, int64_t output_col_stride,
                      int32_t output_width, int32_t* counts, float* scores_out,
                      int64_t scores_row_stride, void* stream) {
  const char* who = "qsa_select_decode";
  if (num_rows < 0 || score_width < 0 || output_width < 0 || num_sequences < 0)
    return fail(QSA_ERR_INVALID, "%s: negative size", who);
  if (num_rows == 0) return QSA_OK;
  if (!q || !k_cache || !page_table || !output || !positions || !sequence_lengths ||
      !token_to_req)
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  if (ratio <= 0) return fail(QSA_ERR_INVALID, "%s: ratio must be positive", who);
  if (physical && (!main_table || main_page_size <= 0))
    return fail(QSA_ERR_INVALID, "%s: physical output needs a block table and page size", who);
  if (head_dim != 64 && head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", who, head_dim);
  if (page_size <= 0 || table_width < 0 || num_blocks < 0)
    return fail(QSA_ERR_INVALID, "%s: bad page geometry", who);
  if (!aligned(q, 16) || q_row_stride % 8 || q_head_stride % 8 || !aligned(k_cache, 16) ||
      cache_block_stride % 8 || cache_token_stride % 8)
    return fail(QSA_ERR_INVALID, "%s: q / key cache need 16-byte aligned rows", who);
  if (decode_query_len <= 0 || num_rows % decode_query_len)
    return fail(QSA_ERR_INVALID, "%s: %d decode rows not a multiple of query len %d", who,
                num_rows, decode_query_len);
  if (num_rows / decode_query_len > num_requests)
    return fail(QSA_ERR_INVALID, "%s: %d decode requests but %d page-table rows", who,
                num_rows / decode_query_len, num_requests);
  if (scores_out && scores_row_stride < score_width)
    return fail(QSA_ERR_INVALID, "%s: scores row stride %lld < width %d", who,
                (long long)scores_row_stride, score_width);
  SelectParams sp = {};
  IndexerParams& p = sp.ix;
  p.q = q;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.heads = num_heads;
  p.dim = head_dim;
  p.k_cache = k_cache;
  p.block_stride = cache_block_stride;
  p.token_stride = cache_token_stride;
  p.num_blocks = num_blocks;
  p.page_size = page_size;
  p.page_div = FastDiv(static_cast<uint32_t>(page_size));
  p.table = page_table;
  p.table_row_stride = table_row_stride;
  p.table_width = table_width;
  p.num_requests = num_requests;
  p.visible = visible;
  p.positions = positions;
  p.seq_lens = sequence_lengths;
  p.num_sequences = num_sequences;
  p.token_to_req = token_to_req;
  p.ratio = ratio;
  p.query_start_loc = nullptr;
  p.decode_query_len = decode_query_len;
  p.max_query_len = decode_query_len;
  p.query_offset = 0;
  p.num_rows = num_rows;
  p.weights = weights;
  p.w_row_stride = weight_row_stride;
  p.w_head_stride = weight_head_stride;
  p.scale = scale;
  p.logits = nullptr;
  p.logits_row_stride = 0;
  p.logits_width = score_width;
  p.err = device_error_word();
  TopkParams& t = sp.tk;
  t.rows = num_rows;
  t.width = score_width;
  t.positions = positions;
  t.seq_lens = sequence_lengths;
  t.num_requests = num_sequences;
  t.token_to_req = token_to_req;
  t.table = main_table;
  t.table_row_stride = main_table_row_stride;
  t.table_width = physical ? main_table_width : 0;
  t.output = output;
  t.out_row_stride = output_row_stride;
  t.out_col_stride = output_col_stride;
  t.out_width = output_width;
  t.counts = counts;
  t.ratio = ratio;
  t.page_size = physical ? main_page_size : 1;
  t.page_div = FastDiv(static_cast<uint32_t>(t.page_size));
  t.physical = physical ? 1 : 0;
  t.aligned_blocks = (physical && main_page_size % ratio == 0) ? 1 : 0;
  t.expand = 1;
  t.topk = output_width / ratio;
  sp.score_width = score_width;
  sp.scores_out = scores_out;
  sp.scores_row_stride = scores_row_stride;
  const char* why = "unsupported shape";
  const cudaError_t e = launch_select_decode(sp, static_cast<cudaStream_t>(stream), &why);
  if (e == cudaErrorNotSupported)
    return fail(QSA_ERR_UNSUPPORTED,
                "%s: outside the fused kernel's range (%s); use qsa_indexer_scores + "
                "qsa_topk_expand", who, why);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

int qsa_visible_blocks(const int64_t* positions, const int32_t* sequence_lengths,
                       int32_t num_requests, const int32_t* token_to_req, int32_t rows,
                       int32_t ratio, int32_t* visible, void* stream) {
  const char* who = "qsa_visible_blocks";
  if (rows < 0 || ratio <= 0) return fail(QSA_ERR_INVALID, "%s: bad rows / ratio", who);
  if (rows == 0) return QSA_OK;
  if (!positions || !sequence_lengths || !token_to_req || !visible)
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  cudaError_t e = launch_visible_blocks(positions, sequence_lengths, num_requests, token_to_req,
                                        rows, ratio, visible, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

// ---------------------------------------------------------------- prepare
int qsa_prepare(const void* index_qk, int64_t index_row_stride, int32_t num_tokens,
                int32_t num_index_heads, int32_t index_head_dim, const int64_t* positions,
                int64_t positions_stride, const void* q_norm_weight, const void* k_norm_weight,
                const void* cos_sin_cache, int64_t cos_sin_rows, int32_t rotary_dim, float eps,
                void* index_q_out, void* state_cache, int64_t state_block_stride,
                int64_t state_token_stride, int64_t state_blocks, int32_t state_size,
                const int64_t* state_slots, const int32_t* state_table,
                int64_t state_table_stride, const int32_t* query_start_loc,
                int32_t num_requests, const int64_t* logical_positions, void* compressed_cache,
                int64_t compressed_block_stride, int64_t compressed_token_stride,
                int64_t compressed_blocks, int32_t compressed_page_size,
                const int64_t* compressed_slots, const int32_t* k_work, int32_t num_k_work,
                int32_t compress_ratio, const void* main_key, int64_t main_key_token_stride,
                int64_t main_key_head_stride, int64_t main_key_dim_stride,
                const void* main_value, int64_t main_value_token_stride,
                int64_t main_value_head_stride, int64_t main_value_dim_stride,
                void* main_key_cache, int64_t main_key_cache_block_stride,
                int64_t main_key_cache_token_stride, int64_t main_key_cache_head_stride,
                int64_t main_key_cache_dim_stride, void* main_value_cache,
                int64_t main_value_cache_block_stride, int64_t main_value_cache_token_stride,
                int64_t main_value_cache_head_stride, int64_t main_value_cache_dim_stride,
                int64_t main_blocks, int32_t main_page_size, const int64_t* main_slots,
                int32_t num_main_kv_heads, int32_t main_head_dim, void* stream) {
  const char* who = "qsa_prepare";
  if (num_tokens < 0 || num_k_work < 0 || num_index_heads <= 0 || num_main_kv_heads < 0 ||
      num_requests < 0)
    return fail(QSA_ERR_INVALID, "%s: negative or zero sizes", who);
  if (index_head_dim != 64 && index_head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, "%s: index head dim %d (64 or 128 supported)", who,
                index_head_dim);
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > index_head_dim)
    return fail(QSA_ERR_INVALID, "%s: rotary dim %d must be even and in [2, %d]", who,
                rotary_dim, index_head_dim);
  if (compress_ratio <= 0 || state_size <= 0 || compressed_page_size <= 0 ||
      (num_main_kv_heads > 0 && (main_page_size <= 0 || main_head_dim <= 0)))
    return fail(QSA_ERR_INVALID, "%s: ratio, ring size and page sizes must be positive", who);
  if (num_tokens == 0 && num_k_work == 0) return QSA_OK;
  if (!index_qk || !positions || !q_norm_weight || !k_norm_weight || !cos_sin_cache ||
      !index_q_out)
    return fail(QSA_ERR_INVALID, "%s: null index projection / weights / rotary cache", who);
  if (num_k_work > 0 && (!state_cache || !state_slots || !state_table || !query_start_loc ||
                         !logical_positions || !compressed_cache || !compressed_slots || !k_work))
    return fail(QSA_ERR_INVALID, "%s: null compression metadata or cache", who);
  if (num_main_kv_heads > 0 && num_tokens > 0 &&
      (!main_key || !main_value || !main_key_cache || !main_value_cache || !main_slots))
    return fail(QSA_ERR_INVALID, "%s: null main K/V or cache", who);
  if (index_row_stride < static_cast<int64_t>(num_index_heads + 1) * index_head_dim)
    return fail(QSA_ERR_INVALID, "%s: index row stride %lld < (heads + 1) * dim", who,
                (long long)index_row_stride);
  // rows are read and written as bf16 pairs
  if (!aligned(index_qk, 4) || index_row_stride % 2 || !aligned(index_q_out, 4) ||
      (num_k_work > 0 && (!aligned(state_cache, 4) || state_block_stride % 2 ||
                          state_token_stride % 2 || !aligned(compressed_cache, 4) ||
                          compressed_block_stride % 2 || compressed_token_stride % 2)))
    return fail(QSA_ERR_INVALID, "%s: index rows must be 4-byte aligned with even strides", who);
  PrepareParams p{};
  p.index_qk = static_cast<const __nv_bfloat16*>(index_qk);
  p.index_row_stride = index_row_stride;
  p.num_tokens = num_tokens;
  p.heads = num_index_heads;
  p.dim = index_head_dim;
  p.positions = positions;
  p.positions_stride = positions_stride;
  p.q_weight = static_cast<const __nv_bfloat16*>(q_norm_weight);
  p.k_weight = static_cast<const __nv_bfloat16*>(k_norm_weight);
  p.cos_sin = static_cast<const __nv_bfloat16*>(cos_sin_cache);
  p.cos_sin_rows = cos_sin_rows;
  p.rotary = rotary_dim;
  p.eps = eps;
  p.index_q_out = static_cast<__nv_bfloat16*>(index_q_out);
  p.state_cache = static_cast<__nv_bfloat16*>(state_cache);
  p.state_block_stride = state_block_stride;
  p.state_token_stride = state_token_stride;
  p.state_size = state_size;
  p.state_blocks = state_blocks;
  p.state_slots = state_slots;
  p.state_table = state_table;
  p.state_table_stride = state_table_stride;
  p.query_start_loc = query_start_loc;
  p.num_requests = num_requests;
  p.logical_positions = logical_positions;
  p.compressed_cache = static_cast<__nv_bfloat16*>(compressed_cache);
  p.comp_block_stride = compressed_block_stride;
  p.comp_token_stride = compressed_token_stride;
  p.comp_page = compressed_page_size;
  p.comp_blocks = compressed_blocks;
  p.compressed_slots = compressed_slots;
  p.k_work = k_work;
  p.num_k_work = num_k_work;
  p.ratio = compress_ratio;
  p.main_key = static_cast<const __nv_bfloat16*>(main_key);
  p.main_value = static_cast<const __nv_bfloat16*>(main_value);
  p.main_key_cache = static_cast<__nv_bfloat16*>(main_key_cache);
  p.main_value_cache = static_cast<__nv_bfloat16*>(main_value_cache);
  const int64_t mk[3] = {main_key_token_stride, main_key_head_stride, main_key_dim_stride};
  const int64_t mv[3] = {main_value_token_stride, main_value_head_stride, main_value_dim_stride};
  const int64_t kc[4] = {main_key_cache_block_stride, main_key_cache_token_stride,
                         main_key_cache_head_stride, main_key_cache_dim_stride};
  const int64_t vc[4] = {main_value_cache_block_stride, main_value_cache_token_stride,
                         main_value_cache_head_stride, main_value_cache_dim_stride};
  bool vec = main_head_dim % 8 == 0 && aligned(main_key, 16) && aligned(main_value, 16) &&
             aligned(main_key_cache, 16) && aligned(main_value_cache, 16);
  for (int i = 0; i < 3; ++i) {
    p.mk_stride[i] = mk[i];
    p.mv_stride[i] = mv[i];
    vec = vec && (i == 2 ? mk[i] == 1 && mv[i] == 1 : mk[i] % 8 == 0 && mv[i] % 8 == 0);
  }
  for (int i = 0; i < 4; ++i) {
    p.kc_stride[i] = kc[i];
    p.vc_stride[i] = vc[i];
    vec = vec && (i == 3 ? kc[i] == 1 && vc[i] == 1 : kc[i] % 8 == 0 && vc[i] % 8 == 0);
  }
  p.main_slots = main_slots;
  p.kv_heads = num_main_kv_heads;
  p.main_dim = main_head_dim;
  p.main_page = main_page_size;
  p.main_blocks = main_blocks;
  p.main_vec = vec ? 1 : 0;
  p.err = device_error_word();
  cudaError_t e = launch_prepare(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

// ----------------------------------------------------------------- rotary
int qsa_rotary(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t num_q_heads,
               void* q_out, int64_t q_out_row_stride, int64_t q_out_head_stride, const void* k,
               int64_t k_row_stride, int64_t k_head_stride, int32_t num_kv_heads, void* k_out,
               int64_t k_out_row_stride, int64_t k_out_head_stride, const void* v,
               int64_t v_row_stride, int64_t v_head_stride, void* k_cache, int64_t k_block_stride,
               int64_t k_token_stride, int64_t k_cache_head_stride, void* v_cache,
               int64_t v_block_stride, int64_t v_token_stride, int64_t v_cache_head_stride,
               int64_t num_blocks, int32_t page_size, const int64_t* slots, int64_t slots_stride,
               int32_t num_tokens, int32_t head_dim, const int64_t* positions,
               int64_t positions_stride, const double* frequencies, int32_t rotary_dim,
               float factor, int32_t interleaved, int32_t inverse, int32_t dtype, void* stream) {
  const char* who = "qsa_rotary";
  if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads < 0)
    return fail(QSA_ERR_INVALID, "%s: negative size", who);
  if (dtype != QSA_DTYPE_BF16 && dtype != QSA_DTYPE_F16 && dtype != QSA_DTYPE_F32)
    return fail(QSA_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (head_dim <= 0 || head_dim > 1024)
    return fail(QSA_ERR_UNSUPPORTED, "%s: head_dim %d (1..1024 supported)", who, head_dim);
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(QSA_ERR_INVALID, "%s: rotary dim %d must be even and in [2, %d]", who, rotary_dim,
                head_dim);
  if (static_cast<int64_t>(num_q_heads) + 2 * static_cast<int64_t>(num_kv_heads) > 65536)
    return fail(QSA_ERR_UNSUPPORTED, "%s: more than 65536 heads", who);
  if (num_tokens == 0 || (num_q_heads == 0 && num_kv_heads == 0)) return QSA_OK;
  if (!positions || !frequencies || (num_q_heads > 0 && (!q || !q_out)) ||
      (num_kv_heads > 0 && !k))
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  const bool store = slots != nullptr;
  if (num_kv_heads > 0) {
    if (store ? (!v || !k_cache || !v_cache) : !k_out)
      return fail(QSA_ERR_INVALID, "%s: null key / value destination", who);
    if (store && (page_size <= 0 || num_blocks < 0))
      return fail(QSA_ERR_INVALID, "%s: bad page geometry", who);
  }
  const int64_t size = dtype == QSA_DTYPE_F32 ? 4 : 2, chunk = 16 / size;
  const void* ptrs[] = {q, q_out, k, store ? k_cache : k_out, v, v_cache};
  const bool used[] = {num_q_heads > 0, num_q_heads > 0, num_kv_heads > 0, num_kv_heads > 0,
                       num_kv_heads > 0 && store, num_kv_heads > 0 && store};
  const int64_t strides[][3] = {
      {q_row_stride, q_head_stride, 0}, {q_out_row_stride, q_out_head_stride, 0},
      {k_row_stride, k_head_stride, 0},
      {store ? k_block_stride : k_out_row_stride, store ? k_token_stride : 0,
       store ? k_cache_head_stride : k_out_head_stride},
      {v_row_stride, v_head_stride, 0}, {v_block_stride, v_token_stride, v_cache_head_stride}};
  // the pairs' halves, and the dims past them, in whole chunks
  bool vec = head_dim % chunk == 0 && rotary_dim % (interleaved ? chunk : 2 * chunk) == 0;
  for (int i = 0; i < 6; ++i) {
    if (!used[i]) continue;
    if (!aligned(ptrs[i], size))
      return fail(QSA_ERR_INVALID, "%s: a tensor is not aligned to its elements", who);
    vec = vec && aligned(ptrs[i], 16) && strides[i][0] % chunk == 0 && strides[i][1] % chunk == 0 &&
          strides[i][2] % chunk == 0;
  }
  RotaryParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.k_row_stride = k_row_stride;
  p.k_head_stride = k_head_stride;
  p.v_row_stride = v_row_stride;
  p.v_head_stride = v_head_stride;
  p.q_out = q_out;
  p.k_out = k_out;
  p.qo_row_stride = q_out_row_stride;
  p.qo_head_stride = q_out_head_stride;
  p.ko_row_stride = k_out_row_stride;
  p.ko_head_stride = k_out_head_stride;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.kc_block_stride = k_block_stride;
  p.kc_token_stride = k_token_stride;
  p.kc_head_stride = k_cache_head_stride;
  p.vc_block_stride = v_block_stride;
  p.vc_token_stride = v_token_stride;
  p.vc_head_stride = v_cache_head_stride;
  p.num_blocks = num_blocks;
  p.page_size = store && page_size > 0 ? page_size : 1;
  p.page_div = FastDiv(static_cast<uint32_t>(p.page_size));
  p.slots = slots;
  p.slot_stride = slots_stride;
  p.num_tokens = num_tokens;
  p.q_heads = num_q_heads;
  p.kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.positions = positions;
  p.positions_stride = positions_stride;
  p.frequencies = frequencies;
  p.rotary_dim = rotary_dim;
  p.factor = factor;
  p.interleaved = interleaved ? 1 : 0;
  p.inverse = inverse ? 1 : 0;
  p.dtype = dtype;
  p.vec = vec ? 1 : 0;
  p.q_in_place = q == q_out && q_row_stride == q_out_row_stride &&
                 q_head_stride == q_out_head_stride;
  p.k_in_place = !store && k == k_out && k_row_stride == k_out_row_stride &&
                 k_head_stride == k_out_head_stride;
  p.err = device_error_word();
  cudaError_t e = launch_rotary(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

// ------------------------------------------------------------ cache moves
// The caches, tables and copy width of a move; a status other than QSA_OK has
// its message set.
static int move_common(MoveParams& p, const char* who, void* k_cache, int64_t k_block_stride,
                       int64_t k_token_stride, int64_t k_head_stride, void* v_cache,
                       int64_t v_block_stride, int64_t v_token_stride, int64_t v_head_stride,
                       int64_t num_blocks, int32_t page_size, int32_t num_kv_heads,
                       int32_t head_dim, int32_t dtype, const int32_t* block_table,
                       int64_t table_stride, int32_t table_width, const int32_t* out_table,
                       int64_t out_table_stride, int32_t out_table_width, int32_t requests) {
  if (dtype != QSA_DTYPE_BF16 && dtype != QSA_DTYPE_F16 && dtype != QSA_DTYPE_F32)
    return fail(QSA_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (requests < 0 || num_kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || num_blocks < 0 ||
      table_width < 0 || out_table_width < 0)
    return fail(QSA_ERR_INVALID, "%s: bad sizes", who);
  if (static_cast<int64_t>(requests) * num_kv_heads > 65535)
    return fail(QSA_ERR_UNSUPPORTED, "%s: %d requests x %d heads exceed 65535", who, requests,
                num_kv_heads);
  if (requests == 0) return QSA_OK;
  if (!k_cache || !v_cache || !block_table) return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  const int64_t size = dtype == QSA_DTYPE_F32 ? 4 : 2;
  const int64_t bytes[] = {k_block_stride * size, k_token_stride * size, k_head_stride * size,
                           v_block_stride * size, v_token_stride * size, v_head_stride * size,
                           head_dim * size};
  if (!aligned(k_cache, size) || !aligned(v_cache, size))
    return fail(QSA_ERR_INVALID, "%s: a cache is not aligned to its elements", who);
  int64_t unit = 16;
  for (const void* c : {k_cache, v_cache})
    while (!aligned(c, unit)) unit /= unit == 16 ? 4 : 2;
  for (const int64_t n : bytes)
    while (n % unit) unit /= unit == 16 ? 4 : 2;
  if (bytes[6] / unit > move_max_row_units())
    return fail(QSA_ERR_UNSUPPORTED, "%s: rows of %lld units of %lld bytes exceed %d", who,
                (long long)(bytes[6] / unit), (long long)unit, move_max_row_units());
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_block = bytes[0];
  p.k_token = bytes[1];
  p.k_head = bytes[2];
  p.v_block = bytes[3];
  p.v_token = bytes[4];
  p.v_head = bytes[5];
  p.row_bytes = static_cast<int>(bytes[6]);
  p.unit = static_cast<int>(unit);
  p.num_blocks = num_blocks;
  p.page_size = page_size;
  p.page_div = FastDiv(static_cast<uint32_t>(page_size));
  p.requests = requests;
  p.kv_heads = num_kv_heads;
  p.head_div = FastDiv(static_cast<uint32_t>(num_kv_heads));
  p.table = block_table;
  p.table_stride = table_stride;
  p.table_width = table_width;
  p.in_place = out_table == nullptr || out_table == block_table;
  p.out_table = p.in_place ? block_table : out_table;
  p.out_table_stride = p.in_place ? table_stride : out_table_stride;
  p.out_table_width = p.in_place ? table_width : out_table_width;
  p.err = device_error_word();
  return QSA_OK;
}

int qsa_cache_compact(void* k_cache, int64_t k_block_stride, int64_t k_token_stride,
                      int64_t k_head_stride, void* v_cache, int64_t v_block_stride,
                      int64_t v_token_stride, int64_t v_head_stride, int64_t num_blocks,
                      int32_t page_size, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                      const int32_t* block_table, int64_t table_row_stride, int32_t table_width,
                      const int32_t* out_table, int64_t out_table_row_stride,
                      int32_t out_table_width, int32_t num_requests, const int32_t* indices,
                      int64_t indices_request_stride, int64_t indices_head_stride, int32_t count,
                      const int32_t* starts, void* stream) {
  const char* who = "qsa_cache_compact";
  MoveParams p = {};
  const int status = move_common(
      p, who, k_cache, k_block_stride, k_token_stride, k_head_stride, v_cache, v_block_stride,
      v_token_stride, v_head_stride, num_blocks, page_size, num_kv_heads, head_dim, dtype,
      block_table, table_row_stride, table_width, out_table, out_table_row_stride, out_table_width,
      num_requests);
  if (status != QSA_OK) return status;
  if (count < 0) return fail(QSA_ERR_INVALID, "%s: negative count", who);
  if (count == 0 || num_requests == 0) return QSA_OK;
  if (!indices) return fail(QSA_ERR_INVALID, "%s: null indices", who);
  p.count = count;
  p.indices = indices;
  p.idx_req_stride = indices_request_stride;
  p.idx_head_stride = indices_head_stride;
  p.list_heads = num_kv_heads;
  p.list_div = p.head_div;
  p.starts = starts;
  cudaError_t e = launch_cache_compact(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

static size_t evict_chosen_offset(int32_t requests, int32_t list_heads) {
  return (static_cast<size_t>(requests) * list_heads * sizeof(int32_t) + 255) / 256 * 256;
}

size_t qsa_cache_evict_workspace_bytes(int32_t num_requests, int32_t list_heads, int32_t budget,
                                       int32_t sinks, int32_t recent) {
  if (num_requests <= 0 || list_heads <= 0 || sinks < 0 || recent < 0 ||
      static_cast<int64_t>(budget) < static_cast<int64_t>(sinks) + recent)
    return 0;  // no launch for these shapes
  return evict_chosen_offset(num_requests, list_heads) +
         static_cast<size_t>(num_requests) * list_heads * (budget - sinks - recent) *
             sizeof(int32_t);
}

int qsa_cache_evict(const float* weights, int64_t weights_request_stride,
                    int64_t weights_head_stride, int32_t list_heads, int32_t capacity,
                    const int32_t* seq_lens, int32_t num_requests, int32_t budget, int32_t sinks,
                    int32_t recent, void* k_cache, int64_t k_block_stride, int64_t k_token_stride,
                    int64_t k_head_stride, void* v_cache, int64_t v_block_stride,
                    int64_t v_token_stride, int64_t v_head_stride, int64_t num_blocks,
                    int32_t page_size, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                    const int32_t* block_table, int64_t table_row_stride, int32_t table_width,
                    const int32_t* out_table, int64_t out_table_row_stride,
                    int32_t out_table_width, float* weights_out, int64_t weights_out_request_stride,
                    int64_t weights_out_head_stride, int32_t* kept, int32_t* lengths_out,
                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "qsa_cache_evict";
  MoveParams p = {};
  const int status = move_common(
      p, who, k_cache, k_block_stride, k_token_stride, k_head_stride, v_cache, v_block_stride,
      v_token_stride, v_head_stride, num_blocks, page_size, num_kv_heads, head_dim, dtype,
      block_table, table_row_stride, table_width, out_table, out_table_row_stride, out_table_width,
      num_requests);
  if (status != QSA_OK) return status;
  if (list_heads != 1 && list_heads != num_kv_heads)
    return fail(QSA_ERR_INVALID, "%s: weights of %d heads (1 or %d expected)", who, list_heads,
                num_kv_heads);
  if (capacity < 0 || budget < 0 || sinks < 0 || recent < 0 ||
      static_cast<int64_t>(sinks) + recent > budget)
    return fail(QSA_ERR_INVALID, "%s: sinks %d + recent %d must fit the budget %d", who, sinks,
                recent, budget);
  if (num_requests == 0) return QSA_OK;
  if ((capacity > 0 && (!weights || !weights_out)) || !seq_lens || (budget > 0 && !kept) ||
      !lengths_out)
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  if (list_heads > 1 && num_requests > 1 &&
      weights_request_stride != weights_head_stride * list_heads)
    return fail(QSA_ERR_INVALID, "%s: weights' (request, head) rows must be evenly spaced", who);
  const int64_t row_stride = list_heads > 1 ? weights_head_stride : weights_request_stride;
  const int chosen = budget - sinks - recent;
  if (capacity > budget && chosen > 0) {
    if (capacity - sinks - recent > topk_max_width())
      return fail(QSA_ERR_UNSUPPORTED, "%s: %d tokens to choose from exceed %d", who,
                  capacity - sinks - recent, topk_max_width());
    if ((num_requests > 1 || list_heads > 1) && row_stride < capacity)
      return fail(QSA_ERR_INVALID, "%s: weights row stride %lld < %d", who, (long long)row_stride,
                  capacity);
  }
  const size_t need =
      qsa_cache_evict_workspace_bytes(num_requests, list_heads, budget, sinks, recent);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(QSA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu required", who, workspace_bytes,
                need);
  if (!aligned(workspace, 256))
    return fail(QSA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
  p.count = budget;
  p.list_heads = list_heads;
  p.list_div = FastDiv(static_cast<uint32_t>(list_heads));
  p.evict = 1;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  p.capacity = capacity;
  p.seq_lens = seq_lens;
  int32_t* middle = static_cast<int32_t*>(workspace);
  int32_t* list = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) +
                                             evict_chosen_offset(num_requests, list_heads));
  p.chosen = list;
  p.chosen_width = chosen;
  p.weights = weights;
  p.w_req_stride = weights_request_stride;
  p.w_head_stride = weights_head_stride;
  p.weights_out = weights_out;
  p.wo_req_stride = weights_out_request_stride;
  p.wo_head_stride = weights_out_head_stride;
  p.kept = kept;
  cudaError_t e = launch_cache_evict(p, lengths_out, middle, list,
                                     static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

// --------------------------------------- attention of drafted-token trees
// What qsa_tree_attention and qsa_attention_weights share; the value cache is
// null for the latter.
static int tree_common(TreeParams& p, const char* who, const void* q, int64_t q_row_stride,
                       int64_t q_head_stride, int32_t rows, int32_t num_q_heads, int32_t head_dim,
                       int32_t dtype, const void* k_cache, int64_t k_block_stride,
                       int64_t k_token_stride, int64_t k_head_stride, int32_t num_blocks,
                       int32_t page_size, int32_t num_kv_heads, const int32_t* block_table,
                       int64_t table_row_stride, int32_t table_width, int32_t num_requests,
                       const int32_t* seq_lens, const int32_t* query_start_loc,
                       const uint8_t* tree_mask, int64_t mask_row_stride, int32_t mask_width,
                       int32_t max_query_len, float scale) {
  if (rows < 0 || num_requests < 0 || mask_width < 0)
    return fail(QSA_ERR_INVALID, "%s: negative size", who);
  if (dtype != QSA_DTYPE_BF16 && dtype != QSA_DTYPE_F16)
    return fail(QSA_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 supported)", who, dtype);
  if (head_dim <= 0 || head_dim % 8 || head_dim > 256)
    return fail(QSA_ERR_UNSUPPORTED, "%s: head_dim %d (multiples of 8 up to 256 supported)", who,
                head_dim);
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(QSA_ERR_INVALID, "%s: %d query heads not a multiple of %d kv heads", who,
                num_q_heads, num_kv_heads);
  if (num_kv_heads > 65535 || static_cast<int64_t>(num_requests) * num_kv_heads > 65535)
    return fail(QSA_ERR_UNSUPPORTED, "%s: %d requests x %d heads exceed 65535", who, num_requests,
                num_kv_heads);
  if (page_size <= 0 || num_blocks < 0 || table_width < 0)
    return fail(QSA_ERR_INVALID, "%s: bad page geometry", who);
  if (static_cast<int64_t>(table_width) * page_size > (int64_t{1} << 30))
    return fail(QSA_ERR_UNSUPPORTED, "%s: tables of more than 2^30 tokens", who);
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return fail(QSA_ERR_INVALID, "%s: scale must be positive and finite", who);
  if (num_requests == 0) return QSA_OK;
  if (max_query_len <= 0) return fail(QSA_ERR_INVALID, "%s: max_query_len must be positive", who);
  if ((rows > 0 && !q) || !k_cache || !block_table || !seq_lens || !query_start_loc)
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(k_cache, 16) || k_block_stride % 8 || k_token_stride % 8 || k_head_stride % 8)
    return fail(QSA_ERR_INVALID, "%s: cache rows must be 16-byte aligned", who);
  if (rows > 0 && (!aligned(q, 16) || q_row_stride % 8 || q_head_stride % 8))
    return fail(QSA_ERR_INVALID, "%s: q head rows must be 16-byte aligned", who);
  p.q = q;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.rows = rows;
  p.q_heads = num_q_heads;
  p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.dim = head_dim;
  p.dtype = dtype;
  p.k_cache = k_cache;
  p.k_block_stride = k_block_stride;
  p.k_token_stride = k_token_stride;
  p.k_head_stride = k_head_stride;
  p.num_blocks = num_blocks;
  p.page_size = page_size;
  p.page_div = FastDiv(static_cast<uint32_t>(page_size));
  p.table = block_table;
  p.table_stride = table_row_stride;
  p.table_width = table_width;
  p.requests = num_requests;
  p.seq_lens = seq_lens;
  p.query_start_loc = query_start_loc;
  p.mask = tree_mask;
  p.mask_stride = mask_row_stride;
  p.mask_width = mask_width;
  p.scale = scale;
  p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  p.max_query_len = std::min(max_query_len, std::max(rows, 1));
  p.err = device_error_word();
  return QSA_OK;
}

size_t qsa_tree_attention_workspace_bytes(int32_t rows, int32_t num_requests, int32_t num_q_heads,
                                          int32_t num_kv_heads, int32_t head_dim,
                                          int32_t max_query_len) {
  if (rows <= 0 || num_requests <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads || max_query_len <= 0)
    return 0;  // no launch for these shapes
  return tree_attention_workspace(rows, num_requests, num_q_heads, num_kv_heads, head_dim,
                                  max_query_len);
}

int qsa_tree_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t rows,
                       int32_t num_q_heads, int32_t head_dim, int32_t dtype, const void* k_cache,
                       int64_t k_block_stride, int64_t k_token_stride, int64_t k_head_stride,
                       const void* v_cache, int64_t v_block_stride, int64_t v_token_stride,
                       int64_t v_head_stride, int32_t num_blocks, int32_t page_size,
                       int32_t num_kv_heads, const int32_t* block_table, int64_t table_row_stride,
                       int32_t table_width, int32_t num_requests, const int32_t* seq_lens,
                       const int32_t* query_start_loc, const uint8_t* tree_mask,
                       int64_t mask_row_stride, int32_t mask_width, int32_t max_query_len,
                       float scale, void* out, int64_t out_row_stride, int64_t out_head_stride,
                       float* lse, int64_t lse_row_stride, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const char* who = "qsa_tree_attention";
  TreeParams p = {};
  const int status = tree_common(p, who, q, q_row_stride, q_head_stride, rows, num_q_heads,
                                 head_dim, dtype, k_cache, k_block_stride, k_token_stride,
                                 k_head_stride, num_blocks, page_size, num_kv_heads, block_table,
                                 table_row_stride, table_width, num_requests, seq_lens,
                                 query_start_loc, tree_mask, mask_row_stride, mask_width,
                                 max_query_len, scale);
  if (status != QSA_OK) return status;
  if (rows == 0 || num_requests == 0) return QSA_OK;
  if (!v_cache || !out) return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(v_cache, 16) || v_block_stride % 8 || v_token_stride % 8 || v_head_stride % 8)
    return fail(QSA_ERR_INVALID, "%s: cache rows must be 16-byte aligned", who);
  if (!aligned(out, 2)) return fail(QSA_ERR_INVALID, "%s: out must be 2-byte aligned", who);
  const size_t need = tree_attention_workspace(rows, num_requests, num_q_heads, num_kv_heads,
                                               head_dim, max_query_len);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(QSA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu required", who, workspace_bytes,
                need);
  if (need > 0 && !aligned(workspace, 256))
    return fail(QSA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
  p.v_cache = v_cache;
  p.v_block_stride = v_block_stride;
  p.v_token_stride = v_token_stride;
  p.v_head_stride = v_head_stride;
  p.out = out;
  p.out_row_stride = out_row_stride;
  p.out_head_stride = out_head_stride;
  p.out_vec = aligned(out, 16) && out_row_stride % 8 == 0 && out_head_stride % 8 == 0;
  p.lse = lse;
  p.lse_row_stride = lse_row_stride;
  p.workspace = workspace;
  cudaError_t e = launch_tree_attention(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

int qsa_attention_weights(const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t rows,
                          int32_t num_q_heads, int32_t head_dim, int32_t dtype,
                          const void* k_cache, int64_t k_block_stride, int64_t k_token_stride,
                          int64_t k_head_stride, int32_t num_blocks, int32_t page_size,
                          int32_t num_kv_heads, const int32_t* block_table,
                          int64_t table_row_stride, int32_t table_width, int32_t num_requests,
                          const int32_t* seq_lens, const int32_t* query_start_loc,
                          const uint8_t* tree_mask, int64_t mask_row_stride, int32_t mask_width,
                          int32_t max_query_len, float scale, const float* lse,
                          int64_t lse_row_stride, const float* row_factors,
                          int64_t row_factors_stride, const float* weights,
                          int64_t weights_request_stride, int64_t weights_head_stride,
                          float* weights_out, int64_t weights_out_request_stride,
                          int64_t weights_out_head_stride, int32_t capacity, void* stream) {
  const char* who = "qsa_attention_weights";
  TreeParams p = {};
  const int status = tree_common(p, who, q, q_row_stride, q_head_stride, rows, num_q_heads,
                                 head_dim, dtype, k_cache, k_block_stride, k_token_stride,
                                 k_head_stride, num_blocks, page_size, num_kv_heads, block_table,
                                 table_row_stride, table_width, num_requests, seq_lens,
                                 query_start_loc, tree_mask, mask_row_stride, mask_width,
                                 max_query_len, scale);
  if (status != QSA_OK) return status;
  if (capacity < 0) return fail(QSA_ERR_INVALID, "%s: negative capacity", who);
  if (num_requests == 0 || capacity == 0) return QSA_OK;
  if ((rows > 0 && !lse) || !weights || !weights_out) return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  p.lse = const_cast<float*>(lse);
  p.lse_row_stride = lse_row_stride;
  p.row_factors = row_factors;
  p.factor_stride = row_factors_stride;
  p.weights = weights;
  p.w_req_stride = weights_request_stride;
  p.w_head_stride = weights_head_stride;
  p.weights_out = weights_out;
  p.wo_req_stride = weights_out_request_stride;
  p.wo_head_stride = weights_out_head_stride;
  p.capacity = capacity;
  cudaError_t e = launch_attention_weights(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

// -------------------------------------------------------------- attention
size_t qsa_sparse_attention_workspace_bytes(int32_t rows, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t head_dim,
                                            int32_t topk_width, int32_t use_decode_kernel) {
  if (rows <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      topk_width < 0)
    return 0;  // no launch for these shapes (qsa_sparse_attention rejects them)
  return plan_attention(rows, num_q_heads, num_kv_heads, head_dim, topk_width, use_decode_kernel)
      .workspace_bytes;
}

int qsa_sparse_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                         int32_t rows, int32_t num_q_heads, int32_t head_dim,
                         const void* k_cache, int64_t k_block_stride, int64_t k_token_stride,
                         int64_t k_head_stride, const void* v_cache, int64_t v_block_stride,
                         int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                         int32_t page_size, int32_t num_kv_heads, const int32_t* indices,
                         int64_t indices_row_stride, int32_t topk_width,
                         const int32_t* block_table, int64_t table_row_stride,
                         int32_t table_width, int32_t num_requests,
                         const int32_t* token_to_req, const int32_t* valid_counts,
                         const void* gate, int64_t gate_row_stride, int64_t gate_head_stride,
                         int64_t gate_dim_stride, void* out, int64_t out_row_stride,
                         int64_t out_head_stride, int32_t indices_are_physical,
                         int32_t use_decode_kernel, void* workspace, size_t workspace_bytes,
                         void* stream) {
  const char* who = "qsa_sparse_attention";
  if (rows < 0 || topk_width < 0) return fail(QSA_ERR_INVALID, "%s: negative size", who);
  if (rows == 0) return QSA_OK;
  if (!q || !k_cache || !v_cache || !indices || !out)
    return fail(QSA_ERR_INVALID, "%s: null pointer", who);
  if (!indices_are_physical && (!block_table || !token_to_req))
    return fail(QSA_ERR_INVALID, "%s: logical indices need block_table and token_to_req", who);
  if (head_dim != 64 && head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", who, head_dim);
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(QSA_ERR_INVALID, "%s: %d query heads not a multiple of %d kv heads", who,
                num_q_heads, num_kv_heads);
  const int group = num_q_heads / num_kv_heads;
  if (group > 16)
    return fail(QSA_ERR_UNSUPPORTED, "%s: GQA group %d > 16", who, group);
  if (page_size <= 0 || num_blocks < 0) return fail(QSA_ERR_INVALID, "%s: bad page geometry", who);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || k_block_stride % 8 ||
      k_token_stride % 8 || k_head_stride % 8 || v_block_stride % 8 || v_token_stride % 8 ||
      v_head_stride % 8)
    return fail(QSA_ERR_INVALID, "%s: K/V cache rows must be 16-byte aligned", who);
  if (!aligned(q, 16) || q_row_stride % 8 || q_head_stride % 8)
    return fail(QSA_ERR_INVALID, "%s: q head rows must be 16-byte aligned", who);
  if (!aligned(out, 4) || out_row_stride % 2 || out_head_stride % 2)
    return fail(QSA_ERR_INVALID, "%s: out rows must be 4-byte aligned", who);
  const AttnPlan plan =
      plan_attention(rows, num_q_heads, num_kv_heads, head_dim, topk_width, use_decode_kernel);
  if (plan.workspace_bytes > 0 && (workspace == nullptr || workspace_bytes < plan.workspace_bytes))
    return fail(QSA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu required", who, workspace_bytes,
                plan.workspace_bytes);
  if (plan.workspace_bytes > 0 && !aligned(workspace, 256))
    return fail(QSA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
  AttnParams p = {};
  p.q = q;
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.rows = rows;
  p.q_heads = num_q_heads;
  p.dim = head_dim;
  p.k_cache = k_cache;
  p.k_block_stride = k_block_stride;
  p.k_token_stride = k_token_stride;
  p.k_head_stride = k_head_stride;
  p.v_cache = v_cache;
  p.v_block_stride = v_block_stride;
  p.v_token_stride = v_token_stride;
  p.v_head_stride = v_head_stride;
  p.num_blocks = num_blocks;
  p.page_size = page_size;
  p.num_slots = static_cast<uint32_t>(
      std::min<int64_t>(static_cast<int64_t>(num_blocks) * page_size, 0xffffffffll));
  p.page_div = FastDiv(static_cast<uint32_t>(page_size));
  p.kv_heads = num_kv_heads;
  p.indices = indices;
  p.indices_row_stride = indices_row_stride;
  p.topk_width = topk_width;
  p.block_table = block_table;
  p.table_row_stride = table_row_stride;
  p.table_width = table_width;
  p.num_requests = num_requests;
  p.token_to_req = token_to_req;
  p.valid_counts = valid_counts;
  p.gate = gate;
  p.gate_row_stride = gate_row_stride;
  p.gate_head_stride = gate_head_stride;
  p.gate_dim_stride = gate_dim_stride;
  p.out = out;
  p.out_row_stride = out_row_stride;
  p.out_head_stride = out_head_stride;
  p.scale_log2 = static_cast<float>(std::pow(static_cast<double>(head_dim), -0.5) *
                                    1.4426950408889634);
  p.physical = indices_are_physical ? 1 : 0;
  // 2: each token's K||V rows of consecutive KV heads form one run (the
  //    [blocks, page, H_kv, K||V] layout); 1: K||V adjacent per head; 0: apart.
  const bool fused = (static_cast<const char*>(v_cache) ==
                      static_cast<const char*>(k_cache) + 2 * head_dim) &&
                     k_block_stride == v_block_stride && k_token_stride == v_token_stride &&
                     k_head_stride == v_head_stride;
  p.kv_fused = fused ? (k_head_stride == 2 * head_dim ? 2 : 1) : 0;
  p.slot_contig = k_block_stride == static_cast<int64_t>(page_size) * k_token_stride &&
                  k_token_stride == static_cast<int64_t>(num_kv_heads) * k_head_stride;
  p.gate_vec = gate != nullptr && gate_dim_stride == 1 && aligned(gate, 16) &&
               gate_row_stride % 8 == 0 && gate_head_stride % 8 == 0;
  p.out_vec = aligned(out, 16) && out_row_stride % 8 == 0 && out_head_stride % 8 == 0;
  p.pair_tiles = plan.pair_tiles;
  p.sk_ctas = plan.ctas;
  p.sk_units = plan.units;
  p.heads_per_unit = plan.heads_per_unit;
  p.partials = plan.partials;
  p.merge_pieces = plan.merge_pieces;
  if (plan.partials > 0) {
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.lse_offset);
  }
  p.err = device_error_word();
  cudaError_t e = launch_attention(p, plan.split, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, who);
  return QSA_OK;
}

}  // extern "C"
