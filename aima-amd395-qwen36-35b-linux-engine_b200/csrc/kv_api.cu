// C ABI of the full-attention cache and of the verification of drafted tokens (contract in include/aima_moe.h).
#include "kv_attention.cuh"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <new>

struct aima_moe_kv {
  std::mutex mutex;
  int device = 0;
  int sm_count = 0;
  aima_moe_kv_config config{};
  aima::KvShape shape{};
  float scale_log2 = 0.0f;
  aima::KvLayer layers[AIMA_MOE_KV_MAX_LAYERS]{};
  aima::KvMaps maps[AIMA_MOE_KV_MAX_LAYERS]{};
  bool bound[AIMA_MOE_KV_MAX_LAYERS]{};
  const float* rotation = nullptr;     // the caller's
  int positions = 0;
  int* status = nullptr;               // the workspace: 256 bytes, then the attention's
  bool owns = false;                   // whether prepare allocated it
  cudaStream_t last_stream = nullptr;
};

namespace aima {
void set_last_error_message(const char* message);
}

namespace {

int kv_fail(int status, const char* format, ...) {
  char text[256];
  va_list args;
  va_start(args, format);
  std::vsnprintf(text, sizeof text, format, args);
  va_end(args);
  aima::set_last_error_message(text);
  return status;
}

int kv_fail_cuda(cudaError_t error, const char* what) {
  char text[256];
  std::snprintf(text, sizeof text, "%s: %s", what, cudaGetErrorString(error));
  aima::set_last_error_message(text);
  (void)cudaGetLastError();
  return static_cast<int>(error);
}

bool misaligned(const void* pointer) { return reinterpret_cast<uintptr_t>(pointer) % 16 != 0; }

// A device that is the current one for the span of a call: the default stream belongs to whichever that is.
struct OnDevice {
  int before = -1;
  cudaError_t error;
  explicit OnDevice(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before == device) before = -1;
    else if (error == cudaSuccess) error = cudaSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0) (void)cudaSetDevice(before);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
};

int check_config(const aima_moe_kv_config* c) {
  if (c == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: config is null");
  if (c->struct_bytes != sizeof(aima_moe_kv_config))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_kv_config size mismatch: got %u, built for %zu", c->struct_bytes, sizeof(aima_moe_kv_config));
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return kv_fail(AIMA_MOE_ERR_UNSUPPORTED, "kv: head_dim %u is not 64, 128 or 256", c->head_dim);
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
    return kv_fail(AIMA_MOE_ERR_UNSUPPORTED, "kv: page_tokens %u is not 16, 32, 64 or 128", c->page_tokens);
  if (c->kv_heads == 0 || c->kv_heads > 128 || c->q_heads == 0 || c->q_heads % c->kv_heads != 0 || c->q_heads / c->kv_heads > 128)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: %u query heads over %u key/value heads (1 .. 128, a whole ratio of at most 128)", c->q_heads, c->kv_heads);
  if (c->rotary_dim > c->head_dim || c->rotary_dim % 16 != 0)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: rotary_dim %u is not a multiple of 16 up to head_dim", c->rotary_dim);
  if (c->pages == 0 || static_cast<uint64_t>(c->pages) * c->kv_heads * c->page_tokens >= (1ull << 31))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: pages is 0, or pages * kv_heads * page_tokens is not below 2^31");
  if (c->layers == 0 || c->layers > AIMA_MOE_KV_MAX_LAYERS)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: layers must be 1 .. %d", AIMA_MOE_KV_MAX_LAYERS);
  if (c->max_sequences == 0 || c->max_sequences > AIMA_MOE_KV_MAX_SEQUENCES)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: max_sequences must be 1 .. %d", AIMA_MOE_KV_MAX_SEQUENCES);
  if (!(c->softmax_scale >= 0.0f) || !std::isfinite(c->softmax_scale))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: softmax_scale must be finite and not negative");
  return AIMA_MOE_OK;
}

aima::KvShape shape_of(const aima_moe_kv_config& c) {
  int shift = 4;
  while ((1u << shift) < c.page_tokens) ++shift;
  return aima::KvShape{static_cast<int>(c.q_heads), static_cast<int>(c.kv_heads), static_cast<int>(c.q_heads / c.kv_heads),
                       static_cast<int>(c.head_dim), static_cast<int>(c.rotary_dim), static_cast<int>(c.page_tokens), shift,
                       static_cast<int>(c.pages)};
}
uint64_t workspace_bytes(const aima::KvShape& shape) { return 256 + aima::kv_workspace_bytes(shape); }

int check_device_pointer(const void* pointer, int device, const char* name) {
  cudaPointerAttributes attributes{};
  const cudaError_t error = cudaPointerGetAttributes(&attributes, pointer);
  if (error != cudaSuccess) return kv_fail_cuda(error, "cudaPointerGetAttributes");
  if ((attributes.type != cudaMemoryTypeDevice && attributes.type != cudaMemoryTypeManaged) || attributes.device != device)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: %s is not memory of the handle's device", name);
  return AIMA_MOE_OK;
}

int check_batch(const aima_moe_kv* h, const aima_moe_kv_batch* b, aima::KvBatch* out) {
  if (b == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: batch is null");
  if (b->struct_bytes != sizeof(aima_moe_kv_batch))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_kv_batch size mismatch: got %u, built for %zu", b->struct_bytes, sizeof(aima_moe_kv_batch));
  if (b->sequences == 0 || b->sequences > h->config.max_sequences)
    return kv_fail(AIMA_MOE_ERR_CAPACITY, "kv: %u sequences, prepared for 1 .. %u", b->sequences, h->config.max_sequences);
  if (b->tokens == 0 || b->tokens > (1u << 24) || b->max_new_tokens == 0 || b->max_new_tokens > b->tokens)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: tokens must be 1 .. 2^24 and max_new_tokens 1 .. tokens");
  if (b->row_offsets == nullptr && static_cast<uint64_t>(b->sequences) * b->max_new_tokens != b->tokens)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: without row_offsets tokens must be sequences * max_new_tokens");
  if (b->table_columns == 0 || static_cast<uint64_t>(b->table_columns) * h->config.page_tokens >= (1ull << 30))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: table_columns is 0 or table_columns * page_tokens is not below 2^30");
  if (b->page_table == nullptr || b->lengths == nullptr)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: page_table or lengths is null");
  *out = aima::KvBatch{b->page_table, b->row_offsets, b->lengths, static_cast<int>(b->sequences), static_cast<int>(b->tokens),
                       static_cast<int>(b->max_new_tokens), static_cast<int>(b->table_columns)};
  return AIMA_MOE_OK;
}

int check_rows(const aima_moe_kv_rows* rows, const char* name, int tokens, int heads, int head_dim, aima::KvRows* out) {
  if (rows == nullptr || rows->data == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: %s is null", name);
  // what a single head or row has as its stride means nothing
  const uint64_t head_stride = heads > 1 ? rows->head_stride : tokens > 1 ? rows->row_stride : head_dim;
  const uint64_t row_stride = tokens > 1 ? rows->row_stride : head_stride * heads;
  if (misaligned(rows->data) || row_stride % 8 != 0 || head_stride % 8 != 0)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: %s must be 16-byte aligned with strides that are multiples of 8 elements", name);
  if (row_stride >= (1ull << 36) || head_stride >= (1ull << 36))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: a stride of %s is too large", name);
  *out = aima::KvRows{static_cast<const __nv_bfloat16*>(rows->data), static_cast<long long>(row_stride), static_cast<long long>(head_stride)};
  return AIMA_MOE_OK;
}

// Whether the span of an input's rows and the contiguous output share bytes.
bool overlaps(const aima::KvRows& x, int heads, const void* out, const aima::KvShape& shape, int tokens) {
  const char* x0 = reinterpret_cast<const char*>(x.data);
  const char* x1 = reinterpret_cast<const char*>(x.data + (tokens - 1) * x.row_stride + (heads - 1) * x.head_stride + shape.head_dim);
  const char* o0 = static_cast<const char*>(out);
  const char* o1 = o0 + 2ull * tokens * shape.q_heads * shape.head_dim;
  return x0 < o1 && o0 < x1;
}

int check_launch(aima_moe_kv* h, uint32_t layer) {
  if (h == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: handle is null");
  if (layer >= h->config.layers) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: layer %u of %u", layer, h->config.layers);
  if (!h->bound[layer]) return kv_fail(AIMA_MOE_ERR_NOT_BOUND, "kv: layer %u has no cache tensors", layer);
  int device = -1;
  const cudaError_t error = cudaGetDevice(&device);
  if (error != cudaSuccess) return kv_fail_cuda(error, "cudaGetDevice");
  if (device != h->device)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: the handle is of device %d, the current one is %d", h->device, device);
  return AIMA_MOE_OK;
}

}  // namespace

extern "C" {

#define AIMA_EXPORT __attribute__((visibility("default")))

AIMA_EXPORT int aima_moe_kv_query_workspace(const aima_moe_kv_config* config, uint64_t* bytes) {
  if (bytes == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: bytes is null");
  if (const int status = check_config(config); status != AIMA_MOE_OK) return status;
  *bytes = workspace_bytes(shape_of(*config));
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_prepare(const aima_moe_kv_config* config, aima_moe_kv** out) {
  if (out == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: handle is null");
  *out = nullptr;
  if (const int status = check_config(config); status != AIMA_MOE_OK) return status;
  int device = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error != cudaSuccess) {
    (void)cudaGetLastError();
    return kv_fail(AIMA_MOE_ERR_NO_DEVICE, "kv: no CUDA device (there is no CPU fallback)");
  }
  int major = 0, sm_count = 0;
  error = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (error == cudaSuccess) error = cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device);
  if (error != cudaSuccess) return kv_fail_cuda(error, "cudaDeviceGetAttribute");
  if (major != 10) return kv_fail(AIMA_MOE_ERR_NO_DEVICE, "kv: needs an sm_100 device");
  aima_moe_kv* h = new (std::nothrow) aima_moe_kv();
  if (h == nullptr) return kv_fail(AIMA_MOE_ERR_INTERNAL, "kv: out of host memory");
  h->device = device;
  h->sm_count = sm_count;
  h->config = *config;
  h->shape = shape_of(*config);
  const double scale = config->softmax_scale != 0.0f ? config->softmax_scale : 1.0 / std::sqrt(static_cast<double>(config->head_dim));
  h->scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  const uint64_t bytes = workspace_bytes(h->shape);
  if (config->workspace != nullptr) {
    int status = AIMA_MOE_OK;
    if (reinterpret_cast<uintptr_t>(config->workspace) % 256 != 0 || config->workspace_bytes < bytes)
      status = kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: the workspace is not 256-byte aligned or has less than %llu bytes",
                       static_cast<unsigned long long>(bytes));
    else
      status = check_device_pointer(config->workspace, device, "the workspace");
    if (status != AIMA_MOE_OK) {
      delete h;
      return status;
    }
    h->status = static_cast<int*>(config->workspace);
  } else {
    error = cudaMalloc(&h->status, bytes);
    h->owns = true;
  }
  // here and now: the launches may come on streams that do not wait for the default one
  if (error == cudaSuccess) error = cudaMemsetAsync(h->status, 0, 256 + aima::kv_counter_bytes(), cudaStreamPerThread);
  if (error == cudaSuccess) error = cudaStreamSynchronize(cudaStreamPerThread);
  if (error != cudaSuccess) {
    if (h->owns) cudaFree(h->status);
    delete h;
    return kv_fail_cuda(error, "allocation of the kv workspace");
  }
  *out = h;
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_bind_layer(aima_moe_kv* h, uint32_t layer, const aima_moe_kv_layer* t) {
  if (h == nullptr || t == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: handle or tensors is null");
  if (t->struct_bytes != sizeof(aima_moe_kv_layer))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_kv_layer size mismatch: got %u, built for %zu", t->struct_bytes, sizeof(aima_moe_kv_layer));
  if (layer >= h->config.layers) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: layer %u of %u", layer, h->config.layers);
  std::lock_guard<std::mutex> lock(h->mutex);
  const uint64_t scales = 4ull * h->config.pages * h->config.kv_heads;
  const uint64_t codes = scales / 4 * h->config.page_tokens * h->config.head_dim;
  const struct { const void* pointer; uint64_t bytes, want; const char* name; } all[4] = {
      {t->keys, t->keys_bytes, codes, "keys"}, {t->values, t->values_bytes, codes, "values"},
      {t->key_scales, t->key_scales_bytes, scales, "key_scales"}, {t->value_scales, t->value_scales_bytes, scales, "value_scales"}};
  for (const auto& x : all) {
    if (x.pointer == nullptr || misaligned(x.pointer))
      return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: %s is null or not 16-byte aligned", x.name);
    if (x.bytes != x.want)
      return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: %s has %llu bytes, expected %llu", x.name, static_cast<unsigned long long>(x.bytes),
                     static_cast<unsigned long long>(x.want));
    if (const int status = check_device_pointer(x.pointer, h->device, x.name); status != AIMA_MOE_OK) return status;
  }
  const aima::KvLayer bound{static_cast<uint8_t*>(t->keys), static_cast<uint8_t*>(t->values), static_cast<float*>(t->key_scales),
                                   static_cast<float*>(t->value_scales)};
  if (!aima::kv_make_maps(h->shape, bound, &h->maps[layer])) return kv_fail(AIMA_MOE_ERR_INTERNAL, "kv: tensor maps of the cache could not be made");
  h->layers[layer] = bound;
  h->bound[layer] = true;
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_set_rotation(aima_moe_kv* h, const void* table, uint32_t positions) {
  if (h == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: handle is null");
  if (table == nullptr || misaligned(table) || positions == 0 || positions >= (1u << 30))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: the rotation table is null, not 16-byte aligned, or has no positions");
  if (const int status = check_device_pointer(table, h->device, "the rotation table"); status != AIMA_MOE_OK) return status;
  std::lock_guard<std::mutex> lock(h->mutex);
  h->rotation = static_cast<const float*>(table);
  h->positions = static_cast<int>(positions);
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_append_launch(aima_moe_kv* h, uint32_t layer, const aima_moe_kv_batch* batch, const aima_moe_kv_rows* k,
                                          const aima_moe_kv_rows* v, const aima_moe_kv_rows* q, void* q_out, void* stream) {
  if (const int status = check_launch(h, layer); status != AIMA_MOE_OK) return status;
  std::lock_guard<std::mutex> lock(h->mutex);
  aima::KvAppend a{};
  a.shape = h->shape;
  a.layer = h->layers[layer];
  if (const int status = check_batch(h, batch, &a.batch); status != AIMA_MOE_OK) return status;
  if (const int status = check_rows(k, "k", a.batch.tokens, h->shape.kv_heads, h->shape.head_dim, &a.k); status != AIMA_MOE_OK) return status;
  if (const int status = check_rows(v, "v", a.batch.tokens, h->shape.kv_heads, h->shape.head_dim, &a.v); status != AIMA_MOE_OK) return status;
  if (q != nullptr && q->data != nullptr) {
    if (const int status = check_rows(q, "q", a.batch.tokens, h->shape.q_heads, h->shape.head_dim, &a.q); status != AIMA_MOE_OK) return status;
    if (q_out == nullptr || misaligned(q_out)) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: q_out is null or not 16-byte aligned");
    if (overlaps(a.q, h->shape.q_heads, q_out, h->shape, a.batch.tokens)) return kv_fail(AIMA_MOE_ERR_ALIAS, "kv: q_out overlaps q");
    // the blocks that write it run beside those that read k and v, twice
    if (overlaps(a.k, h->shape.kv_heads, q_out, h->shape, a.batch.tokens) || overlaps(a.v, h->shape.kv_heads, q_out, h->shape, a.batch.tokens))
      return kv_fail(AIMA_MOE_ERR_ALIAS, "kv: q_out overlaps k or v");
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
  }
  if (h->shape.rotary > 0 && h->rotation == nullptr) return kv_fail(AIMA_MOE_ERR_NOT_BOUND, "kv: no rotation table was set");
  a.rotation = h->rotation;
  a.positions = h->positions;
  a.status = h->status;
  const cudaError_t error = aima::kv_append(a, static_cast<cudaStream_t>(stream));
  if (error != cudaSuccess) return kv_fail_cuda(error, "kv append launch");
  h->last_stream = static_cast<cudaStream_t>(stream);
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_attention_launch(aima_moe_kv* h, uint32_t layer, const aima_moe_kv_batch* batch, const aima_moe_kv_rows* q,
                                             void* out, void* stream) {
  if (const int status = check_launch(h, layer); status != AIMA_MOE_OK) return status;
  std::lock_guard<std::mutex> lock(h->mutex);
  aima::KvAttention a{};
  a.shape = h->shape;
  a.layer = h->layers[layer];
  if (const int status = check_batch(h, batch, &a.batch); status != AIMA_MOE_OK) return status;
  if (const int status = check_rows(q, "q", a.batch.tokens, h->shape.q_heads, h->shape.head_dim, &a.q); status != AIMA_MOE_OK) return status;
  if (out == nullptr || misaligned(out)) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: out is null or not 16-byte aligned");
  if (overlaps(a.q, h->shape.q_heads, out, h->shape, a.batch.tokens)) return kv_fail(AIMA_MOE_ERR_ALIAS, "kv: out overlaps q");
  a.out = static_cast<__nv_bfloat16*>(out);
  a.scale_log2 = h->scale_log2;
  a.status = h->status;
  const cudaError_t error = aima::kv_attention(a, h->maps[layer], reinterpret_cast<uint8_t*>(h->status) + 256, h->sm_count, static_cast<cudaStream_t>(stream));
  if (error != cudaSuccess) return kv_fail_cuda(error, "kv attention launch");
  h->last_stream = static_cast<cudaStream_t>(stream);
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_sync(aima_moe_kv* h) {
  if (h == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: handle is null");
  std::lock_guard<std::mutex> lock(h->mutex);
  const OnDevice scope(h->device);
  if (scope.error != cudaSuccess) return kv_fail_cuda(scope.error, "cudaSetDevice");
  int status = 0;
  cudaError_t error = cudaMemcpyAsync(&status, h->status, sizeof status, cudaMemcpyDeviceToHost, h->last_stream);
  if (error == cudaSuccess) error = cudaStreamSynchronize(h->last_stream);
  if (error == cudaSuccess && status != 0) {
    // after a wait that ran out the counters of the joins may be anything; else they are left to what may be under way elsewhere
    const size_t bytes = (status & aima::kKvTimeout) != 0 ? 256 + aima::kv_counter_bytes() : sizeof status;
    error = cudaMemsetAsync(h->status, 0, bytes, h->last_stream);
    if (error == cudaSuccess) error = cudaStreamSynchronize(h->last_stream);
  }
  if (error != cudaSuccess) return kv_fail_cuda(error, "kv sync");
  if ((status & aima::kKvTimeout) != 0) return kv_fail(AIMA_MOE_ERR_TIMEOUT, "kv: a bounded wait ran out, the output is incomplete");
  if ((status & aima::kKvBadBatch) != 0)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "kv: a page number, length, row offset or position of a batch was out of range");
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_kv_release(aima_moe_kv* h) {
  if (h == nullptr) return AIMA_MOE_OK;
  if (h->owns) cudaFree(h->status);
  delete h;
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_verify_drafts_launch(const aima_moe_verify_drafts* call, void* stream) {
  if (call == nullptr) return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "verify: call is null");
  const aima_moe_verify_drafts& c = *call;
  if (c.struct_bytes != sizeof(aima_moe_verify_drafts))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_verify_drafts size mismatch: got %u, built for %zu", c.struct_bytes, sizeof(aima_moe_verify_drafts));
  if (c.sequences == 0 || c.sequences > 65535 || c.max_drafts > 64 || c.vocabulary == 0 || c.vocabulary > (1u << 22))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "verify: sequences must be 1 .. 65535, max_drafts at most 64, vocabulary 1 .. 2^22");
  if (c.target == nullptr || c.uniforms == nullptr || c.accepted == nullptr || c.tokens == nullptr || (c.max_drafts > 0 && c.draft_tokens == nullptr))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "verify: target, uniforms, draft_tokens, accepted or tokens is null");
  if ((c.cache_lengths == nullptr) != (c.new_lengths == nullptr))
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "verify: cache_lengths and new_lengths go together");
  if (reinterpret_cast<uintptr_t>(c.target) % 4 != 0 || reinterpret_cast<uintptr_t>(c.draft) % 4 != 0)
    return kv_fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "verify: target and draft must be aligned to their elements");
  int device = 0, major = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error == cudaSuccess) error = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (error != cudaSuccess) {
    (void)cudaGetLastError();
    return kv_fail(AIMA_MOE_ERR_NO_DEVICE, "verify: no CUDA device (there is no CPU fallback)");
  }
  if (major != 10) return kv_fail(AIMA_MOE_ERR_NO_DEVICE, "verify: needs an sm_100 device");
  error = aima::verify_drafts(c, static_cast<cudaStream_t>(stream));
  if (error != cudaSuccess) return kv_fail_cuda(error, "verify launch");
  return AIMA_MOE_OK;
}

}  // extern "C"
