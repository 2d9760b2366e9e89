// C ABI of the linear-attention layers and of the head norm (contract in include/aima_moe.h).
#include "host_checks.cuh"
#include "linear.cuh"

#include <cmath>
#include <mutex>
#include <new>

struct aima_moe_linear {
  std::mutex mutex;
  int device = 0;
  int sm_count = 0;
  aima_moe_linear_config config{};
  aima_moe_linear_layer layers[AIMA_MOE_MAX_LAYERS]{};
  bool bound[AIMA_MOE_MAX_LAYERS]{};
  int* status = nullptr;               // the workspace: 256 bytes, then the delta rule's
  bool owns = false;                   // whether prepare allocated it
  cudaStream_t last_stream = nullptr;
};

namespace {

using aima::fail;
using aima::fail_cuda;
using aima::misaligned;
using aima::OnDevice;

constexpr uint64_t kDim = AIMA_MOE_LINEAR_HEAD_DIM;

int check_config(const aima_moe_linear_config* c) {
  if (c == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: config is null");
  if (c->struct_bytes != sizeof(aima_moe_linear_config))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_linear_config size mismatch: got %u, built for %zu", c->struct_bytes, sizeof(aima_moe_linear_config));
  if (c->head_dim != kDim) return fail(AIMA_MOE_ERR_UNSUPPORTED, "linear: head_dim %u is not 128", c->head_dim);
  if (c->k_heads == 0 || c->k_heads > 128 || c->v_heads == 0 || c->v_heads > 256 || c->v_heads % c->k_heads != 0)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: %u value heads over %u key heads (1 .. 128 key heads, up to 256 value heads, a whole ratio)", c->v_heads,
                c->k_heads);
  if (c->conv_width < 2 || c->conv_width > 4) return fail(AIMA_MOE_ERR_UNSUPPORTED, "linear: conv_width %u is not 2 .. 4", c->conv_width);
  if (c->slots == 0 || c->slots > (1u << 20)) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: slots must be 1 .. 2^20");
  if (c->layers == 0 || c->layers > AIMA_MOE_MAX_LAYERS) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: layers must be 1 .. %d", AIMA_MOE_MAX_LAYERS);
  if (c->max_sequences == 0 || c->max_sequences > 1024) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: max_sequences must be 1 .. 1024");
  if (c->max_tokens == 0 || c->max_tokens > (1u << 20)) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: max_tokens must be 1 .. 2^20");
  if (!(c->eps >= 0.0f) || !std::isfinite(c->eps)) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: eps must be finite and not negative");
  return AIMA_MOE_OK;
}

uint64_t channels_of(const aima_moe_linear_config& c) { return (2ull * c.k_heads + c.v_heads) * kDim; }
uint64_t workspace_bytes(const aima_moe_linear_config& c) {
  return 256 + (c.max_tokens > aima::kLinearStepRows ? aima::linear_chunk_workspace(c.k_heads, c.v_heads, c.max_tokens, c.max_sequences) : 0);
}

int check_device_pointer(const void* pointer, int device, const char* name) {
  cudaPointerAttributes attributes{};
  const cudaError_t error = cudaPointerGetAttributes(&attributes, pointer);
  if (error != cudaSuccess) return fail_cuda(error, "cudaPointerGetAttributes");
  if ((attributes.type != cudaMemoryTypeDevice && attributes.type != cudaMemoryTypeManaged) || attributes.device != device)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: %s is not memory of the handle's device", name);
  return AIMA_MOE_OK;
}

int check_launch(aima_moe_linear* h, uint32_t layer) {
  if (h == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: handle is null");
  if (layer >= h->config.layers) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: layer %u of %u", layer, h->config.layers);
  if (!h->bound[layer]) return fail(AIMA_MOE_ERR_NOT_BOUND, "linear: layer %u has no tensors", layer);
  int device = -1;
  const cudaError_t error = cudaGetDevice(&device);
  if (error != cudaSuccess) return fail_cuda(error, "cudaGetDevice");
  if (device != h->device)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: the handle is of device %d, the current one is %d", h->device, device);
  return AIMA_MOE_OK;
}

int check_batch(const aima_moe_linear* h, const aima_moe_linear_batch* b, aima::LinearBatch* out) {
  if (b == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: batch is null");
  if (b->struct_bytes != sizeof(aima_moe_linear_batch))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_linear_batch size mismatch: got %u, built for %zu", b->struct_bytes, sizeof(aima_moe_linear_batch));
  if (b->sequences == 0 || b->sequences > h->config.max_sequences)
    return fail(AIMA_MOE_ERR_CAPACITY, "linear: %u sequences, prepared for 1 .. %u", b->sequences, h->config.max_sequences);
  if (b->tokens == 0 || b->tokens > h->config.max_tokens)
    return fail(AIMA_MOE_ERR_CAPACITY, "linear: %u tokens, prepared for 1 .. %u", b->tokens, h->config.max_tokens);
  if (b->max_new_tokens == 0 || b->max_new_tokens > b->tokens)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: max_new_tokens must be 1 .. tokens");
  if (b->row_offsets == nullptr && static_cast<uint64_t>(b->sequences) * b->max_new_tokens != b->tokens)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: without row_offsets tokens must be sequences * max_new_tokens");
  if (b->slots == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: slots is null");
  *out = aima::LinearBatch{b->slots, b->row_offsets, b->lengths, b->keep, static_cast<int>(b->sequences), static_cast<int>(b->tokens),
                           static_cast<int>(b->max_new_tokens), static_cast<int>(h->config.slots)};
  return AIMA_MOE_OK;
}

int check_rows(const char* what, const aima_moe_kv_rows& rows, const char* name, uint64_t tokens, uint64_t heads, uint64_t dim, aima::KvRows* out) {
  if (rows.data == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
  // what a single head or row has as its stride means nothing
  const uint64_t head_stride = heads > 1 ? rows.head_stride : dim;
  const uint64_t row_stride = tokens > 1 ? rows.row_stride : 0;
  if (misaligned(rows.data) || row_stride % 8 != 0 || head_stride % 8 != 0)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "%s: %s must be 16-byte aligned with strides that are multiples of 8 elements", what, name);
  if (row_stride >= (1ull << 36) || head_stride >= (1ull << 36))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "%s: a stride of %s is too large", what, name);
  *out = aima::KvRows{static_cast<const __nv_bfloat16*>(rows.data), static_cast<long long>(row_stride), static_cast<long long>(head_stride)};
  return AIMA_MOE_OK;
}

// Whether the span of strided rows and `bytes` bytes from `out` on share any.
bool overlaps(const __nv_bfloat16* data, uint64_t tokens, uint64_t row_stride, uint64_t heads, uint64_t head_stride, uint64_t dim, const void* out,
              uint64_t bytes) {
  const char* x0 = reinterpret_cast<const char*>(data);
  const char* x1 = reinterpret_cast<const char*>(data + (tokens - 1) * row_stride + (heads - 1) * head_stride + dim);
  const char* o0 = static_cast<const char*>(out);
  return x0 < o0 + bytes && o0 < x1;
}
bool overlaps(const aima::KvRows& x, uint64_t tokens, uint64_t heads, uint64_t dim, const void* out, uint64_t bytes) {
  return overlaps(x.data, tokens, static_cast<uint64_t>(x.row_stride), heads, static_cast<uint64_t>(x.head_stride), dim, out, bytes);
}

}  // namespace

extern "C" {

#define AIMA_EXPORT __attribute__((visibility("default")))

AIMA_EXPORT int aima_moe_linear_query_workspace(const aima_moe_linear_config* config, uint64_t* bytes) {
  if (bytes == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: bytes is null");
  if (const int status = check_config(config); status != AIMA_MOE_OK) return status;
  *bytes = workspace_bytes(*config);
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_linear_prepare(const aima_moe_linear_config* config, aima_moe_linear** out) {
  if (out == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: handle is null");
  *out = nullptr;
  if (const int status = check_config(config); status != AIMA_MOE_OK) return status;
  int device = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(AIMA_MOE_ERR_NO_DEVICE, "linear: no CUDA device (there is no CPU fallback)");
  }
  int major = 0, sm_count = 0;
  error = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (error == cudaSuccess) error = cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device);
  if (error != cudaSuccess) return fail_cuda(error, "cudaDeviceGetAttribute");
  if (major != 10) return fail(AIMA_MOE_ERR_NO_DEVICE, "linear: needs an sm_100 device");
  aima_moe_linear* h = new (std::nothrow) aima_moe_linear();
  if (h == nullptr) return fail(AIMA_MOE_ERR_INTERNAL, "linear: out of host memory");
  h->device = device;
  h->sm_count = sm_count;
  h->config = *config;
  if (h->config.eps == 0.0f) h->config.eps = 1.0e-6f;
  const uint64_t bytes = workspace_bytes(*config);
  if (config->workspace != nullptr) {
    int status = AIMA_MOE_OK;
    if (reinterpret_cast<uintptr_t>(config->workspace) % 256 != 0 || config->workspace_bytes < bytes)
      status = fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: the workspace is not 256-byte aligned or has less than %llu bytes",
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
  if (error == cudaSuccess) error = cudaMemsetAsync(h->status, 0, 256, cudaStreamPerThread);
  if (error == cudaSuccess) error = cudaStreamSynchronize(cudaStreamPerThread);
  if (error != cudaSuccess) {
    if (h->owns) cudaFree(h->status);
    delete h;
    return fail_cuda(error, "allocation of the linear workspace");
  }
  *out = h;
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_linear_bind_layer(aima_moe_linear* h, uint32_t layer, const aima_moe_linear_layer* t) {
  if (h == nullptr || t == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: handle or tensors is null");
  if (t->struct_bytes != sizeof(aima_moe_linear_layer))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_linear_layer size mismatch: got %u, built for %zu", t->struct_bytes, sizeof(aima_moe_linear_layer));
  if (layer >= h->config.layers) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: layer %u of %u", layer, h->config.layers);
  std::lock_guard<std::mutex> lock(h->mutex);
  const aima_moe_linear_config& c = h->config;
  const uint64_t channels = channels_of(c);
  const struct { const void* pointer; uint64_t bytes, want; const char* name; } all[6] = {
      {t->conv_weight, t->conv_weight_bytes, channels * c.conv_width * 2, "conv_weight"},
      {t->conv_states, t->conv_states_bytes, channels * (c.conv_width - 1) * 2 * c.slots, "conv_states"},
      {t->states, t->states_bytes, kDim * kDim * 4 * c.v_heads * c.slots, "states"},
      {t->a_log, t->a_log_bytes, 4ull * c.v_heads, "a_log"},
      {t->dt_bias, t->dt_bias_bytes, 4ull * c.v_heads, "dt_bias"},
      {t->norm_weight, t->norm_weight_bytes, 2 * kDim, "norm_weight"}};
  for (const auto& x : all) {
    if (x.pointer == nullptr) continue;
    if (misaligned(x.pointer)) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: %s is not 16-byte aligned", x.name);
    if (x.bytes != x.want)
      return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: %s has %llu bytes, expected %llu", x.name, static_cast<unsigned long long>(x.bytes),
                  static_cast<unsigned long long>(x.want));
    if (const int status = check_device_pointer(x.pointer, h->device, x.name); status != AIMA_MOE_OK) return status;
  }
  if ((t->conv_weight == nullptr) != (t->conv_states == nullptr))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: conv_weight and conv_states go together");
  if ((t->states == nullptr) != (t->a_log == nullptr) || (t->states == nullptr) != (t->dt_bias == nullptr))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: states, a_log and dt_bias go together");
  h->layers[layer] = *t;
  h->bound[layer] = true;
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_linear_conv_launch(aima_moe_linear* h, uint32_t layer, const aima_moe_linear_batch* batch, const void* x, uint64_t x_row_stride,
                                            void* out, void* stream) {
  if (const int status = check_launch(h, layer); status != AIMA_MOE_OK) return status;
  std::lock_guard<std::mutex> lock(h->mutex);
  const aima_moe_linear_layer& t = h->layers[layer];
  if (t.conv_weight == nullptr) return fail(AIMA_MOE_ERR_NOT_BOUND, "linear: layer %u has no conv_weight", layer);
  aima::LinearConv a{};
  if (const int status = check_batch(h, batch, &a.batch); status != AIMA_MOE_OK) return status;
  const uint64_t channels = channels_of(h->config), tokens = batch->tokens;
  aima::KvRows rows{};
  if (const int status = check_rows("linear", aima_moe_kv_rows{x, x_row_stride, 0}, "x", tokens, 1, channels, &rows); status != AIMA_MOE_OK) return status;
  if (out == nullptr || misaligned(out)) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: out is null or not 16-byte aligned");
  if (overlaps(rows, tokens, 1, channels, out, 2 * tokens * channels)) return fail(AIMA_MOE_ERR_ALIAS, "linear: out overlaps x");
  a.channels = static_cast<int>(channels);
  a.width = static_cast<int>(h->config.conv_width);
  a.x = rows.data;
  a.x_stride = rows.row_stride;
  a.weight = static_cast<const __nv_bfloat16*>(t.conv_weight);
  a.states = static_cast<__nv_bfloat16*>(t.conv_states);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.status = h->status;
  const cudaError_t error = aima::linear_conv(a, static_cast<cudaStream_t>(stream));
  if (error != cudaSuccess) return fail_cuda(error, "linear convolution launch");
  h->last_stream = static_cast<cudaStream_t>(stream);
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_linear_delta_launch(aima_moe_linear* h, uint32_t layer, const aima_moe_linear_batch* batch, const aima_moe_linear_delta* call,
                                             void* stream) {
  if (const int status = check_launch(h, layer); status != AIMA_MOE_OK) return status;
  if (call == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: call is null");
  if (call->struct_bytes != sizeof(aima_moe_linear_delta))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_linear_delta size mismatch: got %u, built for %zu", call->struct_bytes, sizeof(aima_moe_linear_delta));
  std::lock_guard<std::mutex> lock(h->mutex);
  const aima_moe_linear_layer& t = h->layers[layer];
  if (t.states == nullptr) return fail(AIMA_MOE_ERR_NOT_BOUND, "linear: layer %u has no states", layer);
  aima::LinearDelta a{};
  if (const int status = check_batch(h, batch, &a.batch); status != AIMA_MOE_OK) return status;
  const uint64_t tokens = batch->tokens, k_heads = h->config.k_heads, v_heads = h->config.v_heads;
  const struct { const aima_moe_kv_rows* from; aima::KvRows* to; uint64_t heads; const char* name; } inputs[4] = {
      {&call->q, &a.q, k_heads, "q"}, {&call->k, &a.k, k_heads, "k"}, {&call->v, &a.v, v_heads, "v"}, {&call->gate, &a.gate, v_heads, "gate"}};
  if (call->out != nullptr && misaligned(call->out)) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: out is not 16-byte aligned");
  const uint64_t out_bytes = 2 * tokens * v_heads * kDim;
  for (const auto& x : inputs) {
    if (x.to == &a.gate && x.from->data == nullptr) continue;
    if (const int status = check_rows("linear", *x.from, x.name, tokens, x.heads, kDim, x.to); status != AIMA_MOE_OK) return status;
    if (call->out != nullptr && overlaps(*x.to, tokens, x.heads, kDim, call->out, out_bytes)) return fail(AIMA_MOE_ERR_ALIAS, "linear: out overlaps %s", x.name);
  }
  if (call->gate.data != nullptr && t.norm_weight == nullptr) return fail(AIMA_MOE_ERR_NOT_BOUND, "linear: layer %u has no norm_weight", layer);
  const struct { const void* data; uint64_t stride; const char* name; } numbers[2] = {{call->a, call->a_row_stride, "a"}, {call->b, call->b_row_stride, "b"}};
  for (const auto& x : numbers) {
    if (x.data == nullptr || reinterpret_cast<uintptr_t>(x.data) % 2 != 0 || x.stride >= (1ull << 36))
      return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: %s is null, not aligned to its elements, or its stride is too large", x.name);
    if (call->out != nullptr && overlaps(static_cast<const __nv_bfloat16*>(x.data), tokens, tokens > 1 ? x.stride : 0, 1, 0, v_heads, call->out, out_bytes))
      return fail(AIMA_MOE_ERR_ALIAS, "linear: out overlaps %s", x.name);
  }
  a.k_heads = static_cast<int>(k_heads);
  a.v_heads = static_cast<int>(v_heads);
  a.group = static_cast<int>(v_heads / k_heads);
  a.a = static_cast<const __nv_bfloat16*>(call->a);
  a.b = static_cast<const __nv_bfloat16*>(call->b);
  a.a_stride = static_cast<long long>(call->a_row_stride);
  a.b_stride = static_cast<long long>(call->b_row_stride);
  a.a_log = static_cast<const float*>(t.a_log);
  a.dt_bias = static_cast<const float*>(t.dt_bias);
  a.norm_weight = static_cast<const __nv_bfloat16*>(t.norm_weight);
  a.eps = h->config.eps;
  a.states = static_cast<float*>(t.states);
  a.out = static_cast<__nv_bfloat16*>(call->out);
  a.status = h->status;
  // Sequences of few rows go token by token, longer ones in chunks; a batch that may have both takes both launches.
  cudaError_t error = cudaSuccess;
  const bool chunks = a.batch.max_new > aima::kLinearStepRows, steps = !chunks || (a.batch.sequences > 1 && a.batch.offsets != nullptr);
  if (steps) error = aima::linear_step(a, chunks ? aima::kLinearStepRows : a.batch.max_new, h->sm_count, static_cast<cudaStream_t>(stream));
  if (error == cudaSuccess && chunks)
    error = aima::linear_chunks(a, steps ? aima::kLinearStepRows : 0, reinterpret_cast<uint8_t*>(h->status) + 256, h->sm_count, static_cast<cudaStream_t>(stream));
  if (error != cudaSuccess) return fail_cuda(error, "linear delta launch");
  h->last_stream = static_cast<cudaStream_t>(stream);
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_linear_sync(aima_moe_linear* h) {
  if (h == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: handle is null");
  std::lock_guard<std::mutex> lock(h->mutex);
  const OnDevice scope(h->device);
  if (scope.error != cudaSuccess) return fail_cuda(scope.error, "cudaSetDevice");
  int status = 0;
  cudaError_t error = cudaMemcpyAsync(&status, h->status, sizeof status, cudaMemcpyDeviceToHost, h->last_stream);
  if (error == cudaSuccess) error = cudaStreamSynchronize(h->last_stream);
  if (error == cudaSuccess && status != 0) {
    error = cudaMemsetAsync(h->status, 0, sizeof status, h->last_stream);
    if (error == cudaSuccess) error = cudaStreamSynchronize(h->last_stream);
  }
  if (error != cudaSuccess) return fail_cuda(error, "linear sync");
  if ((status & aima::kLinearTimeout) != 0) return fail(AIMA_MOE_ERR_TIMEOUT, "linear: a bounded wait ran out, outputs and states are incomplete");
  if ((status & aima::kLinearBadBatch) != 0)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "linear: a slot, row offset or length of a batch was out of range");
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_linear_release(aima_moe_linear* h) {
  if (h == nullptr) return AIMA_MOE_OK;
  if (h->owns) cudaFree(h->status);
  delete h;
  return AIMA_MOE_OK;
}

AIMA_EXPORT int aima_moe_head_norm_launch(const aima_moe_head_norm* call, void* stream) {
  if (call == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "head norm: call is null");
  const aima_moe_head_norm& c = *call;
  if (c.struct_bytes != sizeof(aima_moe_head_norm))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "aima_moe_head_norm size mismatch: got %u, built for %zu", c.struct_bytes, sizeof(aima_moe_head_norm));
  if (c.tokens == 0 || c.tokens > (1u << 24) || c.heads == 0 || c.heads > 1024)
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "head norm: tokens must be 1 .. 2^24, heads 1 .. 1024");
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail(AIMA_MOE_ERR_UNSUPPORTED, "head norm: head_dim %u is not 64, 128 or 256", c.head_dim);
  if (c.activation > AIMA_MOE_GATE_SIGMOID || (c.activation == AIMA_MOE_GATE_NONE) != (c.gate.data == nullptr))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "head norm: activation is not one of AIMA_MOE_GATE_*, or does not go with the gate");
  if (c.weight == nullptr && c.gate.data == nullptr) return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "head norm: neither weight nor gate");
  if (!(c.eps >= 0.0f) || !std::isfinite(c.eps) || !std::isfinite(c.weight_offset))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "head norm: eps must be finite and not negative, weight_offset finite");
  if (c.out == nullptr || misaligned(c.out) || misaligned(c.weight))
    return fail(AIMA_MOE_ERR_INVALID_ARGUMENT, "head norm: out is null, or out or weight not 16-byte aligned");
  const uint64_t tokens = c.tokens, heads = c.heads, dim = c.head_dim, bytes = 2 * tokens * heads * dim;
  aima::HeadNorm a{};
  if (const int status = check_rows("head norm", c.x, "x", tokens, heads, dim, &a.x); status != AIMA_MOE_OK) return status;
  const bool in_place = c.out == c.x.data && (heads == 1 || c.x.head_stride == dim) && (tokens == 1 || c.x.row_stride == heads * dim);
  if (!in_place && overlaps(a.x, tokens, heads, dim, c.out, bytes)) return fail(AIMA_MOE_ERR_ALIAS, "head norm: out overlaps x");
  if (c.gate.data != nullptr) {
    if (const int status = check_rows("head norm", c.gate, "gate", tokens, heads, dim, &a.gate); status != AIMA_MOE_OK) return status;
    if (overlaps(a.gate, tokens, heads, dim, c.out, bytes)) return fail(AIMA_MOE_ERR_ALIAS, "head norm: out overlaps the gate");
  }
  if (c.weight != nullptr && overlaps(static_cast<const __nv_bfloat16*>(c.weight), 1, 0, 1, 0, dim, c.out, bytes))
    return fail(AIMA_MOE_ERR_ALIAS, "head norm: out overlaps weight");
  int device = 0, major = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error == cudaSuccess) error = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (error != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(AIMA_MOE_ERR_NO_DEVICE, "head norm: no CUDA device (there is no CPU fallback)");
  }
  if (major != 10) return fail(AIMA_MOE_ERR_NO_DEVICE, "head norm: needs an sm_100 device");
  a.tokens = static_cast<int>(c.tokens);
  a.heads = static_cast<int>(c.heads);
  a.dim = static_cast<int>(c.head_dim);
  a.activation = static_cast<int>(c.activation);
  a.offset = c.weight_offset;
  a.eps = c.eps;
  a.weight = static_cast<const __nv_bfloat16*>(c.weight);
  a.out = static_cast<__nv_bfloat16*>(c.out);
  error = aima::head_norm(a, static_cast<cudaStream_t>(stream));
  if (error != cudaSuccess) return fail_cuda(error, "head norm launch");
  return AIMA_MOE_OK;
}

}  // extern "C"
