// Full-attention cache: what its kernels and their C ABI (kv_api.cu) share.
#pragma once

#include "../../include/aima_moe.h"
#include "common.cuh"

#include <cuda.h>

namespace aima {

// Bits of a handle's status word.
constexpr int kKvBadBatch = 1;       // a page number, length, row offset or position outside its range
constexpr int kKvTimeout = 2;        // a bounded wait ran out

constexpr int kKvMinExponent = -64;  // of a scale: values below 2^-73 of a page that has nothing larger become zero
constexpr int kKvMaxExponent = 120;  // 448 * 2^119 is below the largest BF16 values
constexpr uint8_t kKvNan = 0x7f;     // e4m3 NaN

// 2^e, e in -126 .. 127
__device__ __forceinline__ float kv_exp2(int e) { return __int_as_float((e + 127) << 23); }
// The exponent of a scale: the least e in its range with amax <= 448 * 2^e, from amax = 1.m * 2^x and 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv_scale_exponent(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return amax == 0.0f ? kKvMinExponent : min(max(e, kKvMinExponent), kKvMaxExponent);
}

// floor(log2 x) of a normal number
__device__ __forceinline__ int kv_float_exponent(float x) { return ((__float_as_int(x) >> 23) & 255) - 127; }

struct KvLayer {
  uint8_t* keys;           // [pages, kv_heads, page_tokens, head_dim] e4m3
  uint8_t* values;
  float* key_scales;       // [pages, kv_heads]
  float* value_scales;
};

struct KvBatch {
  const int* table;        // [sequences, columns]
  const int* offsets;      // [sequences + 1] or nullptr: max_new rows each
  const int* lengths;      // [sequences]
  int sequences, tokens, max_new, columns;
};

struct KvShape {
  int q_heads, kv_heads, group, head_dim, rotary, page_tokens, page_shift, pages;
};

struct KvRows {
  const __nv_bfloat16* data;
  long long row_stride, head_stride;
};

// One sequence of a batch as every kernel reads it.  Offsets and lengths come from the device, so they are held to their
// ranges here: a sequence that breaks them has no tokens, and `bad` is set.
struct KvSequence {
  int row0, rows;          // its rows of q, k and v
  int length;              // tokens in the cache with them
  bool bad;
};
__device__ __forceinline__ KvSequence kv_sequence(const KvBatch& b, const KvShape& shape, int s) {
  KvSequence out;
  out.row0 = b.offsets != nullptr ? b.offsets[s] : s * b.max_new;
  const int end = b.offsets != nullptr ? b.offsets[s + 1] : out.row0 + b.max_new;
  out.length = b.lengths[s];
  out.rows = end - out.row0;
  out.bad = out.row0 < 0 || end > b.tokens || out.rows < 0 || out.rows > b.max_new || out.length < 0 ||
            out.length > (static_cast<long long>(b.columns) << shape.page_shift);
  if (out.bad) {
    out.length = 0;
    if (out.row0 < 0 || end > b.tokens || out.rows < 0 || out.rows > b.max_new) out.row0 = out.rows = 0;
  }
  return out;
}

struct KvAppend {
  KvShape shape;
  KvLayer layer;
  KvBatch batch;
  KvRows k, v, q;          // q.data may be nullptr
  __nv_bfloat16* q_out;
  const float* rotation;   // [positions, rotary]
  int positions;
  int* status;
};
cudaError_t kv_append(const KvAppend& args, cudaStream_t stream);

struct KvAttention {
  KvShape shape;
  KvLayer layer;
  KvBatch batch;
  KvRows q;
  __nv_bfloat16* out;
  float scale_log2;        // softmax scale * log2(e)
  int* status;
};
struct KvMaps;             // tensor maps of a layer's cache
size_t kv_workspace_bytes(const KvShape& shape);
size_t kv_counter_bytes();  // at its begin, zero between launches
bool kv_make_maps(const KvShape& shape, const KvLayer& layer, KvMaps* maps);
cudaError_t kv_attention(const KvAttention& args, const KvMaps& maps, void* workspace, int sm_count, cudaStream_t stream);

cudaError_t verify_drafts(const aima_moe_verify_drafts& call, cudaStream_t stream);

}  // namespace aima
