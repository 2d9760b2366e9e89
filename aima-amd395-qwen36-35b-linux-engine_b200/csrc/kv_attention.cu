// Attention of a batch's rows over the paged 8-bit cache: the choice of the kernel, the tensor maps and the workspace.
#include "kv_attention.cuh"

#include <algorithm>
#include <cudaTypedefs.h>

namespace aima {
namespace {

// Up to so many rows the few-row kernel.  us with it and with the prompt kernel, heads of 256: 8 rows, one sequence of 32768 positions 15.8
// and 22.8, 64 of up to 8192 78 and 110; 16 rows 23.4 and 31, 103 and 110 .. 122, but 16 of 4111 31 and 26.  Heads of 128, 64 of up
// to 8192: 8 rows 195 and 231 .. 264, 16 rows 285 and 234 .. 261, 16 rows and 16 of 4111 54 and 46.  Heads of 64, 64 of up to 8192: 8 rows
// 193 and 207, 16 rows 309 and 207, one of 32768 36 and 30.  In a form that took 40 rows it needed 138 for 16 sequences of 4111, where
// the prompt kernel needs 29.
constexpr int decode_rows(int head_dim) { return head_dim == 256 ? 16 : 8; }

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* pointer = nullptr;
    cudaDriverEntryPointQueryResult query;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &pointer, cudaEnableDefault, &query) != cudaSuccess || query != cudaDriverEntryPointSuccess)
      pointer = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(pointer);
  }();
  return fn;
}

size_t round256(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t sums_bytes(const KvShape& shape) { return round256(2ull * kKvMaxBlocks * kKvPartRows * shape.head_dim * sizeof(float)); }
size_t weights_bytes() { return round256(2ull * kKvMaxBlocks * kKvPartRows * sizeof(float4)); }

}  // namespace

size_t kv_counter_bytes() { return round256(2ull * kKvMaxBlocks * sizeof(unsigned)); }
size_t kv_workspace_bytes(const KvShape& shape) {
  return kv_counter_bytes() + weights_bytes() + sums_bytes(shape) + sizeof(KvStart) * (kKvMaxBlocks + 1);
}

bool kv_make_maps(const KvShape& shape, const KvLayer& layer, KvMaps* maps) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = encode_fn();
  if (encode == nullptr) return false;
  const int row_bytes = shape.head_dim >= 128 ? 128 : 64;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(shape.head_dim),
                              static_cast<cuuint64_t>(shape.pages) * shape.kv_heads * shape.page_tokens};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(shape.head_dim)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(row_bytes), static_cast<cuuint32_t>(shape.page_tokens)};
  const cuuint32_t step[2] = {1, 1};
  for (int i = 0; i < 2; ++i) {
    if (encode(i == 0 ? &maps->keys : &maps->values, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, i == 0 ? layer.keys : layer.values, dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  return true;
}

bool kv_make_query_map(const KvAttention& a, int tile_tokens, CUtensorMap* map) {
  const PFN_cuTensorMapEncodeTiled_v12000 encode = encode_fn();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.shape.head_dim), static_cast<cuuint64_t>(a.shape.q_heads), static_cast<cuuint64_t>(a.batch.tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.q.head_stride) * 2, static_cast<cuuint64_t>(a.q.row_stride) * 2};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(a.shape.head_dim >= 128 ? 64 : 32), static_cast<cuuint32_t>(a.shape.group),
                             static_cast<cuuint32_t>(tile_tokens)};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(a.q.data), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t kv_attention(const KvAttention& a, const KvMaps& maps, void* workspace, int sm_count, cudaStream_t stream) {
  KvAttentionPlan plan{};
  plan.a = a;
  uint8_t* cursor = static_cast<uint8_t*>(workspace);
  plan.work.arrived = reinterpret_cast<unsigned*>(cursor); cursor += kv_counter_bytes();
  plan.work.weights = reinterpret_cast<float4*>(cursor); cursor += weights_bytes();
  plan.work.sums = reinterpret_cast<float*>(cursor); cursor += sums_bytes(a.shape);
  plan.work.starts = reinterpret_cast<KvStart*>(cursor);
  plan.blocks = sm_count < kKvMaxBlocks ? sm_count : kKvMaxBlocks;
  plan.tile_rows = static_cast<int>(std::min(static_cast<long long>(a.batch.max_new) * a.shape.group, 1ll << 30));
  plan.tile_tokens = kKvTile / a.shape.group;
  plan.query_map = kv_query_map_fits(a.q);
  plan.wait_limit_ns = kWaitBudgetNs;
  return plan.tile_rows <= decode_rows(a.shape.head_dim) ? kv_decode(plan, maps, stream) : kv_prompt(plan, maps, stream);
}

}  // namespace aima
