// Attention of a batch's rows over the paged 8-bit cache: the choice of the kernel, the tensor maps, the workspace, and the join
// of the few-row kernel's parts.
#include "kv_attention.cuh"

#include <algorithm>
#include <cudaTypedefs.h>

namespace aima {
namespace {

// Puts the parts of divided units together, and writes zeros for rows of sequences without anything in the cache.  One block
// per (sequence, key/value head, row); a float4 of the head per thread, 1024 / kDim parts at a time.
template <int kDim>
__global__ void __launch_bounds__(256)
kv_join_kernel(const KvAttentionPlan plan) {
  constexpr int kGroups = 256 / (kDim / 4);
  __shared__ float factor[kKvMaxBlocks];
  __shared__ float warp_top[8], warp_sum[8];
  __shared__ float4 joined[256];
  pdl_enter();
  const KvAttention& a = plan.a;
  const int row = blockIdx.x % plan.tile_rows;
  const int head = (blockIdx.x / plan.tile_rows) % a.shape.kv_heads;
  const int s = blockIdx.x / (plan.tile_rows * a.shape.kv_heads);
  const KvSequence seq = kv_sequence(a.batch, a.shape, s);
  if (row >= seq.rows * a.shape.group) return;
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  const int piece = thread % (kDim / 4), group = thread / (kDim / 4);
  __nv_bfloat16* out = a.out + ((seq.row0 + row / a.shape.group) * static_cast<long long>(a.shape.q_heads) + head * a.shape.group + row % a.shape.group) * kDim;
  const long long total = plan.work.prefix[a.batch.sequences];
  const long long tiles = (plan.work.prefix[s + 1] - plan.work.prefix[s]) / a.shape.kv_heads;
  if (tiles == 0) {
    if (thread < kDim / 4) reinterpret_cast<uint2*>(out)[thread] = make_uint2(0, 0);
    return;
  }
  const long long first = plan.work.prefix[s] + head * tiles;
  const int block0 = kv_block_of(total, first, plan.blocks), block1 = kv_block_of(total, first + tiles - 1, plan.blocks);
  if (block0 == block1) return;
  const int parts = block1 - block0 + 1;
  auto part_of = [&](int p) { return kv_part(first, kv_block_begin(total, block0 + p, plan.blocks), block0 + p); };
  float2 mine = make_float2(-INFINITY, 0.0f);
  if (thread < parts) mine = plan.work.weights[static_cast<size_t>(part_of(thread)) * plan.work.rows_per_part + row];
  float top = mine.x;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
  top = warp_top[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) top = fmaxf(top, warp_top[w]);
  // a part without a maximum has seen nothing, or nothing but NaN
  const float f = thread < parts ? exp2f(mine.x - (top == -INFINITY ? 0.0f : top)) : 0.0f;
  float sum = mine.x == -INFINITY ? mine.y : mine.y * f;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (thread < parts) factor[thread] = f;
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  sum = warp_sum[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) sum += warp_sum[w];
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
  for (int p = group; p < parts; p += kGroups) {
    const float4 x = *reinterpret_cast<const float4*>(plan.work.sums + (static_cast<size_t>(part_of(p)) * plan.work.rows_per_part + row) * kDim + 4 * piece);
    const float w = factor[p];
    acc.x = fmaf(x.x, w, acc.x);
    acc.y = fmaf(x.y, w, acc.y);
    acc.z = fmaf(x.z, w, acc.z);
    acc.w = fmaf(x.w, w, acc.w);
  }
  joined[thread] = acc;
  __syncthreads();
  if (group == 0) {
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      const float4 x = joined[g * (kDim / 4) + piece];
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inverse, acc.y * inverse), hi = __floats2bfloat162_rn(acc.z * inverse, acc.w * inverse);
    uint2 w;
    w.x = *reinterpret_cast<uint32_t*>(&lo);
    w.y = *reinterpret_cast<uint32_t*>(&hi);
    reinterpret_cast<uint2*>(out)[piece] = w;
  }
}

constexpr int kDecodeRows = 16;
constexpr int kPartRows = 128;

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

template <int kDim>
cudaError_t launch(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream) {
  const KvAttention& a = plan.a;
  if (plan.tile_rows <= kDecodeRows) {
    cudaError_t error = kv_decode(plan, maps, stream);
    if (error != cudaSuccess) return error;
    const long long blocks = static_cast<long long>(a.batch.sequences) * a.shape.kv_heads * plan.tile_rows;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return launch_pdl(kv_join_kernel<kDim>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, plan);
  }
  return kv_prompt(plan, maps, stream);
}

size_t round256(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t sums_bytes(const KvShape& shape) { return round256(2ull * kKvMaxBlocks * kPartRows * shape.head_dim * sizeof(float)); }
size_t weights_bytes() { return round256(2ull * kKvMaxBlocks * kPartRows * sizeof(float2)); }

}  // namespace

size_t kv_workspace_bytes(const KvShape& shape, int max_sequences) {
  return sums_bytes(shape) + weights_bytes() + round256(sizeof(long long) * (max_sequences + 1)) + sizeof(KvStart) * (kKvMaxBlocks + 1);
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

cudaError_t kv_attention(const KvAttention& a, const KvMaps& maps, void* workspace, int max_sequences, int sm_count, cudaStream_t stream) {
  KvAttentionPlan plan{};
  plan.a = a;
  uint8_t* cursor = static_cast<uint8_t*>(workspace);
  plan.work.sums = reinterpret_cast<float*>(cursor); cursor += sums_bytes(a.shape);
  plan.work.weights = reinterpret_cast<float2*>(cursor); cursor += weights_bytes();
  plan.work.prefix = reinterpret_cast<long long*>(cursor); cursor += round256(sizeof(long long) * (max_sequences + 1));
  plan.work.starts = reinterpret_cast<KvStart*>(cursor);
  plan.work.rows_per_part = kPartRows;
  plan.blocks = sm_count < kKvMaxBlocks ? sm_count : kKvMaxBlocks;
  plan.tile_rows = static_cast<int>(std::min(static_cast<long long>(a.batch.max_new) * a.shape.group, 1ll << 30));
  plan.tile_tokens = kKvTile / a.shape.group;
  plan.wait_limit_ns = kWaitBudgetNs;
  switch (a.shape.head_dim) {
    case 64: return launch<64>(plan, maps, stream);
    case 128: return launch<128>(plan, maps, stream);
    default: return launch<256>(plan, maps, stream);
  }
}

}  // namespace aima
