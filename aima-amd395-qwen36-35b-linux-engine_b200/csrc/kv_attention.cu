// Attention of a batch's rows over the paged 8-bit cache: a plain form on CUDA cores.
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  j <= position of the row
// One block per (row, query head); its warps take every eighth position, a lane holds kDim / 32 elements of the head, and the
// running maxima, sums and outputs of the warps are joined at the end.
#include "kv_attention.cuh"

#include <cudaTypedefs.h>

#include <cuda_fp8.h>

namespace aima {
namespace {

constexpr int kWarps = 8;

template <int kPer>
__device__ __forceinline__ void load_codes(const uint8_t* at, float* x) {
  if (kPer == 8) {
    const uint2 c = *reinterpret_cast<const uint2*>(at);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i % kPer] = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 255u), __NV_E4M3)));
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(at[i], __NV_E4M3)));
  }
}

template <int kDim>
__global__ void __launch_bounds__(kWarps * 32)
kv_attention_plain_kernel(const KvAttention a) {
  constexpr int kPer = kDim / 32;
  __shared__ float part_out[kWarps][kDim];
  __shared__ float part_max[kWarps], part_sum[kWarps];
  const int head = blockIdx.x % a.shape.q_heads;
  const int row = blockIdx.x / a.shape.q_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int low = 0, high = a.batch.sequences;
  if (a.batch.offsets == nullptr) {
    low = row / a.batch.max_new;
  } else {
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (a.batch.offsets[mid] <= row) low = mid; else high = mid;
    }
  }
  const KvSequence seq = kv_sequence(a.batch, a.shape, low);
  if (seq.bad && threadIdx.x == 0) atomicOr(a.status, kKvBadBatch);
  if (row < seq.row0 || row >= seq.row0 + seq.rows) return;
  const int position = seq.length - seq.rows + row - seq.row0;
  float q[kPer], out[kPer], top = -INFINITY, sum = 0.0f;
  const __nv_bfloat16* at = a.q.data + row * a.q.row_stride + head * a.q.head_stride + lane * kPer;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    q[i] = __bfloat162float(at[i]);
    out[i] = 0.0f;
  }
  for (int j = warp; j <= position; j += kWarps) {
    const int page = a.batch.table[static_cast<size_t>(low) * a.batch.columns + (j >> a.shape.page_shift)];
    if (page < 0 || page >= a.shape.pages) {
      if (lane == 0) atomicOr(a.status, kKvBadBatch);
      continue;
    }
    const size_t scale_at = static_cast<size_t>(page) * a.shape.kv_heads + head / a.shape.group;
    const size_t element = (scale_at * a.shape.page_tokens + (j & (a.shape.page_tokens - 1))) * kDim + lane * kPer;
    float k[kPer], v[kPer];
    load_codes<kPer>(a.layer.keys + element, k);
    load_codes<kPer>(a.layer.values + element, v);
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) dot = fmaf(q[i], k[i], dot);
    dot = butterfly_sum(dot) * (a.layer.key_scales[scale_at] * a.scale_log2);
    const float new_top = fmaxf(top, dot);
    const float keep = new_top == -INFINITY ? 1.0f : exp2f(top - new_top);
    const float p = new_top == -INFINITY ? dot - dot : exp2f(dot - new_top);
    top = new_top;
    sum = sum * keep + p;
    const float weight = p * a.layer.value_scales[scale_at];
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[i] = fmaf(weight, v[i], out[i] * keep);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) part_out[warp][lane * kPer + i] = out[i];
  if (lane == 0) {
    part_max[warp] = top;
    part_sum[warp] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kDim; i += blockDim.x) {
    float m = -INFINITY;
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, part_max[w]);
    float total = 0.0f, value = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
      const float f = part_max[w] == -INFINITY ? (part_sum[w] == 0.0f ? 0.0f : 1.0f) : exp2f(part_max[w] - m);
      total = fmaf(part_sum[w], f, total);
      value = fmaf(part_out[w][i], f, value);
    }
    a.out[(static_cast<size_t>(row) * a.shape.q_heads + head) * kDim + i] = __float2bfloat16_rn(total == 0.0f ? 0.0f : value / total);
  }
}

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

constexpr int kDecodeRows = 64;
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
  const long long blocks = static_cast<long long>(a.batch.tokens) * a.shape.q_heads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  kv_attention_plain_kernel<kDim><<<static_cast<unsigned>(blocks), kWarps * 32, 0, stream>>>(a);
  return cudaGetLastError();
}

size_t round256(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t sums_bytes(const KvShape& shape) { return round256(2ull * kKvMaxBlocks * kPartRows * shape.head_dim * sizeof(float)); }
size_t weights_bytes() { return round256(2ull * kKvMaxBlocks * kPartRows * sizeof(float2)); }

}  // namespace

size_t kv_workspace_bytes(const KvShape& shape, int max_sequences) {
  return sums_bytes(shape) + weights_bytes() + round256(sizeof(long long) * (max_sequences + 1));
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

cudaError_t kv_attention(const KvAttention& a, const KvMaps& maps, void* workspace, int sm_count, cudaStream_t stream) {
  KvAttentionPlan plan{};
  plan.a = a;
  uint8_t* cursor = static_cast<uint8_t*>(workspace);
  plan.work.sums = reinterpret_cast<float*>(cursor); cursor += sums_bytes(a.shape);
  plan.work.weights = reinterpret_cast<float2*>(cursor); cursor += weights_bytes();
  plan.work.prefix = reinterpret_cast<long long*>(cursor);
  plan.work.rows_per_part = kPartRows;
  plan.blocks = sm_count < kKvMaxBlocks ? sm_count : kKvMaxBlocks;
  plan.tile_rows = a.batch.max_new * a.shape.group;
  plan.wait_limit_ns = kWaitBudgetNs;
  switch (a.shape.head_dim) {
    case 64: return launch<64>(plan, maps, stream);
    case 128: return launch<128>(plan, maps, stream);
    default: return launch<256>(plan, maps, stream);
  }
}

}  // namespace aima
