// Attention of a batch's rows over the paged 8-bit cache: a plain form on CUDA cores.
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  j <= position of the row
// One block per (row, query head); its warps take every eighth position, a lane holds kDim / 32 elements of the head, and the
// running maxima, sums and outputs of the warps are joined at the end.
#include "kv_cache.cuh"

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

}  // namespace

cudaError_t kv_attention(const KvAttention& a, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(a.batch.tokens) * a.shape.q_heads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const unsigned grid = static_cast<unsigned>(blocks);
  switch (a.shape.head_dim) {
    case 64: kv_attention_plain_kernel<64><<<grid, kWarps * 32, 0, stream>>>(a); break;
    case 128: kv_attention_plain_kernel<128><<<grid, kWarps * 32, 0, stream>>>(a); break;
    default: kv_attention_plain_kernel<256><<<grid, kWarps * 32, 0, stream>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace aima
