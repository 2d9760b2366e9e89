// Norm of each head with an optional gate: y = x / sqrt(mean(x^2) + eps) * (w + offset) * act(z), or x * act(z) alone.
//
// A head of 64, 128 or 256 lies in 8, 16 or 32 neighbouring lanes, eight elements each: one load per lane and tensor, the sum of
// squares by shuffles inside them.  All of it is bytes.
#include "linear.cuh"

namespace aima {
namespace {

constexpr int kNormThreads = 256;

template <int kDim, bool kNorm, int kActivation>
__global__ void __launch_bounds__(kNormThreads) head_norm_kernel(const HeadNorm a) {
  constexpr int kLanes = kDim / 8;                       // of a head
  const int lane = threadIdx.x % kLanes;
  const long long unit = static_cast<long long>(blockIdx.x) * (kNormThreads / kLanes) + threadIdx.x / kLanes;
  const bool live = unit < static_cast<long long>(a.tokens) * a.heads;
  const int row = live ? static_cast<int>(unit / a.heads) : 0, head = live ? static_cast<int>(unit - static_cast<long long>(row) * a.heads) : 0;
  const uint4 raw = *reinterpret_cast<const uint4*>(a.x.data + row * a.x.row_stride + head * a.x.head_stride + 8 * lane);
  uint4 gate = make_uint4(0, 0, 0, 0);
  if (kActivation != AIMA_MOE_GATE_NONE) gate = *reinterpret_cast<const uint4*>(a.gate.data + row * a.gate.row_stride + head * a.gate.head_stride + 8 * lane);
  float x[8];
  unpack8(raw, x);
  if (kNorm) {
    float w[8], sum = 0.0f;
    unpack8(*reinterpret_cast<const uint4*>(a.weight + 8 * lane), w);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float scale = __frsqrt_rn(fmaf(sum, 1.0f / kDim, a.eps));
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * scale * (w[j] + a.offset);
  }
  if (kActivation != AIMA_MOE_GATE_NONE) {
    float z[8];
    unpack8(gate, z);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= kActivation == AIMA_MOE_GATE_SILU ? z[j] * linear_sigmoid(z[j]) : linear_sigmoid(z[j]);
  }
  if (live)
    *reinterpret_cast<uint4*>(a.out + unit * kDim + 8 * lane) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

template <int kDim>
cudaError_t launch(const HeadNorm& a, cudaStream_t stream) {
  const long long units = static_cast<long long>(a.tokens) * a.heads;
  const unsigned grid = static_cast<unsigned>((units * (kDim / 8) + kNormThreads - 1) / kNormThreads);
  if (a.weight == nullptr) {
    if (a.activation == AIMA_MOE_GATE_SILU) head_norm_kernel<kDim, false, AIMA_MOE_GATE_SILU><<<grid, kNormThreads, 0, stream>>>(a);
    else head_norm_kernel<kDim, false, AIMA_MOE_GATE_SIGMOID><<<grid, kNormThreads, 0, stream>>>(a);
  } else if (a.activation == AIMA_MOE_GATE_NONE) {
    head_norm_kernel<kDim, true, AIMA_MOE_GATE_NONE><<<grid, kNormThreads, 0, stream>>>(a);
  } else if (a.activation == AIMA_MOE_GATE_SILU) {
    head_norm_kernel<kDim, true, AIMA_MOE_GATE_SILU><<<grid, kNormThreads, 0, stream>>>(a);
  } else {
    head_norm_kernel<kDim, true, AIMA_MOE_GATE_SIGMOID><<<grid, kNormThreads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t head_norm(const HeadNorm& a, cudaStream_t stream) {
  return a.dim == 64 ? launch<64>(a, stream) : a.dim == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace aima
