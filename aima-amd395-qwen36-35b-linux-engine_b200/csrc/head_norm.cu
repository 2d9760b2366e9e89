// Norm of each head with an optional gate: y = x / sqrt(mean(x^2) + eps) * (w + offset) * act(z), or x * act(z) alone.
//
// A head of 64, 128 or 256 lies in 8, 16 or 32 neighbouring lanes, eight elements each: one load per lane and tensor, the sum of
// squares by shuffles inside them.  All of it is bytes: with 8192 tokens of 16 heads of 256 the norm moves 134 MB in 25.9 us and the
// sigmoid gate 201 MB in 32.8 us (5.2 and 6.1 TB/s); norm and silu gate of 32 heads of 128, 201 MB in 37.9 us (5.3 TB/s), take
// 56 % of the exponentials and reciprocals that the multiprocessors can do and 78 % of the instructions.
#include "linear.cuh"

namespace aima {
namespace {

constexpr int kNormThreads = 128;

template <int kDim, bool kNorm, int kActivation, int kUnits>
__global__ void __launch_bounds__(kNormThreads) head_norm_kernel(const HeadNorm a, const int units) {
  constexpr int kLanes = kDim / 8, kPerBlock = kNormThreads / kLanes;          // lanes of a head, heads that a block takes at a time
  const int lane = threadIdx.x % kLanes;
  uint4 raw[kUnits], gate[kUnits];
  int unit[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    unit[u] = (static_cast<int>(blockIdx.x) * kUnits + u) * kPerBlock + static_cast<int>(threadIdx.x) / kLanes;
    const int at = min(unit[u], units - 1), row = at / a.heads, head = at - row * a.heads;
    raw[u] = *reinterpret_cast<const uint4*>(a.x.data + row * a.x.row_stride + head * a.x.head_stride + 8 * lane);
    if (kActivation != AIMA_MOE_GATE_NONE) gate[u] = *reinterpret_cast<const uint4*>(a.gate.data + row * a.gate.row_stride + head * a.gate.head_stride + 8 * lane);
  }
  float w[8];
  if (kNorm) {
    unpack8(*reinterpret_cast<const uint4*>(a.weight + 8 * lane), w);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] += a.offset;
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    float x[8];
    unpack8(raw[u], x);
    if (kNorm) {
      const auto mean = [&](float eps) {     // of the squares, with eps
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        return fmaf(sum, 1.0f / kDim, eps);
      };
      float square = mean(a.eps);
      if (__any_sync(0xffffffffu, !linear_norm_holds(square))) {
        const float by = linear_norm_shift(square);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= by;
        square = mean(a.eps * by * by);
      }
      const float scale = __frsqrt_rn(square);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * scale * w[j];
    }
    if (kActivation != AIMA_MOE_GATE_NONE) {
      float z[8];
      unpack8(gate[u], z);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= kActivation == AIMA_MOE_GATE_SILU ? linear_silu(z[j]) : linear_sigmoid(z[j]);
    }
    if (unit[u] < units)
      *reinterpret_cast<uint4*>(a.out + static_cast<long long>(unit[u]) * kDim + 8 * lane) =
          make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  }
}

// Heads that a thread has under way.  us with one / two, tokens of 16 heads on a stream of them: norms of 256 at 64 tokens 2.1 / 2.3,
// at 1024 5.1 / 5.1, at 2048 8.6 / 8.2, at 8192 28.7 / 25.9; norms of 64 at 2048 3.7 / 3.8, at 4096 5.5 / 5.4, at 16384 15.2 / 14.3; sigmoid
// gate of 256 at 1024 6.4 / 6.4, at 2048 10.3 / 10.2, at 8192 34.1 / 33.8; norm and silu gate of 128 at 1024 4.0 / 4.3, at 1500 5.3 / 5.2,
// at 2048 6.8 / 6.8, at 4096 11.6 / 11.3, at 16384 38.9 / 36.2, at 32768 73.7 / 68.1; norm and sigmoid gate of 128 at 1024 4.4 / 4.6, at 4096
// 11.4 / 10.9, at 32768 72.7 / 66.6.  So two from twenty blocks of one a multiprocessor (148) on.  Four are no faster: norm and silu gate at
// 4096 12.0, at 32768 69.6.
template <int kDim, bool kNorm, int kActivation>
void launch_units(const HeadNorm& a, cudaStream_t stream) {
  constexpr int kPerBlock = kNormThreads / (kDim / 8);
  const int units = a.tokens * a.heads;
  if (units > 20 * 148 * kPerBlock)
    head_norm_kernel<kDim, kNorm, kActivation, 2><<<(units + 2 * kPerBlock - 1) / (2 * kPerBlock), kNormThreads, 0, stream>>>(a, units);
  else
    head_norm_kernel<kDim, kNorm, kActivation, 1><<<(units + kPerBlock - 1) / kPerBlock, kNormThreads, 0, stream>>>(a, units);
}

template <int kDim>
void launch(const HeadNorm& a, cudaStream_t stream) {
  if (a.weight == nullptr) {
    if (a.activation == AIMA_MOE_GATE_SILU) launch_units<kDim, false, AIMA_MOE_GATE_SILU>(a, stream);
    else launch_units<kDim, false, AIMA_MOE_GATE_SIGMOID>(a, stream);
  } else if (a.activation == AIMA_MOE_GATE_NONE) {
    launch_units<kDim, true, AIMA_MOE_GATE_NONE>(a, stream);
  } else if (a.activation == AIMA_MOE_GATE_SILU) {
    launch_units<kDim, true, AIMA_MOE_GATE_SILU>(a, stream);
  } else {
    launch_units<kDim, true, AIMA_MOE_GATE_SIGMOID>(a, stream);
  }
}

}  // namespace

cudaError_t head_norm(const HeadNorm& all, cudaStream_t stream) {
  // launches of at most 2^30 heads, which 32 bits count
  const int most = (1 << 30) / all.heads;
  for (int begin = 0; begin < all.tokens; begin += most) {
    HeadNorm a = all;
    a.tokens = all.tokens - begin < most ? all.tokens - begin : most;
    a.x.data += begin * a.x.row_stride;
    if (a.gate.data != nullptr) a.gate.data += begin * a.gate.row_stride;
    a.out += static_cast<long long>(begin) * a.heads * a.dim;
    if (a.dim == 64) launch<64>(a, stream);
    else if (a.dim == 128) launch<128>(a, stream);
    else launch<256>(a, stream);
    const cudaError_t error = cudaGetLastError();
    if (error != cudaSuccess) return error;
  }
  return cudaSuccess;
}

}  // namespace aima
