// Short causal convolution of a linear-attention layer: y[t, c] = silu(sum_j w[c, j] x[t - (W - 1) + j, c]) for W of 2 .. 4, and
// the state, the last W - 1 inputs of a sequence.
//
// A thread takes eight channels of a run of rows and keeps the last W - 1 rows in registers, so an input is read once and once
// more at each run's begin.  Runs begin with a sequence, so only a sequence's first run reads its state; the same threads write it,
// after that, from the inputs themselves.
#include "linear.cuh"

namespace aima {
namespace {

constexpr int kConvThreads = 128;
constexpr int kConvRows = 16;        // of a run

template <int kWidth>
__global__ void __launch_bounds__(kConvThreads) linear_conv_kernel(const LinearConv a) {
  const LinearBatch& b = a.batch;
  if (blockIdx.x == 0 && blockIdx.y == 0) linear_report(b, a.status, threadIdx.x, kConvThreads);
  int s, run;
  if (!linear_find_run<kConvThreads>(b, kConvRows, blockIdx.x, &s, &run)) return;
  const LinearSequence seq = linear_sequence(b, s);
  const int channel = 8 * (static_cast<int>(blockIdx.y) * kConvThreads + static_cast<int>(threadIdx.x));
  const int begin = run * kConvRows, end = min(begin + kConvRows, seq.rows);
  if (begin >= end || channel >= a.channels) return;
  const __nv_bfloat16* x = a.x + seq.row0 * a.x_stride + channel;
  __nv_bfloat16* out = a.out + static_cast<long long>(seq.row0) * a.channels + channel;
  float w[8][kWidth];
  {
    uint4 raw[kWidth];
#pragma unroll
    for (int i = 0; i < kWidth; ++i) raw[i] = *reinterpret_cast<const uint4*>(a.weight + static_cast<long long>(channel) * kWidth + 8 * i);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      float part[8];
      unpack8(raw[i], part);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[(8 * i + j) / kWidth][(8 * i + j) % kWidth] = part[j];
    }
  }
  // rows before the first active one are zeros, or what the slot holds
  const int first = seq.first;
  const long long slot_base = (static_cast<long long>(max(seq.slot, 0)) * (kWidth - 1)) * a.channels + channel;
  const auto before = [&](int row) {        // row < first, above first - kWidth
    return seq.fresh || seq.slot < 0 ? make_uint4(0, 0, 0, 0)
                                     : *reinterpret_cast<const uint4*>(a.states + slot_base + static_cast<long long>(row - first + kWidth - 1) * a.channels);
  };
  const auto input = [&](int row) { return *reinterpret_cast<const uint4*>(x + row * a.x_stride); };
  // For begin <= first only the run with the first row may look at the state; a run behind it begins at least kConvRows later.
  const int start = max(begin, first);
  uint4 window[kWidth - 1];
#pragma unroll
  for (int i = 0; i < kWidth - 1; ++i) {
    const int row = start - (kWidth - 1) + i;
    window[i] = row < first ? before(row) : input(row);
  }
  if (begin == 0 && seq.kept > first) {     // fresh sequences may have inactive rows in front: none of them enters the state
    uint4 last[kWidth - 1];
#pragma unroll
    for (int i = 0; i < kWidth - 1; ++i) {
      const int row = seq.kept - (kWidth - 1) + i;
      last[i] = row < first ? before(row) : input(row);
    }
#pragma unroll
    for (int i = 0; i < kWidth - 1; ++i) *reinterpret_cast<uint4*>(a.states + slot_base + static_cast<long long>(i) * a.channels) = last[i];
  }
  for (int row = begin; row < min(end, start); ++row)
    *reinterpret_cast<uint4*>(out + static_cast<long long>(row) * a.channels) = make_uint4(0, 0, 0, 0);
  float past[kWidth - 1][8];
#pragma unroll
  for (int i = 0; i < kWidth - 1; ++i) unpack8(window[i], past[i]);
  for (int row = start; row < end; ++row) {
    float now[8], y[8];
    unpack8(input(row), now);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float sum = past[0][j] * w[j][0];
#pragma unroll
      for (int i = 1; i < kWidth - 1; ++i) sum = fmaf(past[i][j], w[j][i], sum);
      sum = fmaf(now[j], w[j][kWidth - 1], sum);
      y[j] = sum * linear_sigmoid(sum);
#pragma unroll
      for (int i = 0; i + 1 < kWidth - 1; ++i) past[i][j] = past[i + 1][j];
      past[kWidth - 2][j] = now[j];
    }
    *reinterpret_cast<uint4*>(out + static_cast<long long>(row) * a.channels) =
        make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
  }
}

}  // namespace

cudaError_t linear_conv(const LinearConv& a, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(linear_runs(a.batch, kConvRows)), (a.channels / 8 + kConvThreads - 1) / kConvThreads);
  switch (a.width) {
    case 2: linear_conv_kernel<2><<<grid, kConvThreads, 0, stream>>>(a); break;
    case 3: linear_conv_kernel<3><<<grid, kConvThreads, 0, stream>>>(a); break;
    default: linear_conv_kernel<4><<<grid, kConvThreads, 0, stream>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace aima
