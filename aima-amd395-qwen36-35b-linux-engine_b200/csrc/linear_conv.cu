// Short causal convolution of a linear-attention layer: y[t, c] = silu(sum_j w[c, j] x[t - (W - 1) + j, c]) for W of 2 .. 4, and
// the state, the last W - 1 inputs of a sequence.
//
// A thread takes eight channels of a run of 16 rows, four at a time: the next four are under way while these are widened, two channels
// at a time, summed and put back in their own place.  Runs begin with a sequence, so only a sequence's first run reads its state; the same threads
// write it, after that, from the inputs themselves.
//
// 8192 tokens of 8192 channels move 268 MB in 57.0 us (4.7 TB/s): two channels an instruction, else two thirds of the issue slots
// (59.4 us).  No one part is full: 61 % of the pipe for exponentials and reciprocals, 57 % of the issue slots, and 20 of 64 warps, more of which
// the registers have no room for.  Earlier forms: runs of 8 rows with all loads first 65.7 us, four channels a
// thread 76.9.
#include "linear.cuh"

namespace aima {
namespace {

constexpr int kConvThreads = 128;
constexpr int kConvRows = 16;        // of a run
constexpr int kConvStep = 4;         // of them at a time

template <int kWidth>
__global__ void __launch_bounds__(kConvThreads, 5) linear_conv_kernel(const LinearConv a) {
  const LinearBatch& b = a.batch;
  if (blockIdx.x == 0 && blockIdx.y == 0) linear_report(b, a.status, threadIdx.x, kConvThreads);
  int s, run;
  if (!linear_find_run<kConvThreads>(b, kConvRows, blockIdx.x, &s, &run)) return;
  const LinearSequence seq = linear_sequence(b, s);
  const int channel = 8 * (static_cast<int>(blockIdx.y) * kConvThreads + static_cast<int>(threadIdx.x));
  const int begin = run * kConvRows, end = min(begin + kConvRows, seq.rows);
  if (begin >= end || channel >= a.channels) return;
  constexpr int kBefore = kWidth - 1;
  const __nv_bfloat16* x = a.x + seq.row0 * a.x_stride + channel;
  // rows before the first active one are zeros, or what the slot holds
  const int first = seq.first;
  const long long slot_base = (static_cast<long long>(max(seq.slot, 0)) * kBefore) * a.channels + channel;
  const auto value = [&](int row) {
    if (row >= end) return make_uint4(0, 0, 0, 0);
    if (row >= first) return *reinterpret_cast<const uint4*>(x + row * a.x_stride);
    if (seq.fresh || seq.slot < 0 || row < first - kBefore) return make_uint4(0, 0, 0, 0);
    return *reinterpret_cast<const uint4*>(a.states + slot_base + static_cast<long long>(row - first + kBefore) * a.channels);
  };
  uint4 rows[kBefore + kConvStep], next[kConvStep], weights[kWidth];
#pragma unroll
  for (int i = 0; i < kBefore + kConvStep; ++i) rows[i] = value(begin - kBefore + i);
#pragma unroll
  for (int i = 0; i < kWidth; ++i) weights[i] = *reinterpret_cast<const uint4*>(a.weight + static_cast<long long>(channel) * kWidth + 8 * i);
  if (begin == 0 && seq.kept > first) {     // fresh sequences may have inactive rows in front: none of them enters the state
    uint4 last[kBefore];
#pragma unroll
    for (int i = 0; i < kBefore; ++i) {
      const int row = seq.kept - kBefore + i;
      last[i] = row >= first ? *reinterpret_cast<const uint4*>(x + row * a.x_stride) : value(row);
    }
#pragma unroll
    for (int i = 0; i < kBefore; ++i) *reinterpret_cast<uint4*>(a.states + slot_base + static_cast<long long>(i) * a.channels) = last[i];
  }
  __nv_bfloat16* out = a.out + static_cast<long long>(seq.row0 + begin) * a.channels + channel;
  const __nv_bfloat16* from = x + (begin + kConvStep) * a.x_stride;
#pragma unroll 1
  for (int row = begin; row < end; row += kConvStep) {
    // the next rows; after the first step they are all behind the first active one, unless that one comes late
    if (row + kConvStep >= first && row + 2 * kConvStep <= end) {
#pragma unroll
      for (int i = 0; i < kConvStep; ++i, from += a.x_stride) next[i] = *reinterpret_cast<const uint4*>(from);
    } else {
#pragma unroll
      for (int i = 0; i < kConvStep; ++i) next[i] = value(row + kConvStep + i);
      from += kConvStep * a.x_stride;
    }
    uint4 y[kConvStep];
#pragma unroll
    for (int j = 0; j < 4; ++j) {             // channels 2 j, 2 j + 1
      const auto weight = [&](int at) {       // of the thread's, eight to a vector
        const uint32_t word = (&weights[at / 8].x)[(at % 8) / 2];
        return at % 2 == 0 ? bf16_lo(word) : bf16_hi(word);
      };
      Pair w[kWidth], in[kBefore + kConvStep];
#pragma unroll
      for (int i = 0; i < kWidth; ++i) w[i] = Pair(weight(2 * j * kWidth + i), weight((2 * j + 1) * kWidth + i));
#pragma unroll
      for (int i = 0; i < kBefore + kConvStep; ++i) in[i] = bf16_pair((&rows[i].x)[j]);
#pragma unroll
      for (int r = 0; r < kConvStep; ++r) {
        Pair sum = in[r] * w[0];
#pragma unroll
        for (int i = 1; i < kWidth; ++i) sum = fma2(in[r + i], w[i], sum);
        (&y[r].x)[j] = pack_bf16((sum * Pair(0.25f, 0.25f)) * linear_four_sigmoid(sum));
      }
    }
#pragma unroll
    for (int r = 0; r < kConvStep; ++r, out += a.channels)
      if (row + r < end) *reinterpret_cast<uint4*>(out) = row + r < first ? make_uint4(0, 0, 0, 0) : y[r];
#pragma unroll
    for (int i = 0; i < kBefore; ++i) rows[i] = rows[kConvStep + i];
#pragma unroll
    for (int i = 0; i < kConvStep; ++i) rows[kBefore + i] = next[i];
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
