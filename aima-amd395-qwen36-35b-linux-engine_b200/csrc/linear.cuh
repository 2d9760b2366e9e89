// Linear-attention layers: what their kernels and their C ABI (linear_api.cu) share.
#pragma once

#include "../../include/aima_moe.h"
#include "common.cuh"
#include "kv_cache.cuh"

namespace aima {

constexpr int kLinearDim = AIMA_MOE_LINEAR_HEAD_DIM;
constexpr int kLinearBadBatch = 1;   // bits of a handle's status word
constexpr int kLinearTimeout = 2;

struct LinearBatch {
  const int* slots;        // [sequences]
  const int* offsets;      // [sequences + 1] or nullptr: max_new rows each
  const int* lengths;      // [sequences] or nullptr
  const int* keep;         // [sequences] or nullptr
  int sequences, tokens, max_new;
  int slot_count;          // of the handle
};

// One sequence of a batch as every kernel reads it.  Its numbers come from the device, so they are held to their ranges here: a
// sequence that breaks them has no rows, and `bad` is set.
struct LinearSequence {
  int row0, rows;
  int slot;                // -1: not there
  int first;               // its first row that is active: rows before position 0, or of a sequence that is not there, are not
  int kept;                // rows that enter the state; nothing does unless this is above `first`
  bool fresh;              // begins with zeros, not with what its slot holds
  bool bad;
};
__device__ __forceinline__ LinearSequence linear_sequence(const LinearBatch& b, int s) {
  LinearSequence out;
  out.row0 = b.offsets != nullptr ? b.offsets[s] : s * b.max_new;
  const int end = b.offsets != nullptr ? b.offsets[s + 1] : out.row0 + b.max_new;
  out.slot = b.slots[s];
  const int length = b.lengths != nullptr ? b.lengths[s] : -1;
  const int kept = b.keep != nullptr ? b.keep[s] : b.max_new;
  out.rows = end - out.row0;
  out.bad = out.row0 < 0 || end > b.tokens || out.rows < 0 || out.rows > b.max_new || out.slot < -1 || out.slot >= b.slot_count ||
            (b.lengths != nullptr && length < 0);
  if (out.bad) out.row0 = out.rows = 0;
  out.fresh = b.lengths != nullptr && length <= out.rows;
  out.first = out.slot < 0 || out.bad ? out.rows : out.fresh ? out.rows - length : 0;
  out.kept = min(max(kept, 0), out.rows);
  return out;
}

// Runs of `per` rows of the sequences, one after the other: how many there can be.
inline long long linear_runs(const LinearBatch& b, int per) {
  const long long each = (b.max_new + per - 1) / per;
  const long long most = each * b.sequences;
  const long long ragged = (b.tokens + per - 1) / per + static_cast<long long>(b.sequences);
  return b.offsets != nullptr && each > 1 && ragged < most ? ragged : most;
}
// The sequence and the run in it that is number `index` of them, found by a whole block of kThreads threads; false: there is none.
// Where linear_runs counts each sequence's most, a division says it; else the block adds up the runs of all sequences.
template <int kThreads>
__device__ __forceinline__ bool linear_find_run(const LinearBatch& b, int per, int index, int* sequence, int* run) {
  const int each = (b.max_new + per - 1) / per;
  if (b.offsets == nullptr || each == 1 || (b.tokens + per - 1) / per + b.sequences >= each * static_cast<long long>(b.sequences)) {
    *sequence = index / each;
    *run = index - *sequence * each;
    return true;
  }
  __shared__ int sums[kThreads / 32];
  __shared__ int found[2];
  const int t = static_cast<int>(threadIdx.x), lane = t & 31;
  const int share = (b.sequences + kThreads - 1) / kThreads;
  const int first = t * share, last = min(first + share, b.sequences);
  int mine = 0;
  for (int s = first; s < last; ++s) mine += (linear_sequence(b, s).rows + per - 1) / per;
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) sums[t >> 5] = upto;
  if (t == 0) found[0] = -1;
  __syncthreads();
  for (int w = 0; w < (t >> 5); ++w) upto += sums[w];
  if (upto - mine <= index && index < upto) {
    int at = upto - mine;
    for (int s = first; s < last; ++s) {
      const int runs = (linear_sequence(b, s).rows + per - 1) / per;
      if (index < at + runs) {
        found[0] = s;
        found[1] = index - at;
        break;
      }
      at += runs;
    }
  }
  __syncthreads();
  *sequence = found[0];
  *run = found[1];
  return found[0] >= 0;
}
// One block looks all sequences over.
__device__ __forceinline__ void linear_report(const LinearBatch& b, int* status, int thread, int threads) {
  for (int s = thread; s < b.sequences; s += threads)
    if (linear_sequence(b, s).bad) atomicOr(status, kLinearBadBatch);
}

struct Pair {                  // two FP32 numbers that one instruction takes
  unsigned long long bits;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(x), "f"(y)); }
  __device__ __forceinline__ float2 values() const {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(bits));
    return v;
  }
};
__device__ __forceinline__ Pair operator*(const Pair& a, const Pair& b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
  return d;
}
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
  return d;
}
__device__ __forceinline__ Pair fma2(const Pair& a, const Pair& b, const Pair& c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return d;
}

// Whether a sum or mean of squares, with eps, is one that a norm can go by: 2^-100 .. below infinity.
__device__ __forceinline__ bool linear_norm_holds(float squares) { return __float_as_uint(squares) - 0x0d800000u < 0x7f800000u - 0x0d800000u; }
// What the numbers have to be multiplied by before they are squared, else 1.  Beyond FP32 there were numbers from 2^60 on, and what is left
// of them has squares of at most 2^96; so small, squares may have been lost.  eps goes with the factor's square.
__device__ __forceinline__ float linear_norm_shift(float squares) { return !(squares < INFINITY) ? 0x1p-80f : squares < 0x1p-100f ? 0x1p80f : 1.0f; }

// 4 / (1 + e^-x), to a few units of the last place: of a quarter of the denominator, so that the reciprocal is a normal number
__device__ __forceinline__ float linear_four_sigmoid(float x) {
  float quarter, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(quarter) : "f"(fmaf(x, -1.4426950408889634f, -2.0f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(quarter + 0.25f));
  return y;
}
__device__ __forceinline__ float linear_sigmoid(float x) { return 0.25f * linear_four_sigmoid(x); }
__device__ __forceinline__ float linear_silu(float x) { return (0.25f * x) * linear_four_sigmoid(x); }
// for two numbers
__device__ __forceinline__ Pair linear_four_sigmoid(const Pair& x) {
  const float2 exponent = fma2(x, Pair(-1.4426950408889634f, -1.4426950408889634f), Pair(-2.0f, -2.0f)).values();
  float a, b;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(exponent.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(exponent.y));
  const float2 quarter = (Pair(a, b) + Pair(0.25f, 0.25f)).values();
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(quarter.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(quarter.y));
  return Pair(a, b);
}
__device__ __forceinline__ Pair bf16_pair(uint32_t word) { return Pair(bf16_lo(word), bf16_hi(word)); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(const Pair& x) {
  const float2 v = x.values();
  return pack_bf16(v.x, v.y);
}

struct LinearConv {
  LinearBatch batch;
  int channels, width;
  const __nv_bfloat16* x;
  long long x_stride;
  const __nv_bfloat16* weight;
  __nv_bfloat16* states;
  __nv_bfloat16* out;
  int* status;
};
cudaError_t linear_conv(const LinearConv& args, cudaStream_t stream);

struct LinearDelta {
  LinearBatch batch;
  int k_heads, v_heads, group;
  KvRows q, k, v, gate;               // gate.data may be nullptr
  const __nv_bfloat16* a;
  const __nv_bfloat16* b;
  long long a_stride, b_stride;
  const float* a_log;
  const float* dt_bias;
  const __nv_bfloat16* norm_weight;
  float eps;
  float* states;
  __nv_bfloat16* out;                 // may be nullptr
  int* status;
};
// Rows of a sequence up to which it is taken token by token.  us token by token / in chunks, captured, 32 heads with gate: one sequence of
// 16 rows 12.8 / 20.2, of 24 17.5 / 20.2, of 28 20.4 / 20.2, of 32 22.3 / 20.1; eight 20.1 / 31.8, 27.6 / 32.0, 31.8 / 32.2, 34.9 / 32.0; 64
// 130 / 219, 184 / 222, 210 / 224, 236 / 223.
constexpr int kLinearStepRows = 28;
// Sequences of at most max_rows rows.
cudaError_t linear_step(const LinearDelta& args, int max_rows, int sm_count, cudaStream_t stream);
size_t linear_chunk_workspace(int k_heads, int v_heads, int max_tokens, int max_sequences);
// Sequences of more than min_rows rows.
cudaError_t linear_chunks(const LinearDelta& args, int min_rows, void* workspace, int sm_count, cudaStream_t stream);

struct HeadNorm {
  int tokens, heads, dim, activation;
  float offset, eps;
  KvRows x, gate;
  const __nv_bfloat16* weight;
  __nv_bfloat16* out;
};
cudaError_t head_norm(const HeadNorm& args, cudaStream_t stream);

}  // namespace aima
