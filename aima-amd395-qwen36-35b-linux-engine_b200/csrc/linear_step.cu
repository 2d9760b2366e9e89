// The gated delta rule token by token: the form for single tokens and drafts.
//
//   S <- e^g S;  d = beta (v - S^T k);  S <- S + k d^T;  o = S^T q
// Both products with the state are taken before it changes, from one pass over it: with r = S^T k and p = S^T q of the old state,
//   d = beta (v - e^g r),   o = e^g p + (k.q) d,   S <- e^g S + k d^T.
//
// A block has the state of one head of one sequence in registers, read and written once however many tokens there are.  A warp has
// 16 columns (value elements) of it and all 128 rows: four columns and 16 rows a lane, so the sums over the rows stay in the warp
// and warps need not wait for each other between tokens.
#include "linear.cuh"

namespace aima {
namespace {

constexpr int kStepThreads = 256;
constexpr int kStepRows = 16;            // tokens prepared at a time

struct __align__(16) StepRow {
  float k[kLinearDim], q[kLinearDim];
  float v[kLinearDim];                   // then the token's output
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  return make_float4(bf16_lo(raw.x), bf16_hi(raw.x), bf16_lo(raw.y), bf16_hi(raw.y));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float4& v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}
__device__ __forceinline__ float dot4(const float4& a, const float4& b) { return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, a.x * b.x))); }
__device__ __forceinline__ float4 scaled(const float4& a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }

__global__ void __launch_bounds__(kStepThreads, 2) linear_step_kernel(const LinearDelta a, int max_rows) {
  __shared__ StepRow rows[kStepRows];
  __shared__ float decay[kStepRows], rate[kStepRows], overlap[kStepRows];
  const int head = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const LinearSequence seq = linear_sequence(a.batch, blockIdx.y);
  if (seq.bad && head == 0 && threadIdx.x == 0) atomicOr(a.status, kLinearBadBatch);
  if (seq.rows > max_rows) return;
  // rows that have to be gone through: the active ones, without outputs only those that stay
  const int end = a.out != nullptr ? seq.rows : min(seq.rows, seq.kept);
  if (a.out != nullptr)
    for (int i = threadIdx.x; i < min(seq.first, end) * (kLinearDim / 8); i += kStepThreads)
      *reinterpret_cast<uint4*>(a.out + (static_cast<long long>(seq.row0 + i / (kLinearDim / 8)) * a.v_heads + head) * kLinearDim + 8 * (i % (kLinearDim / 8))) =
          make_uint4(0, 0, 0, 0);
  if (seq.first >= end) return;

  // this lane's part of the state: rows 32 i + 4 part + j, columns column .. column + 3
  const int part = lane >> 2, column = 16 * warp + 4 * (lane & 3);
  float* state = a.states + ((static_cast<long long>(seq.slot) * a.v_heads + head) * kLinearDim) * kLinearDim + column;
  float4 s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      s[i][j] = seq.fresh ? make_float4(0, 0, 0, 0) : *reinterpret_cast<const float4*>(state + (32 * i + 4 * part + j) * kLinearDim);

  const int k_head = head / a.group;
  for (int begin = seq.first; begin < end; begin += kStepRows) {
    const int count = min(kStepRows, end - begin);
    for (int t = warp; t < count; t += kStepThreads / 32) {
      const long long row = seq.row0 + begin + t;
      const float4 k = load4(a.k.data + row * a.k.row_stride + k_head * a.k.head_stride + 4 * lane);
      const float4 q = load4(a.q.data + row * a.q.row_stride + k_head * a.q.head_stride + 4 * lane);
      const float4 v = load4(a.v.data + row * a.v.row_stride + head * a.v.head_stride + 4 * lane);
      const float kk = warp_sum(dot4(k, k)), qq = warp_sum(dot4(q, q));
      const float4 ku = scaled(k, __frsqrt_rn(kk + a.eps));
      const float4 qu = scaled(q, __frsqrt_rn(qq + a.eps) * 0.08838834764831845f);
      const float kq = warp_sum(dot4(ku, qu));
      *reinterpret_cast<float4*>(&rows[t].k[4 * lane]) = ku;
      *reinterpret_cast<float4*>(&rows[t].q[4 * lane]) = qu;
      *reinterpret_cast<float4*>(&rows[t].v[4 * lane]) = v;
      if (lane == 0) {
        const float x = __bfloat162float(a.a[row * a.a_stride + head]) + a.dt_bias[head];
        decay[t] = expf(-expf(a.a_log[head]) * (x > 20.0f ? x : log1pf(expf(x))));
        rate[t] = 1.0f / (1.0f + expf(-__bfloat162float(a.b[row * a.b_stride + head])));
        overlap[t] = kq;
      }
    }
    __syncthreads();
    for (int t = 0; t < count; ++t) {
      float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};        // of S^T k, then of S^T q, for four columns
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 k4 = *reinterpret_cast<const float4*>(&rows[t].k[32 * i + 4 * part]);
        const float4 q4 = *reinterpret_cast<const float4*>(&rows[t].q[32 * i + 4 * part]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float kj = (&k4.x)[j], qj = (&q4.x)[j];
          sums[0] = fmaf(s[i][j].x, kj, sums[0]);
          sums[1] = fmaf(s[i][j].y, kj, sums[1]);
          sums[2] = fmaf(s[i][j].z, kj, sums[2]);
          sums[3] = fmaf(s[i][j].w, kj, sums[3]);
          sums[4] = fmaf(s[i][j].x, qj, sums[4]);
          sums[5] = fmaf(s[i][j].y, qj, sums[5]);
          sums[6] = fmaf(s[i][j].z, qj, sums[6]);
          sums[7] = fmaf(s[i][j].w, qj, sums[7]);
        }
      }
      // part p ends with the total of sums[p]
      float half[4], quarter[2];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float keep = (lane & 16) != 0 ? sums[4 + c] : sums[c], send = (lane & 16) != 0 ? sums[c] : sums[4 + c];
        half[c] = keep + __shfl_xor_sync(0xffffffffu, send, 16);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float keep = (lane & 8) != 0 ? half[2 + c] : half[c], send = (lane & 8) != 0 ? half[c] : half[2 + c];
        quarter[c] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
      }
      const float keep = (lane & 4) != 0 ? quarter[1] : quarter[0], send = (lane & 4) != 0 ? quarter[0] : quarter[1];
      const float total = keep + __shfl_xor_sync(0xffffffffu, send, 4);
      const float e = decay[t];
      const int mine = column + (part & 3);                              // the column whose total this lane has
      float d = rate[t] * (rows[t].v[mine] - e * total);                 // of use in parts 0 .. 3
      d = __shfl_sync(0xffffffffu, d, lane & 15);
      if (part >= 4) rows[t].v[mine] = fmaf(overlap[t], d, e * total);   // its value element has been read: by lanes that the shuffle waited for
      const float d0 = __shfl_sync(0xffffffffu, d, lane & 3), d1 = __shfl_sync(0xffffffffu, d, (lane & 3) | 4);
      const float d2 = __shfl_sync(0xffffffffu, d, (lane & 3) | 8), d3 = __shfl_sync(0xffffffffu, d, (lane & 3) | 12);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 k4 = *reinterpret_cast<const float4*>(&rows[t].k[32 * i + 4 * part]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float kj = (&k4.x)[j];
          s[i][j].x = fmaf(kj, d0, e * s[i][j].x);
          s[i][j].y = fmaf(kj, d1, e * s[i][j].y);
          s[i][j].z = fmaf(kj, d2, e * s[i][j].z);
          s[i][j].w = fmaf(kj, d3, e * s[i][j].w);
        }
      }
      if (begin + t + 1 == seq.kept) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(state + (32 * i + 4 * part + j) * kLinearDim) = s[i][j];
      }
    }
    __syncthreads();
    if (a.out != nullptr) {
      for (int t = warp; t < count; t += kStepThreads / 32) {
        const long long row = seq.row0 + begin + t;
        float4 o = *reinterpret_cast<const float4*>(&rows[t].v[4 * lane]);
        if (a.gate.data != nullptr) {
          const float4 z = load4(a.gate.data + row * a.gate.row_stride + head * a.gate.head_stride + 4 * lane);
          const float4 w = load4(a.norm_weight + 4 * lane);
          const float scale = __frsqrt_rn(fmaf(warp_sum(dot4(o, o)), 1.0f / kLinearDim, a.eps));
          o.x *= scale * w.x * linear_silu(z.x);
          o.y *= scale * w.y * linear_silu(z.y);
          o.z *= scale * w.z * linear_silu(z.z);
          o.w *= scale * w.w * linear_silu(z.w);
        }
        store4(a.out + (row * a.v_heads + head) * kLinearDim + 4 * lane, o);
      }
    }
    __syncthreads();
  }
}

}  // namespace

cudaError_t linear_step(const LinearDelta& a, int max_rows, cudaStream_t stream) {
  linear_step_kernel<<<dim3(a.v_heads, a.batch.sequences), kStepThreads, 0, stream>>>(a, max_rows);
  return cudaGetLastError();
}

}  // namespace aima
