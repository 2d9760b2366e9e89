// The gated delta rule token by token: the form for single tokens and drafts.
//
//   S <- e^g S;  d = beta (v - S^T k);  S <- S + k d^T;  o = S^T q
// Both products with the state are taken before it changes, from one pass over it: with r = S^T k and p = S^T q of the old state,
//   d = beta (v - e^g r),   o = e^g p + (k.q) d,   S <- e^g S + k d^T.
// The state is held divided by what it has decayed by so far, S / E, so that a token costs three products for an element instead of
// four: E <- e^g E, S / E <- S / E + k (d / E)^T.  Once E falls below 2^-16 the state takes it up, and with every token that a
// warp's columns have a product with the state or a correction above 2^80 for: S / E may then be beyond FP32 where S is not.  What stays divided
// grows by less than 28 * 2^96 so, which is no step of the largest numbers.
//
// A block takes one head of one sequence after the other: its state goes through registers once however many tokens there are.  A warp
// has 16 columns (value elements) of it and all 128 rows: four columns and 16 rows a lane, so the sums over the rows stay in the warp
// and warps need not wait for each other between tokens.  The next head's state is asked into L2 and its first tokens into registers
// while this one is gone through.
//
// One token is bytes: 64 sequences of 32 heads read and write 268 MB in 48.7 us (5.5 TB/s).  More tokens are the arithmetic and the waits
// of a token, 1600 cycles for two heads at a time on a multiprocessor: 16 tokens of each of those heads take 135 us, with four
// products for an element 143.
#include "linear.cuh"

#include <algorithm>

namespace aima {
namespace {

constexpr int kStepThreads = 256, kStepWarps = kStepThreads / 32;
constexpr int kStepRows = 8;             // tokens prepared at a time, a warp each
constexpr int kStepUnits = 1024;         // heads of a block: 1024 sequences of 256 heads on 296 blocks are 886
constexpr uint32_t kStateBytes = kLinearDim * kLinearDim * sizeof(float);

struct __align__(16) StepRow {
  float k[kLinearDim], q[kLinearDim];
  float v[kLinearDim];                   // then the token's output
  uint2 gate[32];
};
struct __align__(16) StepMemory {
  StepRow rows[kStepRows];
  float decay[kStepRows], rate[kStepRows], overlap[kStepRows];
  struct Unit {
    int head, slot;                      // slot: ~slot of a sequence that begins with zeros
    int row0, rows, kept;                // its rows, those that enter the state
  } units[kStepUnits];
  int counts[kStepWarps];
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
// x and its squares with eps, both times what makes them numbers that the norm can take
__device__ __forceinline__ void normable(float4* x, float* squares, float eps) {
  const float by = linear_norm_shift(*squares);
  if (by != 1.0f) {                        // the same for all lanes
    *x = scaled(*x, by);
    *squares = warp_sum(dot4(*x, *x)) + eps * by * by;
  }
}

__device__ __forceinline__ uint2 load_raw(const __nv_bfloat16* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ float4 widened(const uint2& raw) { return make_float4(bf16_lo(raw.x), bf16_hi(raw.x), bf16_lo(raw.y), bf16_hi(raw.y)); }

// A token as it lies in memory, four elements a lane.
struct StepToken {
  uint2 k, q, v, gate;
  __nv_bfloat16 a, b;
};

__global__ void __launch_bounds__(kStepThreads, 2) linear_step_kernel(const LinearDelta a, int max_rows) {
  __shared__ StepMemory m;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // this block's heads that have rows; a thread looks at one, and gives its inactive rows their zeros
  const int all = a.v_heads * a.batch.sequences;
  int units = 0;
  for (int base = blockIdx.x; base < all; base += static_cast<int>(gridDim.x) * kStepThreads) {
    const int unit = base + static_cast<int>(threadIdx.x * gridDim.x);
    bool is = false;
    StepMemory::Unit mine{};
    if (unit < all) {
      const LinearSequence seq = linear_sequence(a.batch, unit / a.v_heads);
      // rows that have to be gone through: the active ones, without outputs only those that stay
      const int head = unit % a.v_heads, end = a.out != nullptr ? seq.rows : min(seq.rows, seq.kept);
      mine = StepMemory::Unit{head, seq.fresh ? ~seq.slot : seq.slot, seq.row0 + seq.first, end - seq.first, seq.kept - seq.first};
      if (seq.bad && head == 0) atomicOr(a.status, kLinearBadBatch);
      is = seq.rows <= max_rows && seq.first < end;
      if (a.out != nullptr && seq.rows <= max_rows) {
        for (int i = 0; i < min(seq.first, end) * (kLinearDim / 8); ++i)
          *reinterpret_cast<uint4*>(a.out + (static_cast<long long>(seq.row0 + i / (kLinearDim / 8)) * a.v_heads + head) * kLinearDim + 8 * (i % (kLinearDim / 8))) =
              make_uint4(0, 0, 0, 0);
      }
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, is);
    if (lane == 0) m.counts[warp] = __popc(votes);
    __syncthreads();
    int at = units + __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < kStepWarps; ++w) {
      if (w < warp) at += m.counts[w];
      units += m.counts[w];
    }
    if (is) m.units[at] = mine;
    __syncthreads();
  }
  if (units == 0) return;

  const auto state_of = [&](const StepMemory::Unit& u) {
    return a.states + (static_cast<long long>(u.slot < 0 ? ~u.slot : u.slot) * a.v_heads + u.head) * kLinearDim * kLinearDim;
  };
  const auto fetch_token = [&](const StepMemory::Unit& u, int row, StepToken* token) {
    const int k_head = u.head / a.group;
    const long long at = u.row0 + row;
    token->k = load_raw(a.k.data + at * a.k.row_stride + k_head * a.k.head_stride + 4 * lane);
    token->q = load_raw(a.q.data + at * a.q.row_stride + k_head * a.q.head_stride + 4 * lane);
    token->v = load_raw(a.v.data + at * a.v.row_stride + u.head * a.v.head_stride + 4 * lane);
    if (a.gate.data != nullptr && a.out != nullptr) token->gate = load_raw(a.gate.data + at * a.gate.row_stride + u.head * a.gate.head_stride + 4 * lane);
    token->a = a.a[at * a.a_stride + u.head];
    token->b = a.b[at * a.b_stride + u.head];
  };
  StepToken token{};
  if (warp < m.units[0].rows) fetch_token(m.units[0], warp, &token);
  const int part = lane >> 2, column = 16 * warp + 4 * (lane & 3);           // rows 32 i + 4 part + j, columns column .. column + 3
  for (int i = 0; i < units; ++i) {
    const StepMemory::Unit& u = m.units[i];
    Pair s[4][2][4];                     // of two rows, four columns; times `scale`
    float scale = 1.0f;
    {
      const float* state = state_of(u) + column;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4* from = reinterpret_cast<const float4*>(state + (32 * r + 4 * part + 2 * j) * kLinearDim);
          const float4 x = u.slot < 0 ? make_float4(0, 0, 0, 0) : from[0], y = u.slot < 0 ? make_float4(0, 0, 0, 0) : from[kLinearDim / 4];
          s[r][j][0] = Pair(x.x, y.x);
          s[r][j][1] = Pair(x.y, y.y);
          s[r][j][2] = Pair(x.z, y.z);
          s[r][j][3] = Pair(x.w, y.w);
        }
    }
    if (threadIdx.x == 0 && i + 1 < units && m.units[i + 1].slot >= 0) prefetch_l2(state_of(m.units[i + 1]), kStateBytes);
    for (int begin = 0; begin < u.rows; begin += kStepRows) {
      const int count = min(kStepRows, u.rows - begin);
      if (warp < count) {
        float4 k = widened(token.k), q = widened(token.q);
        float kk = warp_sum(dot4(k, k)) + a.eps, qq = warp_sum(dot4(q, q)) + a.eps;
        if (!(fmaxf(kk, qq) < INFINITY && fminf(kk, qq) >= 0x1p-100f)) {
          normable(&k, &kk, a.eps);
          normable(&q, &qq, a.eps);
        }
        const float4 ku = scaled(k, __frsqrt_rn(kk));
        const float4 qu = scaled(q, __frsqrt_rn(qq) * 0.08838834764831845f);
        const float kq = warp_sum(dot4(ku, qu));
        StepRow& row = m.rows[warp];
        *reinterpret_cast<float4*>(&row.k[4 * lane]) = ku;
        *reinterpret_cast<float4*>(&row.q[4 * lane]) = qu;
        *reinterpret_cast<float4*>(&row.v[4 * lane]) = widened(token.v);
        row.gate[lane] = token.gate;
        if (lane == 0) {
          const float x = __bfloat162float(token.a) + a.dt_bias[u.head];
          m.decay[warp] = expf(-expf(a.a_log[u.head]) * (x > 20.0f ? x : log1pf(expf(x))));
          m.rate[warp] = 1.0f / (1.0f + expf(-__bfloat162float(token.b)));
          m.overlap[warp] = kq;
        }
      }
      __syncthreads();
      // the next tokens, or the first ones of the next head, while these are gone through
      if (begin + kStepRows < u.rows) {
        if (begin + kStepRows + warp < u.rows) fetch_token(u, begin + kStepRows + warp, &token);
      } else if (i + 1 < units && warp < m.units[i + 1].rows) {
        fetch_token(m.units[i + 1], warp, &token);
      }
      for (int t = 0; t < count; ++t) {
        Pair dots[8];                      // S^T k, then S^T q, for four columns: over even rows, over odd ones
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 k4 = *reinterpret_cast<const float4*>(&m.rows[t].k[32 * r + 4 * part]);
          const float4 q4 = *reinterpret_cast<const float4*>(&m.rows[t].q[32 * r + 4 * part]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const Pair k2 = j == 0 ? Pair(k4.x, k4.y) : Pair(k4.z, k4.w), q2 = j == 0 ? Pair(q4.x, q4.y) : Pair(q4.z, q4.w);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              dots[c] = r + j == 0 ? s[r][j][c] * k2 : fma2(s[r][j][c], k2, dots[c]);
              dots[4 + c] = r + j == 0 ? s[r][j][c] * q2 : fma2(s[r][j][c], q2, dots[4 + c]);
            }
          }
        }
        float sums[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float2 x = dots[c].values();
          sums[c] = x.x + x.y;
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
        const float e = scale * m.decay[t];
        const int mine = column + (part & 3);                              // the column whose total this lane has
        float d = m.rate[t] * (m.rows[t].v[mine] - e * total);             // of use in parts 0 .. 3
        const bool large = __any_sync(0xffffffffu, fmaxf(fabsf(d), fabsf(total)) > 0x1p80f);
        d = __shfl_sync(0xffffffffu, d, lane & 15);
        if (part >= 4) m.rows[t].v[mine] = fmaf(m.overlap[t], d, e * total);   // its value element has been read: by lanes that the shuffle waited for
        const float d0 = __shfl_sync(0xffffffffu, d, lane & 3), d1 = __shfl_sync(0xffffffffu, d, (lane & 3) | 4);
        const float d2 = __shfl_sync(0xffffffffu, d, (lane & 3) | 8), d3 = __shfl_sync(0xffffffffu, d, (lane & 3) | 12);
        scale = e;
        if (e < 0x1p-16f || large) {
#pragma unroll
          for (int i = 0; i < 32; ++i) (&s[0][0][0])[i] = (&s[0][0][0])[i] * Pair(e, e);
          scale = 1.0f;
        }
        const float back = 1.0f / scale;
        const Pair add[4] = {Pair(d0 * back, d0 * back), Pair(d1 * back, d1 * back), Pair(d2 * back, d2 * back), Pair(d3 * back, d3 * back)};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float4 k4 = *reinterpret_cast<const float4*>(&m.rows[t].k[32 * r + 4 * part]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const Pair k2 = j == 0 ? Pair(k4.x, k4.y) : Pair(k4.z, k4.w);
#pragma unroll
            for (int c = 0; c < 4; ++c) s[r][j][c] = fma2(k2, add[c], s[r][j][c]);
          }
        }
        if (begin + t + 1 == u.kept) {
          float* state = state_of(u) + column;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float4* to = reinterpret_cast<float4*>(state + (32 * r + 4 * part + 2 * j) * kLinearDim);
              const Pair by(scale, scale);
              const float2 x = (s[r][j][0] * by).values(), y = (s[r][j][1] * by).values(), z = (s[r][j][2] * by).values(), w = (s[r][j][3] * by).values();
              to[0] = make_float4(x.x, y.x, z.x, w.x);
              to[kLinearDim / 4] = make_float4(x.y, y.y, z.y, w.y);
            }
        }
      }
      __syncthreads();
      if (a.out != nullptr && warp < count) {
        const long long row = u.row0 + begin + warp;
        float4 o = *reinterpret_cast<const float4*>(&m.rows[warp].v[4 * lane]);
        if (a.gate.data != nullptr) {
          const float4 z = widened(m.rows[warp].gate[lane]);
          const float4 w = load4(a.norm_weight + 4 * lane);
          float square = fmaf(warp_sum(dot4(o, o)), 1.0f / kLinearDim, a.eps);
          if (!linear_norm_holds(square)) {
            const float by = linear_norm_shift(square);
            o = scaled(o, by);
            square = fmaf(warp_sum(dot4(o, o)), 1.0f / kLinearDim, a.eps * by * by);
          }
          const float scale = __frsqrt_rn(square);
          o.x *= scale * w.x * linear_silu(z.x);
          o.y *= scale * w.y * linear_silu(z.y);
          o.z *= scale * w.z * linear_silu(z.z);
          o.w *= scale * w.w * linear_silu(z.w);
        }
        store4(a.out + (row * a.v_heads + u.head) * kLinearDim + 4 * lane, o);
      }
      __syncwarp();                       // a warp's row is its own until the next tokens are prepared
    }
  }
}

}  // namespace

cudaError_t linear_step(const LinearDelta& a, int max_rows, int sm_count, cudaStream_t stream) {
  // Two blocks a multiprocessor, and more only where a block could not list its heads.  us so / with a block for each head, captured, 32
  // heads: 64 sequences 46.6 / 54.1, 256 sequences 167 / 200, 16 sequences of 5 tokens 17.3 / 18.4, 32 sequences 23.0 / 23.8.
  const int units = a.v_heads * a.batch.sequences, blocks = std::max(std::min(units, 2 * sm_count), (units + kStepUnits - 1) / kStepUnits);
  linear_step_kernel<<<blocks, kStepThreads, 0, stream>>>(a, max_rows);
  return cudaGetLastError();
}

}  // namespace aima
