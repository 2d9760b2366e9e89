// The gated delta rule in chunks, first kernel: what a chunk needs that does not depend on the state (formulas in linear_chunk.cuh).
//
// A block takes a chunk and a key head.  k and q are scaled by a power of two per row to f16; one product of [k; q] with k gives k.k
// and q.k of all pairs of tokens, exactly but for the order of the sums.  Then, for every value head of that key head: sums of g
// (64 bits, kept as two FP32 numbers, so that differences of large sums keep theirs), decays, the scores, and the inverse of the unit
// lower triangle 1 + A by blocks of 16: the diagonal's by substitution, those below from T_ij = -T_ii sum_k A_ik T_kj.
#include "linear_chunk.cuh"

namespace aima {
namespace {

constexpr int kPrepareThreads = 256;
constexpr int kHeadsAtOnce = 8;                 // a warp each for their sums
constexpr int kRow = kChunk + 4;                // of a matrix in shared memory

struct __align__(1024) PrepareMemory {
  uint8_t pair[kChunkPairBytes];
  float overlap[kChunk * kRow];                 // A
  float inverse[kChunk * kRow];                 // T
  float partial[3 * 16 * 20];                   // of three blocks
  float length[2 * kChunk];                     // 1 / |k|, then 1 / |q|, of the scaled rows
  int broken[2 * kChunk];                       // rows that are not finite
  float sum_high[kHeadsAtOnce][kChunk], sum_low[kHeadsAtOnce][kChunk];         // log2(e) G
  float rate[kHeadsAtOnce][kChunk];             // beta, 0 for a row that is not finite
  unsigned long long done;
  uint32_t tmem;
  int abort_flag;
};

__device__ __forceinline__ float quarter_max(float v) {          // over 16 lanes
#pragma unroll
  for (int d = 8; d >= 1; d /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float quarter_sum(float v) {
#pragma unroll
  for (int d = 8; d >= 1; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__global__ void __launch_bounds__(kPrepareThreads) linear_prepare_kernel(const ChunkPlan plan) {
  extern __shared__ uint8_t raw[];
  PrepareMemory& m = *reinterpret_cast<PrepareMemory*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const LinearDelta& a = plan.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k_head = blockIdx.x, tile = blockIdx.y;
  if (tile == 0 && k_head == 0) linear_report(a.batch, a.status, threadIdx.x, kPrepareThreads);

  // the sequence and chunk of this tile
  __shared__ int found[2];
  __shared__ int sums[kPrepareThreads / 32];
  {
    const int share = (a.batch.sequences + kPrepareThreads - 1) / kPrepareThreads;
    const int first = threadIdx.x * share, last = min(first + share, a.batch.sequences);
    int mine = 0;
    for (int s = first; s < last; ++s) mine += chunks_of(linear_sequence(a.batch, s), plan.min_rows);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    if (threadIdx.x == 0) {
      found[0] = -1;
      m.abort_flag = 0;
      mbar_init(smem_u32(&m.done), 1);
      mbar_fence_init();
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += sums[w];
    int at = upto - mine;
    if (at <= tile && tile < upto) {
      for (int s = first; s < last; ++s) {
        const int chunks = chunks_of(linear_sequence(a.batch, s), plan.min_rows);
        if (tile < at + chunks) {
          found[0] = s;
          found[1] = tile - at;
          break;
        }
        at += chunks;
      }
    }
    __syncthreads();
  }
  if (found[0] < 0) return;
  const LinearSequence seq = linear_sequence(a.batch, found[0]);
  const int begin = seq.first + found[1] * kChunk;
  const int rows = min(kChunk, seq.rows - begin);
  const int kept = min(max(seq.kept - begin, 0), rows);
  const long long row0 = seq.row0 + begin;
  if (warp == 0) tmem_alloc(smem_u32(&m.tmem), 64);

  // k's rows, then q's: 16 lanes a row, eight rows a thread
  uint8_t* pair = plan.pairs + (static_cast<size_t>(tile) * a.k_heads + k_head) * kChunkPairBytes;
  {
    const int piece = lane & 15, half = lane >> 4;
    uint4 data[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 16 * i + 2 * warp + half, t = r & (kChunk - 1);
      const KvRows& from = r < kChunk ? a.k : a.q;
      data[i] = t < rows ? *reinterpret_cast<const uint4*>(from.data + (row0 + t) * from.row_stride + k_head * from.head_stride + 8 * piece) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 16 * i + 2 * warp + half;
      float x[8];
      unpack8(data[i], x);
      float largest = 0.0f;
      bool finite = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        largest = fmaxf(largest, fabsf(x[j]));
        finite = finite && fabsf(x[j]) < INFINITY;
      }
      largest = quarter_max(finite ? largest : INFINITY);
      const bool broken = !(largest < INFINITY);
      // 2^-e with 2^e <= max < 2^(e + 1); a row of zeros, subnormal or broken: e as near as may be
      const int e = broken ? 0 : min(max(kv_float_exponent(largest), -126), 126);
      const float scale = kv_exp2(-e);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = broken ? 0.0f : x[j] * scale;
        sum = fmaf(x[j], x[j], sum);
      }
      sum = quarter_sum(sum);
      if (piece == 0) {
        // 2^e / sqrt(|x|^2 + eps) from |x 2^-e|^2; 2^-2e in two steps
        m.length[r] = broken ? 0.0f : 1.0f / sqrtf(sum + a.eps * scale * scale);
        m.broken[r] = broken;
      }
      const uint4 packed = make_uint4(cvt_f16x2(x[0], x[1]), cvt_f16x2(x[2], x[3]), cvt_f16x2(x[4], x[5]), cvt_f16x2(x[6], x[7]));
      const uint32_t at = (piece >> 3) * kChunkPanelBytes + swizzled(r, piece & 7);
      *reinterpret_cast<uint4*>(m.pair + at) = packed;
      *reinterpret_cast<uint4*>(pair + at) = packed;
    }
  }
  fence_async_proxy();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m.tmem;
  if (warp == 0) {
    if (elect_one()) {
      constexpr uint32_t kForm = instr_desc_f8(kF16, kF16, 0, 0, 128, kChunk);
      const uint32_t base = smem_u32(m.pair);
#pragma unroll
      for (int k = 0; k < kLinearDim / 16; ++k) {
        const uint64_t desc = smem_desc_rows<128>(base + (k / 4) * kChunkPanelBytes) + ((k % 4) * 32 >> 4);
        umma_f16_ss(tmem, desc, desc, kForm, k != 0);
      }
      umma_commit(smem_u32(&m.done));
    }
    __syncwarp();
  }

  const int half = warp >> 2, row = (warp & 3) * 32 + lane;         // row of [k; q], columns 32 half ..
  float dots[32];
  bool alive = true;
  for (int base = 0; base < a.group; base += kHeadsAtOnce) {
    const int heads = min(kHeadsAtOnce, a.group - base);
    if (warp < heads) {
      const int head = k_head * a.group + base + warp;
      ChunkNumbers* numbers = reinterpret_cast<ChunkNumbers*>(plan.heads + (static_cast<size_t>(tile) * a.v_heads + head) * kChunkHeadBytes + kChunkNumbersAt);
      float g[2], beta[2];
      bool broken[2];
      const float slope = expf(a.a_log[head]) * 1.44269504088896341f, bias = a.dt_bias[head];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        g[i] = beta[i] = 0.0f;
        broken[i] = false;
        if (t < rows) {
          const float x = __bfloat162float(a.a[(row0 + t) * a.a_stride + head]) + bias;
          g[i] = -slope * (x > 20.0f ? x : log1pf(expf(x)));
          beta[i] = 1.0f / (1.0f + expf(-__bfloat162float(a.b[(row0 + t) * a.b_stride + head])));
          broken[i] = m.broken[t] != 0 || g[i] != g[i] || beta[i] != beta[i];
          if (broken[i]) g[i] = beta[i] = 0.0f;
          g[i] = fmaxf(g[i], -1.0e6f);                   // e^g is 0 long before
        }
      }
      double upto = static_cast<double>(g[0]) + g[1];
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const double x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
      const double total[2] = {upto - g[1], upto};
      const double last = __shfl_sync(0xffffffffu, upto, 31);          // rows behind the last have g = 0
      const double last_kept_pair0 = __shfl_sync(0xffffffffu, total[0], max(kept - 1, 0) >> 1), last_kept_pair1 = __shfl_sync(0xffffffffu, total[1], max(kept - 1, 0) >> 1);
      const double last_kept = kept == 0 ? 0.0 : ((kept - 1) & 1) != 0 ? last_kept_pair1 : last_kept_pair0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        const float high = static_cast<float>(total[i]);
        m.sum_high[warp][t] = high;
        m.sum_low[warp][t] = static_cast<float>(total[i] - high);
        m.rate[warp][t] = beta[i];
        const float k_length = m.length[t], q_length = m.length[kChunk + t], reach = exp2f(high);
        const bool there = t < rows;
        numbers->rate[t] = beta[i];
        numbers->enter[t] = broken[i] ? NAN : there ? -(beta[i] * reach * k_length) : 0.0f;
        numbers->stay[t] = there ? exp2f(static_cast<float>(last - total[i])) * k_length : 0.0f;
        numbers->read[t] = !there ? 0.0f : m.broken[kChunk + t] != 0 ? NAN : reach * q_length;
        numbers->stay_kept[t] = t < kept ? exp2f(static_cast<float>(last_kept - total[i])) * k_length : 0.0f;
      }
      if (lane == 0) {
        numbers->decay = exp2f(static_cast<float>(last));
        numbers->decay_kept = exp2f(static_cast<float>(last_kept));
      }
    }
    if (base == 0) {
      alive = mbar_wait_bounded_warp(smem_u32(&m.done), 0, &m.abort_flag, plan.wait_limit_ns);
      tc_fence_after();
      tmem_ld32(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 32 * half, reinterpret_cast<uint32_t*>(dots));
      tmem_ld_wait();
    }
    __syncthreads();
    for (int h = 0; h < heads; ++h) {
      const int head = k_head * a.group + base + h;
      uint8_t* out = plan.heads + (static_cast<size_t>(tile) * a.v_heads + head) * kChunkHeadBytes;
      // A, and the scores
      {
        const int t = row & (kChunk - 1);
        const bool is_k = row < kChunk;
        const float high = m.sum_high[h][t], low = m.sum_low[h][t];
        const float factor = is_k ? m.rate[h][t] * m.length[t] : m.length[row];
        float x[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int c = 32 * half + j;
          const float apart = fminf((high - m.sum_high[h][c]) + (low - m.sum_low[h][c]), 0.0f);          // above 0 only where nothing is taken
          x[j] = (is_k ? c < t : c <= t) ? factor * m.length[c] * dots[j] * fast_exp2(apart) : 0.0f;
        }
        if (is_k) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(&m.overlap[t * kRow + 32 * half + j]) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_f16(x[j + 2 * i], x[j + 2 * i + 1], &hi[i], &lo[i]);
            const uint32_t at = 2 * kChunkMatrixBytes + swizzled(t, (32 * half + j) / 8);
            *reinterpret_cast<uint4*>(out + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(out + kChunkMatrixBytes + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      }
      __syncthreads();
      // the diagonal's blocks: a column a thread; zeros above them
      if (threadIdx.x < 64) {
        const int b = threadIdx.x >> 4, j = threadIdx.x & 15;
        const float* at = &m.overlap[16 * b * kRow + 16 * b];
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float sum = i == j ? 1.0f : 0.0f;
#pragma unroll
          for (int k = 0; k < i; ++k) sum = fmaf(-at[i * kRow + k], x[k], sum);
          x[i] = sum;
          m.inverse[(16 * b + i) * kRow + 16 * b + j] = sum;
        }
      }
      __syncthreads();
      // block diagonals below: thread = block, row, four columns
      const int b = threadIdx.x >> 6, i = (threadIdx.x >> 2) & 15, q = 4 * (threadIdx.x & 3);
#pragma unroll
      for (int d = 1; d < 4; ++d) {
        const bool mine = b < 4 - d;
        const int bi = b + d, bj = b;
        float4 sum = make_float4(0, 0, 0, 0);
        if (mine) {
          for (int k = 16 * bj; k < 16 * bi; ++k) {
            const float w = m.overlap[(16 * bi + i) * kRow + k];
            const float4 y = *reinterpret_cast<const float4*>(&m.inverse[k * kRow + 16 * bj + q]);
            sum.x = fmaf(w, y.x, sum.x);
            sum.y = fmaf(w, y.y, sum.y);
            sum.z = fmaf(w, y.z, sum.z);
            sum.w = fmaf(w, y.w, sum.w);
          }
          *reinterpret_cast<float4*>(&m.partial[(b * 16 + i) * 20 + q]) = sum;
        }
        __syncthreads();
        if (mine) {
          sum = make_float4(0, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float w = m.inverse[(16 * bi + i) * kRow + 16 * bi + k];
            const float4 y = *reinterpret_cast<const float4*>(&m.partial[(b * 16 + k) * 20 + q]);
            sum.x = fmaf(-w, y.x, sum.x);
            sum.y = fmaf(-w, y.y, sum.y);
            sum.z = fmaf(-w, y.z, sum.z);
            sum.w = fmaf(-w, y.w, sum.w);
          }
          *reinterpret_cast<float4*>(&m.inverse[(16 * bi + i) * kRow + 16 * bj + q]) = sum;
        }
        __syncthreads();
      }
      // in two terms: row i, sixteen columns a thread
      {
        const int r = threadIdx.x >> 2, c = 16 * (threadIdx.x & 3);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int column = c + 8 * p + 2 * j;
            const float2 x = column / 16 <= r / 16 ? *reinterpret_cast<const float2*>(&m.inverse[r * kRow + column]) : make_float2(0.0f, 0.0f);
            split_f16(x.x, x.y, &hi[j], &lo[j]);
          }
          const uint32_t at = swizzled(r, (c + 8 * p) / 8);
          *reinterpret_cast<uint4*>(out + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(out + kChunkMatrixBytes + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      __syncthreads();
    }
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  if (!alive && lane == 0) atomicOr(a.status, kLinearTimeout);
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 64);
  }
}

}  // namespace

cudaError_t linear_prepare(const ChunkPlan& plan, cudaStream_t stream) {
  constexpr int kBytes = static_cast<int>(sizeof(PrepareMemory)) + 1024;
  const cudaError_t error = opt_in_dynamic_smem<linear_prepare_kernel>(kBytes);
  if (error != cudaSuccess) return error;
  linear_prepare_kernel<<<dim3(plan.a.k_heads, plan.tiles), kPrepareThreads, kBytes, stream>>>(plan);
  return cudaGetLastError();
}

}  // namespace aima
