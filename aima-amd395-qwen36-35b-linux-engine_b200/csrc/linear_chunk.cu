// The gated delta rule in chunks, second kernel: a sequence's chunks one after the other, a block per value head (formulas in
// linear_chunk.cuh).
//
// Everything is transposed: the value elements are the M side of all five products, one to a lane of tensor memory and to a thread of
// each warp group, so what a product leaves is scaled, split and handed to the next one by the thread that holds it.  A operands
// (state, right side, corrections) go through tensor memory, B operands (k, q, T, scores) lie in shared memory as the first kernel wrote
// them.  Per chunk:
//   R = S^T k, Q = S^T q    ->  right side beta v - enter R  ->  D = (right side) T^T
//   S <- decay S + (stay D) k,  O = D scores^T               ->  o = (read Q + O) / sqrt(128)
// Two warp groups have 32 tokens or 64 key elements each of that chain, a third the output, one warp issues products, one loads.
#include "linear_chunk.cuh"

#include <algorithm>

namespace aima {
namespace {

constexpr int kChainWarps = 8, kOutWarps = 4;
constexpr int kChunkThreads = 32 * (kChainWarps + kOutWarps + 4);          // four warp groups; the last one issues products and loads
// registers of a thread: 128 at launch, in all as many as there are
constexpr int kChainRegisters = 168, kOutRegisters = 136, kIssueRegisters = 40;
static_assert(2 * kChainRegisters + kOutRegisters + kIssueRegisters <= 4 * 128, "the warp groups share what the block was launched with");
constexpr int kStages = 2;
constexpr int kStageValues = kChunkPairBytes + kChunkHeadBytes;           // v: 64 rows of 256 bytes
constexpr int kStageBytes = (kStageValues + kChunk * kLinearDim * 2 + 1023) / 1024 * 1024;
constexpr int kOutRow = kLinearDim + 4;

// columns of tensor memory
constexpr uint32_t kStateAt = 0, kHighAt = 128, kLowAt = 192, kDotsAt = 256, kReadAt = 320, kEnterAt = 384, kFreshAt = 448;

struct __align__(1024) ChunkMemory {
  uint8_t stages[kStages][kStageBytes];
  float out[kChunk * kOutRow];
  float largest[2][kLinearDim];           // of a column of the state or of what comes, by warp group
  float scale[2][kLinearDim];             // the power of two of a column, by parity of the chunk
  int broken[2][kLinearDim];              // the first token of the chunk whose right side is not finite
  int sums[kChunkThreads / 32];
  unsigned long long full[kStages], empty[kStages];
  unsigned long long state_ready, dots_full, enter_ready, fresh_full, stay_ready, state_full, out_full, dots_empty;
  uint32_t tmem;
  int abort_flag;
};

__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* r) {
  tmem_ld32(taddr, reinterpret_cast<uint32_t*>(r));
  tmem_ld32(taddr + 32, reinterpret_cast<uint32_t*>(r) + 32);
}
__device__ __forceinline__ void chain_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void out_barrier() { asm volatile("bar.sync 2, 128;" ::: "memory"); }
// mbar_wait_bounded_warp without a call: the numbers that are alive across one would go to memory.
__device__ __forceinline__ bool wait_inline(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned long long limit_ns) {
  if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  const unsigned long long start = global_timer_ns();
  while (!__all_sync(0xffffffffu, mbar_test(bar, parity))) {
    if (__any_sync(0xffffffffu, *abort_flag != 0 || global_timer_ns() - start > limit_ns)) {
      *abort_flag = kStatusTimeoutMbarrier;
      return false;
    }
  }
  return true;
}
// a warp's word that what it stored to tensor memory, or loaded from it, is done
__device__ __forceinline__ void warp_arrive(unsigned long long* bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_u32(bar));
}

__global__ void __launch_bounds__(kChunkThreads, 1) linear_chunk_kernel(const ChunkPlan plan) {
  extern __shared__ uint8_t raw[];
  ChunkMemory& m = *reinterpret_cast<ChunkMemory*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const LinearDelta& a = plan.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x;
  const LinearSequence seq = linear_sequence(a.batch, blockIdx.y);
  if (seq.rows <= plan.min_rows) return;
  if (a.out != nullptr && !plan.kept_only) {          // rows that are not active
    for (int i = threadIdx.x; i < seq.first * (kLinearDim / 8); i += kChunkThreads)
      *reinterpret_cast<uint4*>(a.out + (static_cast<long long>(seq.row0 + i / (kLinearDim / 8)) * a.v_heads + head) * kLinearDim + 8 * (i % (kLinearDim / 8))) =
          make_uint4(0, 0, 0, 0);
  }
  const int limit = plan.kept_only ? seq.kept : seq.rows;                  // rows that are gone through
  const int chunks = (limit - seq.first + kChunk - 1) / kChunk;
  if (limit <= seq.first) return;

  // its first tile
  int tile0 = 0;
  {
    int mine = 0;
    for (int s = threadIdx.x; s < static_cast<int>(blockIdx.y); s += kChunkThreads) mine += chunks_of(linear_sequence(a.batch, s), plan.min_rows);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) m.sums[warp] = mine;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&m.full[i]), 1);
      mbar_init(smem_u32(&m.empty[i]), 1 + kChainWarps + kOutWarps);
    }
    mbar_init(smem_u32(&m.state_ready), kChainWarps);
    mbar_init(smem_u32(&m.dots_full), 1);
    mbar_init(smem_u32(&m.enter_ready), kChainWarps);
    mbar_init(smem_u32(&m.fresh_full), 1);
    mbar_init(smem_u32(&m.stay_ready), kChainWarps);
    mbar_init(smem_u32(&m.state_full), 1);
    mbar_init(smem_u32(&m.out_full), 1);
    mbar_init(smem_u32(&m.dots_empty), kOutWarps);
    m.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kChainWarps + kOutWarps) tmem_alloc(smem_u32(&m.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  for (int w = 0; w < kChunkThreads / 32; ++w) tile0 += m.sums[w];
  const uint32_t tmem = m.tmem;
  const bool fits = tile0 + chunks_of(seq, plan.min_rows) <= plan.tiles;       // not if sequences overlap, which the first kernel reports
  const int n = fits ? chunks : 0;
  if (!fits && threadIdx.x == 0) atomicOr(a.status, kLinearBadBatch);
  volatile int* abort_flag = &m.abort_flag;
  auto wait = [&](unsigned long long* bar, int phase) { return wait_inline(smem_u32(bar), phase & 1, abort_flag, plan.wait_limit_ns); };
  const long long row0 = static_cast<long long>(seq.row0) + seq.first;
  const int rows = limit - seq.first;                                          // of all chunks
  float* const state = a.states + (static_cast<long long>(seq.slot) * a.v_heads + head) * kLinearDim * kLinearDim;

  if (warp < kChainWarps) {
    // ------------------------------ the chain ------------------------------
    more_registers<kChainRegisters>();
    // No wait that runs out leaves this loop: the warps meet at barriers, and every wait after the first that ran out ends at once.
    const int group = warp >> 2, column = (warp & 3) * 32 + lane;              // a value element
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float s[64];                                                               // key elements 64 group ..
    float scale = 1.0f;
    if (seq.fresh || n == 0) {
#pragma unroll
      for (int i = 0; i < 64; ++i) s[i] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < 64; ++i) s[i] = state[(64 * group + i) * kLinearDim + column];
    }
    uint32_t v[16];                                                            // tokens 32 group .., two in a word
    for (int c = 0; c <= n; ++c) {
      const uint8_t* stage = m.stages[c % kStages];
      const ChunkNumbers& numbers = *reinterpret_cast<const ChunkNumbers*>(stage + kChunkPairBytes + kChunkNumbersAt);
      if (c < n) {
        wait(&m.full[c % kStages], c / kStages);
        const uint16_t* values = reinterpret_cast<const uint16_t*>(stage + kStageValues) + 32 * group * kLinearDim + column;
        const int there = rows - c * kChunk - 32 * group;
        if (there >= 32) {
#pragma unroll
          for (int t = 0; t < 32; t += 2) v[t / 2] = values[t * kLinearDim] | static_cast<uint32_t>(values[(t + 1) * kLinearDim]) << 16;
        } else {
#pragma unroll
          for (int t = 0; t < 32; t += 2) {
            const uint32_t v0 = t < there ? values[t * kLinearDim] : 0, v1 = t + 1 < there ? values[(t + 1) * kLinearDim] : 0;
            v[t / 2] = v0 | v1 << 16;
          }
        }
      }
      if (c > 0) {
        wait(&m.state_full, c - 1);
        tc_fence_after();
        tmem_ld64(lanes + kStateAt + 64 * group, s);
        tmem_ld_wait();
        if (m.broken[(c - 1) & 1][column] < kChunk) {
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] = NAN;
        }
      }
      if (c == n) break;
      // the column's power of two
      {
        uint32_t most = 0;
#pragma unroll
        for (int t = 0; t < 16; ++t) most = __vmaxu2(most, v[t] & 0x7fff7fffu);
        most = max(most & 0xffffu, most >> 16);
        if (most >= 0x7f80u) {                                                 // not of numbers that are not finite
          most = 0;
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            const uint32_t low = v[t] & 0x7fffu, high = (v[t] >> 16) & 0x7fffu;
            if (low < 0x7f80u) most = max(most, low);
            if (high < 0x7f80u) most = max(most, high);
          }
        }
        float largest = bf16_bits_to_float(static_cast<uint16_t>(most)) * scale;
#pragma unroll
        for (int i = 0; i < 64; i += 2) largest = max3_abs(largest, s[i], s[i + 1]);
        m.largest[group][column] = largest;
        if (group == 0) m.broken[c & 1][column] = kChunk;
        chain_barrier();
        largest = fmaxf(largest, m.largest[group ^ 1][column]);
        if ((largest > 512.0f || largest < 0.5f) && largest > 0.0f && largest < INFINITY) {
          const int now = kv_float_exponent(scale), next = min(max(now + 4 - kv_float_exponent(largest), -120), 100);
          const float up = kv_exp2(max(min(next - now, 126), -126));
          scale = kv_exp2(next);
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] *= up;
        }
        if (group == 0) m.scale[c & 1][column] = scale;
      }
      // the state in two terms, and decayed for the sum that follows
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t high[16], low[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) split_f16(s[32 * b + 2 * i], s[32 * b + 2 * i + 1], &high[i], &low[i]);
        tmem_st16(lanes + kHighAt + 32 * group + 16 * b, high);
        tmem_st16(lanes + kLowAt + 32 * group + 16 * b, low);
      }
      tmem_st_wait();
      warp_arrive(&m.state_ready, lane);
      {
        const float decay = plan.kept_only ? numbers.decay_kept : numbers.decay;
        // for a chunk that ends before its last row the numbers of the kept ones are those of all
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] *= decay;
        tmem_st32(lanes + kStateAt + 64 * group, reinterpret_cast<uint32_t*>(s));
        tmem_st32(lanes + kStateAt + 64 * group + 32, reinterpret_cast<uint32_t*>(s) + 32);
      }
      // the right side
      {
        float r[32];
        wait(&m.dots_full, c);
        tc_fence_after();
        tmem_ld32(lanes + kDotsAt + 32 * group, reinterpret_cast<uint32_t*>(r));
        tmem_ld_wait();
        const int there = rows - c * kChunk - 32 * group;
        float check = 0.0f;
#pragma unroll
        for (int t = 0; t < 32; ++t) {
          const float2 e = numbers.enter[32 * group + t];
          const float value = (t & 1) != 0 ? bf16_hi(v[t / 2]) : bf16_lo(v[t / 2]);
          r[t] = fmaf(-e.y, r[t], e.x * scale * value);
          if (plan.kept_only && t >= there) r[t] = 0.0f;                       // not a row that is gone through
          check = fmaf(r[t], 0.0f, check);
        }
        if (check != 0.0f) {
          int first = kChunk;
#pragma unroll
          for (int t = 31; t >= 0; --t) {
            if (!(fabsf(r[t]) < INFINITY)) {
              first = 32 * group + t;
              r[t] = 0.0f;
            }
          }
          atomicMin(&m.broken[c & 1][column], first);
        }
        uint32_t high[16], low[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) split_f16(r[2 * i], r[2 * i + 1], &high[i], &low[i]);
        tmem_st16(lanes + kEnterAt + 16 * group, high);
        tmem_st16(lanes + kEnterAt + 32 + 16 * group, low);
        tmem_st_wait();
        warp_arrive(&m.enter_ready, lane);
      }
      // the corrections
      {
        float d[32];
        wait(&m.fresh_full, c);
        tc_fence_after();
        tmem_ld32(lanes + kDotsAt + 32 * group, reinterpret_cast<uint32_t*>(d));
        tmem_ld_wait();
        uint32_t high[16], low[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) split_f16(d[2 * i], d[2 * i + 1], &high[i], &low[i]);
        tmem_st16(lanes + kFreshAt + 16 * group, high);
        tmem_st16(lanes + kFreshAt + 32 + 16 * group, low);
        const float* stay = plan.kept_only ? numbers.stay_kept : numbers.stay;
#pragma unroll
        for (int t = 0; t < 32; ++t) d[t] *= stay[32 * group + t];
#pragma unroll
        for (int i = 0; i < 16; ++i) split_f16(d[2 * i], d[2 * i + 1], &high[i], &low[i]);
        tmem_st16(lanes + kEnterAt + 16 * group, high);
        tmem_st16(lanes + kEnterAt + 32 + 16 * group, low);
        tmem_st_wait();
        warp_arrive(&m.stay_ready, lane);
        if (lane == 0) mbar_arrive(smem_u32(&m.empty[c % kStages]));
      }
    }
    if (n > 0 && plan.store && seq.kept > seq.first) {
      const float back = kv_exp2(-kv_float_exponent(scale));
#pragma unroll
      for (int i = 0; i < 64; ++i) state[(64 * group + i) * kLinearDim + column] = s[i] * back;
    }
  } else if (warp < kChainWarps + kOutWarps) {
    // ------------------------------ outputs ------------------------------
    more_registers<kOutRegisters>();
    const int w = warp - kChainWarps, column = w * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const bool outputs = a.out != nullptr && !plan.kept_only, gated = outputs && a.gate.data != nullptr;
    const int half = lane >> 4, piece = lane & 15;
    uint4 weights = make_uint4(0, 0, 0, 0);
    if (gated) weights = *reinterpret_cast<const uint4*>(a.norm_weight + 8 * piece);
    for (int c = 0; c < n; ++c) {
      const uint8_t* stage = m.stages[c % kStages];
      const ChunkNumbers& numbers = *reinterpret_cast<const ChunkNumbers*>(stage + kChunkPairBytes + kChunkNumbersAt);
      // the gate's rows come while the chunk is under way: 16 lanes a row, eight rows a thread
      const int there = min(kChunk, rows - c * kChunk);
      uint4 gate[8];
      if (gated) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = 8 * i + 2 * w + half;
          if (t < there) gate[i] = *reinterpret_cast<const uint4*>(a.gate.data + (row0 + c * kChunk + t) * a.gate.row_stride + head * a.gate.head_stride + 8 * piece);
        }
      }
      wait(&m.out_full, c);
      tc_fence_after();
      if (outputs) {
        const float back = kv_exp2(-kv_float_exponent(m.scale[c & 1][column])) * 0.08838834764831845f;
        const int broken = m.broken[c & 1][column];
        out_barrier();                                                         // the rows of the chunk before have been read
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float o[32], q[32];
          tmem_ld32(lanes + kDotsAt + 32 * h, reinterpret_cast<uint32_t*>(o));
          tmem_ld32(lanes + kReadAt + 32 * h, reinterpret_cast<uint32_t*>(q));
          tmem_ld_wait();
          if (h == 1) warp_arrive(&m.dots_empty, lane);
#pragma unroll
          for (int t = 0; t < 32; ++t) {
            const float x = fmaf(numbers.read[32 * h + t], q[t], o[t]) * back;
            m.out[(32 * h + t) * kOutRow + column] = 32 * h + t < broken ? x : NAN;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&m.empty[c % kStages]));
        out_barrier();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = 8 * i + 2 * w + half;
          float o[8];
          *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(&m.out[t * kOutRow + 8 * piece]);
          *reinterpret_cast<float4*>(o + 4) = *reinterpret_cast<const float4*>(&m.out[t * kOutRow + 8 * piece + 4]);
          if (gated) {
            float sum = 0.0f, z[8], weight[8];
            unpack8(weights, weight);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(o[j], o[j], sum);
#pragma unroll
            for (int d = 8; d >= 1; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const float factor = __frsqrt_rn(fmaf(sum, 1.0f / kLinearDim, a.eps));
            unpack8(gate[i], z);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] *= factor * weight[j] * (z[j] * linear_sigmoid(z[j]));
          }
          if (t < there)
            *reinterpret_cast<uint4*>(a.out + ((row0 + c * kChunk + t) * a.v_heads + head) * kLinearDim + 8 * piece) =
                make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        }
      } else {
        warp_arrive(&m.dots_empty, lane);
        if (lane == 0) mbar_arrive(smem_u32(&m.empty[c % kStages]));
      }
    }
  } else {
    fewer_registers<kIssueRegisters>();
    if (warp == kChainWarps + kOutWarps) {
      // ------------------------------ products ------------------------------
      // Products of different shapes need not run in the order of issue: one that reads or writes what another wrote waits for its commit.
      constexpr uint32_t kNarrow = instr_desc_f8(kF16, kF16, 0, 0, 128, kChunk);
      constexpr uint32_t kWide = instr_desc_f8(kF16, kF16, 0, 1, 128, kLinearDim);
      const uint32_t base = smem_u32(m.stages[0]);
      for (int c = 0; c < n; ++c) {
        const uint32_t pair = base + (c % kStages) * kStageBytes, inverse = pair + kChunkPairBytes, scores = inverse + 2 * kChunkMatrixBytes;
        if (!wait(&m.full[c % kStages], c / kStages) || !wait(&m.state_ready, c) || (c > 0 && !wait(&m.dots_empty, c - 1))) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int k = 0; k < kLinearDim / 16; ++k)
              umma_f16_ts(tmem + kDotsAt, tmem + (term == 0 ? kHighAt : kLowAt) + 8 * k,
                          smem_desc_rows<128>(pair + (k / 4) * kChunkPanelBytes) + ((k % 4) * 32 >> 4), kNarrow, (term | k) != 0);
          umma_commit(smem_u32(&m.dots_full));
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int k = 0; k < kLinearDim / 16; ++k)
              umma_f16_ts(tmem + kReadAt, tmem + (term == 0 ? kHighAt : kLowAt) + 8 * k,
                          smem_desc_rows<128>(pair + (k / 4) * kChunkPanelBytes + kChunk * 128) + ((k % 4) * 32 >> 4), kNarrow, (term | k) != 0);
        }
        __syncwarp();
        if (!wait(&m.enter_ready, c)) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int term = 0; term < 3; ++term)                                   // both terms by T's first, the first by T's second
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k)
              umma_f16_ts(tmem + kDotsAt, tmem + kEnterAt + (term == 1 ? 32 : 0) + 8 * k,
                          smem_desc_rows<128>(inverse + (term == 2 ? kChunkMatrixBytes : 0)) + (k * 32 >> 4), kNarrow, (term | k) != 0);
          umma_commit(smem_u32(&m.fresh_full));
        }
        __syncwarp();
        if (!wait(&m.stay_ready, c)) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k)
              umma_f16_ts(tmem + kStateAt, tmem + kEnterAt + 32 * term + 8 * k, smem_desc_rows<128>(pair + k * 16 * 128, kChunkPanelBytes), kWide, 1);
          umma_commit(smem_u32(&m.state_full));
#pragma unroll
          for (int term = 0; term < 3; ++term)
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k)
              umma_f16_ts(tmem + kDotsAt, tmem + kFreshAt + (term == 1 ? 32 : 0) + 8 * k,
                          smem_desc_rows<128>(scores + (term == 2 ? kChunkMatrixBytes : 0)) + (k * 32 >> 4), kNarrow, (term | k) != 0);
          umma_commit(smem_u32(&m.out_full));
          umma_commit(smem_u32(&m.empty[c % kStages]));
        }
        __syncwarp();
      }
    } else if (warp == kChainWarps + kOutWarps + 1) {
      // ------------------------------ loads ------------------------------
      int c = 0;
      for (; c < n; ++c) {
        const int slot = c % kStages;
        if (!wait(&m.empty[slot], c / kStages + 1)) break;
        const uint32_t to = smem_u32(m.stages[slot]), bar = smem_u32(&m.full[slot]);
        const int there = min(kChunk, rows - c * kChunk);
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, kStageValues + there * 2 * kLinearDim);
          const size_t tile = static_cast<size_t>(tile0 + c);
          bulk_g2s(to, plan.pairs + (tile * a.k_heads + head / a.group) * kChunkPairBytes, kChunkPairBytes, bar);
          bulk_g2s(to + kChunkPairBytes, plan.heads + (tile * a.v_heads + head) * kChunkHeadBytes, kChunkHeadBytes, bar);
        }
        __syncwarp();
        for (int t = lane; t < there; t += 32)
          bulk_g2s(to + kStageValues + t * 2 * kLinearDim, a.v.data + (row0 + c * kChunk + t) * a.v.row_stride + head * a.v.head_stride, 2 * kLinearDim, bar);
      }
      if (*abort_flag != 0) {                // what is in flight lands before the block leaves
        volatile int ignore = 0;
        for (int i = max(0, c - kStages); i < c; ++i) wait_inline(smem_u32(&m.full[i % kStages]), (i / kStages) & 1, &ignore, kWaitBudgetNs);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(a.status, kLinearTimeout);
  if (warp == kChainWarps + kOutWarps) tmem_dealloc(tmem, 512);
}

size_t tiles_of(int tokens, int sequences, int min_rows) {
  return static_cast<size_t>(tokens / kChunk) + std::min(sequences, tokens / (min_rows + 1));
}

}  // namespace

size_t linear_chunk_workspace(int k_heads, int v_heads, int max_tokens, int max_sequences) {
  const size_t tiles = std::max<size_t>(tiles_of(max_tokens, max_sequences, kLinearStepRows), tiles_of(max_tokens, 1, 0));
  return tiles * (static_cast<size_t>(k_heads) * kChunkPairBytes + static_cast<size_t>(v_heads) * kChunkHeadBytes);
}

cudaError_t linear_chunks(const LinearDelta& a, int min_rows, void* workspace, cudaStream_t stream) {
  ChunkPlan plan{};
  plan.a = a;
  plan.min_rows = min_rows;
  plan.tiles = static_cast<int>(tiles_of(a.batch.tokens, a.batch.sequences, min_rows));
  plan.pairs = static_cast<uint8_t*>(workspace);
  plan.heads = plan.pairs + static_cast<size_t>(plan.tiles) * a.k_heads * kChunkPairBytes;
  plan.wait_limit_ns = kWaitBudgetNs;
  cudaError_t error = linear_prepare(plan, stream);
  if (error != cudaSuccess) return error;
  constexpr int kBytes = static_cast<int>(sizeof(ChunkMemory)) + 1024;
  error = opt_in_dynamic_smem<linear_chunk_kernel>(kBytes);
  if (error != cudaSuccess) return error;
  const dim3 grid(a.v_heads, a.batch.sequences);
  // with rows that are computed but do not stay, once for the outputs and once for the states
  plan.kept_only = a.out == nullptr;
  plan.store = a.out == nullptr || a.batch.keep == nullptr;
  linear_chunk_kernel<<<grid, kChunkThreads, kBytes, stream>>>(plan);
  if (a.out != nullptr && a.batch.keep != nullptr) {
    plan.kept_only = plan.store = 1;
    linear_chunk_kernel<<<grid, kChunkThreads, kBytes, stream>>>(plan);
  }
  return cudaGetLastError();
}

}  // namespace aima
