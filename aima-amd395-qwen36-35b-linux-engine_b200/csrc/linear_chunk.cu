// The gated delta rule in chunks, second kernel: a sequence's chunks one after the other, a block per value head (formulas in
// linear_chunk.cuh).
//
// Everything is transposed: the value elements are the M side of all five products, one to a lane of tensor memory and to a thread of
// each warp group, so what a product leaves is scaled, split and handed to the next one by the thread that holds it.  A operands
// (state, right side, corrections) go through tensor memory, B operands (k, q, T, scores) lie in shared memory as the first kernel wrote
// them.  Per chunk:
//   R = S^T k, Q = S^T q    ->  right side beta v - enter R  ->  D = (right side) T^T
//   S <- decay S + (stay D) k,  O = D scores^T               ->  o = (read Q + O) / sqrt(128)
// Four warp groups have 16 tokens or 32 key elements each of that chain.  What does not depend on the chain is put where it waits for a
// product: the outputs of the chunk before are taken from tensor memory and turned into rows while R runs, and normed and written while D
// and S run; warps of their own for that cannot keep up, there being room for three beside the one that issues products.  One warp issues products, three load.  T and the
// scores are triangles, whose products begin with the row that is not zero.
//
// The chain bounds it: three products that wait for one another, with loads, splits and stores of all 16 warps in between.  A chunk
// takes 6000 cycles without outputs, 7900 with them and 9750 with the gate; its products alone take 1300 and 2000.  8192 tokens of 32
// heads with gate, from the end of one launch to the next: first kernel 84 us, first pass 100, join 12, second pass 198.
//
// Few heads leave multiprocessors idle, so a sequence's chunks are cut into segments then.  What a segment does to the state is
// S <- M S + B: a first pass finds the state behind the first segment, and M (values of zero, the identity as state) and B (a state of
// zeros) of those between the first and the last; the states at all borders follow from them, and a second pass goes through all segments
// at once.  The first pass has no outputs and takes 0.6 of the time of the second.  The first segment has no part in the products of M
// and B, so a multiprocessor that goes through two of half the length is done when the others are: it may be shorter.
#include "linear_chunk.cuh"

#include <algorithm>
#include <cuda_fp16.h>

namespace aima {
namespace {

constexpr int kGroups = 4, kChainWarps = 4 * kGroups;                      // groups of four warps, one for each 32 lanes of tensor memory
constexpr int kChunkThreads = 32 * (kChainWarps + 4);
constexpr int kTokens = kChunk / kGroups, kKeys = kLinearDim / kGroups;    // of a group
constexpr int kTokenSteps = kTokens / 16;                                  // of products over tokens, by when their operands come
constexpr int kStages = 2;
constexpr int kStageValues = kChunkPairBytes + kChunkHeadBytes;           // v: 64 rows of 256 bytes, zeros behind the last
constexpr int kStageBytes = (kStageValues + kChunk * kLinearDim * 2 + 1023) / 1024 * 1024;
constexpr int kOutRow = kLinearDim + 4;
constexpr int kOutRows = 2 * kChainWarps, kOutPasses = kChunk / kOutRows;   // rows that the groups write at a time, 16 lanes a row

// Columns of tensor memory.  Operands lie as eight columns of first and eight of second terms for every 16 elements of K: what a warp
// splits at a time and a step of a product takes.  O is left where the corrections of the state were.
constexpr uint32_t kStateAt = 0, kTermsAt = 128, kFreshAt = 256, kDotsAt = 320, kReadAt = 384, kEnterAt = 448;
__device__ __forceinline__ constexpr uint32_t operand(int k, int term) { return 16 * k + 8 * term; }

struct __align__(1024) ChunkMemory {
  uint8_t stages[kStages][kStageBytes];
  float out[kChunk * kOutRow];
  float largest[kGroups][kLinearDim];     // of a column of the state, by warp group
  float largest_value[kStages][2][kLinearDim];   // of a column of v, by the warp that brought the rows; not of numbers that are not finite
  float scale[2][kLinearDim];             // the power of two of a column, by parity of the chunk
  int broken[2][kLinearDim];              // the first token of the chunk whose right side is not finite
  float read[2][kChunk];                  // of ChunkNumbers, for when its stage is gone
  float weight[kLinearDim];               // a quarter of the norm's
  int sums[kChunkThreads / 32];
  unsigned long long full[kStages], empty[kStages], values_full[kStages];
  unsigned long long state_ready[2], dots_full, enter_ready[kTokenSteps], fresh_full, stay_ready[kTokenSteps], state_full, fresh_ready, out_full, out_taken;
  uint32_t tmem;
  int abort_flag;
};

// The launches of a call may begin before the one before them has ended: each waits here for its results, on every way out.
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_barrier() { asm volatile("bar.sync 1, %0;" :: "n"(32 * kChainWarps) : "memory"); }
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

// What is at a head's `borders`: the states before the segments, then B and M of those between the first and the last.
__device__ __forceinline__ float* border(const ChunkPlan& plan, int sequence, int head, int which) {
  return plan.borders + ((static_cast<size_t>(sequence) * plan.a.v_heads + head) * kMaxBorders + which) * kLinearDim * kLinearDim;
}
__device__ __forceinline__ int border_b(int segment) { return kMaxSegments + 2 * segment; }
__device__ __forceinline__ int border_m(int segment) { return kMaxSegments + 2 * segment + 1; }

// kOutput: all rows of a segment, the state behind the last if plan.store says so.  kKept: the states alone, for the rows that enter them.
// kTransfer: the first pass over segments.
enum ChunkMode { kOutput, kKept, kTransfer };
template <ChunkMode kMode>
__global__ void __launch_bounds__(kChunkThreads, 1) linear_chunk_kernel(const ChunkPlan plan) {
  constexpr bool kOutputs = kMode == kOutput;
  extern __shared__ uint8_t raw[];
  ChunkMemory& m = *reinterpret_cast<ChunkMemory*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const LinearDelta& a = plan.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x;
  launch_may_follow();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&m.full[i]), 1);
      mbar_init(smem_u32(&m.empty[i]), 1 + kChainWarps);
      mbar_init(smem_u32(&m.values_full[i]), 2);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&m.state_ready[i]), kChainWarps);
    for (int i = 0; i < kTokenSteps; ++i) {
      mbar_init(smem_u32(&m.enter_ready[i]), kChainWarps);
      mbar_init(smem_u32(&m.stay_ready[i]), kChainWarps);
    }
    mbar_init(smem_u32(&m.dots_full), 1);
    mbar_init(smem_u32(&m.fresh_full), 1);
    mbar_init(smem_u32(&m.state_full), 1);
    mbar_init(smem_u32(&m.fresh_ready), kChainWarps);
    mbar_init(smem_u32(&m.out_full), 1);
    mbar_init(smem_u32(&m.out_taken), kChainWarps);
    m.abort_flag = 0;
    mbar_fence_init();
  }
  const LinearSequence seq = linear_sequence(a.batch, blockIdx.y);
  if (seq.rows <= plan.min_rows) {
    wait_for_launch_before();
    return;
  }
  // segment, and for the first pass whether its M is wanted
  const int job = static_cast<int>(gridDim.z - 1 - blockIdx.z);            // the first segment, which may be shorter, is begun last
  const int segment = kMode == kTransfer ? (job + 1) / 2 : job;
  const bool transfer = kMode == kTransfer && segment > 0 && job % 2 == 0;
  if (kOutputs && segment == 0) {                     // rows that are not active
    for (int i = threadIdx.x; i < seq.first * (kLinearDim / 8); i += kChunkThreads)
      *reinterpret_cast<uint4*>(a.out + (static_cast<long long>(seq.row0 + i / (kLinearDim / 8)) * a.v_heads + head) * kLinearDim + 8 * (i % (kLinearDim / 8))) =
          make_uint4(0, 0, 0, 0);
  }
  const int limit = kMode == kKept ? seq.kept : seq.rows;                  // rows that are gone through
  const int all_chunks = (limit - seq.first + kChunk - 1) / kChunk;
  const Segments cut(plan.segments, plan.first, all_chunks);
  const int chunk0 = cut.begin(segment), chunks = min(cut.begin(segment + 1), all_chunks) - chunk0;
  if (limit <= seq.first || chunks <= 0) {
    wait_for_launch_before();
    return;
  }

  // its first tile
  int tile0 = 0;
  {
    int mine = 0;
    for (int s = threadIdx.x; s < static_cast<int>(blockIdx.y); s += kChunkThreads) mine += chunks_of(linear_sequence(a.batch, s), plan.min_rows);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) m.sums[warp] = mine;
  }
  if (warp == kChainWarps) tmem_alloc(smem_u32(&m.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  for (int w = 0; w < kChunkThreads / 32; ++w) tile0 += m.sums[w];
  wait_for_launch_before();
  constexpr uint32_t tmem = 0;               // all 512 columns begin at 0
  const bool fits = tile0 + chunks_of(seq, plan.min_rows) <= plan.tiles;       // not if sequences overlap, which the first kernel reports
  const int n = fits ? chunks : 0;
  if (!fits && threadIdx.x == 0) atomicOr(a.status, kLinearBadBatch);
  volatile int* abort_flag = &m.abort_flag;
  auto wait = [&](unsigned long long* bar, int phase) { return wait_inline(smem_u32(bar), phase & 1, abort_flag, plan.wait_limit_ns); };
  tile0 += chunk0;
  const long long row0 = static_cast<long long>(seq.row0) + seq.first + chunk0 * kChunk;
  const int rows = limit - seq.first - chunk0 * kChunk;                        // of all its chunks, and behind them

  if (warp < kChainWarps) {
    // ------------------------------ the chain ------------------------------
    // No wait that runs out leaves this loop: the warps meet at barriers, and every wait after the first that ran out ends at once.
    const int group = warp >> 2, column = (warp & 3) * 32 + lane;              // a value element
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const long long part = kKeys * group * kLinearDim + column;                // of a state
    float* const state = a.states + (static_cast<long long>(seq.slot) * a.v_heads + head) * kLinearDim * kLinearDim + part;
    const bool gated = kOutputs && a.gate.data != nullptr;
    // rows of the output: 16 lanes a row
    const int out_row = 2 * warp + (lane >> 4), piece = lane & 15;

    // O and Q of chunk c as rows in shared memory
    auto take_outputs = [&](int c) {
      const float back = kv_exp2(-kv_float_exponent(m.scale[c & 1][column])) * 0.08838834764831845f;
      const int broken = m.broken[c & 1][column];
      wait(&m.out_full, c);
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < kTokens / 16; ++b) {
        const int token = kTokens * group + 16 * b;
        Pair o[8], q[8];
        tmem_ld16(lanes + kEnterAt + token, reinterpret_cast<uint32_t*>(o));
        tmem_ld16(lanes + kReadAt + token, reinterpret_cast<uint32_t*>(q));
        tmem_ld_wait();
        if (b == kTokens / 16 - 1) warp_arrive(&m.out_taken, lane);
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
          const float4 read = *reinterpret_cast<const float4*>(&m.read[c & 1][token + t]);
          const float2 x = (fma2(Pair(read.x, read.y), q[t / 2], o[t / 2]) * Pair(back, back)).values();
          const float2 y = (fma2(Pair(read.z, read.w), q[t / 2 + 1], o[t / 2 + 1]) * Pair(back, back)).values();
          float* to = &m.out[(token + t) * kOutRow + column];
          to[0] = x.x;
          to[kOutRow] = x.y;
          to[2 * kOutRow] = y.x;
          to[3 * kOutRow] = y.y;
        }
      }
      for (int t = max(broken, kTokens * group); t < kTokens * (group + 1); ++t) m.out[t * kOutRow + column] = NAN;
    };
    // half of the rows that a thread has of chunk c, from shared memory to the output
    auto gate_at = [&](int c, int i) {                                         // of row i
      const int t = min(kOutRows * i + out_row, rows - c * kChunk - 1);
      return *reinterpret_cast<const uint4*>(a.gate.data + (row0 + c * kChunk + t) * a.gate.row_stride + head * a.gate.head_stride + 8 * piece);
    };
    auto write_rows = [&](int c, int which, const uint4* gates) {
      constexpr int kRows = kOutPasses / 2;
      float o[kRows][8], sum[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const float* from = &m.out[(kOutRows * (kRows * which + i) + out_row) * kOutRow + 8 * piece];
        *reinterpret_cast<float4*>(o[i]) = *reinterpret_cast<const float4*>(from);
        *reinterpret_cast<float4*>(o[i] + 4) = *reinterpret_cast<const float4*>(from + 4);
      }
      if (gated) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          sum[i] = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[i] = fmaf(o[i][j], o[i][j], sum[i]);
        }
#pragma unroll
        for (int d = 8; d >= 1; d /= 2)
#pragma unroll
          for (int i = 0; i < kRows; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
        float weight[8];
        *reinterpret_cast<float4*>(weight) = *reinterpret_cast<const float4*>(&m.weight[8 * piece]);
        *reinterpret_cast<float4*>(weight + 4) = *reinterpret_cast<const float4*>(&m.weight[8 * piece + 4]);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          float square = fmaf(sum[i], 1.0f / kLinearDim, a.eps);
          if (!linear_norm_holds(square)) {                                    // for the 16 lanes of a row
            const float by = linear_norm_shift(square);
            square = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[i][j] *= by;
              square = fmaf(o[i][j], o[i][j], square);
            }
#pragma unroll
            for (int d = 8; d >= 1; d /= 2) square += __shfl_xor_sync(0xffffu << (lane & 16), square, d);
            square = fmaf(square, 1.0f / kLinearDim, a.eps * by * by);
          }
          const float factor = rsqrtf(square);
          float z[8];
          unpack8(gates[kRows * which + i], z);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[i][j] *= (factor * weight[j]) * (z[j] * linear_four_sigmoid(z[j]));
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int t = c * kChunk + kOutRows * (kRows * which + i) + out_row;
        if (t < rows)
          *reinterpret_cast<uint4*>(a.out + ((row0 + t) * a.v_heads + head) * kLinearDim + 8 * piece) =
              make_uint4(pack_bf16(o[i][0], o[i][1]), pack_bf16(o[i][2], o[i][3]), pack_bf16(o[i][4], o[i][5]), pack_bf16(o[i][6], o[i][7]));
      }
    };

    Pair s[kKeys / 2];                                                         // key elements kKeys group ..
    float scale = 1.0f;
    {
      // where the state comes from; nullptr: zeros, or the identity.  With segments the first pass keeps the first one's: the second
      // pass's last segment may write the state before its first one has begun.
      const float* before = n == 0 || seq.fresh ? nullptr : state;
      if (kOutputs && plan.segments > 1) before = border(plan, blockIdx.y, head, segment) + part;
      if (kMode == kTransfer && segment > 0) before = nullptr;
      if (before != nullptr) {
#pragma unroll
        for (int i = 0; i < kKeys; i += 2) s[i / 2] = Pair(before[i * kLinearDim], before[(i + 1) * kLinearDim]);
      } else {
        const int one = transfer ? column - kKeys * group : -1;                // where the identity has its element
#pragma unroll
        for (int i = 0; i < kKeys; i += 2) s[i / 2] = Pair(i == one ? 1.0f : 0.0f, i + 1 == one ? 1.0f : 0.0f);
      }
      if (gated && group == 0) m.weight[column] = 0.25f * __bfloat162float(a.norm_weight[column]);
      float largest = 0.0f;
#pragma unroll
      for (int i = 0; i < kKeys / 2; ++i) largest = max3_abs(largest, s[i].values().x, s[i].values().y);
      m.largest[group][column] = largest;
      if (kMode == kTransfer && segment == 0 && n > 0) {
        float* const first = border(plan, blockIdx.y, head, 0) + part;
#pragma unroll
        for (int i = 0; i < kKeys / 2; ++i) {
          const float2 x = s[i].values();
          first[2 * i * kLinearDim] = x.x;
          first[(2 * i + 1) * kLinearDim] = x.y;
        }
      }
      chain_barrier();
    }
    auto load_state = [&](int c) {                                             // after chunk c
      wait(&m.state_full, c);
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < kKeys / 16; ++b) tmem_ld16(lanes + kStateAt + kKeys * group + 16 * b, reinterpret_cast<uint32_t*>(s + 8 * b));
      tmem_ld_wait();
      if (m.broken[c & 1][column] < kChunk) {
#pragma unroll
        for (int i = 0; i < kKeys / 2; ++i) s[i] = Pair(NAN, NAN);
      }
    };
    float value_before = 0.0f;
    for (int c = 0; c < n; ++c) {
      const uint8_t* stage = m.stages[c % kStages];
      const ChunkNumbers& numbers = *reinterpret_cast<const ChunkNumbers*>(stage + kChunkPairBytes + kChunkNumbersAt);
      const int there = rows - c * kChunk;                                     // tokens
      wait(&m.values_full[c % kStages], c / kStages);
      // The column's power of two, from the largest of the state one chunk ago and of the values since: the state is at most
      // sqrt(128) of it longer with 64 of them added, so that 140 times the largest bounds all that is held in 16 bits here.
      bool rescale;
      float up = 1.0f;
      {
        const float value = fmaxf(m.largest_value[c % kStages][0][column], m.largest_value[c % kStages][1][column]);
        float largest = fmaxf(value, value_before);
#pragma unroll
        for (int i = 0; i < kGroups; ++i) largest = fmaxf(largest, m.largest[i][column]);
        const float held = largest * scale;
        value_before = value;
        rescale = !(held <= 256.0f && held >= 0.5f) && largest > 0.0f && largest < INFINITY;
        if (rescale) {
          const int now = kv_float_exponent(scale), next = min(max(3 - kv_float_exponent(largest), -120), 100);
          up = kv_exp2(max(min(next - now, 126), -126));
          scale = kv_exp2(next);
        }
        if (group == 0) {                     // what two chunks ago was left here has been read
          m.scale[c & 1][column] = scale;
          m.broken[c & 1][column] = kChunk;
        }
      }
      if (c > 0) load_state(c - 1);
      if (rescale) {
#pragma unroll
        for (int i = 0; i < kKeys / 2; ++i) s[i] = s[i] * Pair(up, up);
      }
      // the state in two terms, and decayed for the sum that follows; products begin with the first half of each group's elements
#pragma unroll
      for (int b = 0; b < kKeys / 16; ++b) {
        uint32_t terms[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) split_f16(s[8 * b + i], &terms[i], &terms[8 + i]);
        tmem_st16(lanes + kTermsAt + kKeys * group + 16 * b, terms);
        if (b % (kKeys / 32) == kKeys / 32 - 1) {
          tmem_st_wait();
          warp_arrive(&m.state_ready[b / (kKeys / 32)], lane);
        }
      }
      float largest_here = 0.0f;
      {
        const float decay = kMode == kKept ? numbers.decay_kept : numbers.decay;
#pragma unroll
        for (int b = 0; b < kKeys / 16; ++b) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 x = s[8 * b + i].values();
            largest_here = max3_abs(largest_here, x.x, x.y);
            s[8 * b + i] = s[8 * b + i] * Pair(decay, decay);
          }
          tmem_st16(lanes + kStateAt + kKeys * group + 16 * b, reinterpret_cast<uint32_t*>(s + 8 * b));
        }
        largest_here *= kv_exp2(-kv_float_exponent(scale));
      }
      if (kOutputs && c > 0) {
        wait(&m.state_ready[1], c);           // all warps are done with the rows that lie in shared memory
        take_outputs(c - 1);
      }
      Pair given[kTokens / 2];                                                 // beta v of tokens kTokens group .., what of the right side can wait here
      {
        const uint16_t* values = reinterpret_cast<const uint16_t*>(stage + kStageValues) + kTokens * group * kLinearDim + column;
#pragma unroll
        for (int t = 0; t < kTokens; t += 4) {
          const float4 rate = *reinterpret_cast<const float4*>(&numbers.rate[kTokens * group + t]);
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(static_cast<uint32_t>(values[(t + i) * kLinearDim]) << 16);
          given[t / 2] = Pair(rate.x, rate.y) * (Pair(x[0], x[1]) * Pair(scale, scale));
          given[t / 2 + 1] = Pair(rate.z, rate.w) * (Pair(x[2], x[3]) * Pair(scale, scale));
        }
      }
      uint4 gates[kOutPasses];
      if (gated && c > 0) {
#pragma unroll
        for (int i = 0; i < kOutPasses; ++i) gates[i] = gate_at(c - 1, i);
      }
      wait(&m.dots_full, c);
      tc_fence_after();
      m.largest[group][column] = largest_here;                                 // all warps have read what the chunk before left here
      // the right side
      {
        Pair all[kTokens / 2];             // read before the first products write there
#pragma unroll
        for (int b = 0; b < kTokens / 16; ++b) tmem_ld16(lanes + kDotsAt + kTokens * group + 16 * b, reinterpret_cast<uint32_t*>(all + 8 * b));
        tmem_ld_wait();
#pragma unroll
        for (int b = 0; b < kTokens / 16; ++b) {
          const int token = kTokens * group + 16 * b;
          Pair* const r = all + 8 * b;
          uint32_t terms[16];
          __half2 check = __half2half2(__ushort_as_half(0));
#pragma unroll
          for (int t = 0; t < 16; t += 4) {
            const float4 enter = *reinterpret_cast<const float4*>(&numbers.enter[token + t]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int j = t / 2 + i;
              r[j] = fma2(i == 0 ? Pair(enter.x, enter.y) : Pair(enter.z, enter.w), r[j], given[8 * b + j]);
              split_f16(r[j], &terms[j], &terms[8 + j]);
              check = __hfma2(*reinterpret_cast<const __half2*>(&terms[j]), __half2half2(__ushort_as_half(0)), check);
            }
          }
          if ((*reinterpret_cast<const uint32_t*>(&check) & 0x7fff7fffu) != 0) {
            int first = kChunk;
#pragma unroll
            for (int j = 7; j >= 0; --j) {
              float2 x = r[j].values();
              if (!(fabsf(x.y) < INFINITY)) {
                if (token + 2 * j + 1 < there) first = token + 2 * j + 1;      // rows that are not gone through say nothing
                x.y = 0.0f;
              }
              if (!(fabsf(x.x) < INFINITY)) {
                if (token + 2 * j < there) first = token + 2 * j;
                x.x = 0.0f;
              }
              split_f16(x.x, x.y, &terms[j], &terms[8 + j]);
            }
            atomicMin(&m.broken[c & 1][column], first);
          }
          tmem_st16(lanes + kEnterAt + token, terms);
          tmem_st_wait();
          warp_arrive(&m.enter_ready[b], lane);
        }
      }
      if (kOutputs && c > 0) {
        wait(&m.enter_ready[kTokenSteps - 1], c);                              // all warps' part of the rows is there
        write_rows(c - 1, 0, gates);
      }
      // the corrections
      {
        Pair d[kTokens / 2];
        float4 stay[kTokens / 4];
#pragma unroll
        for (int t = 0; t < kTokens; t += 4)
          stay[t / 4] = *reinterpret_cast<const float4*>((kMode == kKept ? numbers.stay_kept : numbers.stay) + kTokens * group + t);
        wait(&m.fresh_full, c);
        tc_fence_after();
        uint32_t terms[16];
#pragma unroll
        for (int b = 0; b < kTokens / 16; ++b) tmem_ld16(lanes + kDotsAt + kTokens * group + 16 * b, reinterpret_cast<uint32_t*>(d + 8 * b));
        tmem_ld_wait();
#pragma unroll
        for (int b = 0; b < kTokens / 16; ++b) {
#pragma unroll
          for (int t = 0; t < 16; t += 4) {
            const float4 x = stay[4 * b + t / 4];
            const int j = t / 2;
            split_f16(d[8 * b + j] * Pair(x.x, x.y), &terms[j], &terms[8 + j]);
            split_f16(d[8 * b + j + 1] * Pair(x.z, x.w), &terms[j + 1], &terms[8 + j + 1]);
          }
          tmem_st16(lanes + kEnterAt + kTokens * group + 16 * b, terms);
          tmem_st_wait();
          warp_arrive(&m.stay_ready[b], lane);
        }
        if (kOutputs) {
          if (column < kTokens) m.read[c & 1][kTokens * group + column] = numbers.read[kTokens * group + column];
#pragma unroll
          for (int b = 0; b < kTokens / 16; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) split_f16(d[8 * b + i], &terms[i], &terms[8 + i]);
            tmem_st16(lanes + kFreshAt + kTokens * group + 16 * b, terms);
          }
          tmem_st_wait();
          warp_arrive(&m.fresh_ready, lane);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&m.empty[c % kStages]));
      }
      if (kOutputs && c > 0) write_rows(c - 1, 1, gates);
    }
    if (n > 0) {
      load_state(n - 1);
      float* after = nullptr;
      if (kMode == kTransfer) after = border(plan, blockIdx.y, head, segment == 0 ? 1 : transfer ? border_m(segment) : border_b(segment)) + part;
      else if (plan.store && seq.kept > seq.first && chunk0 + chunks == all_chunks) after = state;
      if (after != nullptr) {
        const float back = kv_exp2(-kv_float_exponent(scale));
#pragma unroll
        for (int i = 0; i < kKeys / 2; ++i) {
          const float2 x = s[i].values();
          after[2 * i * kLinearDim] = x.x * back;
          after[(2 * i + 1) * kLinearDim] = x.y * back;
        }
      }
      if (kOutputs) {
        uint4 gates[kOutPasses];
        if (gated) {
#pragma unroll
          for (int i = 0; i < kOutPasses; ++i) gates[i] = gate_at(n - 1, i);
        }
        chain_barrier();
        take_outputs(n - 1);
        chain_barrier();
        write_rows(n - 1, 0, gates);
        write_rows(n - 1, 1, gates);
      }
    }
  } else if (warp == kChainWarps) {
    // ------------------------------ products ------------------------------
    // Products of different shapes need not run in the order of issue: one that reads or writes what another wrote waits for its commit.
    // A step with N = 64 takes 32 cycles, one with 128 takes 64.  What the chain waits for goes first.
    constexpr uint32_t kNarrow = instr_desc_f8(kF16, kF16, 0, 0, 128, kChunk), kUpdate = instr_desc_f8(kF16, kF16, 0, 1, 128, kLinearDim);
    // T and the scores are triangles: tokens 16 k .. add to what they and those behind them have, and to nothing before
    const auto below = [](int k) { return instr_desc_f8(kF16, kF16, 0, 0, 128, kChunk - 16 * k); };
    // descriptors: those of a stage's begin, to which constants are added (an address takes their low 14 bits)
    const uint32_t base = smem_u32(m.stages[0]);
    for (int c = 0; c < n; ++c) {
      const uint32_t at = base + (c % kStages) * kStageBytes;
      const uint64_t rows_desc = smem_desc_rows<128>(at), update_desc = smem_desc_rows<128>(at, kChunkPanelBytes);
      auto dots = [&](int half, uint32_t to, uint32_t rows_at) {                  // of a half of each group's key elements
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i)
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int term = 0; term < 2; ++term) {
              const int k = g * (kKeys / 16) + half * (kKeys / 32) + i;
              umma_f16_ts(to, kTermsAt + operand(k, term), rows_desc + ((rows_at + (k / 4) * kChunkPanelBytes + (k % 4) * 32) >> 4), kNarrow,
                          (half | i | g | term) != 0);
            }
      };
      if (!wait(&m.full[c % kStages], c / kStages) || !wait(&m.state_ready[0], c)) break;
      tc_fence_after();
      if (elect_one()) dots(0, kDotsAt, 0);
      __syncwarp();
      if (!wait(&m.state_ready[1], c)) break;
      tc_fence_after();
      if (elect_one()) {
        dots(1, kDotsAt, 0);
        umma_commit(smem_u32(&m.dots_full));
      }
      __syncwarp();
      if (kOutputs) {
        if (c > 0 && !wait(&m.out_taken, c - 1)) break;
        tc_fence_after();
        if (elect_one()) {
          dots(0, kReadAt, kChunk * 128);
          dots(1, kReadAt, kChunk * 128);
        }
        __syncwarp();
      }
      bool alive = true;
#pragma unroll
      for (int step = 0; step < kTokenSteps && alive; ++step) {                   // of each group's tokens
        alive = wait(&m.enter_ready[step], c);
        tc_fence_after();
        if (alive && elect_one()) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int term = 0; term < 3; ++term) {                                // both terms by T's first, the first by T's second
              const int k = g * kTokenSteps + step;
              umma_f16_ts(kDotsAt + 16 * k, kEnterAt + operand(k, term == 1),
                          rows_desc + ((kChunkPairBytes + (term == 2 ? kChunkMatrixBytes : 0) + k * (16 * 128 + 32)) >> 4), below(k), (k | term) != 0);
            }
          if (step == kTokenSteps - 1) umma_commit(smem_u32(&m.fresh_full));
        }
        __syncwarp();
      }
#pragma unroll
      for (int step = 0; step < kTokenSteps && alive; ++step) {
        alive = wait(&m.stay_ready[step], c);
        tc_fence_after();
        if (alive && elect_one()) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int term = 0; term < 2; ++term) {
              const int k = g * kTokenSteps + step;
              umma_f16_ts(kStateAt, kEnterAt + operand(k, term), update_desc + ((k * 16 * 128) >> 4), kUpdate, 1);
            }
          if (step == kTokenSteps - 1) {
            umma_commit(smem_u32(&m.state_full));
            if (!kOutputs) umma_commit(smem_u32(&m.empty[c % kStages]));
          }
        }
        __syncwarp();
      }
      if (!alive) break;
      if (kOutputs) {
        if (!wait(&m.fresh_ready, c) || !wait(&m.state_full, c)) break;           // O goes where the state's corrections are read
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int term = 0; term < 3; ++term)                                    // both terms by the scores' first, the first by their second
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k)
              umma_f16_ts(kEnterAt + 16 * k, kFreshAt + operand(k, term == 1),
                          rows_desc + ((kChunkPairBytes + (term == 2 ? 3 : 2) * kChunkMatrixBytes + k * (16 * 128 + 32)) >> 4), below(k), (term | k) != 0);
          umma_commit(smem_u32(&m.out_full));
          umma_commit(smem_u32(&m.empty[c % kStages]));
        }
        __syncwarp();
      }
    }
  } else if (warp == kChainWarps + 1) {
    // ------------------------------ loads ------------------------------
    int c = 0;
    for (; c < n; ++c) {
      const int slot = c % kStages;
      if (!wait(&m.empty[slot], c / kStages + 1)) break;
      const uint32_t to = smem_u32(m.stages[slot]), bar = smem_u32(&m.full[slot]);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, kStageValues);
        const size_t tile = static_cast<size_t>(tile0 + c);
        bulk_g2s(to, plan.pairs + (tile * a.k_heads + head / a.group) * kChunkPairBytes, kChunkPairBytes, bar);
        bulk_g2s(to + kChunkPairBytes, plan.heads + (tile * a.v_heads + head) * kChunkHeadBytes, kChunkHeadBytes, bar);
      }
      __syncwarp();
    }
    if (*abort_flag != 0) {                // what is in flight lands before the block leaves
      volatile int ignore = 0;
      for (int i = max(0, c - kStages); i < c; ++i) wait_inline(smem_u32(&m.full[i % kStages]), (i / kStages) & 1, &ignore, kWaitBudgetNs);
    }
  } else {
    // ------------------------------ values, and the largest of each column ------------------------------
    // 16 lanes a row, 16 rows a thread.  (A copy of 256 bytes for each row took 70 cycles to issue, 5000 for the chunk.)
    const int which = warp & 1, piece = lane & 15, first = 2 * which + (lane >> 4);
    const __nv_bfloat16* from = a.v.data + (row0 + first) * a.v.row_stride + head * a.v.head_stride + 8 * piece;
    for (int c = 0; c < n; ++c) {
      const int slot = c % kStages, there = min(kChunk, rows - c * kChunk) - first;
      uint8_t* const to = m.stages[slot] + kStageValues + first * 2 * kLinearDim + piece * 16;
      wait(&m.empty[slot], c / kStages + 1);
      const uint32_t at = smem_u32(to);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool is = !transfer && 4 * i < there;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(at + i * 4 * 2 * kLinearDim), "l"(is ? from : a.v.data), "r"(is ? 16 : 0) : "memory");
        from += 4 * a.v.row_stride;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      uint32_t most[4] = {0, 0, 0, 0};
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(to + i * 4 * 2 * kLinearDim);
#pragma unroll
        for (int j = 0; j < 4; ++j) most[j] = __vmaxu2(most[j], (&x.x)[j] & 0x7fff7fffu);
      }
      if (__vmaxu2(__vmaxu2(most[0], most[1]), __vmaxu2(most[2], most[3])) != __vminu2(__vmaxu2(__vmaxu2(most[0], most[1]), __vmaxu2(most[2], most[3])), 0x7f7f7f7fu)) {
        most[0] = most[1] = most[2] = most[3] = 0;
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(to + i * 4 * 2 * kLinearDim);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t y = (&x.x)[j] & 0x7fff7fffu;
            if ((y & 0xffffu) >= 0x7f80u) y &= 0xffff0000u;
            if (y >= 0x7f800000u) y &= 0xffffu;
            most[j] = __vmaxu2(most[j], y);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) most[j] = __vmaxu2(most[j], __shfl_xor_sync(0xffffffffu, most[j], 16));
      if (lane < 16) {
        float4* largest = reinterpret_cast<float4*>(&m.largest_value[slot][which][8 * piece]);
        largest[0] = make_float4(bf16_lo(most[0]), bf16_hi(most[0]), bf16_lo(most[1]), bf16_hi(most[1]));
        largest[1] = make_float4(bf16_lo(most[2]), bf16_hi(most[2]), bf16_lo(most[3]), bf16_hi(most[3]));
      }
      wait(&m.full[slot], c / kStages);                                           // for those that wait for this alone
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&m.values_full[slot]));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(a.status, kLinearTimeout);
  if (warp == kChainWarps) tmem_dealloc(tmem, 512);
}

// The states before the segments from the first pass: S_(j + 1) = M_j S_j + B_j, a block per head and 32 columns.  A thread
// takes 4 x 4 elements and half of the sum: 8 loads from shared memory for 64 products.  The next M is on its way meanwhile.
constexpr int kJoinThreads = 512, kJoinColumns = 32, kJoinRow = kLinearDim + 4;
struct __align__(16) JoinMemory {
  float transfer[2][kLinearDim * kJoinRow];
  float before[kLinearDim][kJoinColumns], other[kLinearDim][kJoinColumns];
};
__global__ void __launch_bounds__(kJoinThreads, 1) linear_join_kernel(const ChunkPlan plan) {
  extern __shared__ uint8_t raw[];
  JoinMemory& m = *reinterpret_cast<JoinMemory*>(raw);
  const int head = blockIdx.x, sequence = blockIdx.y, begin = static_cast<int>(blockIdx.z) * kJoinColumns;
  const int column = 4 * (threadIdx.x & 7), first = (threadIdx.x >> 3) & 31, part = threadIdx.x >> 8;        // rows first + 32 i
  const LinearSequence seq = linear_sequence(plan.a.batch, sequence);
  const int chunks = chunks_of(seq, plan.min_rows);
  const Segments cut(plan.segments, plan.first, chunks);
  launch_may_follow();
  wait_for_launch_before();
  const auto there = [&](int j) { return j + 1 < plan.segments && cut.begin(j + 1) < chunks; };
  const auto fetch = [&](int j) {
    const float* from = border(plan, sequence, head, border_m(j));
#pragma unroll
    for (int i = 0; i < kLinearDim * kLinearDim / 4 / kJoinThreads; ++i) {
      const int at = i * kJoinThreads + static_cast<int>(threadIdx.x), row = at / (kLinearDim / 4), piece = at % (kLinearDim / 4);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(&m.transfer[j & 1][row * kJoinRow + 4 * piece])), "l"(from + 4 * at) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (!there(1)) return;
  fetch(1);
  if (part == 0) {
    const float* from = border(plan, sequence, head, 1) + begin;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4*>(&m.before[first + 32 * i][column]) = *reinterpret_cast<const float4*>(from + (first + 32 * i) * kLinearDim + column);
  }
  for (int j = 1; there(j); ++j) {
    float4 sum[4];
    const float* add = border(plan, sequence, head, border_b(j)) + begin;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = part == 0 ? *reinterpret_cast<const float4*>(add + (first + 32 * i) * kLinearDim + column) : make_float4(0, 0, 0, 0);
    if (there(j + 1)) fetch(j + 1);
    if (there(j + 1)) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
#pragma unroll 4
    for (int k = part * (kLinearDim / 2); k < (part + 1) * (kLinearDim / 2); k += 4) {
      float4 x[4];
#pragma unroll
      for (int l = 0; l < 4; ++l) x[l] = *reinterpret_cast<const float4*>(&m.before[k + l][column]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(&m.transfer[j & 1][(first + 32 * i) * kJoinRow + k]);
#pragma unroll
        for (int l = 0; l < 4; ++l) {
          const float z = (&y.x)[l];
          sum[i].x = fmaf(z, x[l].x, sum[i].x);
          sum[i].y = fmaf(z, x[l].y, sum[i].y);
          sum[i].z = fmaf(z, x[l].z, sum[i].z);
          sum[i].w = fmaf(z, x[l].w, sum[i].w);
        }
      }
    }
    if (part != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(&m.other[first + 32 * i][column]) = sum[i];
    }
    __syncthreads();                       // the states are read; what M lay in is free for the one after the next
    if (part == 0) {
      float* to = border(plan, sequence, head, j + 1) + begin;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(&m.other[first + 32 * i][column]);
        const float4 x = make_float4(sum[i].x + y.x, sum[i].y + y.y, sum[i].z + y.z, sum[i].w + y.w);
        *reinterpret_cast<float4*>(to + (first + 32 * i) * kLinearDim + column) = x;
        *reinterpret_cast<float4*>(&m.before[first + 32 * i][column]) = x;
      }
    }
  }
}

}  // namespace

size_t linear_chunk_workspace(int k_heads, int v_heads, int max_tokens, int max_sequences) {
  return chunk_workspace(k_heads, v_heads, max_tokens, max_sequences, kLinearStepRows, kChunkPairBytes, kChunkHeadBytes);
}

cudaError_t linear_chunks(const LinearDelta& a, int min_rows, void* workspace, int sm_count, cudaStream_t stream) {
  ChunkPlan plan{};
  plan.a = a;
  plan.min_rows = min_rows;
  const ChunkLayout layout = chunk_layout(a.k_heads, a.v_heads, a.batch.tokens, a.batch.sequences, a.batch.max_new, min_rows, sm_count, kChunkPairBytes,
                                          kChunkHeadBytes);
  const Cut cut = layout.cut;
  plan.tiles = static_cast<int>(layout.tiles);
  plan.borders = static_cast<float*>(workspace);
  plan.pairs = static_cast<uint8_t*>(workspace) + layout.pairs_at;
  plan.heads = static_cast<uint8_t*>(workspace) + layout.heads_at;
  plan.wait_limit_ns = kWaitBudgetNs;
  cudaError_t error = linear_prepare(plan, sm_count, stream);
  constexpr int kBytes = static_cast<int>(sizeof(ChunkMemory)) + 1024;
  if (error == cudaSuccess) error = opt_in_dynamic_smem<linear_chunk_kernel<kOutput>>(kBytes);
  if (error == cudaSuccess) error = opt_in_dynamic_smem<linear_chunk_kernel<kKept>>(kBytes);
  if (error == cudaSuccess) error = opt_in_dynamic_smem<linear_chunk_kernel<kTransfer>>(kBytes);
  if (error == cudaSuccess) error = opt_in_dynamic_smem<linear_join_kernel>(sizeof(JoinMemory));
  if (error != cudaSuccess) return error;
  const auto grid = [&](int parts) { return dim3(a.v_heads, a.batch.sequences, parts); };
  // with rows that are computed but do not stay, once for the outputs and once for the states
  if (a.out != nullptr) {
    plan.store = a.batch.keep == nullptr;
    plan.segments = cut.segments;
    plan.first = cut.first;
    if (cut.segments > 1) error = launch_pdl(linear_chunk_kernel<kTransfer>, grid(2 * cut.segments - 3), kChunkThreads, kBytes, stream, plan);
    if (error == cudaSuccess && cut.segments > 2)
      error = launch_pdl(linear_join_kernel, grid(kLinearDim / kJoinColumns), kJoinThreads, sizeof(JoinMemory), stream, plan);
    if (error == cudaSuccess) error = launch_pdl(linear_chunk_kernel<kOutput>, grid(cut.segments), kChunkThreads, kBytes, stream, plan);
  }
  if (error == cudaSuccess && (a.out == nullptr || a.batch.keep != nullptr)) {
    plan.store = plan.segments = 1;
    plan.first = 8;
    error = launch_pdl(linear_chunk_kernel<kKept>, grid(1), kChunkThreads, kBytes, stream, plan);
  }
  return error;
}

}  // namespace aima
