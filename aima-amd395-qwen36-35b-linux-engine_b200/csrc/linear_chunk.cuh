// The gated delta rule in chunks of 64 tokens: what its two kernels share.
//
// With G_t the sum of g over a chunk's tokens up to t, S the state before the chunk and T = (1 + A)^-1,
// A_ij = beta_i e^(G_i - G_j) k_i.k_j for j < i, the corrections of all tokens of the chunk are
//   d = T (beta v - beta e^G (S^T k)),
// and with them
//   o_i = e^G_i S^T q_i + sum_(j <= i) e^(G_i - G_j) (q_i.k_j) d_j,      S <- e^G_63 S + sum_j e^(G_63 - G_j) k_j d_j^T.
//
// linear_prepare_kernel makes, for all chunks at once, what does not depend on the state; linear_chunk_kernel goes through a
// sequence's chunks one after the other, one block per value head.
//
// 16-bit operands.  q and k are held as f16 numbers times a power of two per row, 1 <= max < 2: exact, but for elements below 2^-17 of a
// row's largest, which are off by 2^-25 of it at the most.  The lengths by which they are divided stay outside, in FP32.  State, corrections,
// T and the scores are held in two f16 terms, 22 bits: where a value is corrected away within a chunk, what is left is a small
// difference of what the products add up, in the outputs too.  A state column and what is added to it share a power of two that keeps them between 2^-1
// and 2^9 at their largest, so that both terms have all their bits.
#pragma once

#include "linear.cuh"
#include "linear_segments.cuh"
#include "tcgen05.cuh"

namespace aima {

constexpr int kChunkPairBytes = 2 * kChunk * kLinearDim * 2;     // k and q of a chunk: two panels of 64 elements, k's rows, then q's, 128-byte swizzle
constexpr int kChunkPanelBytes = kChunkPairBytes / 2;
static_assert(kBorderBytes == static_cast<size_t>(kMaxBorders) * kLinearDim * kLinearDim * sizeof(float));
constexpr int kChunkMatrixBytes = kChunk * kChunk * 2;           // T's first terms, its second, the scores' first, their second: rows of 128 bytes, swizzled
constexpr int kChunkNumbersAt = 4 * kChunkMatrixBytes;
struct ChunkNumbers {                                            // of a chunk and value head
  float rate[kChunk];          // beta
  float enter[kChunk];         // -beta e^G / |k|
  float stay[kChunk];          // e^(G_last - G) / |k|
  float read[kChunk];          // e^G / |q|
  float stay_kept[kChunk];     // as `stay`, for the last token that enters the state; 0 behind it
  float decay, decay_kept;     // e^G_last, and of the last that enters
  float pad[2];
};
constexpr int kChunkHeadBytes = kChunkNumbersAt + (static_cast<int>(sizeof(ChunkNumbers)) + 127) / 128 * 128;

struct ChunkPlan {
  LinearDelta a;
  int min_rows;                // sequences with more rows than this are taken here
  int tiles;                   // that `pairs` and `heads` have room for
  int store;                   // whether the states are written
  int segments, first;         // that a sequence's chunks are cut into, and eighths of the others' length that the first has
  float* borders;              // [sequences, v_heads, kMaxBorders, 128, 128]: see linear_chunk.cu
  uint8_t* pairs;              // [tiles, k_heads, kChunkPairBytes]
  uint8_t* heads;              // [tiles, v_heads, kChunkHeadBytes]
  unsigned long long wait_limit_ns;
};

// Chunks of a sequence: of its active rows, if it is taken here.
__device__ __forceinline__ int chunks_of(const LinearSequence& s, int min_rows) {
  return s.rows > min_rows ? (s.rows - s.first + kChunk - 1) / kChunk : 0;
}

__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }      // 16-byte pieces of 128-byte rows

__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
         "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
// x as two f16 numbers whose sum has 22 bits of it: pairs of them
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t* high, uint32_t* low) {
  *high = cvt_f16x2(x0, x1);
  float l0, l1;                // x - high, exactly
  asm("{\n\t.reg .b16 l, u, m;\n\tmov.b32 {l, u}, %2;\n\tmov.b16 m, 0xBC00;\n\t"
      "fma.rn.f32.f16 %0, l, m, %3;\n\tfma.rn.f32.f16 %1, u, m, %4;\n\t}"
      : "=f"(l0), "=f"(l1) : "r"(*high), "f"(x0), "f"(x1));
  *low = cvt_f16x2(l0, l1);
}
__device__ __forceinline__ void split_f16(const Pair& x, uint32_t* high, uint32_t* low) {
  const float2 v = x.values();
  split_f16(v.x, v.y, high, low);
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float y;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ void launch_may_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
cudaError_t linear_prepare(const ChunkPlan& plan, int sm_count, cudaStream_t stream);

}  // namespace aima
