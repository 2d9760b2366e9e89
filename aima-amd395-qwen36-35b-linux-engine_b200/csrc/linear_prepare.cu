// The gated delta rule in chunks, first kernel: what a chunk needs that does not depend on the state (formulas in linear_chunk.cuh).
//
// A block takes a chunk and a key head.  k and q are scaled by a power of two per row to f16; one product of [k; q] with k gives k.k
// and q.k of all pairs of tokens, exactly but for the order of the sums.  Then, for every value head of that key head:
// sums of g (64 bits, kept as two FP32 numbers, so that differences of large sums keep theirs), decays, the scores, and the inverse of
// the unit lower triangle 1 + A by blocks of 16.  Decays between tokens of different blocks are products of two, from a token to its
// block's first and from that to the other token, which spares three quarters of the exponentials.  The diagonal's blocks are inverted
// by substitution; those below follow, a warp per column of blocks, from
//   X_i = T_ij = -T_ii (A_ij T_jj + sum_(j < k < i) A_ik X_k),
// transposed: the accumulators of each product are the first operand of the next as they lie in the warp's registers.  All operands
// have two f16 terms.
//
// Two blocks a multiprocessor go through all tiles, the next one's rows on their way.  Barriers and the latency of the substitution bound
// it (40 % of the issue slots, 2.6 TB/s): 8192 tokens of 16 key and 32 value heads take 84 us, of them 34 for the bytes.  Three blocks with 80
// registers spill and are no faster (86); two heads in every phase with half of the barriers are slower (93).
#include "linear_chunk.cuh"

#include <algorithm>

namespace aima {
namespace {

constexpr int kRowWarps = 6, kGateWarps = 2;
constexpr int kPrepareThreads = 32 * (kRowWarps + kGateWarps);
constexpr int kHeadsAtOnce = kGateWarps;        // whose gates are taken together
constexpr int kHalfRow = kChunk + 8;            // of a 16-bit matrix in shared memory
constexpr int kBlockRow = 20;                   // of a block of the diagonal

struct __align__(16) Terms {                    // a matrix in two terms, without swizzle
  uint16_t of[2][kChunk * kHalfRow];
};
struct __align__(1024) PrepareMemory {
  uint8_t rows[kChunkPairBytes];                // k and q of the next tile as they come, in the places that their pieces get
  union {
    uint8_t pair[kChunkPairBytes];              // until its products are there
    struct {
      Terms overlap, scores;                    // A, q.k
    };
  };
  Terms inverse;                                // T
  float diagonal[4][16 * kBlockRow];            // A's
  float length[2 * kChunk];                     // 1 / |k|, then 1 / |q|, of the scaled rows
  int broken[2 * kChunk];                       // rows that are not finite
  float sum_high[kHeadsAtOnce][kChunk], sum_low[kHeadsAtOnce][kChunk];         // log2(e) G
  float rate[kHeadsAtOnce][kChunk];             // beta, 0 for a token whose gates are not numbers
  float down[kHeadsAtOnce][kChunk];             // decay from a block's first token to a token of it
  float across[kHeadsAtOnce][4][kChunk];        // from a token to the first one of its own block or a later one, over |k|; 0 for earlier ones
  int steep[kHeadsAtOnce][4];                   // a block whose own decays are too small for that
  struct Tile {
    int row0, rows, kept;                       // its first row, its rows, those that enter the state
  } tiles[2];                                   // by turn
  int sums[kPrepareThreads / 32];
  unsigned long long done;
  uint32_t tmem;
  int abort_flag;
};

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// 16 x 16 of a matrix in two terms as a first operand, transposed
__device__ __forceinline__ void load_transposed(const uint16_t* at, int lane, uint32_t* a) {
  // tiles of 8: (rows 0, columns 0), (rows 0, columns 8), (rows 8, columns 0), (rows 8, columns 8) of the matrix
  const uint32_t from = smem_u32(at + ((lane & 7) + (lane >> 4) * 8) * kHalfRow + ((lane >> 3) & 1) * 8);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(from) : "memory");
}
// the other way
__device__ __forceinline__ void store_transposed(uint16_t* at, int lane, const uint32_t* a) {
  const uint32_t to = smem_u32(at + ((lane & 7) + (lane >> 4) * 8) * kHalfRow + ((lane >> 3) & 1) * 8);
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" :: "r"(to), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]) : "memory");
}
// d[2][4] (16 x 16) += x y^T of x in two terms (first operand) and a 16 x 16 block y in two terms
__device__ __forceinline__ void add_product(float (*d)[4], const uint32_t (*x)[4], const Terms& y, int row, int column, int lane) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    uint32_t b[2][2];
#pragma unroll
    for (int term = 0; term < 2; ++term) {
      const uint16_t* from = &y.of[term][(row + 8 * n + (lane >> 2)) * kHalfRow + column + 2 * (lane & 3)];
      b[term][0] = *reinterpret_cast<const uint32_t*>(from);
      b[term][1] = *reinterpret_cast<const uint32_t*>(from + 8);
    }
    mma_f16(d[n], x[0], b[0]);
    mma_f16(d[n], x[1], b[0]);
    mma_f16(d[n], x[0], b[1]);
  }
}
// accumulators times `sign` as a first operand in two terms
__device__ __forceinline__ void as_operand(const float (*d)[4], float sign, uint32_t (*x)[4]) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    split_f16(sign * d[n][0], sign * d[n][1], &x[0][2 * n], &x[1][2 * n]);
    split_f16(sign * d[n][2], sign * d[n][3], &x[0][2 * n + 1], &x[1][2 * n + 1]);
  }
}

// A lower triangle in two terms to where the second kernel takes it from, by some of the threads; the blocks above it are not read there.
__device__ __forceinline__ void write_terms(const Terms& from, uint8_t* to, int thread, int threads) {
#pragma unroll 4
  for (int i = thread; i < 2 * kChunk * 8; i += threads) {
    const int piece = i & 7, r = (i >> 3) & (kChunk - 1), term = i >> 9;
    if (piece / 2 <= r / 16)
      *reinterpret_cast<uint4*>(to + term * kChunkMatrixBytes + swizzled(r, piece)) = *reinterpret_cast<const uint4*>(&from.of[term][r * kHalfRow + 8 * piece]);
  }
}
// where the gates wait for the lengths of k
__device__ __forceinline__ void lengths_barrier() { asm volatile("bar.sync 1, %0;" :: "n"(kPrepareThreads) : "memory"); }

__global__ void __launch_bounds__(kPrepareThreads, 2) linear_prepare_kernel(const ChunkPlan plan) {
  extern __shared__ uint8_t raw[];
  PrepareMemory& m = *reinterpret_cast<PrepareMemory*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const LinearDelta& a = plan.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  launch_may_follow();
  if (blockIdx.x == 0) linear_report(a.batch, a.status, threadIdx.x, kPrepareThreads);
  if (warp == 0) tmem_alloc(smem_u32(&m.tmem), 64);
  if (threadIdx.x == 0) {
    m.abort_flag = 0;
    mbar_init(smem_u32(&m.done), 1);
    mbar_fence_init();
  }
  // a thread knows the tiles of some sequences
  const int share = (a.batch.sequences + kPrepareThreads - 1) / kPrepareThreads;
  const int first_mine = threadIdx.x * share, last_mine = min(first_mine + share, a.batch.sequences);
  int all = 0, upto = 0;
  {
    int mine = 0;
    for (int s = first_mine; s < last_mine; ++s) mine += chunks_of(linear_sequence(a.batch, s), plan.min_rows);
    upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    if (lane == 31) m.sums[warp] = upto;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    for (int w = 0; w < kPrepareThreads / 32; ++w) {
      if (w < warp) upto += m.sums[w];
      all += m.sums[w];
    }
    all = min(all, plan.tiles);
    upto -= mine;                                                    // those before this thread's
  }
  const uint32_t tmem = m.tmem;
  // the sequence and rows of a tile, by the thread that knows it
  const auto look_up = [&](int tile, int turn) {
    if (first_mine >= last_mine || tile < upto || tile >= all) return;
    int at = upto;
    for (int s = first_mine; s < last_mine; ++s) {
      const LinearSequence seq = linear_sequence(a.batch, s);
      const int chunks = chunks_of(seq, plan.min_rows);
      if (tile < at + chunks) {
        const int begin = seq.first + (tile - at) * kChunk, rows = min(kChunk, seq.rows - begin);
        m.tiles[turn] = PrepareMemory::Tile{seq.row0 + begin, rows, min(max(seq.kept - begin, 0), rows)};
        return;
      }
      at += chunks;
    }
  };
  // k's rows, then q's: four lanes a row, eight rows a warp at a time; a thread goes on with what it copied itself
  constexpr int kParts = 2 * kChunk / 8, kPasses = (kParts + kRowWarps - 1) / kRowWarps;
  const auto place = [&](int r, int p) {                             // of piece p of this lane
    const int piece = 4 * p + (lane & 3);
    return (piece >> 3) * kChunkPanelBytes + swizzled(r, piece & 7);
  };
  const auto fetch_rows = [&](int k_head, int row0, int rows) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = 8 * (warp + i * kRowWarps) + (lane >> 2), t = r & (kChunk - 1);
      if (8 * (warp + i * kRowWarps) >= 2 * kChunk) break;
      const KvRows& from = r < kChunk ? a.k : a.q;
      const bool there = t < rows;
      const __nv_bfloat16* at = there ? from.data + static_cast<long long>(row0 + t) * from.row_stride + k_head * from.head_stride + 8 * (lane & 3) : from.data;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::
                     "r"(smem_u32(m.rows + place(r, p))), "l"(there ? at + 32 * p : at), "r"(there ? 16 : 0) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // a and b of two tokens a lane
  const auto fetch_gates = [&](int head, int row0, int rows, float* x, float* y) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = y[i] = 0.0f;
      if (2 * lane + i < rows) {
        const long long at = row0 + 2 * lane + i;
        x[i] = __bfloat162float(a.a[at * a.a_stride + head]);
        y[i] = __bfloat162float(a.b[at * a.b_stride + head]);
      }
    }
  };
  const int half = warp >> 2, row = (warp & 3) * 32 + lane, token = row & (kChunk - 1), block = token >> 4;
  const int step_tile = static_cast<int>(gridDim.x) / a.k_heads, step_head = static_cast<int>(gridDim.x) - step_tile * a.k_heads;
  int tile_after = static_cast<int>(blockIdx.x) / a.k_heads, k_head_after = static_cast<int>(blockIdx.x) - tile_after * a.k_heads;
  PrepareMemory::Tile next{};
  float next_a[2], next_b[2];                                        // of a gate warp's first head
  if (tile_after < all) {
    look_up(tile_after, 0);
    __syncthreads();
    next = m.tiles[0];
    if (warp < kRowWarps) fetch_rows(k_head_after, next.row0, next.rows);
    else if (warp - kRowWarps < a.group) fetch_gates(k_head_after * a.group + warp - kRowWarps, next.row0, next.rows, next_a, next_b);
  }
  bool alive = true;
  for (int turn = 0; tile_after < all; turn ^= 1) {
    const int tile = tile_after, k_head = k_head_after;
    const int rows = next.rows, kept = next.kept;
    const long long row0 = next.row0;
    tile_after += step_tile;
    k_head_after += step_head;
    if (k_head_after >= a.k_heads) {
      k_head_after -= a.k_heads;
      ++tile_after;
    }
    const bool more = tile_after < all;
    if (more) look_up(tile_after, turn ^ 1);
    for (int base = 0; base < a.group; base += kHeadsAtOnce) {
      const int heads = min(kHeadsAtOnce, a.group - base);
      double total[2] = {0.0, 0.0}, last = 0.0;
      float beta[2] = {0.0f, 0.0f};
      bool broken[2] = {false, false};
      if (warp >= kRowWarps) {
        // sums of g and decays: two tokens a lane, a head a warp
        const int h = warp - kRowWarps, head = k_head * a.group + base + h;
        if (h < heads) {
          float g[2] = {0.0f, 0.0f}, x[2] = {next_a[0], next_a[1]}, y[2] = {next_b[0], next_b[1]};
          if (base != 0) fetch_gates(head, static_cast<int>(row0), rows, x, y);
          const float slope = expf(a.a_log[head]) * 1.44269504088896341f, bias = a.dt_bias[head];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (2 * lane + i < rows) {
              const float z = x[i] + bias;
              g[i] = -slope * (z > 20.0f ? z : log1pf(expf(z)));
              beta[i] = 1.0f / (1.0f + expf(-y[i]));
              broken[i] = g[i] != g[i] || beta[i] != beta[i];
              if (broken[i]) g[i] = beta[i] = 0.0f;
              g[i] = fmaxf(g[i], -1.0e6f);                             // e^g is 0 long before
            }
          }
          double upto = static_cast<double>(g[0]) + g[1];
#pragma unroll
          for (int d = 1; d < 32; d *= 2) {
            const double z = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += z;
          }
          total[0] = upto - g[1];
          total[1] = upto;
          last = __shfl_sync(0xffffffffu, upto, 31);                   // rows behind the last have g = 0
          double first[4];                                             // of each block
#pragma unroll
          for (int b = 0; b < 4; ++b) first[b] = __shfl_sync(0xffffffffu, total[0], 8 * b);
          float across[2][4];                                          // from a token to the first one of blocks 1 .. 3, of its own
          bool own_steep = false;
          const double mine = lane < 8 ? first[0] : lane < 16 ? first[1] : lane < 24 ? first[2] : first[3];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int t = 2 * lane + i;
            const float high = static_cast<float>(total[i]);
            m.sum_high[h][t] = high;
            m.sum_low[h][t] = static_cast<float>(total[i] - high);
            m.rate[h][t] = beta[i];
            // Decay from the block's first token, and its inverse: their products are the decays within the block, so the whole part of
            // the exponent stays apart, and they keep their bits however far the two are from 1.
            const double x = total[i] - mine;
            const int whole = max(__double2int_rn(x), -126);
            const float part = static_cast<float>(x - whole);
            m.down[h][t] = fast_exp2(part) * kv_exp2(whole);
            across[i][3] = fast_exp2(-part) * kv_exp2(-whole);
          }
          const double end[4] = {first[1], first[2], first[3], last};            // a token too far: no matter
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const bool steep = first[b] - end[b] > 64.0;
            if (lane == 0) m.steep[h][b] = steep;
            own_steep = lane >> 3 == b ? steep : own_steep;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (own_steep) across[i][3] = 0.0f;
#pragma unroll
            for (int b = 1; b < 4; ++b) across[i][b - 1] = fast_exp2(static_cast<float>(first[b] - total[i]));
          }
          // with the lengths of k, which the other warps find meanwhile
          if (base == 0) lengths_barrier();
#pragma unroll
          for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int t = 2 * lane + i;
              m.across[h][b][t] = lane >> 3 > b ? 0.0f : (lane >> 3 == b ? across[i][3] : across[i][b == 0 ? 0 : b - 1]) * m.length[t];
            }
          }
        } else if (base == 0) {
          lengths_barrier();
        }
      } else if (base == 0) {
        uint8_t* const pair = plan.pairs + (static_cast<size_t>(tile) * a.k_heads + k_head) * kChunkPairBytes;
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
        for (int i = 0; i < kPasses; ++i) {
          const int r = 8 * (warp + i * kRowWarps) + (lane >> 2);
          if (8 * (warp + i * kRowWarps) >= 2 * kChunk) break;
          uint4 data[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) data[p] = *reinterpret_cast<const uint4*>(m.rows + place(r, p));
          uint32_t most = 0;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            most = __vmaxu2(most, data[p].x & 0x7fff7fffu);
            most = __vmaxu2(most, data[p].y & 0x7fff7fffu);
            most = __vmaxu2(most, data[p].z & 0x7fff7fffu);
            most = __vmaxu2(most, data[p].w & 0x7fff7fffu);
          }
          most = max(most & 0xffffu, most >> 16);
          most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
          const bool bad = most >= 0x7f80u;
          // 2^-e with 2^e <= max < 2^(e + 1); a row of zeros, subnormal or broken: e as near as may be
          const int e = bad ? 0 : min(max(static_cast<int>(most >> 7) - 127, -126), 126);
          const float scale = kv_exp2(-e);
          float sum = 0.0f;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            float x[8];
            unpack8(data[p], x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              x[j] *= scale;
              sum = fmaf(x[j], x[j], sum);
            }
            uint4 packed = make_uint4(cvt_f16x2(x[0], x[1]), cvt_f16x2(x[2], x[3]), cvt_f16x2(x[4], x[5]), cvt_f16x2(x[6], x[7]));
            if (bad) packed = make_uint4(0, 0, 0, 0);
            const uint32_t at = place(r, p);
            *reinterpret_cast<uint4*>(m.pair + at) = packed;
            *reinterpret_cast<uint4*>(pair + at) = packed;
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if ((lane & 3) == 0) {
            // 2^e / sqrt(|x|^2 + eps) from |x 2^-e|^2
            m.length[r] = bad ? 0.0f : 1.0f / sqrtf(sum + a.eps * scale * scale);
            m.broken[r] = bad;
          }
        }
        fence_async_proxy();
        asm volatile("bar.arrive 1, %0;" :: "n"(kPrepareThreads) : "memory");       // the lengths are there, for the gates
        asm volatile("bar.sync 2, %0;" :: "n"(32 * kRowWarps) : "memory");
        if (warp == 0) {
          if (elect_one()) {
            constexpr uint32_t kForm = instr_desc_f8(kF16, kF16, 0, 0, 128, kChunk);
            const uint64_t desc = smem_desc_rows<128>(smem_u32(m.pair));
#pragma unroll
            for (int k = 0; k < kLinearDim / 16; ++k) {
              const uint64_t at = desc + (((k / 4) * kChunkPanelBytes + (k % 4) * 32) >> 4);
              umma_f16_ss(tmem, at, at, kForm, k != 0);
            }
            umma_commit(smem_u32(&m.done));
          }
          __syncwarp();
        }
      }
      if (base == 0) {
        alive = alive & mbar_wait_bounded_warp(smem_u32(&m.done), turn, &m.abort_flag, plan.wait_limit_ns);
        tc_fence_after();
      }
      __syncthreads();                                                 // the gates are there; A and the scores take the rows' place
      if (base == 0 && more) {
        // the next tile's rows and gates, while this one is gone through
        next = m.tiles[turn ^ 1];
        if (warp < kRowWarps) fetch_rows(k_head_after, next.row0, next.rows);
        else if (warp - kRowWarps < a.group) fetch_gates(k_head_after * a.group + warp - kRowWarps, next.row0, next.rows, next_a, next_b);
      }
      if (warp >= kRowWarps && warp - kRowWarps < heads) {
        // what the second kernel multiplies by
        const int head = k_head * a.group + base + warp - kRowWarps;
        ChunkNumbers* numbers = reinterpret_cast<ChunkNumbers*>(plan.heads + (static_cast<size_t>(tile) * a.v_heads + head) * kChunkHeadBytes + kChunkNumbersAt);
        const double pair0 = __shfl_sync(0xffffffffu, total[0], max(kept - 1, 0) >> 1), pair1 = __shfl_sync(0xffffffffu, total[1], max(kept - 1, 0) >> 1);
        const double last_kept = kept == 0 ? 0.0 : ((kept - 1) & 1) != 0 ? pair1 : pair0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = 2 * lane + i;
          const bool there = t < rows;
          const float k_length = m.length[t], q_length = m.length[kChunk + t], reach = exp2f(static_cast<float>(total[i]));
          numbers->rate[t] = beta[i];
          numbers->enter[t] = broken[i] || m.broken[t] != 0 ? NAN : there ? -(beta[i] * reach * k_length) : 0.0f;
          numbers->stay[t] = there ? exp2f(static_cast<float>(last - total[i])) * k_length : 0.0f;
          numbers->read[t] = !there ? 0.0f : m.broken[kChunk + t] != 0 ? NAN : reach * q_length;
          numbers->stay_kept[t] = t < kept ? exp2f(static_cast<float>(last_kept - total[i])) * k_length : 0.0f;
        }
        if (lane == 0) {
          numbers->decay = exp2f(static_cast<float>(last));
          numbers->decay_kept = exp2f(static_cast<float>(last_kept));
        }
      }
#pragma unroll 1
      for (int h = 0; h < heads; ++h) {
        uint8_t* const out = plan.heads + (static_cast<size_t>(tile) * a.v_heads + k_head * a.group + base + h) * kChunkHeadBytes;
        {
          // A, and the scores: a row of [k; q] and 32 columns a thread.  Columns behind the diagonal's block are not looked at again.
          const int beside = (warp & 1) - half;                        // rows of the two blocks that the columns are of: 0, behind them: 1
          if (beside >= 0) {
            const bool is_k = row < kChunk;
            Terms& to = is_k ? m.overlap : m.scores;
            const float own = (is_k ? m.rate[h][token] : 1.0f) * m.length[row], down = own * m.down[h][token];
            const int last_column = is_k ? token - 1 : token;
            const bool steep = m.steep[h][block] != 0;
#pragma unroll
            for (int q = 0; q < 2; ++q) {                              // 16 columns
              const int column = 32 * half + 16 * q;
              float x[16];
              tmem_ld16(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + column, reinterpret_cast<uint32_t*>(x));
              tmem_ld_wait();
              if (beside == 0 && steep && column >> 4 == block) {
                const float high = m.sum_high[h][token], low = m.sum_low[h][token];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  const float apart = fminf((high - m.sum_high[h][column + j]) + (low - m.sum_low[h][column + j]), 0.0f);
                  x[j] *= own * m.length[column + j] * fast_exp2(apart);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  const float4 y = *reinterpret_cast<const float4*>(&m.across[h][block][column + j]);
                  x[j] *= down * y.x;
                  x[j + 1] *= down * y.y;
                  x[j + 2] *= down * y.z;
                  x[j + 3] *= down * y.w;
                }
              }
              if (beside == 0) {
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = column + j <= last_column ? x[j] : 0.0f;
                if (is_k && column >> 4 == block) {
#pragma unroll
                  for (int j = 0; j < 16; j += 4)
                    *reinterpret_cast<float4*>(&m.diagonal[block][(token & 15) * kBlockRow + j]) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                }
              }
#pragma unroll
              for (int j = 0; j < 16; j += 8) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) split_f16(x[j + 2 * i], x[j + 2 * i + 1], &hi[i], &lo[i]);
                *reinterpret_cast<uint4*>(&to.of[0][token * kHalfRow + column + j]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(&to.of[1][token * kHalfRow + column + j]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            }
          }
        }
        __syncthreads();
        if (warp < 2) {
          // the diagonal's blocks: a column a thread
          const int b = 2 * warp + (lane >> 4), j = lane & 15;
          const float* at = m.diagonal[b];
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float y[16], sum = i == j ? 1.0f : 0.0f;
#pragma unroll
            for (int k = 0; k < i; k += 4) *reinterpret_cast<float4*>(y + k) = *reinterpret_cast<const float4*>(&at[i * kBlockRow + k]);
#pragma unroll
            for (int k = 0; k < i; ++k) sum = fmaf(-y[k], x[k], sum);
            x[i] = sum;
          }
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            uint32_t hi, lo;
            split_f16(x[i], x[i + 1], &hi, &lo);
            uint16_t* first = &m.inverse.of[0][(16 * b + i) * kHalfRow + 16 * b + j];
            uint16_t* second = &m.inverse.of[1][(16 * b + i) * kHalfRow + 16 * b + j];
            first[0] = static_cast<uint16_t>(hi);
            first[kHalfRow] = static_cast<uint16_t>(hi >> 16);
            second[0] = static_cast<uint16_t>(lo);
            second[kHalfRow] = static_cast<uint16_t>(lo >> 16);
          }
        } else {
          write_terms(m.scores, out + 2 * kChunkMatrixBytes, threadIdx.x - 64, kPrepareThreads - 64);
        }
        __syncthreads();
        // the blocks below the diagonal's, a column of them a warp
        if (warp < 3) {
          const int j = warp;
          uint32_t x[4][2][4];                                         // x[k]: the block of row j + k, transposed
#pragma unroll
          for (int term = 0; term < 2; ++term) load_transposed(&m.inverse.of[term][16 * j * kHalfRow + 16 * j], lane, x[0][term]);
#pragma unroll
          for (int d = 1; d < 4; ++d) {
            if (j + d < 4) {
              const int i = j + d;
              float sum[2][4] = {};
#pragma unroll
              for (int k = 0; k < d; ++k) add_product(sum, x[k], m.overlap, 16 * i, 16 * (j + k), lane);
              uint32_t y[2][4];
              as_operand(sum, -1.0f, y);
              float z[2][4] = {};
              add_product(z, y, m.inverse, 16 * i, 16 * i, lane);
              as_operand(z, 1.0f, x[d]);
#pragma unroll
              for (int term = 0; term < 2; ++term) store_transposed(&m.inverse.of[term][16 * i * kHalfRow + 16 * j], lane, x[d][term]);
            }
          }
        }
        __syncthreads();
        write_terms(m.inverse, out, threadIdx.x, kPrepareThreads);
      }
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
    }
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

cudaError_t linear_prepare(const ChunkPlan& plan, int sm_count, cudaStream_t stream) {
  constexpr int kBytes = static_cast<int>(sizeof(PrepareMemory)) + 1024;
  const cudaError_t error = opt_in_dynamic_smem<linear_prepare_kernel>(kBytes);
  if (error != cudaSuccess) return error;
  const int jobs = plan.tiles * plan.a.k_heads;
  linear_prepare_kernel<<<std::min(jobs, 2 * sm_count), kPrepareThreads, kBytes, stream>>>(plan);
  return cudaGetLastError();
}

}  // namespace aima
