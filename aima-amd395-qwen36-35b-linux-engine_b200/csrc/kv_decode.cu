// Attention of few rows per sequence (one new token, or a few drafted ones) over the paged 8-bit cache.
//
//   t_j = scale q . k_j  (log2 units) + log2(value scale of j's page),   w_j = 2^(t_j - m)
//   o   = sum_j w_j code(v_j) / sum_j w_j / (value scale of j's page)
// A page's scale of V is carried by the weight, so that V enters the product as the codes that lie in memory; the denominator is
// taken without it (kv_attention.cuh).
//
// Bound: the cache is read once, 2 head_dim bytes per position and key/value head, and the products with the 1 .. 16 rows
// that share them are small.  So the CACHE is the M side of both products, as it comes by TMA, and the rows are the N side:
//   S^T[128 positions, rows]   = K[128, head_dim] . Q^T            K-major A
//   O^T[head_dim, rows]       += V^T[head_dim, 128] . P^T           MN-major A: V's rows are the K dimension
// Nothing is unpacked to 16 bits.  A BF16 query is split into two e4m3 terms, q 2^-e = hi + lo / 16 -- exact but for elements
// below 2^-15 of the row's largest -- that are 2 x rows columns of one product.  A weight becomes an f16, w 2^14, and that three
// e5m2 terms, the upper bytes of it and of what is left of it, times 8 each time: w 2^14 = t0 + t1 / 8 + t2 / 64 to 2^-8.7 of
// itself where it exceeds 2^-28 of the largest and to 2^-36 of the largest below that.  (Without the factors of 8 the last terms of a
// small weight are subnormal; an e4m3 first term with an e5m2 remainder leaves 3 bits below 2^-18, which shows where one position outweighs
// all others and brings nothing.)  The terms are 3 x rows columns of one product, each with its accumulators.  All sums are FP32 in
// tensor memory.
//
// One block per SM; the list of all tiles is cut into equal shares (kv_attention.cuh).  Warp 0 loads tiles by page, warp 1
// issues the products, warps 2 and 3 prepare the queries of the next unit, warps 4-7 (thread = position) do the softmax and
// write the results.  S is double-buffered: the product of the next tile runs under the softmax of this one.  The running
// maximum moves only when a tile's exceeds it by more than kGrow, so the accumulators are rarely rescaled.
//
// Measured: 64 sequences of up to 8192 positions, one token, 16/2 heads of 256 (406 MB) 78 us = 5.2 TB/s, 80 % of a copy; two tokens 103:
// the softmax threads, which also bound heads of 128 (32/8, one token 190 us) and 64 (8/8, 188 us); one sequence of 32768 15.9 us, of which the
// tiles are 3 and the rest is a chain: cuts, queries, first scores, results, join.
#include "kv_attention.cuh"

namespace aima {
namespace {

constexpr int kThreads = 256;
constexpr float kGrow = 0.75f;            // 2^14 * 2^0.75 = 27554: a remainder times 8 rounds to at most 32768
constexpr float kWeightExponent = 14.0f;  // of the weights and of their sum alike
constexpr float kQueryLow = 16.0f;        // a remainder is at most 16: 256 <= 448 (0x4c00 as f16)
constexpr int kMaxPrefix = AIMA_MOE_KV_MAX_SEQUENCES + 1;

template <int kDim, int kRows>
struct Decode {
  static constexpr int kRowBytes = kDim >= 128 ? 128 : 64;
  static constexpr int kPanels = kDim / kRowBytes;
  static constexpr int kPanelBytes = kKvTile * kRowBytes;
  static constexpr int kSlotBytes = kKvTile * kDim;
  static constexpr int kSlots = kDim == 256 ? 6 : 8;
  static constexpr int kWeightRows = (3 * kRows + 15) / 16 * 16;        // N of the second product: three terms, and zeros
  static constexpr int kQueryBytes = 2 * kRows * kDim;
  static constexpr int kWeightBytes = kWeightRows * kKvTile;            // one buffer
  static constexpr int kOutPanels = kDim >= 128 ? kDim / 128 : 1;
  static constexpr int kOutColumn = 4 * kRows;                          // tensor memory: S0 | S1 | per panel the terms
  static constexpr int kQueryAt = kSlots * kSlotBytes;
  static constexpr int kWeightAt = kQueryAt + 2 * kQueryBytes;          // two segments' queries
  static constexpr int kPrefixAt = kWeightAt + 2 * kWeightBytes;
  static constexpr int kSmallAt = (kPrefixAt + kMaxPrefix * 4 + 15) / 16 * 16;
};

struct SegmentInfo {
  int length;               // positions of the sequence
  int rows;                 // rows of the unit
  int row0;                 // of q, the first one's
};

template <int kRows>
struct Small {              // shared memory that is not an operand
  unsigned long long full[8], empty[8];
  unsigned long long s_full[2], s_empty[2], p_full[2], o_done[2], q_full[2], info_empty[2], drain;
  alignas(16) float part[2][kRows][4];  // per row and warp: maxima of a tile (two buffers), sums at the end of a segment
  alignas(16) float low[kRows][4];      // scales far apart: maxima of a tile without them
  float row_scale[2][kRows];
  int limit[2][kRows];      // last position a row sees; -1: none
  long long out_at[2][kRows];
  SegmentInfo info[2];
  int scan[kThreads / 32];
  KvShared shared[2];       // the units divided at the share's begin and at its end
  int verdict;
  uint32_t tmem;
  int abort_flag;
};

// A block's share of the list, unit by unit.
struct Walk {
  const int* prefix;
  int heads;
  int at, end;
  int sequence;
  // the current segment
  int head, tile0, tiles, unit_tiles;
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    while (prefix[sequence + 1] <= at) ++sequence;
    unit_tiles = static_cast<int>(static_cast<uint32_t>(prefix[sequence + 1] - prefix[sequence]) / static_cast<uint32_t>(heads));
    const int within = at - prefix[sequence];
    head = static_cast<int>(static_cast<uint32_t>(within) / static_cast<uint32_t>(unit_tiles));
    tile0 = within - head * unit_tiles;
    tiles = min(unit_tiles - tile0, end - at);
    return true;
  }
  __device__ __forceinline__ void advance() { at += tiles; }
  __device__ __forceinline__ bool whole() const { return tiles == unit_tiles; }
};

// Eight reductions over the 32 lanes at once; lane l returns that of value reduce8_slot(l).
template <bool kMax>
__device__ __forceinline__ float reduce8(const float* v, int lane) {
  auto join = [](float x, float y) { return kMax ? fmaxf(x, y) : x + y; };
  const bool b4 = (lane & 16) != 0, b3 = (lane & 8) != 0, b2 = (lane & 4) != 0;
  float a[4], b[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = join(b4 ? v[j + 4] : v[j], __shfl_xor_sync(0xffffffffu, b4 ? v[j] : v[j + 4], 16));
#pragma unroll
  for (int j = 0; j < 2; ++j) b[j] = join(b3 ? a[j + 2] : a[j], __shfl_xor_sync(0xffffffffu, b3 ? a[j] : a[j + 2], 8));
  float c = join(b2 ? b[1] : b[0], __shfl_xor_sync(0xffffffffu, b2 ? b[0] : b[1], 4));
  c = join(c, __shfl_xor_sync(0xffffffffu, c, 2));
  return join(c, __shfl_xor_sync(0xffffffffu, c, 1));
}
__device__ __forceinline__ void softmax_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// ... and whether x holds in any of its threads
__device__ __forceinline__ bool softmax_barrier_or(bool x) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"(static_cast<uint32_t>(x)) : "memory");
  return any != 0;
}
__device__ __forceinline__ float max4(const float* at) {
  const float4 m = *reinterpret_cast<const float4*>(at);
  return fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
}

template <int kDim, int kRows>
__global__ void __launch_bounds__(kThreads, 1)
kv_decode_kernel(const __grid_constant__ KvMaps maps, const KvAttentionPlan plan) {
  using L = Decode<kDim, kRows>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* generic = smem_raw + (base - smem_u32(smem_raw));
  int* prefix = reinterpret_cast<int*>(generic + L::kPrefixAt);
  Small<kRows>& sm = *reinterpret_cast<Small<kRows>*>(generic + L::kSmallAt);
  volatile int* abort_flag = &sm.abort_flag;
  const KvAttention& a = plan.a;
  const KvShape& shape = a.shape;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 1);
      mbar_init(smem_u32(&sm.empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.s_empty[i]), 4);
      mbar_init(smem_u32(&sm.p_full[i]), 4);
      mbar_init(smem_u32(&sm.o_done[i]), 1);
      mbar_init(smem_u32(&sm.q_full[i]), 2);
      mbar_init(smem_u32(&sm.info_empty[i]), 4);
    }
    mbar_init(smem_u32(&sm.drain), 1);
    sm.abort_flag = 0;
    sm.shared[0].parts = sm.shared[1].parts = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc(smem_u32(&sm.tmem), 512);
  if (L::kWeightRows > 3 * kRows) {           // rows of the weights that are no term
    for (int i = threadIdx.x; i < 2 * L::kWeightBytes / 16; i += kThreads)
      *reinterpret_cast<uint4*>(generic + L::kWeightAt + 16 * i) = make_uint4(0, 0, 0, 0);
    fence_async_proxy();
  }
  pdl_enter();

  // tiles before each sequence; four sequences per thread
  {
    int mine[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = threadIdx.x * 4 + i;
      mine[i] = sum;
      if (s < a.batch.sequences) {
        const KvSequence seq = kv_sequence(a.batch, shape, s);
        if (seq.bad && blockIdx.x == 0) atomicOr(a.status, kKvBadBatch);
        if (seq.rows > 0) sum = min(kKvMaxList + 1, sum + (seq.length + kKvTile - 1) / kKvTile * shape.kv_heads);
      }
    }
    int run = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, run, d);
      if (lane >= d) run = min(kKvMaxList + 1, run + other);
    }
    if (lane == 31) sm.scan[warp] = run;
    __syncthreads();
    int before = run - sum;
    for (int w = 0; w < warp; ++w) before += sm.scan[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = threadIdx.x * 4 + i;
      if (s <= a.batch.sequences) prefix[s] = before + mine[i];
    }
    if (threadIdx.x == kThreads - 1 && a.batch.sequences == kThreads * 4) prefix[kThreads * 4] = before + sum;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  int total = prefix[a.batch.sequences];
  if (total > kKvMaxList) {
    if (threadIdx.x == 0) atomicOr(a.status, kKvBadBatch);
    total = 0;
  }
  const int blocks = min(static_cast<int>(gridDim.x), total);        // with a share; none is empty
  Walk walk;
  walk.prefix = prefix;
  walk.heads = shape.kv_heads;
  walk.at = walk.end = 0;
  if (static_cast<int>(blockIdx.x) < blocks) {
    walk.at = kv_cut(total, blockIdx.x, blocks);
    walk.end = kv_cut(total, blockIdx.x + 1, blocks);
  }
  walk.sequence = 0;
  auto wait = [&](unsigned long long* bar, uint32_t parity) { return mbar_wait_bounded_warp(smem_u32(bar), parity, abort_flag, plan.wait_limit_ns); };
  // Ring of K and V tiles, in the order in which the products take them: K0 K1 V0 K2 V1 .. V(n-2) V(n-1) of a segment.
  auto ring_k = [](int start, int j) { return start + (j == 0 ? 0 : 2 * j - 1); };
  auto ring_v = [](int start, int j, int n) { return start + (j + 1 < n ? 2 * j + 2 : 2 * n - 1); };

  if (warp == 0) {
    // ------------------------------ loads ------------------------------
    const int boxes = (kKvTile >> shape.page_shift) * L::kPanels;     // of a tile; a lane each
    const int my_page = lane / L::kPanels, my_panel = lane % L::kPanels;
    int ring = 0;
    bool alive = true;
    while (alive && walk.next()) {
      const KvSequence seq = kv_sequence(a.batch, shape, walk.sequence);
      const int* table = a.batch.table + static_cast<size_t>(walk.sequence) * a.batch.columns;
      const int pages = (seq.length + shape.page_tokens - 1) >> shape.page_shift;
      auto page_of = [&](int j) {          // of this lane's box; -1: behind the sequence's last, kNoPage: its table has none
        const int column = ((walk.tile0 + j) << (7 - shape.page_shift)) + my_page;
        if (j >= walk.tiles || lane >= boxes || column >= pages) return -1;
        int page = table[column];
        if (page < 0 || page >= shape.pages) {
          atomicOr(a.status, kKvBadBatch);
          page = kNoPage;
        }
        return page;
      };
      auto issue = [&](bool is_k, int page) {
        const int slot = ring % L::kSlots;
        if (!wait(&sm.empty[slot], ((ring / L::kSlots) & 1) ^ 1)) return false;
        const int loads = __popc(__ballot_sync(0xffffffffu, page != -1));
        if (lane == 0) mbar_arrive_expect_tx(smem_u32(&sm.full[slot]), loads * shape.page_tokens * L::kRowBytes);
        __syncwarp();
        if (page != -1)
          tma_load_2d(base + slot * L::kSlotBytes + my_panel * L::kPanelBytes + (my_page << shape.page_shift) * L::kRowBytes,
                      is_k ? &maps.keys : &maps.values, my_panel * L::kRowBytes,
                      page == kNoPage ? -shape.page_tokens : static_cast<int>((static_cast<long long>(page) * shape.kv_heads + walk.head) << shape.page_shift),
                      smem_u32(&sm.full[slot]));
        __syncwarp();
        ++ring;
        return true;
      };
      int page = page_of(0), next = page_of(1);
      alive = issue(true, page);
      for (int j = 0; j < walk.tiles && alive; ++j) {
        if (j + 1 < walk.tiles) alive = issue(true, next);
        alive = alive && issue(false, page);
        page = next;
        next = page_of(j + 2);
      }
      walk.advance();
    }
    if (*abort_flag != 0) {              // what is in flight lands before the block leaves
      volatile int ignore = 0;
      for (int i = max(0, ring - L::kSlots); i < ring; ++i) mbar_wait_bounded(smem_u32(&sm.full[i % L::kSlots]), (i / L::kSlots) & 1, &ignore);
    }
  } else if (warp == 1) {
    // ------------------------------ products ------------------------------
    constexpr uint32_t kScores = instr_desc_f8(kE4m3, kE4m3, 0, 0, 128, 2 * kRows);
    constexpr uint32_t kSums = instr_desc_f8(kE4m3, kE5m2, 1, 0, 128, L::kWeightRows);
    int ring = 0, tile = 0, segment = 0;
    bool alive = true;
    while (alive && walk.next()) {
      const int n = walk.tiles;
      auto scores = [&](int j) {
        const int r = ring_k(ring, j), slot = r % L::kSlots, buffer = (tile + j) & 1;
        if (!wait(&sm.full[slot], (r / L::kSlots) & 1) || !wait(&sm.s_empty[buffer], (((tile + j) >> 1) & 1) ^ 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t k0 = base + slot * L::kSlotBytes, q0 = base + L::kQueryAt + (segment & 1) * L::kQueryBytes;
#pragma unroll
          for (int k = 0; k < kDim / 32; ++k) {
            const int panel = k * 32 / L::kRowBytes, inside = k * 32 % L::kRowBytes;
            umma_f8(tmem + buffer * 2 * kRows, smem_desc_rows<L::kRowBytes>(k0 + panel * L::kPanelBytes) + (inside >> 4),
                    smem_desc_rows<L::kRowBytes>(q0 + panel * 2 * kRows * L::kRowBytes) + (inside >> 4), kScores, k != 0);
          }
          umma_commit(smem_u32(&sm.empty[slot]));
          umma_commit(smem_u32(&sm.s_full[buffer]));
        }
        __syncwarp();
        return true;
      };
      alive = wait(&sm.q_full[segment & 1], (segment >> 1) & 1) && scores(0);
      for (int j = 0; j < n && alive; ++j) {
        if (j + 1 < n && !scores(j + 1)) { alive = false; break; }
        const int r = ring_v(ring, j, n), slot = r % L::kSlots, buffer = (tile + j) & 1;
        if (!wait(&sm.p_full[buffer], ((tile + j) >> 1) & 1) || !wait(&sm.full[slot], (r / L::kSlots) & 1)) { alive = false; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t v0 = base + slot * L::kSlotBytes, p0 = base + L::kWeightAt + buffer * L::kWeightBytes;
#pragma unroll
          for (int panel = 0; panel < L::kOutPanels; ++panel) {
            const uint32_t d = tmem + L::kOutColumn + panel * L::kWeightRows;
#pragma unroll
            for (int k = 0; k < kKvTile / 32; ++k) {
              // head_dim 64: the instruction's upper 64 rows read the next slot (or the queries); nothing reads them
              const uint64_t v = smem_desc_rows<L::kRowBytes>(v0 + panel * L::kPanelBytes + k * 32 * L::kRowBytes, L::kPanelBytes);
              umma_f8(d, v, smem_desc_rows<128>(p0) + k * 2, kSums, (j | k) != 0);
            }
          }
          umma_commit(smem_u32(&sm.empty[slot]));
          umma_commit(smem_u32(&sm.o_done[buffer]));
        }
        __syncwarp();
      }
      ring += 2 * n;
      tile += n;
      ++segment;
      walk.advance();
    }
  } else if (warp < 4) {
    // ------------------------------ queries ------------------------------
    constexpr int kPer = kDim / 32;
    int segment = 0;
    bool alive = true;
    while (alive && walk.next()) {
      const KvSequence seq = kv_sequence(a.batch, shape, walk.sequence);
      const int rows = seq.rows * shape.group, which = segment & 1;
      // empty once the segment before the last has been finished: its products too
      if (!wait(&sm.info_empty[which], ((segment >> 1) & 1) ^ 1)) break;
      if (warp == 2 && lane == 0) sm.info[which] = SegmentInfo{seq.length, rows, seq.row0};
#pragma unroll 1
      for (int r0 = 4 * (warp - 2); r0 < kRows; r0 += 8) {       // four rows side by side: one alone is a chain of 340 cycles
        uint32_t raw[4][kPer / 2];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int r = r0 + b, i = r / shape.group, g = r - i * shape.group;
          const int head = walk.head * shape.group + g;
          const __nv_bfloat16* at = a.q.data + (seq.row0 + i) * a.q.row_stride + head * a.q.head_stride + lane * kPer;
#pragma unroll
          for (int e = 0; e < kPer / 2; ++e) raw[b][e] = 0;
          if (r < rows) {
            if constexpr (kPer == 8) {
              const uint4 v = *reinterpret_cast<const uint4*>(at);
              raw[b][0] = v.x; raw[b][1] = v.y; raw[b][2] = v.z; raw[b][3] = v.w;
            } else if constexpr (kPer == 4) {
              const uint2 v = *reinterpret_cast<const uint2*>(at);
              raw[b][0] = v.x; raw[b][1] = v.y;
            } else {
              raw[b][0] = *reinterpret_cast<const uint32_t*>(at);
            }
          }
          if (lane == 0) {
            sm.limit[which][r] = r < rows ? seq.length - seq.rows + i : -1;
            sm.out_at[which][r] = ((seq.row0 + i) * static_cast<long long>(shape.q_heads) + head) * kDim;
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int r = r0 + b;
          uint32_t largest = 0;            // magnitudes as integers: infinities and NaN come last
#pragma unroll
          for (int e = 0; e < kPer / 2; ++e) largest = max(largest, max(raw[b][e] & 0x7fffu, (raw[b][e] >> 16) & 0x7fffu));
          largest = __reduce_max_sync(0xffffffffu, largest);
          const bool finite = largest < 0x7f80u;
          const int exponent = kv_scale_exponent(__uint_as_float(largest << 16));
          const float inverse = kv_exp2(-exponent);
          uint32_t codes[2][kPer / 2];
#pragma unroll
          for (int e = 0; e < kPer / 2; ++e) {
            const uint32_t h = cvt_f16x2(bf16_lo(raw[b][e]) * inverse, bf16_hi(raw[b][e]) * inverse);
            codes[0][e] = finite ? cvt_e4m3x2_f16x2(h) : kKvNan * 0x0101u;
            codes[1][e] = finite ? cvt_e4m3x2_f16x2(mul_f16x2(sub_f16x2(h, e4m3x2_f16x2(codes[0][e])), 0x4c004c00u)) : 0u;       // times 16
          }
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            const uint32_t* c = codes[term];
            const int row = r + term * kRows, byte = lane * kPer;
            const int panel = byte / L::kRowBytes, inside = byte % L::kRowBytes;
            const int piece = (inside >> 4) ^ (L::kRowBytes == 128 ? row & 7 : (row >> 1) & 3);
            uint8_t* to = generic + L::kQueryAt + which * L::kQueryBytes + (panel * 2 * kRows + row) * L::kRowBytes + piece * 16 + (inside & 15);
            if constexpr (kPer == 8) *reinterpret_cast<uint2*>(to) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
            else if constexpr (kPer == 4) *reinterpret_cast<uint32_t*>(to) = c[0] | (c[1] << 16);
            else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(c[0]);
          }
          if (lane == 0) sm.row_scale[which][r] = kv_exp2(exponent) * a.scale_log2;
        }
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.q_full[which]));
      ++segment;
      walk.advance();
    }
  } else {
    // ------------------------------ softmax and results ------------------------------
    const int quarter = warp - 4, token = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    int ring = 0, tile = 0, segment = 0;
    // No wait that runs out leaves this loop: the other warps of the group meet this one at its barriers, and every wait
    // after the first that ran out ends at once.
    while (walk.next()) {
      const int n = walk.tiles, which = segment & 1;
      const int* table = a.batch.table + static_cast<size_t>(walk.sequence) * a.batch.columns;
      wait(&sm.q_full[which], (segment >> 1) & 1);
      const int length = sm.info[which].length;
      auto page_of = [&](int j) {          // of this thread's position; -1: it has none
        const int position = (walk.tile0 + j) * kKvTile + token;
        if (j >= n || position >= length) return -1;
        const int page = table[position >> shape.page_shift];
        return page < 0 || page >= shape.pages ? -1 : page;
      };
      auto scales_of = [&](int page) {
        if (page < 0) return make_float2(0.0f, 1.0f);
        const size_t at = static_cast<size_t>(page) * shape.kv_heads + walk.head;
        return make_float2(a.layer.key_scales[at], a.layer.value_scales[at]);
      };
      float top[kRows], weights[kRows], low[kRows];      // low: once scales are apart
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        top[r] = low[r] = -INFINITY;
        weights[r] = 0.0f;
      }
      bool apart = false;                  // the same in all threads
      int page = page_of(0), page_next = page_of(1);
      float2 scales = scales_of(page);
      const int page_first = table[(walk.tile0 * kKvTile) >> shape.page_shift];
      const float first = page_first < 0 || page_first >= shape.pages
                              ? 0.0f : static_cast<float>(kv_float_exponent(a.layer.value_scales[static_cast<size_t>(page_first) * shape.kv_heads + walk.head]));
      for (int j = 0; j < n; ++j, ++tile) {
        const int buffer = tile & 1;
        const float2 scales_next = scales_of(page_next);
        const int page_after = page_of(j + 2);
        const int position = page >= 0 ? (walk.tile0 + j) * kKvTile + token : 0x7fffffff;
        const float value_log2 = log2f(scales.y);
        wait(&sm.s_full[buffer], (tile >> 1) & 1);
        tc_fence_after();
        float t[kRows];
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += 8) {
          uint32_t hi[8], lo[8];
          tmem_ld8(tmem + lanes + buffer * 2 * kRows + r0, hi);
          tmem_ld8(tmem + lanes + buffer * 2 * kRows + kRows + r0, lo);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float s = fmaf(__uint_as_float(lo[i]), 1.0f / kQueryLow, __uint_as_float(hi[i]));
            t[r0 + i] = position <= sm.limit[which][r0 + i] ? fmaf(s, scales.x * sm.row_scale[which][r0 + i], value_log2) : -INFINITY;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.s_empty[buffer]));
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += 8) {
          const float m = reduce8<true>(t + r0, lane);
          if ((lane & 3) == 0) sm.part[buffer][r0 + reduce8_slot(lane)][quarter] = m;
        }
        const bool was_apart = apart;
        apart = softmax_barrier_or(apart || (page >= 0 && fabsf(value_log2 - first) > kKvApart));
        if (__builtin_expect(apart, 0)) {
#pragma unroll
          for (int r0 = 0; r0 < kRows; r0 += 8) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = t[r0 + i] - value_log2;
            const float m = reduce8<true>(s, lane);
            if ((lane & 3) == 0) sm.low[r0 + reduce8_slot(lane)][quarter] = m;
          }
          softmax_barrier();
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float from = was_apart ? low[r] : top[r] - first;
            low[r] = fmaxf(from, max4(sm.low[r]));
            if (from != low[r]) weights[r] *= fast_exp2(from - low[r]);
            weights[r] += fast_exp2(t[r] - value_log2 + (kWeightExponent - (low[r] == -INFINITY ? 0.0f : low[r])));
          }
        }
        const float value_inverse = apart ? 0.0f : fast_exp2(first - value_log2);
        auto grown = [&](int r) {          // the reference maximum after this tile
          const float m = max4(sm.part[buffer][r]);
          return m > top[r] + kGrow || (top[r] == -INFINITY && m > top[r]) ? m : top[r];
        };
        bool grows = false;                // the same in all threads
#pragma unroll
        for (int r = 0; r < kRows; ++r) grows = grows || grown(r) != top[r];
        if (grows) {
          if (j > 0) {
            wait(&sm.o_done[buffer ^ 1], ((tile - 1) >> 1) & 1);
            tc_fence_after();
          }
#pragma unroll
          for (int r0 = 0; r0 < kRows; r0 += 8) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float to = grown(r0 + i);
              f[i] = top[r0 + i] == to ? 1.0f : fast_exp2(top[r0 + i] - to);
              if (!apart) weights[r0 + i] *= f[i];
              top[r0 + i] = to;
            }
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < 3 * L::kOutPanels; ++c) {
                const uint32_t at = tmem + lanes + L::kOutColumn + c / 3 * L::kWeightRows + c % 3 * kRows + r0;
                uint32_t o[8];
                tmem_ld8(at, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f[i]);
                tmem_st8(at, o);
              }
            }
          }
          tmem_st_wait();
        }
        // the buffer of the weights is free once the product of two tiles ago has read it
        wait(&sm.o_done[buffer], ((tile >> 1) & 1) ^ 1);
        uint8_t* terms = generic + L::kWeightAt + buffer * L::kWeightBytes;
#pragma unroll
        for (int r = 0; r < kRows; r += 2) {
          float w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            w[i] = fast_exp2(t[r + i] + (kWeightExponent - (top[r + i] == -INFINITY ? 0.0f : top[r + i])));
            weights[r + i] = fmaf(w[i], value_inverse, weights[r + i]);
          }
          uint32_t h = cvt_f16x2(w[0], w[1]);
          const int at = r * 128 + (token & 15), piece = token >> 4;
#pragma unroll
          for (int term = 0; term < 3; ++term) {
            const uint32_t codes = term < 2 ? h : h + 0x00800080u;        // two cut off, the last rounded
            terms[term * kRows * 128 + at + ((piece ^ (r & 7)) << 4)] = static_cast<uint8_t>(codes >> 8);
            terms[term * kRows * 128 + at + 128 + ((piece ^ ((r + 1) & 7)) << 4)] = static_cast<uint8_t>(codes >> 24);
            if (term < 2) h = mul_f16x2(sub_f16x2(h, h & 0xff00ff00u), 0x48004800u);        // times 8
          }
        }
        if (j + 1 == n && (walk.tile0 + n) * kKvTile > length) {
          // behind the sequence's end a page can hold anything, and zero weights do not stop a NaN
          const int r = ring_v(ring, j, n), slot = r % L::kSlots;
          wait(&sm.full[slot], (r / L::kSlots) & 1);
          if ((walk.tile0 + j) * kKvTile + token >= length) {
#pragma unroll
            for (int c = 0; c < kDim / 16; ++c)
              *reinterpret_cast<uint4*>(generic + slot * L::kSlotBytes + (c * 16 / L::kRowBytes) * L::kPanelBytes + token * L::kRowBytes +
                                        c * 16 % L::kRowBytes) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_proxy();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[buffer]));
        page = page_next;
        page_next = page_after;
        scales = scales_next;
      }
      // the unit's sums, or this block's part of them
      const int last = (tile - 1) & 1;
#pragma unroll
      for (int r0 = 0; r0 < kRows; r0 += 8) {
        const float sum = reduce8<false>(weights + r0, lane);
        if ((lane & 3) == 0) sm.part[last ^ 1][r0 + reduce8_slot(lane)][quarter] = sum;
      }
      softmax_barrier();
      wait(&sm.o_done[last], ((tile - 1) >> 1) & 1);
      tc_fence_after();
      const bool whole = walk.whole(), begins = walk.tile0 == 0;
      const size_t part = kv_part_index(blockIdx.x, begins);
      const int rows = sm.info[which].rows;
      if (!whole && token == 0) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 s4 = *reinterpret_cast<const float4*>(sm.part[last ^ 1][r]);
          if (r < rows) *kv_part_weight(plan.work, part, r) = make_float4(top[r], (s4.x + s4.y) + (s4.z + s4.w), apart ? low[r] : top[r] - first, 0.0f);
        }
        // the block of tile t is the last whose cut is not behind it: the one before the first cut at t + 1 or later
        const int first = walk.at - walk.tile0;
        const int block0 = begins ? static_cast<int>(blockIdx.x) : kv_first_cut(first + 1, total, blocks) - 1;
        const int block1 = kv_first_cut(first + walk.unit_tiles, total, blocks) - 1;
        sm.shared[begins ? 1 : 0] = KvShared{block0, block1 - block0 + 1, static_cast<int>(blockIdx.x) - block0, rows, sm.info[which].row0,
                                             walk.head * shape.group};
      }
#pragma unroll 1
      for (int panel = 0; panel < L::kOutPanels; ++panel) {
        const int d = panel * 128 + token;
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += 8) {
          uint32_t o[3][8];
#pragma unroll
          for (int term = 0; term < 3; ++term) tmem_ld8(tmem + lanes + L::kOutColumn + panel * L::kWeightRows + term * kRows + r0, o[term]);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = r0 + i;
            if (r >= rows || d >= kDim) continue;
            const float x = fmaf(__uint_as_float(o[2][i]), 1.0f / 64.0f, fmaf(__uint_as_float(o[1][i]), 1.0f / 8.0f, __uint_as_float(o[0][i])));
            if (whole) {
              const float4 s4 = *reinterpret_cast<const float4*>(sm.part[last ^ 1][r]);
              const float sum = (s4.x + s4.y) + (s4.z + s4.w);
              const float2 back = kv_exp2_factors(!apart ? first : top[r] == -INFINITY ? 0.0f : top[r] - low[r]);
              a.out[sm.out_at[which][r] + d] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : x / sum * back.x * back.y);
            } else {
              kv_part_sum<kDim>(plan.work, part, r, d & ~3)[d & 3] = x;
            }
          }
        }
      }
      tc_fence_before();
      softmax_barrier();                   // part is read by all before the next segment writes it
      if (lane == 0) mbar_arrive(smem_u32(&sm.info_empty[which]));
      ring += 2 * n;
      ++segment;
      walk.advance();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // a wait ran out: the copies have been waited for above, and so are the products under way, by a last commit
    volatile int ignore = 0;
    if (threadIdx.x == 0) atomicOr(a.status, kKvTimeout);
    if (warp == 1 && elect_one()) umma_commit(smem_u32(&sm.drain));
    if (threadIdx.x == 0) mbar_wait_bounded(smem_u32(&sm.drain), 0, &ignore);
    __syncthreads();
  }
  if (warp == 2) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i)
      if (sm.shared[i].parts > 0) kv_arrive(plan.work, sm.shared[i]);
  }
  // sequences without anything in the cache
  for (int s = blockIdx.x; s < a.batch.sequences; s += gridDim.x) {
    if (prefix[s + 1] != prefix[s]) continue;
    const KvSequence seq = kv_sequence(a.batch, shape, s);
    kv_zero_rows<kDim, kThreads>(a, seq.row0, seq.rows);
  }
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (sm.shared[i].parts > 0) kv_join<kDim, kThreads>(a, plan.work, sm.shared[i], plan.wait_limit_ns, &sm.verdict);
  }
}

template <int kDim, int kRows>
cudaError_t launch(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream) {
  constexpr int bytes = kv_smem_bytes(Decode<kDim, kRows>::kSmallAt + static_cast<int>(sizeof(Small<kRows>)) + 1024);
  static_assert(bytes <= 227 * 1024, "more shared memory than a block can have");
  const cudaError_t error = opt_in_dynamic_smem<kv_decode_kernel<kDim, kRows>>(bytes);
  if (error != cudaSuccess) return error;
  return launch_resident(kv_decode_kernel<kDim, kRows>, dim3(plan.blocks), dim3(kThreads), bytes, stream, maps, plan);
}

template <int kDim>
cudaError_t launch_rows(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream) {
  // N of the products: 8 rows in the kernel for 16 take 20.6 us instead of 16.0 (one sequence of 32768), 96 instead of 79 (64 of 8192).
  // Heads of 64 and 128 come with 8 rows at most.
  if constexpr (kDim == 256) {
    if (plan.tile_rows > 8) return launch<kDim, 16>(plan, maps, stream);
  }
  return launch<kDim, 8>(plan, maps, stream);
}

}  // namespace

cudaError_t kv_decode(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream) {
  switch (plan.a.shape.head_dim) {
    case 64: return launch_rows<64>(plan, maps, stream);
    case 128: return launch_rows<128>(plan, maps, stream);
    default: return launch_rows<256>(plan, maps, stream);
  }
}

}  // namespace aima
