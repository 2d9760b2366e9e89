// Attention of many rows per sequence (chunks of prompts) over the paged 8-bit cache.
//
//   t_ij = scale q_i . k_j (log2 units) + log2(value scale of j's page),   w_ij = 2^(t_ij - m_i)
//   o_i  = sum_j w_ij code(v_j) / sum_j w_ij / (value scale of j's page)
// as in kv_decode.cu (and the denominator as in kv_attention.cuh), here with the rows as the M side.  A row tile is up to 128 rows:
// whole new tokens x the query heads that share a key/value head, so that K and V are loaded once for all of them.
//
// Bound: the products, 4 x rows x positions x head_dim flops at the rate of 16-bit ones.  Queries and weights are BF16-like, the
// cache is e4m3, and no operand of mixed width exists.  So Q is split into two 8-bit terms and its product runs twice at twice the rate:
//   q 2^-e  = hi (e4m3) + lo (e5m2)          exact down to 2^-16 (largest 448)
// Weights and values, heads of 256:
//   w 2^9   = three terms (e5m2)             to 2^-8 of itself where it exceeds 2^-9, to 2^-17 below
// An e5m2 number is the upper byte of an f16, so the weights' terms take no conversions; two terms with an e4m3 first one would
// take a fifth less of the tensor cores but hold weights below 2^-13 of the largest to a few bits only, which is not enough where
// one position outweighs all others and brings nothing.  Heads of 64 and 128 (kWide), whose softmax takes longer than their products:
//   w 2^9   = one f16                        to 2^-11 of itself down to 2^-23 of the largest
// with V's codes as f16, which they are exactly, in a second pair of buffers (heads of 256 would need 128 KB for them).  That saves the
// softmax 13 of 23 instructions per four weights and the tensor cores a third of the second product; the softmax warps widen V on
// the way.  4096 tokens of 16384 with 32/8 heads of 128 1235 us in three terms and 1090 this way, with 8/8 of 64 275 and 242 (both before
// the denominator had a reference of its own: now 1090 .. 1113 and 239 .. 249).
// All terms of an operand go into one accumulator.  S[128 rows, 128 positions] = Q K^T with both operands in shared memory;
// O[128, head_dim] += W V with W in tensor memory, where it takes the place of the scores it was made from, and V MN-major.
//
// One block per SM.  Warp 0 loads tiles by page, warp 1 issues the products, warp 3 fetches the scales; warps 4-7 and 8-11 (thread =
// row) each turn half of a tile's scores into weights; two warps with the same rows exchange their maxima in between.
// The scores are double-buffered: the products of one tile run under the softmax of another.
//
// Measured: 8192 tokens of 32768 with 16/2 heads of 256 3.75 ms = 1.03 PFLOP/s at the 1.5 GHz that the power cap leaves, 2560 cycles
// of products in the 3300 of a tile: both operands of Q K^T come from shared memory at its full rate while the next tiles are
// written there.  With heads of 128 a tile takes 2250 cycles, which its softmax needs (a chain of V's widening, maxima, an exchange and 64
// weights per thread on two warps per scheduler), the products 1050: 7 prompts of 1531 .. 2999 with 32/8 heads 354 us.  1024
// tokens of 16/2 heads of 256 alone 28 us, most of it before the first tile and after the last.
#include "kv_attention.cuh"

namespace aima {
namespace {

constexpr int kThreads = 384;
// The reference of a row's weights moves up when a tile's maximum exceeds it by more than kGrow, and down when a tile's maximum
// falls short of it by more than kFall, where the weights get few bits.  It stays within kDepth of the row's maximum so that
// nothing overflows.
constexpr float kGrow = 6.75f;            // 2^9 * 2^6.75 = 55109 <= 57344
// Of three terms the last is subnormal where a weight is small, so a row's first maximum, and one that exceeds all before it by more than
// kJump, is placed kLift above the reference: the other weights of its tile keep 2^-8 of themselves down to 2^-22 of it instead of
// 2^-18, which shows where one position outweighs all others and brings nothing.  The next time that a row of the warp moves, the
// others give the lift back, so that ordinary scores, whose maximum grows slowly, rescale once or twice more per unit.  (Always so
// little room above the maximum: 4096 tokens of 16384 955 -> 1006 us.)  A whole number: the largest weight, which often is a third of
// the row's, then is a power of two and exact; at 2^13.75 it is rounded up by 2^-9.8, in every row.
constexpr float kLift = 4.0f;
constexpr float kJump = 8.0f;
constexpr float kFall = 16.0f;
constexpr float kDepth = 30.0f;
constexpr float kWeightExponent = 9.0f;
constexpr int kScaleSlots = 4;
constexpr int kApart = 256;               // of a tile's marks: value scales of the segment so far are far apart
constexpr int kStageBytes = 32 * 64;      // of a warp: 32 rows x 32 results

template <int kDim>
struct Prompt {
  static constexpr int kRowBytes = kDim >= 128 ? 128 : 64;
  static constexpr int kPanels = kDim / kRowBytes;
  static constexpr int kPanelBytes = kKvTile * kRowBytes;
  static constexpr int kSlotBytes = kKvTile * kDim;
  static constexpr bool kWide = kDim <= 128;                            // weights and values in 16 bits
  static constexpr int kWideBytes = kWide ? kKvTile * kDim * 2 : 0;     // a tile of V, rows of 64 values per panel
  static constexpr int kSlots = kDim == 256 ? 4 : kDim == 128 ? 6 : 8;
  static constexpr int kQueryAt = kSlots * kSlotBytes;                  // hi, then lo
  static constexpr int kWideAt = kQueryAt + 2 * kSlotBytes;
  static constexpr int kStageAt = kWideAt + 2 * kWideBytes;
  static constexpr int kSmallAt = kStageAt + 8 * kStageBytes;
  static constexpr int kScoreColumn = 256;                              // tensor memory: O | S0 | S1
};

struct Small {
  float4 scales[kScaleSlots][8];           // per 16 positions: key scale x softmax scale, log2 of the value scale, 2^e / value scale (0: far apart)
  int2 marks[kScaleSlots];                 // a bit for each 16 positions without a page, and kApart; e
  unsigned long long full[8], empty[8], scales_full[kScaleSlots], scales_empty[kScaleSlots];
  unsigned long long s_full[2], p_full[2], o_done[2], q_raw, q_full, q_empty, drain;
  float row_scale[128];
  float half_top[2][2][128];               // per tile parity, half and row
  float half_low[2][128];                  // scales far apart: the same without them
  float sum[2][2][128];                    // per parity of the unit, half and row
  KvStart cut[2];
  KvShared shared[2];                      // the units divided at the share's begin and at its end
  int verdict;
  uint32_t tmem;
  int abort_flag;
};

// A unit of the list: the rows of `tokens` new tokens of a sequence, for the query heads of one key/value head.
struct KvUnit {
  int tokens;             // new tokens of the row tile
  int first;              // position of the first one (negative: it sees nothing)
  int tiles;              // tiles of the cache that the last one sees
};
__device__ __forceinline__ KvUnit kv_unit(const KvSequence& seq, int row_tile, int tile_tokens) {
  KvUnit u;
  const int before = row_tile * tile_tokens;
  u.tokens = min(tile_tokens, seq.rows - before);
  u.first = seq.length - seq.rows + before;
  u.tiles = max(0, u.first + u.tokens + kKvTile - 1) / kKvTile;
  return u;
}

// A block's share of the list, unit by unit: from one cut to the next.
struct Walk {
  const KvAttentionPlan* plan;
  int sequence, row_tile, head, tile0, tiles;
  int end_sequence, end_row_tile, end_head, end_tile;
  KvSequence seq;
  KvUnit unit;
  int row_tiles;
  __device__ __forceinline__ void begin(const KvAttentionPlan& p, const KvStart& start, const KvStart& end) {
    plan = &p;
    sequence = start.sequence;
    row_tile = start.row_tile;
    head = start.head;
    tile0 = start.tile;
    end_sequence = end.sequence;
    end_row_tile = end.row_tile;
    end_head = end.head;
    end_tile = end.tile;
    seq = KvSequence{start.row0, start.rows, start.length, false};
    row_tiles = (seq.rows + plan->tile_tokens - 1) / plan->tile_tokens;
  }
  __device__ __forceinline__ bool next() {
    for (;;) {
      int most = 0x7fffffff;
      if (sequence == end_sequence && row_tile == end_row_tile && head == end_head) {
        most = end_tile - tile0;
        if (most <= 0) return false;
      }
      if (row_tile < row_tiles) {
        unit = kv_unit(seq, row_tile, plan->tile_tokens);
        tiles = min(unit.tiles - tile0, most);
        if (tiles > 0) return true;
        tile0 = 0;
        if (unit.tiles > 0 && ++head < plan->a.shape.kv_heads) continue;
        head = 0;
        ++row_tile;
      } else {
        row_tile = 0;
        ++sequence;
        seq = kv_sequence(plan->a.batch, plan->a.shape, sequence);
        row_tiles = (seq.rows + plan->tile_tokens - 1) / plan->tile_tokens;
      }
    }
  }
  __device__ __forceinline__ void advance() { tile0 += tiles; }
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// two FP32 operations per instruction
__device__ __forceinline__ unsigned long long both(float2 x) { return __float_as_uint(x.x) | (static_cast<unsigned long long>(__float_as_uint(x.y)) << 32); }
__device__ __forceinline__ float2 both(unsigned long long x) { return make_float2(__uint_as_float(static_cast<uint32_t>(x)), __uint_as_float(static_cast<uint32_t>(x >> 32))); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(both(a)), "l"(both(b)), "l"(both(c)));
  return both(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return both(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return both(r);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^t without the exponential unit: t = n + f with n whole and |f| <= 1/2, 2^f by the polynomial of degree 3 whose largest relative error
// is the least (2^-13.7, found by exchange), 2^n put together from n + 127.  Below -127 it is 0, NaN stays NaN.  A quarter of the
// exponentials of kWide go this way, whose unit would otherwise be busy for 1024 cycles of a tile: 4096 of 16384 with 32/8 heads
// of 128 1192 -> 1150 us, with three eighths 1164, with half 1177; in the three-term form every one of them lost time.
__device__ __forceinline__ float2 exp2_by_polynomial(float2 t) {
  constexpr float kMagic = 12582912.0f + 127.0f;         // 1.5 * 2^23: the sum's low bits are n + 127
  t.x = max_nan(t.x, -127.0f);
  t.y = max_nan(t.y, -127.0f);
  const float2 shifted = add2(t, make_float2(kMagic, kMagic));
  const float2 f = add2(t, fma2(shifted, make_float2(-1.0f, -1.0f), make_float2(kMagic, kMagic)));
  float2 p = fma2(f, make_float2(0.055171665f, 0.055171665f), make_float2(0.24261113f, 0.24261113f));
  p = fma2(p, f, make_float2(0.69326097f, 0.69326097f));
  p = fma2(p, f, make_float2(0.99992806f, 0.99992806f));
  return mul2(p, make_float2(__uint_as_float(__float_as_uint(shifted.x) << 23), __uint_as_float(__float_as_uint(shifted.y) << 23)));
}
// row / group for rows below 128, with inverse = ceil(2^16 / group)
__device__ __forceinline__ int row_token(int row, int inverse) { return (row * inverse) >> 16; }
__device__ __forceinline__ void group_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// Four weights as f16 pairs -> four e5m2 codes of each of three terms: two cut off, the last rounded.
__device__ __forceinline__ void split_weights(uint32_t h0, uint32_t h1, uint32_t* terms, int stride) {
#pragma unroll
  for (int term = 0; term < 2; ++term) {
    terms[term * stride] = __byte_perm(h0, h1, 0x7531);
    h0 = sub_f16x2(h0, h0 & 0xff00ff00u);
    h1 = sub_f16x2(h1, h1 & 0xff00ff00u);
  }
  terms[2 * stride] = __byte_perm(h0 + 0x00800080u, h1 + 0x00800080u, 0x7531);
}

// Cuts the list into shares of equal cost.  The list runs over sequences, their row tiles, the key/value heads and the
// tiles of the cache; a unit costs its tiles and kUnitCost more, for its queries, the first scores that nothing overlaps and
// its results.  A cut within kv_snap tiles of a unit's end moves there: a divided unit costs all that twice, and the join.  Units
// that several cuts divide anyway are left closer to equal shares (of no more than one tile: 16 sequences x 40 rows of 4111 28.7 us
// and 31.0 with two; 1024 tokens, whose units of 1 .. 8 tiles two tiles keep whole, 27.9 and 36.9 with one).  One block; items are row
// tiles, one for a thread at a time.  emit(c, start) is called for the cuts c in [cut0, cut1], by some thread; nothing(item, row0, rows)
// for an item whose rows see nothing.
constexpr int kUnitCost = 3;
__device__ __forceinline__ int kv_snap(int tiles, int total, int blocks) { return static_cast<long long>(tiles) * blocks <= 2ll * total ? 2 : 1; }
template <int kThreadCount>
struct PlanMemory {
  int first_item[AIMA_MOE_KV_MAX_SEQUENCES + 1];
  int warp_sum[kThreadCount / 32];
};
template <int kThreadCount, typename Emit, typename Nothing>
__device__ __forceinline__ void plan_list(const KvAttentionPlan& plan, PlanMemory<kThreadCount>& memory, int cut0, int cut1, Emit emit, Nothing nothing) {
  const KvAttention& a = plan.a;
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  const int heads = a.shape.kv_heads;
  auto scan = [&](int x, int* all) {                     // inclusive, over the block
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x = min(kKvMaxList + 1, x + other);
    }
    __syncthreads();                                     // the scan before has been read
    if (lane == 31) memory.warp_sum[warp] = x;
    __syncthreads();
    *all = 0;
    for (int w = 0; w < kThreadCount / 32; ++w) {
      const int s = memory.warp_sum[w];
      if (w < warp) x = min(kKvMaxList + 1, x + s);
      *all = min(kKvMaxList + 1, *all + s);
    }
    return x;
  };
  int items_so_far = 0;
  for (int s0 = 0; s0 < a.batch.sequences; s0 += kThreadCount) {
    int mine = 0;
    if (s0 + thread < a.batch.sequences) {
      const KvSequence seq = kv_sequence(a.batch, a.shape, s0 + thread);
      if (seq.bad) atomicOr(a.status, kKvBadBatch);
      mine = (seq.rows + plan.tile_tokens - 1) / plan.tile_tokens;
    }
    int all;
    const int upto = scan(mine, &all) + items_so_far;
    if (s0 + thread < a.batch.sequences) memory.first_item[s0 + thread + 1] = upto;
    items_so_far += all;
  }
  if (thread == 0) memory.first_item[0] = 0;
  __syncthreads();
  const int items = items_so_far;
  int total = 0;
  // Items for which the threads suffice need one scan; more are gone through twice, for the total and for the cuts.
  for (int pass = items > kThreadCount ? 0 : 1; pass < 2; ++pass) {
    int before = 0;
    for (int item0 = 0; item0 < items; item0 += kThreadCount) {
      const int item = item0 + thread;
      int s = 0, row_tile = 0;
      KvUnit unit{0, 0, 0};
      KvSequence seq{};
      if (item < items) {
        int low = 0, high = a.batch.sequences;
        while (high - low > 1) {
          const int mid = (low + high) >> 1;
          if (memory.first_item[mid] <= item) low = mid; else high = mid;
        }
        s = low;
        row_tile = item - memory.first_item[s];
        seq = kv_sequence(a.batch, a.shape, s);
        unit = kv_unit(seq, row_tile, plan.tile_tokens);
      }
      const int unit_cost = unit.tiles > 0 ? unit.tiles + kUnitCost : 0;
      const int cost = min(kKvMaxList + 1, unit_cost * heads);
      int all;
      const int end = min(kKvMaxList + 1, scan(cost, &all) + before), begin = end - cost;
      before = min(kKvMaxList + 1, before + all);
      if (items <= kThreadCount) total = before;
      if (pass == 1) {
        if (total > kKvMaxList) {
          atomicOr(a.status, kKvBadBatch);
          continue;
        }
        const int blocks = min(plan.blocks, total);
        // the cuts in (begin, end], and the first one of all
        const int first = unit_cost == 0 ? cut1 + 1 : begin == 0 ? 0 : kv_first_cut(begin + 1, total, blocks);
        const int last = end == total ? cut1 : kv_first_cut(end + 1, total, blocks) - 1;
        for (int c = max(first, cut0); c <= min(last, cut1); ++c) {
          const int cut = kv_cut(total, min(c, blocks), blocks);
          const int head = min(static_cast<int>(static_cast<uint32_t>(cut - begin) / static_cast<uint32_t>(unit_cost)), heads - 1);
          const int unit_begin = begin + head * unit_cost;
          int tile = max(0, cut - unit_begin - kUnitCost);
          const int snap = kv_snap(unit.tiles, total, blocks);
          if (tile <= snap && tile <= unit.tiles - tile) tile = 0;
          else if (unit.tiles - tile <= snap) tile = unit.tiles;
          emit(c, KvStart{unit_begin + (tile > 0 ? kUnitCost + tile : 0), total, blocks, s, row_tile, head, tile, seq.row0, seq.rows, seq.length, {0, 0}});
        }
        if (item < items && unit_cost == 0) nothing(item, seq.row0 + row_tile * plan.tile_tokens, unit.tokens);
      }
    }
    total = before;
  }
  if (total == 0 || total > kKvMaxList) {
    for (int c = cut0 + thread; c <= cut1; c += kThreadCount) emit(c, KvStart{});
  }
}

// For lists of many row tiles: one block writes all cuts.  (Rows that see nothing are left to the blocks of the next launch, which divide
// them: here each row tile would be zeroed by the one thread that has it.)
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads)
kv_plan_kernel(const KvAttentionPlan plan) {
  __shared__ PlanMemory<kPlanThreads> memory;
  pdl_enter();
  plan_list<kPlanThreads>(plan, memory, 0, plan.blocks, [&](int c, const KvStart& start) { plan.work.starts[c] = start; }, [](int, int, int) {});
}

// Zeroes the row tiles that see nothing, this block's share of each sequence's: the first rows of one that has more rows than positions.
// Called by all threads; `memory` holds 2 * AIMA_MOE_KV_MAX_SEQUENCES + 1 numbers.
template <int kDim, int kThreadCount>
__device__ __forceinline__ void zero_unseen(const KvAttentionPlan& plan, int* memory) {
  if (threadIdx.x == 0) memory[0] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < plan.a.batch.sequences; s += kThreadCount) {
    const KvSequence seq = kv_sequence(plan.a.batch, plan.a.shape, s);
    const int rows = seq.length <= 0 ? seq.rows : max(0, seq.rows - seq.length) / plan.tile_tokens * plan.tile_tokens;
    if (rows > 0) {
      const int at = atomicAdd(memory, 1);
      memory[1 + 2 * at] = seq.row0;
      memory[2 + 2 * at] = rows;
    }
  }
  __syncthreads();
  const int count = memory[0], blocks = gridDim.x;
  for (int i = 0; i < count; ++i) {
    const int row0 = memory[1 + 2 * i], rows = memory[2 + 2 * i];
    const int block = static_cast<int>((blockIdx.x + static_cast<uint32_t>(row0)) % gridDim.x);       // not the same few for every short one
    const int begin = static_cast<int>(static_cast<long long>(rows) * block / blocks), end = static_cast<int>(static_cast<long long>(rows) * (block + 1) / blocks);
    if (begin < end) kv_zero_rows<kDim, kThreadCount>(plan.a, row0 + begin, end - begin);
  }
}

// The unit that cut `cut` divides: its blocks.  Cut c lies at total c / blocks, and divides a unit if it leaves more than
// kv_snap tiles of it on either side.
__device__ __forceinline__ void divided_unit(const KvStart& cut, int tiles, int* first_block, int* parts) {
  const int tiles_begin = cut.at - cut.tile, snap = kv_snap(tiles, cut.total, cut.blocks);
  const int first = kv_first_cut(tiles_begin + snap + 1, cut.total, cut.blocks), last = kv_first_cut(tiles_begin + tiles - snap, cut.total, cut.blocks) - 1;
  *first_block = first - 1;
  *parts = last - first + 2;
}

// kPlanned: kv_plan_kernel has left the cuts; else every block finds its own two.
template <int kDim, bool kPlanned>
__global__ void __launch_bounds__(kThreads, 1)
kv_prompt_kernel(const __grid_constant__ KvMaps maps, const __grid_constant__ CUtensorMap queries, const __grid_constant__ KvAttentionPlan plan) {
  using L = Prompt<kDim>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* generic = smem_raw + (base - smem_u32(smem_raw));
  Small& sm = *reinterpret_cast<Small*>(generic + L::kSmallAt);
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
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(smem_u32(&sm.scales_full[s]), 1);
      mbar_init(smem_u32(&sm.scales_empty[s]), 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.p_full[i]), 8);
      mbar_init(smem_u32(&sm.o_done[i]), 1);
    }
    mbar_init(smem_u32(&sm.q_raw), 1);
    mbar_init(smem_u32(&sm.q_full), 8);
    mbar_init(smem_u32(&sm.q_empty), 1);
    mbar_init(smem_u32(&sm.drain), 1);
    sm.abort_flag = 0;
    sm.shared[0].parts = sm.shared[1].parts = 0;
    mbar_fence_init();
  }
  if (warp == 2) tmem_alloc(smem_u32(&sm.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  pdl_enter();

  Walk walk;
  if (kPlanned) {
    if (threadIdx.x < 2) sm.cut[threadIdx.x] = plan.work.starts[blockIdx.x + threadIdx.x];
    zero_unseen<kDim, kThreads>(plan, reinterpret_cast<int*>(generic));        // in the place of the first tiles
    fence_async_proxy();
  } else {
    // in the place of the first tiles
    PlanMemory<kThreads>& memory = *reinterpret_cast<PlanMemory<kThreads>*>(generic);
    int* empty = reinterpret_cast<int*>(generic + sizeof(PlanMemory<kThreads>));         // row, rows of items that see nothing
    empty[2 * threadIdx.x + 1] = 0;
    bool mine = false;
    plan_list<kThreads>(plan, memory, blockIdx.x, blockIdx.x + 1, [&](int c, const KvStart& start) { sm.cut[c - blockIdx.x] = start; },
                        [&](int item, int row0, int rows) {
                          if (item % gridDim.x != blockIdx.x) return;
                          empty[2 * threadIdx.x] = row0;
                          empty[2 * threadIdx.x + 1] = rows;
                          mine = true;
                        });
    if (__syncthreads_or(mine)) {
      for (int i = 0; i < kThreads; ++i) {
        if (empty[2 * i + 1] > 0) kv_zero_rows<kDim, kThreads>(a, empty[2 * i], empty[2 * i + 1]);
      }
    }
    fence_async_proxy();                   // tiles will be written where the plan lay
  }
  __syncthreads();
  walk.begin(plan, sm.cut[0], sm.cut[1]);
  auto wait = [&](unsigned long long* bar, uint32_t parity) { return mbar_wait_bounded_warp(smem_u32(bar), parity, abort_flag, plan.wait_limit_ns); };
  // Ring of K and V tiles, in the order in which the products take them: K0 K1 V0 K2 V1 .. V(n-2) V(n-1) of a segment.
  auto ring_k = [](int first, int j) { return first + (j == 0 ? 0 : 2 * j - 1); };
  auto ring_v = [](int first, int j, int n) { return first + (j + 1 < n ? 2 * j + 2 : 2 * n - 1); };

  // V of a tile from its codes to 16 bits, 16 rows by each of warps 4 .. 11.  Rows behind the sequence's end, where a page can hold
  // anything, become zeros.  Which rows eight lanes have together lets them read and write all banks: with heads of 128 four pieces of
  // rows r and r ^ 5, whose swizzles differ in the bit that tells even pieces from odd ones and in the one that tells halves.
  auto widen = [&](int slot, int buffer, int seen) {
    constexpr bool kLong = kDim == 128;
    constexpr int kSteps = kLong ? 4 : 2;
    const int piece = kLong ? (lane & 3) | ((lane >> 2) & 4) : lane & 3;          // of 16 codes
    const int low = kLong ? (5 * ((lane >> 2) & 1)) ^ ((lane >> 3) & 1) : lane >> 2;
    auto row_of = [&](int b) { return 16 * (warp - 4) + low + (kLong ? 2 * (b & 1) + 8 * (b >> 1) : 8 * b); };
    const uint8_t* from = generic + slot * L::kSlotBytes;
    uint8_t* to = generic + L::kWideAt + buffer * L::kWideBytes + (piece >> 2) * (kKvTile * 128);
    uint4 codes[kSteps];
#pragma unroll
    for (int b = 0; b < kSteps; ++b) {
      const int swizzle = kLong ? low ^ (2 * (b & 1)) : (low >> 1) & 3;
      codes[b] = *reinterpret_cast<const uint4*>(from + row_of(b) * L::kRowBytes + ((piece ^ swizzle) << 4));
    }
    if (seen < kKvTile) {
#pragma unroll
      for (int b = 0; b < kSteps; ++b)
        if (row_of(b) >= seen) codes[b] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < kSteps; ++b) {
      const uint4& c = codes[b];
      const uint32_t even = ((2 * (piece & 3)) ^ (kLong ? low ^ (2 * (b & 1)) : low)) << 4;
      uint8_t* row_at = to + row_of(b) * 128;
      *reinterpret_cast<uint4*>(row_at + even) = make_uint4(e4m3x2_f16x2(c.x), e4m3x2_f16x2(c.x >> 16), e4m3x2_f16x2(c.y), e4m3x2_f16x2(c.y >> 16));
      *reinterpret_cast<uint4*>(row_at + (even ^ 16)) = make_uint4(e4m3x2_f16x2(c.z), e4m3x2_f16x2(c.z >> 16), e4m3x2_f16x2(c.w), e4m3x2_f16x2(c.w >> 16));
    }
    fence_async_proxy();
  };

  if (warp < 4) {
    if (warp == 0) {
      // ------------------------------ loads ------------------------------
      const int boxes = (kKvTile >> shape.page_shift) * L::kPanels;     // of a tile; a lane each
      const int my_page = lane / L::kPanels, my_panel = lane % L::kPanels;
      int ring = 0;
      bool alive = true;
      while (alive && walk.next()) {
        const int* table = a.batch.table + static_cast<size_t>(walk.sequence) * a.batch.columns;
        const int pages = (walk.seq.length + shape.page_tokens - 1) >> shape.page_shift;
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
      constexpr uint32_t kScoresHigh = instr_desc_f8(kE4m3, kE4m3, 0, 0, 128, kKvTile);
      constexpr uint32_t kScoresLow = instr_desc_f8(kE5m2, kE4m3, 0, 0, 128, kKvTile);
      constexpr uint32_t kSums = L::kWide ? instr_desc_f8(kF16, kF16, 0, 1, 128, kDim) : instr_desc_f8(kE5m2, kE4m3, 0, 1, 128, kDim);
      int ring = 0, tile = 0, segment = 0;
      bool alive = true;
      while (alive && walk.next()) {
        const int n = walk.tiles;
        auto scores = [&](int j) {
          // the scores' buffer is free once the product that reads the weights in it has ended: products of different shapes
          // need not run in the order of issue (the wait costs heads of 256 two percent, smaller ones nothing)
          const int r = ring_k(ring, j), slot = r % L::kSlots, buffer = (tile + j) & 1;
          if (!wait(&sm.full[slot], (r / L::kSlots) & 1) || !wait(&sm.o_done[buffer], (((tile + j) >> 1) & 1) ^ 1)) return false;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t k0 = base + slot * L::kSlotBytes, q0 = base + L::kQueryAt;
#pragma unroll
            for (int term = 0; term < 2; ++term) {
#pragma unroll
              for (int k = 0; k < kDim / 32; ++k) {
                const int panel = k * 32 / L::kRowBytes, inside = k * 32 % L::kRowBytes;
                umma_f8(tmem + L::kScoreColumn + buffer * 128,
                        smem_desc_rows<L::kRowBytes>(q0 + term * L::kSlotBytes + panel * L::kPanelBytes) + (inside >> 4),
                        smem_desc_rows<L::kRowBytes>(k0 + panel * L::kPanelBytes) + (inside >> 4), term == 0 ? kScoresHigh : kScoresLow,
                        (term | k) != 0);
              }
            }
            umma_commit(smem_u32(&sm.empty[slot]));
            umma_commit(smem_u32(&sm.s_full[buffer]));
            if (j + 1 == n) umma_commit(smem_u32(&sm.q_empty));
          }
          __syncwarp();
          return true;
        };
        alive = wait(&sm.q_full, segment & 1) && scores(0);
        for (int j = 0; j < n && alive; ++j) {
          if (j + 1 < n && !scores(j + 1)) { alive = false; break; }
          const int r = ring_v(ring, j, n), slot = r % L::kSlots, buffer = (tile + j) & 1;
          if (!wait(&sm.p_full[buffer], ((tile + j) >> 1) & 1) || (!L::kWide && !wait(&sm.full[slot], (r / L::kSlots) & 1))) { alive = false; break; }
          tc_fence_after();
          if (L::kWide) {
            if (lane == 0) mbar_arrive(smem_u32(&sm.empty[slot]));         // its codes have been read
            __syncwarp();
            if (elect_one()) {
              const uint32_t v0 = base + L::kWideAt + buffer * L::kWideBytes, w0 = tmem + L::kScoreColumn + buffer * 128;
#pragma unroll
              for (int k = 0; k < kKvTile / 16; ++k)
                umma_f16_ts(tmem, w0 + (k / 4) * 64 + (k % 4) * 8, smem_desc_rows<128>(v0 + k * 16 * 128, kKvTile * 128), kSums, (j | k) != 0);
              umma_commit(smem_u32(&sm.o_done[buffer]));
            }
          } else if (elect_one()) {
            const uint32_t v0 = base + slot * L::kSlotBytes, w0 = tmem + L::kScoreColumn + buffer * 128;
#pragma unroll
            for (int term = 0; term < 3; ++term) {
#pragma unroll
              for (int k = 0; k < kKvTile / 32; ++k)
                umma_f8_ts(tmem, w0 + k * 32 + term * 8, smem_desc_rows<L::kRowBytes>(v0 + k * 32 * L::kRowBytes, L::kPanelBytes),
                           kSums, (j | term | k) != 0);
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
    } else if (warp == 2) {
      // ------------------------------ queries, as they are ------------------------------
      // A BF16 row of a head is as long as its two terms together and goes where they will lie, kRowBytes at a time, so that it
      // can be converted in place.  Rows behind the unit's last are another unit's or zeros; their results go nowhere.  Queries
      // whose strides a tensor map cannot have are read from where they are by the warps that convert them, which waits for
      // memory four times per unit: 1024 tokens 29.5 us instead of 27.9, no difference from some thousands of positions on.
      int segment = 0;
      for (; walk.next(); ++segment, walk.advance()) {
        if (!wait(&sm.q_empty, (segment & 1) ^ 1)) break;
        if (plan.query_map) {
          if (elect_one()) {
            constexpr int kBoxes = 2 * kDim / L::kRowBytes;
            mbar_arrive_expect_tx(smem_u32(&sm.q_raw), kBoxes * plan.tile_tokens * shape.group * L::kRowBytes);
            for (int i = 0; i < kBoxes; ++i)
              tma_load_3d(base + L::kQueryAt + (i / L::kPanels) * L::kSlotBytes + (i % L::kPanels) * L::kPanelBytes, &queries, i * L::kRowBytes / 2,
                          walk.head * shape.group, walk.seq.row0 + walk.row_tile * plan.tile_tokens, smem_u32(&sm.q_raw));
          }
        } else {
          if (lane == 0) mbar_arrive(smem_u32(&sm.q_raw));
        }
        __syncwarp();
      }
      if (*abort_flag != 0 && segment > 0) {
        volatile int ignore = 0;
        mbar_wait_bounded(smem_u32(&sm.q_raw), (segment - 1) & 1, &ignore);
      }
    } else if (warp == 3) {
      // ------------------------------ scales ------------------------------
      int tile = 0;
      bool alive = true;
      while (alive && walk.next()) {
        const int* table = a.batch.table + static_cast<size_t>(walk.sequence) * a.batch.columns;
        auto fetch = [&](int j) {            // lane g < 8: positions 16 g .. 16 g + 15 of the tile
          const int position = (walk.tile0 + j) * kKvTile + 16 * lane;
          float2 s = make_float2(0.0f, 1.0f);
          if (j < walk.tiles && lane < 8 && position < walk.seq.length) {
            const int page = table[position >> shape.page_shift];
            if (page >= 0 && page < shape.pages) {
              const size_t at = static_cast<size_t>(page) * shape.kv_heads + walk.head;
              s = make_float2(a.layer.key_scales[at], a.layer.value_scales[at]);
            }
          }
          return s;
        };
        float2 s = fetch(0);
        int first = 0;                       // exponent of the first value scale
        bool known = false, apart = false;
        for (int j = 0; j < walk.tiles; ++j, ++tile) {
          const float2 after = fetch(j + 1);
          const int slot = tile % kScaleSlots;
          if (!wait(&sm.scales_empty[slot], ((tile / kScaleSlots) & 1) ^ 1)) { alive = false; break; }
          // positions without a page are marked; their factor only has to be positive
          const bool hole = lane < 8 && s.x == 0.0f;
          const uint32_t holes = __ballot_sync(0xffffffffu, hole);
          if (!known && holes != 0xffu) {
            first = __shfl_sync(0xffffffffu, kv_float_exponent(s.y), __ffs(static_cast<int>(~holes)) - 1);
            known = true;
          }
          const float value_log2 = log2f(s.y), relative = static_cast<float>(first) - value_log2;
          apart = apart || __any_sync(0xffffffffu, lane < 8 && !hole && fabsf(relative) > kKvApart);
          if (lane == 0) sm.marks[slot] = make_int2(static_cast<int>(holes) | (apart ? kApart : 0), first);
          if (lane < 8) sm.scales[slot][lane] = make_float4(s.x > 0.0f ? s.x * a.scale_log2 : 1.0f, value_log2, apart ? 0.0f : fast_exp2(relative), 0.0f);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.scales_full[slot]));
          s = after;
        }
        walk.advance();
      }
    }
  } else {
    // ------------------------------ softmax and results ------------------------------
    const int group = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int group_inverse = (65536 + shape.group - 1) / shape.group;
    int ring = 0, tile = 0, segment = 0;
    // No wait that runs out leaves this loop: the warps meet at barriers, and every wait after the first that ran out ends at once.
    while (walk.next()) {
      const int n = walk.tiles;
      const int rows = walk.unit.tokens * shape.group;
      const int token0 = walk.seq.row0 + walk.row_tile * plan.tile_tokens;
      // Queries: a warp takes every eighth row, four side by side (one alone is a chain of 340 cycles).  BF16 numbers are f16 numbers
      // down to 2^-14 of the row's scale; a row that is not finite becomes NaN.
      wait(&sm.q_raw, segment & 1);
      {
        constexpr int kPer = kDim / 32;
        const int w8 = warp - 4;
        uint8_t* queries_at = generic + L::kQueryAt;
        const int raw_byte = 2 * kPer * lane, byte = kPer * lane;
        const int raw_at = (raw_byte / kDim) * L::kSlotBytes + (raw_byte % kDim / L::kRowBytes) * L::kPanelBytes + raw_byte % L::kRowBytes + w8 * L::kRowBytes;
        // the swizzle takes the row modulo 8, which is the warp
        const int piece = (byte % L::kRowBytes >> 4) ^ (L::kRowBytes == 128 ? w8 : w8 >> 1);
        const int code_at = (byte / L::kRowBytes) * L::kPanelBytes + piece * 16 + (byte & 15) + w8 * L::kRowBytes;
#pragma unroll 1
        for (int i = 0; i < 16 && 8 * i < rows; i += 4) {
          uint32_t raw[4][kPer / 2], codes[4][2][kPer / 2];
          int exponent[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint8_t* from = queries_at + raw_at + 8 * (i + b) * L::kRowBytes;
            if (!plan.query_map) {
              const int r = min(8 * (i + b) + w8, rows - 1), token = row_token(r, group_inverse);
              from = reinterpret_cast<const uint8_t*>(a.q.data + (token0 + token) * a.q.row_stride +
                                                      (walk.head * shape.group + r - token * shape.group) * a.q.head_stride + kPer * lane);
            }
            if constexpr (kPer == 8) {
              const uint4 v = *reinterpret_cast<const uint4*>(from);
              raw[b][0] = v.x; raw[b][1] = v.y; raw[b][2] = v.z; raw[b][3] = v.w;
            } else if constexpr (kPer == 4) {
              const uint2 v = *reinterpret_cast<const uint2*>(from);
              raw[b][0] = v.x; raw[b][1] = v.y;
            } else {
              raw[b][0] = *reinterpret_cast<const uint32_t*>(from);
            }
          }
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            uint32_t largest = 0;          // magnitudes as integers: infinities and NaN come last
#pragma unroll
            for (int e = 0; e < kPer / 2; ++e) largest = __vmaxu2(largest, raw[b][e] & 0x7fff7fffu);
            largest = __reduce_max_sync(0xffffffffu, max(largest & 0xffffu, largest >> 16));           // all lanes have read the row
            exponent[b] = kv_scale_exponent(__uint_as_float(largest << 16));
            const uint32_t inverse = largest < 0x7f80u ? static_cast<uint32_t>(127 - exponent[b]) * 0x00800080u : 0x7fff7fffu;      // two BF16 numbers
            uint32_t h[kPer / 2];
#pragma unroll
            for (int e = 0; e < kPer / 2; ++e) {
              const uint32_t scaled = mul_bf16x2(raw[b][e], inverse);
              h[e] = cvt_f16x2(bf16_lo(scaled), bf16_hi(scaled));
              codes[b][0][e] = cvt_e4m3x2_f16x2(h[e]);
              h[e] = sub_f16x2(h[e], e4m3x2_f16x2(codes[b][0][e])) + 0x00800080u;           // rounded to e5m2, its upper byte
            }
#pragma unroll
            for (int e = 0; e < kPer / 2; e += 2) {
              codes[b][0][e / 2] = __byte_perm(codes[b][0][e], kPer > 2 ? codes[b][0][e + 1 < kPer / 2 ? e + 1 : e] : 0u, 0x5410);
              codes[b][1][e / 2] = __byte_perm(h[e], h[e + 1 < kPer / 2 ? e + 1 : e], 0x7531);
            }
          }
#pragma unroll
          for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int term = 0; term < 2; ++term) {
              const uint32_t* c = codes[b][term];
              uint8_t* to = queries_at + term * L::kSlotBytes + code_at + 8 * (i + b) * L::kRowBytes;
              if constexpr (kPer == 8) *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[1]);
              else if constexpr (kPer == 4) *reinterpret_cast<uint32_t*>(to) = c[0];
              else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(c[0]);
            }
            if (lane == 0) sm.row_scale[8 * (i + b) + w8] = kv_exp2(exponent[b]);
          }
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_full));
        group_barrier();                   // row_scale
      }
      const float row_scale = row < rows ? sm.row_scale[row] : 0.0f;
      const int limit = row < rows ? walk.unit.first + row_token(row, group_inverse) : -1;     // last position the row sees
      float top = -INFINITY, peak = -INFINITY, sum = 0.0f;       // reference and maximum so far; this half's denominator
      float low = -INFINITY;                                     // the denominator's reference once scales are apart
      bool apart = false;
      int first = 0;                                             // e
      float shift = kWeightExponent;                             // less the reference
      for (int j = 0; j < n; ++j, ++tile) {
        const int buffer = tile & 1, slot = tile % kScaleSlots;
        const int position0 = (walk.tile0 + j) * kKvTile;
        const uint32_t scores = tmem + lanes + L::kScoreColumn + buffer * 128;
        // all at once: even a wait that has ended takes 85 cycles to say so
        const bool scales_there = mbar_test(smem_u32(&sm.scales_full[slot]), (tile / kScaleSlots) & 1);
        const bool scores_there = mbar_test(smem_u32(&sm.s_full[buffer]), (tile >> 1) & 1);
        if (L::kWide) {
          const int r = ring_v(ring, j, n), ring_slot = r % L::kSlots;
          const bool codes_there = mbar_test(smem_u32(&sm.full[ring_slot]), (r / L::kSlots) & 1);
          const bool room = mbar_test(smem_u32(&sm.o_done[buffer]), ((tile >> 1) & 1) ^ 1);
          if (!__all_sync(0xffffffffu, codes_there)) wait(&sm.full[ring_slot], (r / L::kSlots) & 1);
          if (!__all_sync(0xffffffffu, room)) wait(&sm.o_done[buffer], ((tile >> 1) & 1) ^ 1);
          widen(ring_slot, buffer, walk.seq.length - position0);
        }
        if (!__all_sync(0xffffffffu, scores_there)) wait(&sm.s_full[buffer], (tile >> 1) & 1);
        if (!__all_sync(0xffffffffu, scales_there)) wait(&sm.scales_full[slot], (tile / kScaleSlots) & 1);
        tc_fence_after();
        const uint32_t half = 64 * group;
        uint32_t s[64];
        tmem_ld32(scores + half, s);
        tmem_ld32(scores + half + 32, s + 32);
        const float4* scales = sm.scales[slot];
        const int2 marks = sm.marks[slot];
        const int holes = marks.x & (kApart - 1);
        first = marks.y;
        const bool masked = position0 + kKvTile - 1 > walk.unit.first || marks.x != 0;        // or scales apart
        // positive, so that a masked score stays -inf
        auto factor_of = [&](int g) { return fmaxf(scales[g].x * row_scale, 1.17549435e-38f); };
        auto mask = [&](uint32_t* x, int first) {          // 32 scores from position `first` of the tile on
          // the diagonal, the sequence's end, or a page that is not there: a bit for each that counts
          const int seen = limit - position0 - first;
          uint32_t bits = seen >= 31 ? 0xffffffffu : seen < 0 ? 0u : (2u << seen) - 1u;
          if ((holes >> (first / 16)) & 1) bits &= 0xffff0000u;
          if ((holes >> (first / 16)) & 2) bits &= 0x0000ffffu;
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if ((bits & (1u << c)) == 0u) x[c] = 0xff800000u;
        };
        auto top_of = [&](const uint32_t* x, int first) {
          float m = -INFINITY;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float a0 = __uint_as_float(x[16 * g]), a1 = __uint_as_float(x[16 * g + 1]);
#pragma unroll
            for (int c = 2; c < 16; c += 4) {
              a0 = fmaxf(fmaxf(a0, __uint_as_float(x[16 * g + c])), __uint_as_float(x[16 * g + c + 1]));
              if (c + 2 < 16) a1 = fmaxf(fmaxf(a1, __uint_as_float(x[16 * g + c + 2])), __uint_as_float(x[16 * g + c + 3]));
            }
            m = fmaxf(m, fmaf(fmaxf(a0, a1), factor_of(first / 16 + g), scales[first / 16 + g].y));
          }
          return m;
        };
        tmem_ld_wait();
        if (masked) {
          mask(s, half);
          mask(s + 32, half + 32);
          if ((marks.x & kApart) != 0) {
            float s_top = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float x = __uint_as_float(s[16 * g]);
#pragma unroll
              for (int c = 1; c < 16; ++c) x = fmaxf(x, __uint_as_float(s[16 * g + c]));
              s_top = fmaxf(s_top, x * factor_of(half / 16 + g));
            }
            sm.half_low[group][row] = s_top;
            asm volatile("bar.sync %0, 64;" :: "r"(2 + quarter) : "memory");
            const float from = apart ? low : top - static_cast<float>(first);
            low = fmaxf(from, fmaxf(s_top, sm.half_low[group ^ 1][row]));
            if (from != low) sum *= fast_exp2(from - low);
            const float low_shift = kWeightExponent - (low == -INFINITY ? 0.0f : low);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
              for (int c = 0; c < 16; ++c) sum += fast_exp2(fmaf(__uint_as_float(s[16 * g + c]), factor_of(half / 16 + g), low_shift));
            }
            apart = true;
          }
        }
        float m = fmaxf(top_of(s, half), top_of(s + 32, half + 32));
        sm.half_top[buffer][group][row] = m;
        asm volatile("bar.sync %0, 64;" :: "r"(2 + quarter) : "memory");
        m = fmaxf(m, sm.half_top[buffer][group ^ 1][row]);
        const bool jumps = m > peak + kJump;
        peak = fmaxf(peak, m);
        const bool falls = m > -INFINITY && fmaxf(m, peak - kDepth) < top - kFall;
        const bool moves = m > top + kGrow || falls;               // the first that is seen is above -inf
        if (__any_sync(0xffffffffu, moves)) {
          float now = top;
          if (falls) now = fmaxf(m, peak - kDepth);
          else if (moves) now = !L::kWide && jumps ? m - kLift : m;
          else if (!L::kWide && peak - top <= kLift) now = fmaxf(top, peak);       // a lift that is given back; a fallen reference stays
          const float f = now != top ? fast_exp2(top - now) : 1.0f;                // top is -inf at first: 0
          if (j > 0) {
            wait(&sm.o_done[buffer ^ 1], ((tile - 1) >> 1) & 1);
            tc_fence_after();
            const uint32_t sums = tmem + lanes + group * (kDim / 2);
#pragma unroll 1
            for (int c = 0; c < kDim / 2; c += 32) {
              uint32_t o[32];
              tmem_ld32(sums + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st32(sums + c, o);
            }
          }
          if (!apart) sum *= f;
          top = now;
          shift = kWeightExponent - (top == -INFINITY ? 0.0f : top);
        }
#pragma unroll
        for (int chunk = 0; chunk < 2; ++chunk) {
          uint32_t terms[24];                 // kWide: 16 pairs of weights
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int at = half / 16 + 2 * chunk + g;
            const float factor = factor_of(at), offset = scales[at].y + shift;
            float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              float w[4];
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                const uint32_t* x = s + 32 * chunk + 16 * g + c + i;
                const float2 t = fma2(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), make_float2(factor, factor), make_float2(offset, offset));
                if (L::kWide && i == 2 && c >= 8) {
                  const float2 e = exp2_by_polynomial(t);
                  w[i] = e.x;
                  w[i + 1] = e.y;
                } else {
                  w[i] = fast_exp2(t.x);
                  w[i + 1] = fast_exp2(t.y);
                }
                part = add2(part, make_float2(w[i], w[i + 1]));
              }
              if (L::kWide) {
                terms[8 * g + c / 2] = cvt_f16x2(w[0], w[1]);
                terms[8 * g + c / 2 + 1] = cvt_f16x2(w[2], w[3]);
              } else {
                split_weights(cvt_f16x2(w[0], w[1]), cvt_f16x2(w[2], w[3]), terms + 4 * g + c / 4, 8);
              }
            }
            sum = fmaf(part.x + part.y, scales[at].z, sum);
          }
          // where the scores of these 32 positions lay (kWide: those of the half's first 32)
#pragma unroll
          for (int term = 0; term < (L::kWide ? 2 : 3); ++term) tmem_st8(scores + half + (L::kWide ? 16 : 32) * chunk + 8 * term, terms + 8 * term);
        }
        tmem_st_wait();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.scales_empty[slot]));
        if (!L::kWide && position0 + kKvTile > walk.seq.length) {
          // behind the sequence's end a page can hold anything, and zero weights do not stop a NaN
          const int r = ring_v(ring, j, n), ring_slot = r % L::kSlots;
          wait(&sm.full[ring_slot], (r / L::kSlots) & 1);
          if (position0 + row >= walk.seq.length) {
#pragma unroll
            for (int i = 0; i < kDim / 32; ++i) {
              const int c = group * (kDim / 32) + i;
              *reinterpret_cast<uint4*>(generic + ring_slot * L::kSlotBytes + (c * 16 / L::kRowBytes) * L::kPanelBytes + row * L::kRowBytes +
                                        c * 16 % L::kRowBytes) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_async_proxy();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[buffer]));
      }
      // the unit's sums, or this block's part of them; each group has half of the columns
      sm.sum[segment & 1][group][row] = sum;
      asm volatile("bar.sync %0, 64;" :: "r"(2 + quarter) : "memory");
      const float total = sm.sum[segment & 1][0][row] + sm.sum[segment & 1][1][row];
      wait(&sm.o_done[(tile - 1) & 1], ((tile - 1) >> 1) & 1);
      tc_fence_after();
      const bool whole = n == walk.unit.tiles, begins = walk.tile0 == 0;
      const size_t part = kv_part_index(blockIdx.x, begins);
      if (!whole) {
        if (group == 0 && row < rows) *kv_part_weight(plan.work, part, row) = make_float4(top, total, apart ? low : top - static_cast<float>(first), 0.0f);
        if (threadIdx.x == 128) {
          KvShared shared{0, 0, 0, rows, token0, walk.head * shape.group};
          divided_unit(sm.cut[begins ? 1 : 0], walk.unit.tiles, &shared.first_block, &shared.parts);
          shared.mine = static_cast<int>(blockIdx.x) - shared.first_block;
          sm.shared[begins ? 1 : 0] = shared;
        }
      }
      const float2 back = kv_exp2_factors(!apart ? static_cast<float>(first) : top == -INFINITY ? 0.0f : top - low);
      const float inverse = total == 0.0f ? 0.0f : back.x / total;
      // 32 columns at a time through shared memory, 16-byte pieces XORed with the row, so that every store writes 64 bytes of
      // eight rows.  (Each thread storing its own row took 5 us per unit.)
      uint8_t* stage = generic + L::kStageAt + (warp - 4) * kStageBytes;
      const uint32_t from = tmem + lanes + group * (kDim / 2);
#pragma unroll 1
      for (int c = 0; c < kDim / 64; ++c) {
        uint32_t x[32];
        tmem_ld32(from + 32 * c, x);
        tmem_ld_wait();
        const int column = group * (kDim / 2) + 32 * c;
        if (whole) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t packed[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(x[8 * k + 2 * i]) * inverse * back.y, __uint_as_float(x[8 * k + 2 * i + 1]) * inverse * back.y);
              packed[i] = *reinterpret_cast<const uint32_t*>(&two);
            }
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 8 * i + (lane >> 2), r = quarter * 32 + at;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + at * 64 + (((lane & 3) ^ ((at >> 1) & 3)) << 4));
            if (r < rows) {
              const int token = row_token(r, group_inverse), g = r - token * shape.group;
              *reinterpret_cast<uint4*>(a.out + (static_cast<long long>(token0 + token) * shape.q_heads + walk.head * shape.group + g) * kDim +
                                        column + 8 * (lane & 3)) = v;
            }
          }
          __syncwarp();
        } else if (row < rows) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            *reinterpret_cast<uint4*>(kv_part_sum<kDim>(plan.work, part, row, column + 4 * k)) = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
        }
      }
      tc_fence_before();
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
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (sm.shared[i].parts > 0) kv_join<kDim, kThreads>(a, plan.work, sm.shared[i], plan.wait_limit_ns, &sm.verdict);
  }
}

template <int kDim, bool kPlanned>
cudaError_t launch_planned(const KvAttentionPlan& plan, const KvMaps& maps, const CUtensorMap& queries, cudaStream_t stream) {
  constexpr int bytes = kv_smem_bytes(Prompt<kDim>::kSmallAt + static_cast<int>(sizeof(Small)) + 1024);
  static_assert(bytes <= 227 * 1024, "more shared memory than a block can have");
  static_assert(sizeof(PlanMemory<kThreads>) + 8 * kThreads <= Prompt<kDim>::kQueryAt, "the plan lies in the ring");
  static_assert(4 * (2 * AIMA_MOE_KV_MAX_SEQUENCES + 1) <= Prompt<kDim>::kQueryAt, "so do the sequences with rows that see nothing");
  const cudaError_t error = opt_in_dynamic_smem<kv_prompt_kernel<kDim, kPlanned>>(bytes);
  if (error != cudaSuccess) return error;
  return launch_resident(kv_prompt_kernel<kDim, kPlanned>, dim3(plan.blocks), dim3(kThreads), bytes, stream, maps, queries, plan);
}

template <int kDim>
cudaError_t launch(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream) {
  // Row tiles at most.  With one for each thread of a block every block can find its share by itself, which saves a launch: 1024
  // tokens 27.9 us and 31.7 with the plan kernel, 4096 tokens 160 .. 164 with either.
  const long long items = plan.a.batch.tokens / plan.tile_tokens + plan.a.batch.sequences;
  CUtensorMap queries{};
  if (plan.query_map && !kv_make_query_map(plan.a, plan.tile_tokens, &queries)) return cudaErrorInvalidValue;
  if (items <= kThreads) return launch_planned<kDim, false>(plan, maps, queries, stream);
  const cudaError_t error = launch_pdl(kv_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, plan);
  return error != cudaSuccess ? error : launch_planned<kDim, true>(plan, maps, queries, stream);
}

}  // namespace

cudaError_t kv_prompt(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream) {
  switch (plan.a.shape.head_dim) {
    case 64: return launch<64>(plan, maps, stream);
    case 128: return launch<128>(plan, maps, stream);
    default: return launch<256>(plan, maps, stream);
  }
}

}  // namespace aima
