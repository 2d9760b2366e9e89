// What the attention kernels over the paged 8-bit cache share: tensor maps, the workspace of units that several blocks work on,
// and the join of their parts.
#pragma once

#include "kv_cache.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace aima {

constexpr int kKvTile = 128;            // positions of the cache per step
// In place of a page number out of range: a box in front of the tensor, which TMA fills with zeros.  The positions are masked, but what
// lies in V is multiplied by their zero weights, and any page that exists may hold NaN there.
constexpr int kNoPage = -2;
constexpr int kKvMaxBlocks = 160;       // blocks of an attention kernel at most (one per SM)
constexpr int kKvPartRows = 128;
constexpr int kKvMaxList = 1 << 24;     // tiles (with the units' own cost) of a launch: shares are computed in 32 bits

// A value's scale vs rides on its weight, w = 2^(s + log2 vs - m), which is relative to the largest of them.  The softmax's denominator
// wants them without it.  While the scales stay within 2^kKvApart of 2^e, the exponent of the first page's, it is the sum of w 2^e / vs,
// relative to 2^l with l = m - e: no weight that counts there is lost in w.  From the first page beyond that on its terms are
// exponentials of their own, 2^(s - l) with a running l: a page of zeros, whose scale is the least, may lie beside one of the
// largest values.  Either way o = 2^(m - l) * (sum of w code) / denominator.
constexpr float kKvApart = 32.0f;

struct KvMaps {
  CUtensorMap keys, values;             // [pages * kv_heads * page_tokens, head_dim] bytes, boxes of one page x up to 128 bytes
};

// Where a block of the prompt kernel begins: the unit and the tile inside it, and the place in the list in units of its cost.
struct alignas(16) KvStart {
  int at, total;
  int blocks;                           // the shares of the list
  int sequence, row_tile, head, tile;
  int row0, rows, length;               // of the sequence
  int unused[2];
};

// A unit is the tiles of the cache that a row tile (up to 128 rows: query heads of one key/value head x new tokens) sees.
// The kernels go through the list of all units' tiles, every block through an equal share; a unit that ends up in several
// blocks leaves its part in the workspace of each, and those blocks put the parts together, each a share of the results
// (kv_join).  A block has two parts: of the unit that it begins in the middle, and of the one that it does not finish.
struct KvWorkspace {
  unsigned* arrived;      // [2 * kKvMaxBlocks], by the block that begins the unit: parts written, parts joined; zero between launches
  float4* weights;        // [2 * kKvMaxBlocks][kKvPartRows]: m, denominator, l
  float* sums;            // [2 * kKvMaxBlocks][head_dim / 4][kKvPartRows][4]
  KvStart* starts;        // [kKvMaxBlocks + 1], for prompts of many row tiles
};

struct KvAttentionPlan {
  KvAttention a;
  KvWorkspace work;
  int blocks;
  int tile_rows;          // rows that a sequence has at most for one key/value head
  int tile_tokens;        // prompts: new tokens of a row tile
  bool query_map;         // prompts: queries come through a tensor map
  unsigned long long wait_limit_ns;
};

// What a block keeps of a unit that it shares with others until it has written its last part; parts = 0: none.
struct KvShared {
  int first_block, parts;       // blocks first_block .. first_block + parts - 1
  int mine;                     // which of the parts this block wrote
  int rows;
  int row0, head;               // of q: the unit's first row and query head
};

// floor(total c / blocks) and ceil(x blocks / total), x <= total <= kKvMaxList
__device__ __forceinline__ int kv_cut(int total, int c, int blocks) { return static_cast<int>(static_cast<uint32_t>(total) * static_cast<uint32_t>(c) / static_cast<uint32_t>(blocks)); }
__device__ __forceinline__ int kv_first_cut(int x, int total, int blocks) {
  return static_cast<int>((static_cast<uint32_t>(x) * static_cast<uint32_t>(blocks) + static_cast<uint32_t>(total) - 1u) / static_cast<uint32_t>(total));
}

__device__ __forceinline__ size_t kv_part_index(int block, bool begins) { return 2 * block + (begins ? 1 : 0); }
// Two factors whose product is 2^d, each within FP32's range.
__device__ __forceinline__ float2 kv_exp2_factors(float d) {
  const float near = fminf(fmaxf(d, -60.0f), 60.0f);
  return make_float2(fast_exp2(near), fast_exp2(d - near));
}
__device__ __forceinline__ float4* kv_part_weight(const KvWorkspace& work, size_t part, int row) { return work.weights + part * kKvPartRows + row; }
template <int kDim>
__device__ __forceinline__ float* kv_part_sum(const KvWorkspace& work, size_t part, int row, int d) {       // d: a multiple of 4
  return work.sums + part * kKvPartRows * kDim + (static_cast<size_t>(d >> 2) * kKvPartRows + row) * 4;
}

// The block's part has been written, before a barrier of the block that this thread has passed.
__device__ __forceinline__ void kv_arrive(const KvWorkspace& work, const KvShared& unit) {
  __threadfence();
  atomicAdd(work.arrived + 2 * unit.first_block, 1u);
}

// Joins a unit's parts: waits until all have been written, then takes the `mine`-th share of its results.  Called by all
// threads of a block.  The blocks of the launch are all resident (it is a cooperative one), and none waits before its own parts
// are written; the wait has its limit all the same.  A result is four neighbouring elements of a row.  Few parts (a row tile of a
// prompt in two or three blocks): a thread keeps to one row, so that the parts' factors are found once, and all blocks share the
// columns.  Many parts (one token's few rows in 74 blocks): 4 .. 32 lanes share the parts of a result.  Either way in the same
// order in every launch.  512 tokens of 4096 (2 or 3 parts of 128 rows) 51 us by rows and 100 by lanes, 16 x 40 rows of 4111 (4 .. 6
// parts) 28.7 and 35.4, 10 x 40 rows of 4000 22.6 and 25.7; with 74 parts a row's factors alone would be 74 loads per thread.
template <int kDim, int kThreads>
__device__ __forceinline__ void kv_join(const KvAttention& a, const KvWorkspace& work, const KvShared& unit, unsigned long long limit_ns, int* verdict) {
  unsigned* arrived = work.arrived + 2 * unit.first_block;
  if (threadIdx.x == 0) {
    const unsigned long long start = global_timer_ns();
    int ok = 1;
    for (;;) {
      unsigned seen;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(arrived) : "memory");
      if (seen >= static_cast<unsigned>(unit.parts)) break;
      if (global_timer_ns() - start > limit_ns) {
        atomicOr(a.status, kKvTimeout);
        ok = 0;
        break;
      }
    }
    *verdict = ok;
  }
  __syncthreads();
  const bool ok = *verdict != 0;
  auto store = [&](int row, int d, const float4& sums, float inverse, float rest) {
    const float4 x = make_float4(sums.x * inverse, sums.y * inverse, sums.z * inverse, sums.w * inverse);
    const int token = row / a.shape.group, g = row - token * a.shape.group;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * rest, x.y * rest), hi = __floats2bfloat162_rn(x.z * rest, x.w * rest);
    *reinterpret_cast<uint2*>(a.out + (static_cast<long long>(unit.row0 + token) * a.shape.q_heads + unit.head + g) * kDim + d) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  };
  // kFew parts at most, kColumns results of a row under way together
  auto by_rows = [&](auto few, auto columns) {
    constexpr int kFew = decltype(few)::value, kColumns = decltype(columns)::value;
    const int at_once = kThreads / unit.rows, row = threadIdx.x % unit.rows;       // kThreads is at least a row tile's rows
    const int end = 4 * (kDim / 4 * (unit.mine + 1) / unit.parts);
    int d = 4 * (kDim / 4 * unit.mine / unit.parts + static_cast<int>(threadIdx.x) / unit.rows);
    if (static_cast<int>(threadIdx.x) >= at_once * unit.rows || d >= end) return;
    float4 x[kColumns][kFew];
    auto load = [&] {
#pragma unroll
      for (int i = 0; i < kColumns; ++i) {
#pragma unroll
        for (int p = 0; p < kFew; ++p) {
          x[i][p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (p < unit.parts && d + 4 * at_once * i < end)
            x[i][p] = __ldcg(reinterpret_cast<const float4*>(kv_part_sum<kDim>(work, kv_part_index(unit.first_block + p, p == 0), row, d + 4 * at_once * i)));
        }
      }
    };
    float4 w[kFew];
#pragma unroll
    for (int p = 0; p < kFew; ++p) {
      w[p] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
      if (p < unit.parts) w[p] = __ldcg(kv_part_weight(work, kv_part_index(unit.first_block + p, p == 0), row));
    }
    load();
    float top = -INFINITY, low = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int p = 0; p < kFew; ++p) {
      top = fmaxf(top, w[p].x);
      low = fmaxf(low, w[p].z);
    }
    if (top == -INFINITY) top = low = 0.0f;                       // nothing seen, or nothing but NaN
#pragma unroll
    for (int p = 0; p < kFew; ++p) {
      sum += w[p].z == -INFINITY ? w[p].y : w[p].y * fast_exp2(w[p].z - low);
      w[p].x = fast_exp2(w[p].x - top);
    }
    const float2 back = kv_exp2_factors(top - low);
    const float inverse = sum == 0.0f ? 0.0f : back.x / sum;
#pragma unroll 1
    for (;;) {
#pragma unroll
      for (int i = 0; i < kColumns; ++i) {
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int p = 0; p < kFew; ++p) {
          acc.x = fmaf(x[i][p].x, w[p].x, acc.x);
          acc.y = fmaf(x[i][p].y, w[p].x, acc.y);
          acc.z = fmaf(x[i][p].z, w[p].x, acc.z);
          acc.w = fmaf(x[i][p].w, w[p].x, acc.w);
        }
        if (d + 4 * at_once * i < end) store(row, d + 4 * at_once * i, acc, inverse, back.y);
      }
      d += 4 * kColumns * at_once;
      if (d >= end) break;
      load();
    }
  };
  constexpr int kMost = 8;
  if (ok && unit.parts <= 4) {
    by_rows(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
  } else if (ok && unit.parts <= kMost) {
    by_rows(std::integral_constant<int, kMost>(), std::integral_constant<int, 2>());
  } else if (ok) {
    int lanes = 4;
    while (lanes < 32 && 4 * lanes < unit.parts) lanes *= 2;
    const int results = unit.rows * (kDim / 4);
    const int begin = results * unit.mine / unit.parts, end = results * (unit.mine + 1) / unit.parts;
    const int lane = threadIdx.x & (lanes - 1), slot = threadIdx.x / lanes;
    for (int i0 = begin; i0 < end; i0 += kThreads / lanes) {
      const int i = min(i0 + slot, end - 1);                      // whole warps stay together
      const int row = i % unit.rows, d = 4 * (i / unit.rows);
      float4 x[5];
      float4 w[5];
      float top = -INFINITY, low = -INFINITY;
#pragma unroll
      for (int k = 0; k < 5; ++k) {
        const int p = lane + k * lanes;
        w[k] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p < unit.parts) {
          const size_t part = kv_part_index(unit.first_block + p, p == 0);
          w[k] = __ldcg(kv_part_weight(work, part, row));
          x[k] = __ldcg(reinterpret_cast<const float4*>(kv_part_sum<kDim>(work, part, row, d)));
        }
        top = fmaxf(top, w[k].x);
        low = fmaxf(low, w[k].z);
      }
      for (int step = lanes >> 1; step >= 1; step >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
        low = fmaxf(low, __shfl_xor_sync(0xffffffffu, low, step));
      }
      if (top == -INFINITY) top = low = 0.0f;                     // nothing seen, or nothing but NaN
      float sum = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < 5; ++k) {
        const float f = fast_exp2(w[k].x - top);
        sum += w[k].z == -INFINITY ? w[k].y : w[k].y * fast_exp2(w[k].z - low);
        acc.x = fmaf(x[k].x, f, acc.x);
        acc.y = fmaf(x[k].y, f, acc.y);
        acc.z = fmaf(x[k].z, f, acc.z);
        acc.w = fmaf(x[k].w, f, acc.w);
      }
      for (int step = lanes >> 1; step >= 1; step >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, step);
        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, step);
        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, step);
        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, step);
        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, step);
      }
      const float2 back = kv_exp2_factors(top - low);
      if (lane == 0 && i0 + slot < end) store(row, d, acc, sum == 0.0f ? 0.0f : back.x / sum, back.y);
    }
  }
  if (ok) {
    // the last to leave puts the counters back
    if (threadIdx.x == 0 && atomicAdd(arrived + 1, 1u) == static_cast<unsigned>(unit.parts) - 1u) {
      arrived[0] = 0;
      arrived[1] = 0;
    }
  }
  __syncthreads();
}

// Rows [row0, row0 + rows) of the output are zero: they see nothing.  Called by all threads of a block.
template <int kDim, int kThreads>
__device__ __noinline__ void kv_zero_rows(const KvAttention& a, int row0, int rows) {
  uint4* out = reinterpret_cast<uint4*>(a.out + static_cast<long long>(row0) * a.shape.q_heads * kDim);
  const long long pieces = static_cast<long long>(rows) * a.shape.q_heads * (kDim / 8);
  for (long long i = threadIdx.x; i < pieces; i += kThreads) out[i] = make_uint4(0, 0, 0, 0);
}

// Shared memory of a block, so much at least that a SM holds one: a second block would wait for the first one's tensor memory, while
// the first may wait for the second one's part of a unit.
constexpr int kv_smem_bytes(int needed) { return needed > 120 * 1024 ? needed : 120 * 1024; }

// Launches a kernel whose blocks are all resident, with programmatic serialisation like launch_pdl.
template <typename... KernelArgs, typename... Args>
inline cudaError_t launch_resident(void (*kernel)(KernelArgs...), dim3 grid, dim3 block, size_t smem_bytes, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem_bytes;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeCooperative;
  attribute[0].val.cooperative = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, kernel, static_cast<KernelArgs>(args)...);
}

// Whether queries of these strides can have a tensor map: each stride is a whole multiple of the one before it, and none is zero.
inline bool kv_query_map_fits(const KvRows& q) { return q.head_stride > 0 && q.row_stride > 0 && q.row_stride % q.head_stride == 0; }
// Map of a call's queries: boxes of kRowBytes x the heads of a key/value head x tile_tokens.
bool kv_make_query_map(const KvAttention& a, int tile_tokens, CUtensorMap* map);
cudaError_t kv_decode(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream);
cudaError_t kv_prompt(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream);

}  // namespace aima
