// What the attention kernels over the paged 8-bit cache share: tensor maps, the division of the work and the join of what
// was divided.
#pragma once

#include "kv_cache.cuh"
#include "tcgen05.cuh"

namespace aima {

constexpr int kKvTile = 128;            // positions of the cache per step
constexpr int kKvMaxBlocks = 160;       // blocks of an attention kernel at most (one per SM)

struct KvMaps {
  CUtensorMap keys, values;             // [pages * kv_heads * page_tokens, head_dim] bytes, boxes of one page x up to 128 bytes
};

// The list of work: for every sequence, head by head and row tile by row tile, the tiles of the cache that its rows see.
// Block c of G takes the tiles [total c / G, total (c + 1) / G) of it, so that all stream the same amount; a unit (the tiles
// of one sequence, head and row tile) that ends up in several blocks leaves its part in the workspace of each, and
// kv_join_kernel puts the parts together.
__host__ __device__ inline long long kv_block_begin(long long total, int block, int blocks) { return total * block / blocks; }
__host__ __device__ inline int kv_block_of(long long total, long long tile, int blocks) {
  return static_cast<int>(((tile + 1) * blocks - 1) / total);
}

// Where a block of the prompt kernel begins: the unit and the tile inside it, and the place in the list in units of its cost.
struct alignas(16) KvStart {
  long long at;
  int sequence, row_tile, head, tile;
  int row0, rows, length, unused;       // of the sequence
};

// One part: rows x head_dim sums in FP32, and per row the reference maximum (log2) and the sum of the weights.
// A block has two: of the unit it begins in the middle (or that covers its whole share), and of the one it does not finish.
struct KvWorkspace {
  float* sums;            // [2 * kKvMaxBlocks][rows_per_part][head_dim]
  float2* weights;        // [2 * kKvMaxBlocks][rows_per_part]: maximum, sum
  long long* prefix;      // few rows: [sequences + 1] tiles before each sequence, left by block 0 for kv_join_kernel
  KvStart* starts;        // prompts: [blocks + 1]
  int rows_per_part;
};
// part of a unit that begins at tile `first` of the list, in block `block`
__host__ __device__ inline int kv_part(long long first, long long block_begin, int block) { return 2 * block + (first >= block_begin ? 1 : 0); }

struct KvAttentionPlan {
  KvAttention a;
  KvWorkspace work;
  int blocks;
  int tile_rows;          // rows (query heads of one key/value head x new tokens) of a row tile
  int tile_tokens;        // prompts: new tokens of a row tile
  unsigned long long wait_limit_ns;
};

// A unit of the prompt kernel: the rows of `tokens` new tokens of a sequence, for the query heads of one key/value head.
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

cudaError_t kv_decode(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream);
cudaError_t kv_prompt(const KvAttentionPlan& plan, const KvMaps& maps, cudaStream_t stream);

}  // namespace aima
