// The gated delta rule in chunks: into how many segments a sequence's chunks are cut, and how a workspace is laid out for it.  Plain
// C++, for the kernels as for the host.
#pragma once

#include <algorithm>
#include <cstddef>

#ifdef __CUDACC__
#define AIMA_HOST_DEVICE __host__ __device__
#else
#define AIMA_HOST_DEVICE
#endif

namespace aima {

constexpr int kChunk = 64;                               // tokens
constexpr int kMaxSegments = 8, kMaxBorders = 3 * kMaxSegments;
constexpr int kMultiprocessors = 148;                    // that the workspace reckons with
constexpr size_t kBorderBytes = static_cast<size_t>(kMaxBorders) * 128 * 128 * sizeof(float);      // of a head of a sequence

struct Cut {
  int segments, first;                                   // first: eighths of the other segments' length that the first one has
};

// Where the segments of `chunks` chunks begin: all are as long, but for the first.
struct Segments {
  int first, per;
  AIMA_HOST_DEVICE Segments(int segments, int eighths, int chunks) {
    const int parts = 8 * (segments - 1) + eighths;
    per = (8 * chunks + parts - 1) / parts;
    const int left = chunks - (segments - 1) * per;
    first = left > 1 ? left : 1;
  }
  AIMA_HOST_DEVICE int begin(int segment) const { return segment == 0 ? 0 : first + (segment - 1) * per; }
};

// Jobs of two lengths on `places` multiprocessors, the long ones first; 0: the long ones do not all find room.
inline int makespan(int long_jobs, int length, int short_jobs, int short_length, int places) {
  if (long_jobs > places || (long_jobs == places && short_jobs > 0)) return 0;
  const int rounds = (short_jobs + places - long_jobs - 1) / std::max(places - long_jobs, 1);
  return std::max(long_jobs > 0 ? length : 0, rounds * short_length);
}

// What the two passes over the segments are estimated to take least with.  us as estimated, with segments of one length, without segments,
// captured: 32 heads, 512 tokens 49.5 / 49.5 / 51.5, 1024 72.4 / 80.0 / 91.4, 2048 123 / 126 / 187, 8192 381 / 422 / 713; 8 heads, 512
// 45.9 / 45.9 / 50.2, 1024 64.5 / 64.5 / 85.4, 8192 184 / 184 / 638; 64 heads, 1024 100 / 100 / 111, 8192 630 / 655 / 799.
// A chunk counts 5 in the second pass (about 5 us), 3 in the first; the first pass's launch and the join 12, and 3 for each product of
// the join.
inline Cut estimated_cut(int heads, int chunks, int places) {
  Cut best{1, 8};
  int least = 5 * chunks;
  if (2 * heads > places) return best;
  for (int g = 2; g <= kMaxSegments && g <= chunks; ++g) {
    for (const int eighths : {8, 4, 3, 2}) {
      const Segments cut(g, eighths, chunks);
      const int one = makespan(2 * (g - 2) * heads, cut.per, heads, cut.first, places);
      const int two = makespan((g - 1) * heads, cut.per, heads, cut.first, places);
      const int time = 3 * one + 5 * two + 12 + 3 * (g - 2);
      if (one > 0 && two > 0 && time < least) {
        least = time;
        best = Cut{g, eighths};
      }
    }
  }
  return best;
}
// Only what kMultiprocessors would be cut for too has room in a workspace.
inline Cut cut_of(int heads, int chunks, int places) {
  if (places < kMultiprocessors && estimated_cut(heads, chunks, kMultiprocessors).segments == 1) return Cut{1, 8};
  return estimated_cut(heads, chunks, std::min(places, kMultiprocessors));
}

// Tiles that sequences of more than min_rows rows each can have.
inline size_t tiles_of(int tokens, int sequences, int min_rows) {
  return static_cast<size_t>(tokens / kChunk) + std::min(sequences, tokens / (min_rows + 1));
}

// A workspace: the states at the borders of segments, if there are segments; then pair_bytes for each tile and key head; then head_bytes for
// each tile and value head.
struct ChunkLayout {
  Cut cut;
  size_t tiles, pairs_at, heads_at, bytes;
};
inline ChunkLayout chunk_layout(int k_heads, int v_heads, int tokens, int sequences, int max_new, int min_rows, int places, size_t pair_bytes,
                                size_t head_bytes) {
  ChunkLayout out{};
  out.cut = cut_of(v_heads * sequences, (max_new + kChunk - 1) / kChunk, places);
  out.tiles = tiles_of(tokens, sequences, min_rows);
  out.pairs_at = out.cut.segments > 1 ? static_cast<size_t>(v_heads) * sequences * kBorderBytes : 0;
  out.heads_at = out.pairs_at + out.tiles * k_heads * pair_bytes;
  out.bytes = out.heads_at + out.tiles * v_heads * head_bytes;
  return out;
}
// Heads of as many sequences as can be cut in a batch of at most max_tokens tokens and max_sequences sequences.
inline int heads_with_borders(int v_heads, int max_tokens, int max_sequences) {
  const int chunks = (max_tokens + kChunk - 1) / kChunk;
  for (int sequences = std::min(max_sequences, kMultiprocessors / 2 / v_heads); sequences > 0; --sequences)
    for (int c = 2; c <= chunks; ++c)
      if (cut_of(v_heads * sequences, c, kMultiprocessors).segments > 1) return v_heads * sequences;
  return 0;
}
// What all batches of a handle find room in; step_rows: rows up to which a sequence of a ragged batch is not taken in chunks.
inline size_t chunk_workspace(int k_heads, int v_heads, int max_tokens, int max_sequences, int step_rows, size_t pair_bytes, size_t head_bytes) {
  const size_t tiles = std::max(tiles_of(max_tokens, max_sequences, step_rows), tiles_of(max_tokens, 1, 0));
  return heads_with_borders(v_heads, max_tokens, max_sequences) * kBorderBytes + tiles * (k_heads * pair_bytes + v_heads * head_bytes);
}

}  // namespace aima
