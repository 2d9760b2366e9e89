// Keys and values of new tokens into the paged 8-bit cache, rotated on the way; the queries with them.
//
//   rot(x)[j]     = x[j] cos_j - x[j + h] sin_j
//   rot(x)[j + h] = x[j + h] cos_j + x[j] sin_j        j < h = rotary / 2, the rest of a head passes through
//   scale         = 2^e, e the least integer with max|x| <= 448 * 2^e over the page's new rows of a head; a page that holds older
//                   rows keeps the scale it has while the new ones fit
//   code          = e4m3(x / scale)
// in FP32, every product, difference and sum rounded on its own.  One rounding leads from the rotated key to its code.
//
// A scale that is a power of two costs a floating-point code nothing in its mantissa, and a page whose scale has to grow
// keeps its codes: dividing them by 2, 4, ... is exact but for those that fall below e4m3's normal range.  So what the cache
// holds hardly depends on whether a page was filled by one call or by sixty-four.
#include "kv_cache.cuh"

#include <cuda_fp8.h>

namespace aima {
namespace {

constexpr int kHeadsPerThread = 8;                  // query heads of a row that share its angles; with four 8192 tokens took 1.8 us more
constexpr long long kApartElements = 1 << 21;       // of queries: more are rotated by a kernel of their own
constexpr int kRotateThreads = 256;
// A thread of the page blocks has up to four vectors of keys and four of values under way.  (Eight: one token 5.8 us instead of 3.9.)
template <int kDim, int kPage>
constexpr int append_threads = kPage * kDim < 256 * 32 ? 256 : kPage * kDim / 32;

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The largest magnitude; NaN if one of the values is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float amax8(const float* x) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
  return m;
}
// of eight BF16 values, whose magnitudes are ordered as integers, NaN last
__device__ __forceinline__ float amax8(const uint4& raw) {
  const uint32_t m = __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu), __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
  return __uint_as_float(max(m & 0xffffu, m >> 16) << 16);
}
// eight values times a power of two -> eight e4m3 codes
__device__ __forceinline__ uint2 codes8(const float* x, float inverse) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * h] * inverse, x[4 * h + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * h + 2] * inverse, x[4 * h + 3] * inverse), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// 1 / scale; powers of two, which is what an append writes, by their exponent
__device__ __forceinline__ float inverse_of(float scale) {
  const int bits = __float_as_int(scale);
  return (bits & 0x7fffff) == 0 && bits > 0 && bits < (254 << 23) ? __int_as_float((254 << 23) - bits) : __frcp_rn(scale);
}

// A vector that this thread has read before; the compiler would keep the first one in registers.
__device__ __forceinline__ uint4 load_again(const void* from) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(from));
  return v;
}

// The eight angles of a vector of the rotated part: cosines and sines of one position.
struct Angles {
  float4 c0, c1, s0, s1;
};
__device__ __forceinline__ Angles load_angles(const float* row, int piece, int half) {
  const float4* c = reinterpret_cast<const float4*>(row) + 2 * (piece < half ? piece : piece - half);
  const float4* s = c + 2 * half;
  return Angles{__ldg(c), __ldg(c + 1), __ldg(s), __ldg(s + 1)};
}
// Vector `piece` (elements 8 piece .. 8 piece + 7) of a head, rotated.  Called by whole groups of kDim / 8 lanes that hold
// one head; the partner's vector comes by shuffle.  half: vectors of one half of the rotated part.
template <int kDim>
__device__ __forceinline__ void rotate8(const uint4& raw, int piece, int half, const Angles& angles, bool active, float* x) {
  const int group0 = (threadIdx.x & 31) & ~(kDim / 8 - 1);
  const bool turns = piece < 2 * half;
  const int partner = turns ? group0 + (piece < half ? piece + half : piece - half) : 0;
  uint4 other;
  other.x = __shfl_sync(0xffffffffu, raw.x, partner);
  other.y = __shfl_sync(0xffffffffu, raw.y, partner);
  other.z = __shfl_sync(0xffffffffu, raw.z, partner);
  other.w = __shfl_sync(0xffffffffu, raw.w, partner);
  unpack8(raw, x);
  if (turns && active) {
    const float c[8] = {angles.c0.x, angles.c0.y, angles.c0.z, angles.c0.w, angles.c1.x, angles.c1.y, angles.c1.z, angles.c1.w};
    const float s[8] = {angles.s0.x, angles.s0.y, angles.s0.z, angles.s0.w, angles.s1.x, angles.s1.y, angles.s1.z, angles.s1.w};
    float y[8];
    unpack8(other, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = __fmul_rn(x[i], c[i]), b = __fmul_rn(y[i], s[i]);
      x[i] = piece < half ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
  }
}

__device__ __forceinline__ int sequence_of_row(const KvBatch& b, int row) {
  if (b.offsets == nullptr) return row / b.max_new;
  int low = 0, high = b.sequences;           // offsets[low] <= row < offsets[high] unless the row is of no sequence
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (b.offsets[mid] <= row) low = mid; else high = mid;
  }
  return low;
}

// Queries: kDim / 8 lanes hold one head of one row, kHeadsPerThread heads at once, which share the row's angles.
template <int kDim, int kThreads>
__device__ __forceinline__ void rotate_queries(const KvAppend& a, long long block) {
  constexpr int kPieces = kDim / 8, kRowsPerPass = kThreads / kPieces;
  const int piece = threadIdx.x % kPieces, slot0 = threadIdx.x / kPieces;
  const KvShape& shape = a.shape;
  const int half = shape.rotary >> 4;
  const int head_groups = (shape.q_heads + kHeadsPerThread - 1) / kHeadsPerThread;
  const long long work = block * kRowsPerPass + slot0;
  const int row = static_cast<int>(min(work / head_groups, static_cast<long long>(a.batch.tokens)));
  const int head0 = static_cast<int>(work % head_groups) * kHeadsPerThread;
  const bool exists = row < a.batch.tokens;
  uint4 raw[kHeadsPerThread];
#pragma unroll
  for (int h = 0; h < kHeadsPerThread; ++h) {
    raw[h] = make_uint4(0, 0, 0, 0);
    if (exists && head0 + h < shape.q_heads)
      raw[h] = __ldcs(reinterpret_cast<const uint4*>(a.q.data + row * a.q.row_stride + (head0 + h) * a.q.head_stride + 8 * piece));
  }
  int position = -1;
  if (exists) {
    const int s = sequence_of_row(a.batch, row);
    const KvSequence seq = kv_sequence(a.batch, shape, s);
    if (!seq.bad && row >= seq.row0 && row < seq.row0 + seq.rows) position = seq.length - seq.rows + row - seq.row0;
  }
  const bool active = position >= 0 && position < a.positions;
  Angles angles{};
  if (active && piece < 2 * half) angles = load_angles(a.rotation + static_cast<size_t>(position) * shape.rotary, piece, half);
#pragma unroll
  for (int h = 0; h < kHeadsPerThread; ++h) {
    float x[8];
    rotate8<kDim>(raw[h], piece, half, angles, active, x);
    uint4 w;
    w.x = static_cast<uint32_t>(float_to_bf16_bits(x[0])) | (static_cast<uint32_t>(float_to_bf16_bits(x[1])) << 16);
    w.y = static_cast<uint32_t>(float_to_bf16_bits(x[2])) | (static_cast<uint32_t>(float_to_bf16_bits(x[3])) << 16);
    w.z = static_cast<uint32_t>(float_to_bf16_bits(x[4])) | (static_cast<uint32_t>(float_to_bf16_bits(x[5])) << 16);
    w.w = static_cast<uint32_t>(float_to_bf16_bits(x[6])) | (static_cast<uint32_t>(float_to_bf16_bits(x[7])) << 16);
    if (exists && head0 + h < shape.q_heads)
      *reinterpret_cast<uint4*>(a.q_out + (static_cast<long long>(row) * shape.q_heads + head0 + h) * kDim + 8 * piece) = w;
  }
}

// One block per (sequence, touched page, head), then blocks for the queries.  A page and head belongs to one block, which goes
// through its new rows twice: for the largest magnitudes, and, with the scale, for the codes.  The second time they come from
// the caches: held in registers they would leave room for one block per SM (8192 tokens 35.8 us instead of 33.4, with 32/8 heads of
// 128 50.7 instead of 45.7; one token 3.9 instead of 4.2).
//
// Bound: bytes.  8192 tokens with 16/2 heads of 256 read 84 MB and write 75 MB; 33.4 us are 4.8 TB/s (the queries' stream, 134 MB, alone
// 27 us).  One token is bound by its launch and three dependent loads (length, page, rows).
template <int kDim, int kPage>
__global__ void __launch_bounds__(append_threads<kDim, kPage>, append_threads<kDim, kPage> > 512 ? 1 : 1024 / append_threads<kDim, kPage>)
kv_append_kernel(const KvAppend a, int page_blocks, int columns_per_sequence) {
  constexpr int kAppendThreads = append_threads<kDim, kPage>;
  constexpr int kPieces = kDim / 8;                                   // 16-byte vectors of a head
  constexpr int kRowsPerPass = kAppendThreads / kPieces;
  constexpr int kPasses = (kPage + kRowsPerPass - 1) / kRowsPerPass;
  __shared__ float warp_amax[2][kAppendThreads / 32];
  const int piece = threadIdx.x % kPieces;
  const int slot0 = threadIdx.x / kPieces;
  const KvShape& shape = a.shape;
  const int half = shape.rotary >> 4;
  pdl_launch_dependents();       // after what came before this kernel has ended: it is launched without the attribute

  if (static_cast<int>(blockIdx.x) < page_blocks) {
    const int head = blockIdx.x % shape.kv_heads;
    const int column_index = (blockIdx.x / shape.kv_heads) % columns_per_sequence;
    const int s = blockIdx.x / (shape.kv_heads * columns_per_sequence);
    const KvSequence seq = kv_sequence(a.batch, shape, s);
    if (seq.bad && threadIdx.x == 0) atomicOr(a.status, kKvBadBatch);
    const int begin = max(0, seq.length - seq.rows);                   // first new position
    const int column = (begin >> shape.page_shift) + column_index;
    const int page_start = column << shape.page_shift;
    const int low = max(begin, page_start), high = min(seq.length, page_start + kPage);
    if (low >= high) return;                                           // the same for the whole block
    const int page = a.batch.table[static_cast<size_t>(s) * a.batch.columns + column];
    if (page < 0 || page >= shape.pages || (shape.rotary > 0 && high > a.positions)) {
      if (threadIdx.x == 0) atomicOr(a.status, kKvBadBatch);
      return;
    }
    const int first_row = seq.row0 + seq.rows - seq.length;            // + position = row
    uint4 kraw[kPasses], vraw[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int position = page_start + slot0 + p * kRowsPerPass;
      kraw[p] = vraw[p] = make_uint4(0, 0, 0, 0);
      if (position >= low && position < high) {
        const long long row = first_row + position;
        kraw[p] = *reinterpret_cast<const uint4*>(a.k.data + row * a.k.row_stride + head * a.k.head_stride + 8 * piece);
        vraw[p] = *reinterpret_cast<const uint4*>(a.v.data + row * a.v.row_stride + head * a.v.head_stride + 8 * piece);
      }
    }
    float kmax = 0.0f, vmax = 0.0f;
    uint32_t poisoned = 0;
    const uint32_t head_lanes = kPieces == 32 ? 0xffffffffu : ((1u << (kPieces & 31)) - 1u) << ((threadIdx.x & 31) & ~(kPieces - 1));
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int position = page_start + slot0 + p * kRowsPerPass;
      const bool active = position >= low && position < high;
      float k[8];
      Angles angles{};
      if (active && piece < 2 * half) angles = load_angles(a.rotation + static_cast<size_t>(position) * shape.rotary, piece, half);
      rotate8<kDim>(kraw[p], piece, half, angles, active, k);
      const float k8 = amax8(k), v8 = amax8(vraw[p]);
      const uint32_t bad = __ballot_sync(0xffffffffu, !(k8 <= 3.402823466e38f && v8 <= 3.402823466e38f));
      if ((bad & head_lanes) != 0) {
        poisoned |= 1u << p;
      } else {
        kmax = fmaxf(kmax, k8);
        vmax = fmaxf(vmax, v8);
      }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
      kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, d));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
    }
    if ((threadIdx.x & 31) == 0) {
      warp_amax[0][threadIdx.x >> 5] = kmax;
      warp_amax[1][threadIdx.x >> 5] = vmax;
    }
    const size_t scale_at = static_cast<size_t>(page) * shape.kv_heads + head;
    const bool held = low > page_start;                                // the page holds older tokens
    float old_scale[2] = {1.0f, 1.0f};
    if (held) {
      old_scale[0] = a.layer.key_scales[scale_at];
      old_scale[1] = a.layer.value_scales[scale_at];
    }
    __syncthreads();
    float scale[2], inverse[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float m = warp_amax[t][0];
#pragma unroll
      for (int w = 1; w < kAppendThreads / 32; ++w) m = fmaxf(m, warp_amax[t][w]);
      // a scale that the page came with stays as it is while the new rows fit, whether it is a power of two or not
      scale[t] = held && m <= 448.0f * old_scale[t] ? old_scale[t] : kv_exp2(kv_scale_exponent(m));
      inverse[t] = inverse_of(scale[t]);
    }
    if (threadIdx.x == 0) {
      a.layer.key_scales[scale_at] = scale[0];
      a.layer.value_scales[scale_at] = scale[1];
    }
    const size_t base = scale_at * kPage * kDim;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int slot = slot0 + p * kRowsPerPass, position = page_start + slot;
      const bool active = position >= low && position < high;
      float k[8], v[8];
      uint4 kagain = make_uint4(0, 0, 0, 0), vagain = kagain;
      if (active) {
        const long long row = first_row + position;
        kagain = load_again(a.k.data + row * a.k.row_stride + head * a.k.head_stride + 8 * piece);
        vagain = load_again(a.v.data + row * a.v.row_stride + head * a.v.head_stride + 8 * piece);
      }
      Angles angles{};
      if (active && piece < 2 * half) angles = load_angles(a.rotation + static_cast<size_t>(position) * shape.rotary, piece, half);
      rotate8<kDim>(kagain, piece, half, angles, active, k);
      unpack8(vagain, v);
      if (active) {
        uint2 kc = codes8(k, inverse[0]), vc = codes8(v, inverse[1]);
        if ((poisoned >> p) & 1u) {
          kc = make_uint2(kKvNan * 0x01010101u, kKvNan * 0x01010101u);
          vc = make_uint2(0, 0);
        }
        *reinterpret_cast<uint2*>(a.layer.keys + base + slot * kDim + 8 * piece) = kc;
        *reinterpret_cast<uint2*>(a.layer.values + base + slot * kDim + 8 * piece) = vc;
      } else if (held && position < low) {
        // an older token: to the larger scale, where there is one
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (scale[t] == old_scale[t]) continue;
          const float ratio = old_scale[t] * inverse[t];
          uint2* at = reinterpret_cast<uint2*>((t == 0 ? a.layer.keys : a.layer.values) + base + slot * kDim + 8 * piece);
          const uint2 codes = *at;
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))) & 255u), __NV_E4M3)));
          *at = codes8(x, ratio);
        }
      }
    }
    return;
  }

  if (a.q.data != nullptr) rotate_queries<kDim, kAppendThreads>(a, static_cast<long long>(blockIdx.x) - page_blocks);
}

template <int kDim>
__global__ void __launch_bounds__(kRotateThreads, 4)
kv_rotate_kernel(const KvAppend a) {
  rotate_queries<kDim, kRotateThreads>(a, blockIdx.x);
  pdl_wait();          // the page kernel has ended when this one does: whoever waits for this one waits for both
}

template <int kDim, int kPage>
cudaError_t launch(const KvAppend& a, cudaStream_t stream) {
  constexpr int kAppendThreads = append_threads<kDim, kPage>;
  const int columns = (a.batch.max_new + kPage - 2) / kPage + 1;      // pages that max_new consecutive tokens can touch
  const long long page_blocks = static_cast<long long>(columns) * a.shape.kv_heads * a.batch.sequences;
  const long long query_work = a.q.data != nullptr ? static_cast<long long>(a.batch.tokens) * ((a.shape.q_heads + kHeadsPerThread - 1) / kHeadsPerThread) : 0;
  // Few queries are rotated by blocks of the same launch.  Many are a stream of their own beside the page blocks, whose registers
  // would leave too few of the stream's bytes in flight.  us together / apart, 16 heads of 256: 256 tokens 5.7 / 6.3, 512 6.0 / 6.4,
  // 1024 8.0 / 6.5, 8192 43 / 33.
  const bool apart = query_work * kHeadsPerThread * kDim > kApartElements;
  const long long query_blocks = apart ? 0 : (query_work + kAppendThreads / (kDim / 8) - 1) / (kAppendThreads / (kDim / 8));
  const long long rotate_blocks = (query_work + kRotateThreads / (kDim / 8) - 1) / (kRotateThreads / (kDim / 8));
  if (page_blocks + query_blocks > 0x7fffffffll || rotate_blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  KvAppend pages = a;
  if (apart) pages.q.data = nullptr;
  kv_append_kernel<kDim, kPage><<<static_cast<unsigned>(page_blocks + query_blocks), kAppendThreads, 0, stream>>>(pages, static_cast<int>(page_blocks), columns);
  const cudaError_t error = cudaGetLastError();
  if (error != cudaSuccess || !apart) return error;
  return launch_pdl(kv_rotate_kernel<kDim>, dim3(static_cast<unsigned>(rotate_blocks)), dim3(kRotateThreads), 0, stream, a);
}

template <int kDim>
cudaError_t launch_page(const KvAppend& a, cudaStream_t stream) {
  switch (a.shape.page_tokens) {
    case 16: return launch<kDim, 16>(a, stream);
    case 32: return launch<kDim, 32>(a, stream);
    case 64: return launch<kDim, 64>(a, stream);
    default: return launch<kDim, 128>(a, stream);
  }
}

}  // namespace

cudaError_t kv_append(const KvAppend& a, cudaStream_t stream) {
  switch (a.shape.head_dim) {
    case 64: return launch_page<64>(a, stream);
    case 128: return launch_page<128>(a, stream);
    default: return launch_page<256>(a, stream);
  }
}

}  // namespace aima
