// Keys and values of new tokens into the paged 8-bit cache, rotated on the way; the queries with them.
//
//   rot(x)[j]     = x[j] cos_j - x[j + h] sin_j
//   rot(x)[j + h] = x[j + h] cos_j + x[j] sin_j        j < h = rotary / 2, the rest of a head passes through
//   scale         = 2^e, e the least integer with max|x| <= 448 * 2^e over the page's rows of a head
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

constexpr int kAppendThreads = 256;

__device__ __forceinline__ bool finite8(const float* x) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) ok = ok && fabsf(x[i]) <= 3.402823466e38f;
  return ok;
}
__device__ __forceinline__ float amax8(const float* x) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
  return m;
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
// exponent of the power of two that is not below a scale
__device__ __forceinline__ int exponent_of(float scale) {
  const int bits = __float_as_int(scale);
  return min(max(((bits >> 23) & 255) - 127 + ((bits & 0x7fffff) != 0 ? 1 : 0), kKvMinExponent), kKvMaxExponent);
}

// Vector `piece` (elements 8 piece .. 8 piece + 7) of a head, rotated.  Called by whole groups of kDim / 8 lanes that hold
// one head; the partner's vector comes by shuffle.
template <int kDim>
__device__ __forceinline__ void rotate8(const uint4& raw, int piece, int rotary, const float* angle, bool active, float* x) {
  const int half = rotary >> 4;              // vectors of one half
  const int group0 = (threadIdx.x & 31) & ~(kDim / 8 - 1);
  const int partner = group0 + (piece < half ? piece + half : piece - half);
  const bool turns = piece < 2 * half;
  uint4 other;
  other.x = __shfl_sync(0xffffffffu, raw.x, turns ? partner : 0);
  other.y = __shfl_sync(0xffffffffu, raw.y, turns ? partner : 0);
  other.z = __shfl_sync(0xffffffffu, raw.z, turns ? partner : 0);
  other.w = __shfl_sync(0xffffffffu, raw.w, turns ? partner : 0);
  unpack8(raw, x);
  if (turns && active) {
    float y[8];
    unpack8(other, y);
    const float* cosine = angle + 8 * (piece < half ? piece : piece - half);
    const float* sine = cosine + 8 * half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = __fmul_rn(x[i], __ldg(cosine + i)), b = __fmul_rn(y[i], __ldg(sine + i));
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

// One block per (sequence, touched page, head), then blocks for the queries.  A page and head belongs to one block, which
// holds all of its new rows in registers between finding the scale and writing the codes: every byte is read once.
template <int kDim, int kPage>
__global__ void __launch_bounds__(kAppendThreads)
kv_append_kernel(const KvAppend a, int page_blocks, int columns_per_sequence) {
  constexpr int kPieces = kDim / 8;                                   // 16-byte vectors of a head
  constexpr int kRowsPerPass = kAppendThreads / kPieces;
  constexpr int kPasses = (kPage + kRowsPerPass - 1) / kRowsPerPass;
  __shared__ float warp_amax[2][kAppendThreads / 32];
  const int piece = threadIdx.x % kPieces;
  const int slot0 = threadIdx.x / kPieces;
  const KvShape& shape = a.shape;

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
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int position = page_start + slot0 + p * kRowsPerPass;
      const bool active = position >= low && position < high;
      float k[8], v[8];
      rotate8<kDim>(kraw[p], piece, shape.rotary, a.rotation + static_cast<size_t>(position) * shape.rotary, active, k);
      unpack8(vraw[p], v);
      int bad = (finite8(k) && finite8(v)) ? 0 : 1;
#pragma unroll
      for (int d = kPieces / 2; d >= 1; d >>= 1) bad |= __shfl_xor_sync(0xffffffffu, bad, d);
      if (bad) {
        poisoned |= 1u << p;
      } else {
        kmax = fmaxf(kmax, amax8(k));
        vmax = fmaxf(vmax, amax8(v));
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
    int exponent[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float m = warp_amax[t][0];
#pragma unroll
      for (int w = 1; w < kAppendThreads / 32; ++w) m = fmaxf(m, warp_amax[t][w]);
      exponent[t] = kv_scale_exponent(m);
      if (held) exponent[t] = max(exponent[t], exponent_of(old_scale[t]));
    }
    if (threadIdx.x == 0) {
      a.layer.key_scales[scale_at] = kv_exp2(exponent[0]);
      a.layer.value_scales[scale_at] = kv_exp2(exponent[1]);
    }
    const size_t base = scale_at * kPage * kDim;
    const float kinv = kv_exp2(-exponent[0]), vinv = kv_exp2(-exponent[1]);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int slot = slot0 + p * kRowsPerPass, position = page_start + slot;
      const bool active = position >= low && position < high;
      float k[8], v[8];
      rotate8<kDim>(kraw[p], piece, shape.rotary, a.rotation + static_cast<size_t>(position) * shape.rotary, active, k);
      unpack8(vraw[p], v);
      if (active) {
        uint2 kc = codes8(k, kinv), vc = codes8(v, vinv);
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
          const float ratio = old_scale[t] * kv_exp2(-exponent[t]);
          if (ratio == 1.0f) continue;
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

  // queries: kPieces lanes hold one head of one row, which stays with its thread for all heads of the row
  if (a.q.data == nullptr) return;
  const int row = (blockIdx.x - page_blocks) * kRowsPerPass + slot0;
  const bool exists = row < a.batch.tokens;
  int position = -1;
  if (exists) {
    const int s = sequence_of_row(a.batch, row);
    const KvSequence seq = kv_sequence(a.batch, shape, s);
    if (!seq.bad && row >= seq.row0 && row < seq.row0 + seq.rows) position = seq.length - seq.rows + row - seq.row0;
  }
  const bool turns = position >= 0 && position < a.positions;
  for (int head = 0; head < shape.q_heads; ++head) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (exists) raw = *reinterpret_cast<const uint4*>(a.q.data + row * a.q.row_stride + head * a.q.head_stride + 8 * piece);
    float x[8];
    rotate8<kDim>(raw, piece, shape.rotary, a.rotation + static_cast<size_t>(max(position, 0)) * shape.rotary, turns, x);
    uint4 w;
    w.x = static_cast<uint32_t>(float_to_bf16_bits(x[0])) | (static_cast<uint32_t>(float_to_bf16_bits(x[1])) << 16);
    w.y = static_cast<uint32_t>(float_to_bf16_bits(x[2])) | (static_cast<uint32_t>(float_to_bf16_bits(x[3])) << 16);
    w.z = static_cast<uint32_t>(float_to_bf16_bits(x[4])) | (static_cast<uint32_t>(float_to_bf16_bits(x[5])) << 16);
    w.w = static_cast<uint32_t>(float_to_bf16_bits(x[6])) | (static_cast<uint32_t>(float_to_bf16_bits(x[7])) << 16);
    if (exists) *reinterpret_cast<uint4*>(a.q_out + (static_cast<long long>(row) * shape.q_heads + head) * kDim + 8 * piece) = w;
  }
}

template <int kDim, int kPage>
cudaError_t launch(const KvAppend& a, cudaStream_t stream) {
  const int columns = (a.batch.max_new + kPage - 2) / kPage + 1;      // pages that max_new consecutive tokens can touch
  const long long page_blocks = static_cast<long long>(columns) * a.shape.kv_heads * a.batch.sequences;
  const int rows_per_block = kAppendThreads / (kDim / 8);
  const long long query_blocks = a.q.data != nullptr ? (a.batch.tokens + rows_per_block - 1) / rows_per_block : 0;
  if (page_blocks + query_blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  kv_append_kernel<kDim, kPage><<<static_cast<unsigned>(page_blocks + query_blocks), kAppendThreads, 0, stream>>>(a, static_cast<int>(page_blocks), columns);
  return cudaGetLastError();
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
