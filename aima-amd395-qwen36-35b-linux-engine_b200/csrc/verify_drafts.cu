// Verification of drafted tokens: acceptance against the target's probabilities, and the token drawn after it.
//
//   accepted   a = the first i with not (u_i q_i(x_i) < p_i(x_i)), or n
//   weights    w_t = p_n(t) if a = n, else max(p_a(t) - q_a(t), 0);  W_t = floor(2^40 w_t)
//   token      the lowest t with sum_{s <= t} W_s > floor(total * floor(2^24 u_n) / 2^24)
// The weights are whole numbers, so their sums are the same in every order: the draw does not depend on how the vocabulary
// is split over threads.  2^22 weights of at most 2^40 stay below 2^62.
#include "kv_cache.cuh"

namespace aima {
namespace {

constexpr int kVerifyThreads = 512;
constexpr int kAhead = 4;                      // steps of a warp whose loads are under way together
constexpr uint32_t kWholeVocabulary = 4096;    // up to here one block per sequence
constexpr uint32_t kResident = 256;            // blocks of the launch that run at once
constexpr uint32_t kLongRun = 32768;           // tokens of a block that are worth a cluster whatever runs beside it

// floor(2^40 w) of w clamped to [0, 1]; NaN counts as 0
__device__ __forceinline__ unsigned long long whole(float w) {
  return static_cast<unsigned long long>(__fmul_rn(fminf(fmaxf(w, 0.0f), 1.0f), 1099511627776.0f));
}

struct Weights {
  const float* p;        // the target's row
  const float* q;        // the draft's row or nullptr
  int without;           // token whose weight is zero (no draft probabilities), or -1
  __device__ __forceinline__ unsigned long long of(float w, float without_q, int t) const {
    w = fmaxf(w, 0.0f);
    if (q != nullptr) w = __fsub_rn(w, fmaxf(without_q, 0.0f));
    return t == without ? 0ull : whole(w);
  }
  // of tokens t .. t + 3, those from `last` on being 0
  template <bool kAligned>
  __device__ __forceinline__ void four(int t, int last, unsigned long long* out) const {
    float4 x = make_float4(0, 0, 0, 0), y = x;
    if (kAligned && t + 4 <= last) {
      x = *reinterpret_cast<const float4*>(p + t);
      if (q != nullptr) y = *reinterpret_cast<const float4*>(q + t);
    } else {
      float* xs = &x.x;
      float* ys = &y.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (t + i < last) {
          xs[i] = p[t + i];
          if (q != nullptr) ys[i] = q[t + i];
        }
      }
    }
    out[0] = of(x.x, y.x, t);
    out[1] = of(x.y, y.y, t + 1);
    out[2] = of(x.z, y.z, t + 2);
    out[3] = of(x.w, y.w, t + 3);
  }
  // the sum over tokens t .. t + 3 of kAhead steps, all loads first
  __device__ __forceinline__ unsigned long long ahead(int t) const {
    float4 x[kAhead], y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = __ldcs(reinterpret_cast<const float4*>(p + t + 128 * i));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) y[i] = q != nullptr ? __ldcs(reinterpret_cast<const float4*>(q + t + 128 * i)) : make_float4(0, 0, 0, 0);
    unsigned long long sum = 0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      sum += of(x[i].x, y[i].x, t + 128 * i);
      sum += of(x[i].y, y[i].y, t + 128 * i + 1);
      sum += of(x[i].z, y[i].z, t + 128 * i + 2);
      sum += of(x[i].w, y[i].w, t + 128 * i + 3);
    }
    return sum;
  }
};

__device__ __forceinline__ void store_u64_in_block(unsigned long long* local, uint32_t rank, unsigned long long value) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(remote), "l"(value) : "memory");
}

// Bound: reading one row (or a row of each) once, 8 bytes per token of the vocabulary with draft probabilities, and for few
// sequences the chain of dependent loads: draft, its probabilities, the row, the found run again.  32 sequences of 248320 (64 MB):
// 16.0 us with the rows in L2, 20.6 us from memory (3.1 TB/s); 148 sequences (294 MB) 63 us (4.7 TB/s); 1 sequence 8.3 us.  The
// loads of four steps are issued together: with one step at a time 17.8 and 10.1 us.
// A cluster of kBlocks per sequence.  The vocabulary is cut into one run of whole 128-token steps per warp; each warp sums its
// run (a float4 per lane and step), the blocks exchange their sums through each other's shared memory, and the warp whose run
// holds the token goes through it a second time.
template <int kBlocks, bool kAligned>
__global__ void __launch_bounds__(kVerifyThreads)
verify_drafts_kernel(const aima_moe_verify_drafts c) {
  constexpr int kWarps = kVerifyThreads / 32;
  __shared__ unsigned long long warp_sum[kWarps], block_sum[2][kBlocks];
  __shared__ int accepted_s;
  if (kBlocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this block runs
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = blockIdx.x / kBlocks, rank = blockIdx.x % kBlocks;
  const int vocabulary = static_cast<int>(c.vocabulary), most = static_cast<int>(c.max_drafts);
  const float* target = static_cast<const float*>(c.target) + s * c.target_sequence_stride;
  const float* draft = c.draft != nullptr ? static_cast<const float*>(c.draft) + s * c.draft_sequence_stride : nullptr;
  const int* x = c.draft_tokens + static_cast<size_t>(s) * most;
  const float* u = c.uniforms + static_cast<size_t>(s) * (most + 1);
  const float uniform = fminf(fmaxf(u[most], 0.0f), 0.99999994f);
  int n = most;
  if (warp == 0) {
    if (c.draft_counts != nullptr) n = min(max(c.draft_counts[s], 0), most);
    int a = n;
    for (int i0 = 0; i0 < n && a == n; i0 += 32) {        // every lane looks at a draft
      const int i = i0 + lane;
      bool stays = true;
      if (i < n) {
        const int t = x[i];
        stays = t >= 0 && t < vocabulary;
        if (stays) {
          const float p = fmaxf(target[i * c.target_row_stride + t], 0.0f);
          const float q = draft != nullptr ? fmaxf(draft[i * c.draft_row_stride + t], 0.0f) : 1.0f;
          stays = __fmul_rn(fmaxf(u[i], 0.0f), q) < p;
        }
      }
      const uint32_t rejected = __ballot_sync(0xffffffffu, !stays);
      if (rejected != 0) a = i0 + __ffs(static_cast<int>(rejected)) - 1;
    }
    if (lane == 0) accepted_s = a;
  }
  __syncthreads();
  const int a = accepted_s;
  if (c.draft_counts != nullptr) n = min(max(c.draft_counts[s], 0), most);
  Weights w;
  w.p = target + a * c.target_row_stride;
  w.q = a < n && draft != nullptr ? draft + a * c.draft_row_stride : nullptr;
  w.without = a < n && draft == nullptr ? x[a] : -1;
  const int steps = (vocabulary + kBlocks * kWarps * 128 - 1) / (kBlocks * kWarps * 128);
  const int first = min(vocabulary, (rank * kWarps + warp) * steps * 128), last = min(vocabulary, first + steps * 128);
  bool found = false;
#pragma unroll 1
  for (int attempt = 0; attempt < 2 && !found; ++attempt) {
    unsigned long long sum = 0;
    int t0 = first;
    if (kAligned) {
      for (; t0 + 128 * kAhead <= last; t0 += 128 * kAhead) sum += w.ahead(t0 + 4 * lane);
    }
    for (; t0 < last; t0 += 128) {
      unsigned long long v[4];
      w.four<kAligned>(t0 + 4 * lane, last, v);
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) warp_sum[warp] = sum;
    // before the first store into another block: it runs
    if (kBlocks > 1 && attempt == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
      unsigned long long mine = lane < kWarps ? warp_sum[lane] : 0ull;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
      if (kBlocks > 1) {
        if (lane < kBlocks) store_u64_in_block(&block_sum[attempt][rank], lane, mine);
      } else if (lane == 0) {
        block_sum[attempt][0] = mine;
      }
    }
    if (kBlocks > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
      __syncthreads();
    }
    unsigned long long total = 0, before = 0;
#pragma unroll
    for (int r = 0; r < kBlocks; ++r) {
      const unsigned long long b = block_sum[attempt][r];
      if (r < rank) before += b;
      total += b;
    }
    if (total != 0) {
      found = true;
      const unsigned long long step = static_cast<unsigned long long>(__fmul_rn(uniform, 16777216.0f));
      const unsigned long long below = (total >> 24) * step + (((total & 0xffffffull) * step) >> 24);
      if (before <= below && below - before < block_sum[attempt][rank]) {
        for (int i = 0; i < warp; ++i) before += warp_sum[i];
        if (before <= below && below - before < sum) {                  // one warp of all: its run holds the token
          for (t0 = first; t0 < last; t0 += 128) {
            unsigned long long v[4];
            w.four<kAligned>(t0 + 4 * lane, last, v);
            const unsigned long long mine = (v[0] + v[1]) + (v[2] + v[3]);
            unsigned long long run = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const unsigned long long other = __shfl_up_sync(0xffffffffu, run, d);
              if (lane >= d) run += other;
            }
            const uint32_t over = __ballot_sync(0xffffffffu, before + run > below);
            if (over != 0) {
              if (lane == __ffs(static_cast<int>(over)) - 1) {
                unsigned long long at = before + run - mine;
                int token = t0 + 4 * lane;
                for (int i = 0; i < 3 && at + v[i] <= below; ++i, ++token) at += v[i];
                c.tokens[static_cast<size_t>(s) * (most + 1) + a] = token;
              }
              break;
            }
            before += __shfl_sync(0xffffffffu, run, 31);
          }
        }
      }
    } else {
      w.q = nullptr;                                                    // nothing left: from the target's row itself
      w.without = -1;
    }
  }
  if (rank == 0) {
    for (int i = threadIdx.x; i <= most; i += blockDim.x) {
      if (i != a || !found) c.tokens[static_cast<size_t>(s) * (most + 1) + i] = i < a ? x[i] : -1;
    }
    if (threadIdx.x == 0) {
      c.accepted[s] = a;
      if (c.new_lengths != nullptr) c.new_lengths[s] = c.cache_lengths[s] - (n - a);
    }
  }
}

template <int kBlocks, bool kAligned>
cudaError_t launch(const aima_moe_verify_drafts& call, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(call.sequences * kBlocks);
  config.blockDim = dim3(kVerifyThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = kBlocks;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, verify_drafts_kernel<kBlocks, kAligned>, call);
}

}  // namespace

cudaError_t verify_drafts(const aima_moe_verify_drafts& call, cudaStream_t stream) {
  const bool aligned = reinterpret_cast<uintptr_t>(call.target) % 16 == 0 && call.target_sequence_stride % 4 == 0 && call.target_row_stride % 4 == 0 &&
                       reinterpret_cast<uintptr_t>(call.draft) % 16 == 0 && call.draft_sequence_stride % 4 == 0 && call.draft_row_stride % 4 == 0;
  // As many blocks per sequence as run at once.  us with 1 / 2 / 4 / 8 blocks, vocabulary 4096: 1 sequence 3.5 / 3.9 / 3.7 / 3.8;
  // 32768: 8 sequences 10.1 / 7.9 / 5.7 / 4.9, 64 10.6 / 8.6 / 6.9 / 10.3, 300 18.2 / 19.7 / 24.7 / 44.3; 131072: 8 sequences
  // 33 / 18 / 12 / 8.0, 148 58 / 37 / 35 / 38.
  uint32_t blocks = call.vocabulary <= kWholeVocabulary ? 1 : 8;
  while (blocks > 1 && call.sequences * blocks > kResident && call.vocabulary / blocks < kLongRun) blocks /= 2;
  switch (blocks) {
    case 8: return aligned ? launch<8, true>(call, stream) : launch<8, false>(call, stream);
    case 4: return aligned ? launch<4, true>(call, stream) : launch<4, false>(call, stream);
    case 2: return aligned ? launch<2, true>(call, stream) : launch<2, false>(call, stream);
    default: return aligned ? launch<1, true>(call, stream) : launch<1, false>(call, stream);
  }
}

}  // namespace aima
