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

constexpr int kVerifyThreads = 1024;

// floor(2^40 w) of w clamped to [0, 1]; NaN counts as 0
__device__ __forceinline__ unsigned long long whole(float w) {
  return static_cast<unsigned long long>(__fmul_rn(fminf(fmaxf(w, 0.0f), 1.0f), 1099511627776.0f));
}

struct Weights {
  const float* p;        // the target's row
  const float* q;        // the draft's row or nullptr
  int without;           // token whose weight is zero (no draft probabilities), or -1
  __device__ __forceinline__ unsigned long long at(int t) const {
    float w = fmaxf(p[t], 0.0f);
    if (q != nullptr) w = __fsub_rn(w, fmaxf(q[t], 0.0f));
    return t == without ? 0ull : whole(w);
  }
};

__global__ void __launch_bounds__(kVerifyThreads)
verify_drafts_kernel(const aima_moe_verify_drafts c) {
  __shared__ unsigned long long warp_sum[kVerifyThreads / 32];
  __shared__ unsigned long long total_s;
  __shared__ int accepted_s, token_s;
  const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int vocabulary = static_cast<int>(c.vocabulary), most = static_cast<int>(c.max_drafts);
  const float* target = static_cast<const float*>(c.target) + s * c.target_sequence_stride;
  const float* draft = c.draft != nullptr ? static_cast<const float*>(c.draft) + s * c.draft_sequence_stride : nullptr;
  const int* x = c.draft_tokens + static_cast<size_t>(s) * most;
  const float* u = c.uniforms + static_cast<size_t>(s) * (most + 1);
  const int n = c.draft_counts != nullptr ? min(max(c.draft_counts[s], 0), most) : most;
  if (threadIdx.x == 0) {
    int a = 0;
    for (; a < n; ++a) {
      const int t = x[a];
      if (t < 0 || t >= vocabulary) break;
      const float p = fmaxf(target[a * c.target_row_stride + t], 0.0f);
      const float q = draft != nullptr ? fmaxf(draft[a * c.draft_row_stride + t], 0.0f) : 1.0f;
      if (!(__fmul_rn(fmaxf(u[a], 0.0f), q) < p)) break;
    }
    accepted_s = a;
  }
  __syncthreads();
  const int a = accepted_s;
  Weights w;
  w.p = target + a * c.target_row_stride;
  w.q = a < n && draft != nullptr ? draft + a * c.draft_row_stride : nullptr;
  w.without = a < n && draft == nullptr ? x[a] : -1;
  const int per_warp = (vocabulary + kVerifyThreads / 32 - 1) / (kVerifyThreads / 32);
  const int first = warp * per_warp, last = min(vocabulary, first + per_warp);
  int token = -1;
  for (int attempt = 0; attempt < 2; ++attempt) {
    unsigned long long sum = 0;
    for (int t = first + lane; t < last; t += 32) sum += w.at(t);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long total = 0;
      for (int i = 0; i < kVerifyThreads / 32; ++i) total += warp_sum[i];
      total_s = total;
    }
    __syncthreads();
    const unsigned long long total = total_s;
    if (total != 0) {
      const float uniform = fminf(fmaxf(u[most], 0.0f), 0.99999994f);
      const unsigned long long step = static_cast<unsigned long long>(__fmul_rn(uniform, 16777216.0f));
      const unsigned long long below = (total >> 24) * step + (((total & 0xffffffull) * step) >> 24);
      unsigned long long before = 0;
      for (int i = 0; i < warp; ++i) before += warp_sum[i];
      if (before <= below && below < before + warp_sum[warp]) {       // one warp: its range holds the token
        for (int t0 = first; t0 < last; t0 += 32) {
          const unsigned long long mine = t0 + lane < last ? w.at(t0 + lane) : 0ull;
          unsigned long long run = mine;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const unsigned long long other = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += other;
          }
          const uint32_t over = __ballot_sync(0xffffffffu, before + run > below);
          if (over != 0) {
            if (lane == 0) token_s = t0 + __ffs(static_cast<int>(over)) - 1;
            break;
          }
          before += __shfl_sync(0xffffffffu, run, 31);
        }
      }
      __syncthreads();
      token = token_s;
      break;
    }
    w.q = nullptr;                                                    // nothing left: from the target's row itself
    w.without = -1;
    __syncthreads();
  }
  for (int i = threadIdx.x; i <= most; i += blockDim.x)
    c.tokens[static_cast<size_t>(s) * (most + 1) + i] = i < a ? x[i] : i == a ? token : -1;
  if (threadIdx.x == 0) {
    c.accepted[s] = a;
    if (c.new_lengths != nullptr) c.new_lengths[s] = c.cache_lengths[s] - (n - a);
  }
}

}  // namespace

cudaError_t verify_drafts(const aima_moe_verify_drafts& call, cudaStream_t stream) {
  verify_drafts_kernel<<<call.sequences, kVerifyThreads, 0, stream>>>(call);
  return cudaGetLastError();
}

}  // namespace aima
