// Test kernel for the join of a unit's parts: one block joins its share of parts that the test has laid out, and says how that ended.
// The counter of the parts written is the test's too, so a part that never comes is a number that stays too small.
#include "kv_attention.cuh"

namespace {

constexpr int kThreads = 256;

template <int kDim>
__global__ void __launch_bounds__(kThreads) join_kernel(const aima::KvAttention a, const aima::KvWorkspace work, const aima::KvShared unit,
                                                        unsigned long long limit_ns, int* verdict_out) {
  __shared__ int verdict;
  aima::kv_join<kDim, kThreads>(a, work, unit, limit_ns, &verdict);
  if (threadIdx.x == 0) *verdict_out = verdict;
}

}  // namespace

extern "C" __attribute__((visibility("default"))) int run_join(void* out, int* status, unsigned* arrived, void* weights, float* sums, int dim,
                                                               int group, int rows, int parts, int mine, unsigned long long limit_ns, int* verdict) {
  aima::KvAttention a{};
  a.shape.q_heads = a.shape.group = group;
  a.shape.kv_heads = 1;
  a.shape.head_dim = dim;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.status = status;
  const aima::KvWorkspace work{arrived, static_cast<float4*>(weights), sums, nullptr};
  const aima::KvShared unit{0, parts, mine, rows, 0, 0};
  if (dim == 64) join_kernel<64><<<1, kThreads>>>(a, work, unit, limit_ns, verdict);
  else join_kernel<256><<<1, kThreads>>>(a, work, unit, limit_ns, verdict);
  const cudaError_t launched = cudaGetLastError();
  return static_cast<int>(launched != cudaSuccess ? launched : cudaDeviceSynchronize());
}
