// A CUDA runtime for linear_api.cu without a device: device memory is the host's, nothing is launched.  Two devices.
#include "../include/aima_moe.h"

#include <cuda_runtime_api.h>

#include <cstdlib>
#include <cstring>

namespace {
int current = 0, owner = 0, launches = 0;
char message[512];
}  // namespace

#define FAKE extern "C" __attribute__((visibility("default")))

FAKE cudaError_t cudaGetDevice(int* device) { *device = current; return cudaSuccess; }
FAKE cudaError_t cudaSetDevice(int device) { current = device; return cudaSuccess; }
FAKE cudaError_t cudaDeviceGetAttribute(int* value, cudaDeviceAttr attribute, int) { *value = attribute == cudaDevAttrComputeCapabilityMajor ? 10 : 148; return cudaSuccess; }
FAKE cudaError_t cudaMalloc(void** pointer, size_t bytes) { owner = current; *pointer = std::aligned_alloc(256, (bytes + 255) / 256 * 256); return cudaSuccess; }
FAKE cudaError_t cudaFree(void* pointer) { std::free(pointer); return cudaSuccess; }
FAKE cudaError_t cudaMemsetAsync(void* at, int value, size_t bytes, cudaStream_t) { std::memset(at, value, bytes); return cudaSuccess; }
FAKE cudaError_t cudaMemcpyAsync(void* to, const void* from, size_t bytes, cudaMemcpyKind, cudaStream_t) { std::memcpy(to, from, bytes); return cudaSuccess; }
FAKE cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
FAKE cudaError_t cudaGetLastError() { return cudaSuccess; }
FAKE const char* cudaGetErrorString(cudaError_t) { return "fake"; }
FAKE cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* attributes, const void*) { attributes->type = cudaMemoryTypeDevice; attributes->device = owner; return cudaSuccess; }
FAKE void** __cudaRegisterFatBinary(void*) { return nullptr; }
FAKE void __cudaRegisterFatBinaryEnd(void**) {}
FAKE void __cudaUnregisterFatBinary(void**) {}

FAKE void fake_device(int device) { current = device; }
FAKE int fake_current() { return current; }
// How many launches there were: convolution 1, token by token 10, chunks 100, head norm 1000 each.
FAKE int fake_launches() { return launches; }
FAKE const char* fake_message() { return message; }

namespace aima {
struct LinearConv;
struct LinearDelta;
struct HeadNorm;
void set_last_error_message(const char* text) { std::strncpy(message, text, sizeof message - 1); }
cudaError_t linear_conv(const LinearConv&, cudaStream_t) { launches += 1; return cudaSuccess; }
cudaError_t linear_step(const LinearDelta&, int, int, cudaStream_t) { launches += 10; return cudaSuccess; }
cudaError_t linear_chunks(const LinearDelta&, int, void*, int, cudaStream_t) { launches += 100; return cudaSuccess; }
cudaError_t head_norm(const HeadNorm&, cudaStream_t) { launches += 1000; return cudaSuccess; }
size_t linear_chunk_workspace(int, int, int max_tokens, int) { return 16ull * static_cast<size_t>(max_tokens); }
}  // namespace aima
