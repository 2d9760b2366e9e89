// A CUDA runtime for kv_api.cu without a device: device memory is the host's, nothing is launched.  Two devices, each with a default
// stream of its own; a test can leave a write under way on a stream, which lands when that stream is next used or waited for.
#include "../include/aima_moe.h"

#include <cuda_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <new>
#include <vector>

namespace {

struct Pending {
  int device;
  cudaStream_t stream;
  int* at;
  int value;
};
std::vector<Pending> pending;
int current = 0, owner = 0, appends = 0;
unsigned long long cleared = 0;
char message[512];

void land(cudaStream_t stream) {
  for (size_t i = 0; i < pending.size();) {
    if (pending[i].stream == stream && (stream != nullptr || pending[i].device == current)) {
      *pending[i].at = pending[i].value;
      pending.erase(pending.begin() + static_cast<long>(i));
    } else {
      ++i;
    }
  }
}

}  // namespace

#define FAKE extern "C" __attribute__((visibility("default")))

FAKE cudaError_t cudaGetDevice(int* device) { *device = current; return cudaSuccess; }
FAKE cudaError_t cudaSetDevice(int device) { current = device; return cudaSuccess; }
FAKE cudaError_t cudaDeviceGetAttribute(int* value, cudaDeviceAttr attribute, int) { *value = attribute == cudaDevAttrComputeCapabilityMajor ? 10 : 148; return cudaSuccess; }
FAKE cudaError_t cudaMalloc(void** pointer, size_t bytes) { owner = current; *pointer = std::aligned_alloc(256, (bytes + 255) / 256 * 256); return cudaSuccess; }
FAKE cudaError_t cudaFree(void* pointer) { std::free(pointer); return cudaSuccess; }
FAKE cudaError_t cudaMemsetAsync(void* at, int value, size_t bytes, cudaStream_t stream) { land(stream); std::memset(at, value, bytes); cleared = bytes; return cudaSuccess; }
FAKE cudaError_t cudaMemcpyAsync(void* to, const void* from, size_t bytes, cudaMemcpyKind, cudaStream_t stream) { land(stream); std::memcpy(to, from, bytes); return cudaSuccess; }
FAKE cudaError_t cudaStreamSynchronize(cudaStream_t stream) { land(stream); return cudaSuccess; }
FAKE cudaError_t cudaDeviceSynchronize() { land(nullptr); return cudaSuccess; }
FAKE cudaError_t cudaGetLastError() { return cudaSuccess; }
FAKE const char* cudaGetErrorString(cudaError_t) { return "fake"; }
FAKE cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* attributes, const void*) { attributes->type = cudaMemoryTypeDevice; attributes->device = owner; return cudaSuccess; }
FAKE void** __cudaRegisterFatBinary(void*) { return nullptr; }
FAKE void __cudaRegisterFatBinaryEnd(void**) {}
FAKE void __cudaUnregisterFatBinary(void**) {}

FAKE void fake_device(int device) { current = device; }
FAKE int fake_current() { return current; }
FAKE void fake_leave(int device, void* stream, int* at, int value) { pending.push_back({device, static_cast<cudaStream_t>(stream), at, value}); }
FAKE int fake_appends() { return appends; }
FAKE unsigned long long fake_cleared() { return cleared; }
FAKE const char* fake_message() { return message; }

namespace aima {
struct KvAppend;
struct KvAttention;
struct KvLayer;
struct KvMaps;
struct KvShape;
void set_last_error_message(const char* text) { std::strncpy(message, text, sizeof message - 1); }
cudaError_t kv_append(const KvAppend&, cudaStream_t) { ++appends; return cudaSuccess; }
cudaError_t kv_attention(const KvAttention&, const KvMaps&, void*, int, cudaStream_t) { return cudaSuccess; }
bool kv_make_maps(const KvShape&, const KvLayer&, KvMaps*) { return true; }
cudaError_t verify_drafts(const aima_moe_verify_drafts&, cudaStream_t) { return cudaSuccess; }
size_t kv_counter_bytes() { return 2048; }
size_t kv_workspace_bytes(const KvShape&) { return 4096; }
}  // namespace aima
