// What the C ABI files check and report on the host.
#pragma once

#include "../../include/aima_moe.h"

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

namespace aima {

void set_last_error_message(const char* message);

inline int fail(int status, const char* format, ...) {
  char text[256];
  va_list args;
  va_start(args, format);
  std::vsnprintf(text, sizeof text, format, args);
  va_end(args);
  set_last_error_message(text);
  return status;
}

inline int fail_cuda(cudaError_t error, const char* what) {
  char text[256];
  std::snprintf(text, sizeof text, "%s: %s", what, cudaGetErrorString(error));
  set_last_error_message(text);
  (void)cudaGetLastError();
  return static_cast<int>(error);
}

inline bool misaligned(const void* pointer) { return reinterpret_cast<uintptr_t>(pointer) % 16 != 0; }

// A device that is the current one for the span of a call: the default stream belongs to whichever that is.
struct OnDevice {
  int before = -1;
  cudaError_t error;
  explicit OnDevice(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before == device) before = -1;
    else if (error == cudaSuccess) error = cudaSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0) (void)cudaSetDevice(before);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
};

}  // namespace aima
