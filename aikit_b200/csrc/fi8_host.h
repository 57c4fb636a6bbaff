// fi8_host.h -- what the C entry points share on the host: the error message
// of the last failing call, the device guard, growable buffers and the device
// context.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>

#include "../../include/fi8.h"

struct fi8_ctx {
  int device = 0;
  int sm_count = 0;
};

namespace fi8 {

// Sets fi8_last_error's message for this thread and returns code.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

#define FI8_CUDA(call, what)                      \
  do {                                            \
    cudaError_t e_ = (call);                      \
    if (e_ != cudaSuccess) return cuda_fail(e_, what); \
  } while (0)

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    cudaGetDevice(&cur);
    if (prev >= 0 && cur != prev) cudaSetDevice(prev);
  }
};

template <typename T>
int ensure_device(T** p, size_t* cap, size_t need, const char* what) {
  if (*cap >= need && *p) return FI8_OK;
  if (*p) cudaFree(*p);
  *p = nullptr;
  *cap = 0;
  const size_t n = std::max<size_t>(need, 1);
  cudaError_t e = cudaMalloc(reinterpret_cast<void**>(p), n * sizeof(T));
  if (e != cudaSuccess) {
    *p = nullptr;
    return cuda_fail(e, what);
  }
  *cap = n;
  return FI8_OK;
}

template <typename T>
int ensure_host(T** p, size_t* cap, size_t need, const char* what) {
  if (*cap >= need && *p) return FI8_OK;
  if (*p) cudaFreeHost(*p);
  *p = nullptr;
  *cap = 0;
  const size_t n = std::max<size_t>(need, 1);
  cudaError_t e = cudaMallocHost(reinterpret_cast<void**>(p), n * sizeof(T));
  if (e != cudaSuccess) {
    *p = nullptr;
    return cuda_fail(e, what);
  }
  *cap = n;
  return FI8_OK;
}

}  // namespace fi8
