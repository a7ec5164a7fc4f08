// paged.cuh -- host-side checks and launch descriptors shared by the paged
// serving operators (paged.cu, paged_attn.cu, sample.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdarg.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "common.cuh"
#include "minicpmo_gpu.h"

namespace mcpo {

inline int paged_error(char* err, size_t cap, const char* fmt, ...) {
  if (err && cap) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, cap, fmt, ap);
    va_end(ap);
  }
  return 0;
}

// Bytes of one value of an activation or cache type; 0: not one of them.
inline size_t paged_type_bytes(int dtype) { return dtype == kF32 ? 4 : dtype == kF16 || dtype == kBF16 ? 2 : 0; }

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Work done once for each device, on the first call made with it current (two
// threads may both do it: it has to be harmless twice).
class OncePerDevice {
  std::atomic<uint64_t> done_{0};

 public:
  template <typename F>
  cudaError_t operator()(F&& work) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (done_.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = work();
    if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

// Whether p is memory of the current device (or managed memory).
bool paged_on_device(const void* p, const char* op, char* err, size_t cap);

// The cache's types, sizes and strides, and that no two rows overlap.
bool paged_cache_ok(const minicpmo_paged_cache* c, const char* op, char* err, size_t cap);

}  // namespace mcpo
