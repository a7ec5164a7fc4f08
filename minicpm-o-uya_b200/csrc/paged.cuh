// paged.cuh -- host-side checks and launch descriptors shared by the paged
// serving operators (paged.cu, paged_attn.cu, sample.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdarg.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

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

// Whether p is memory of the current device (or managed memory).
bool paged_on_device(const void* p, const char* op, char* err, size_t cap);

// The cache's types, sizes and strides, and that no two rows overlap.
bool paged_cache_ok(const minicpmo_paged_cache* c, const char* op, char* err, size_t cap);

}  // namespace mcpo
