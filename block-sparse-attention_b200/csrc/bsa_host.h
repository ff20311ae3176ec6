// Host-side helpers shared by the entry points: thread-local error text, TMA tensor-map encoding
// through the driver entry point (no link-time dependency on libcuda), device queries.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace bsa {

// Asks for a kernel's dynamic shared memory once per device (the call costs as much as a launch's other host work).
// One static object per kernel; concurrent first calls set the same value.
struct SmemAttribute {
  std::atomic<bool> done[64] = {};
  cudaError_t set(const void* kernel, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < 64;
    if (known && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && known) done[dev].store(true, std::memory_order_relaxed);
    return e;
  }
};

// Stores a printf-style message for bsa_last_error() and returns `code`.
int set_error(int code, const char* fmt, ...);

// Encodes a tiled tensor map with 128-byte swizzle and zero fill for out-of-range elements.
//   dims[rank]            extents, innermost first
//   strides_bytes[rank-1] byte strides of dimensions 1..rank-1 (multiples of 16)
//   box[rank]             box extents; box[0] * element size must be 128 bytes
// Returns 0 or a negative bsa_error (message set).
int make_tensor_map(CUtensorMap* map, CUtensorMapDataType dtype, int rank, const void* base,
                    const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                    const char* what);

}  // namespace bsa
