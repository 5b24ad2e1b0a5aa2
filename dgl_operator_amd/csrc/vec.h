// Element types and 16-byte vectors shared by the row kernels.
#pragma once

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "common.h"

namespace doa {

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// what the wave's lanes wrote to LDS is there for its other lanes
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// 16 bytes, also at any 2-byte address: gfx950 loads them all the same
using Chunk = uint32_t __attribute__((ext_vector_type(4)));
typedef Chunk LooseChunk __attribute__((aligned(2)));

// a grid has fewer than 2^32 threads
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1024;

inline hipStream_t stream_of_current() {
  return c10::hip::getCurrentHIPStream().stream();
}

// widest vector of at most 16 bytes that divides a row and keeps its
// alignment, in elements
inline int row_vec(const void* p, int64_t row_elems, int64_t stride_elems,
                   int elem) {
  int v = 16 / elem;
  while (v > 1 && (row_elems % v || stride_elems % v ||
                   reinterpret_cast<uintptr_t>(p) % (v * elem)))
    v /= 2;
  return v;
}

}  // namespace doa

// fp32 / bf16 / fp16 with `T` the device type
#define DOA_FLOAT_TYPES(TYPE, NAME, ...)                                     \
  [&] {                                                                      \
    switch (TYPE) {                                                          \
      case at::kFloat: { using T = float; __VA_ARGS__(); break; }            \
      case at::kBFloat16: { using T = __bf16; __VA_ARGS__(); break; }        \
      case at::kHalf: { using T = _Float16; __VA_ARGS__(); break; }          \
      default:                                                               \
        TORCH_CHECK(false, NAME, ": fp32, bf16 or fp16 expected, got ",      \
                    TYPE);                                                   \
    }                                                                        \
  }()
