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

// the same with no alignment beyond an element's: rows of odd length start
// anywhere, and gfx950 loads 16 bytes from any element's address
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) LooseVec {
  T v[V];
};

// device types of the tensors' types (hardware conversions, unlike c10's)
template <typename T>
struct DeviceT { using type = T; };
template <>
struct DeviceT<c10::Half> { using type = _Float16; };
template <>
struct DeviceT<c10::BFloat16> { using type = __bf16; };

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
