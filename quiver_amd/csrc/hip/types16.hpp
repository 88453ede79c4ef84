// Element types of the encoder operators (fp32, fp16, bf16) and their loads and stores by whole vectors.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "common.hpp"

namespace qvh {

using half_t = _Float16;
using bhalf_t = __bf16;

inline size_t dtype_size(int dtype) { return dtype == QVH_FP32 ? 4 : 2; }

inline void require_dtype(const char* who, int dtype) {
  QVH_REQUIRE(dtype == QVH_FP32 || dtype == QVH_FP16 || dtype == QVH_BF16,
              std::string(who) + ": dtype must be QVH_FP32, QVH_FP16 or QVH_BF16");
}

/// Calls f with a null pointer of the element type that `dtype` names.
template <class F>
void with_dtype(int dtype, F&& f) {
  if (dtype == QVH_FP32) return f(static_cast<float*>(nullptr));
  if (dtype == QVH_FP16) return f(static_cast<half_t*>(nullptr));
  f(static_cast<bhalf_t*>(nullptr));
}

/// V elements of T moved as one access (V * sizeof(T) <= 16, a power of two).
template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <class T, int V>
__device__ __forceinline__ void load_floats(const T* p, float (&out)[V]) {
  const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = static_cast<float>(k.v[i]);
}

/// Rounds to nearest even, once.
template <class T, int V>
__device__ __forceinline__ void store_floats(T* p, const float (&in)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = static_cast<T>(in[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = k;
}

/// The largest power of two of elements, at most 16 bytes, that divides the row length, the row
/// strides and the base addresses.
inline int vector_width(size_t elem, std::initializer_list<uint64_t> lengths, std::initializer_list<const void*> bases) {
  uint64_t bits = 16 / elem;
  for (uint64_t n : lengths) bits |= n;
  for (const void* p : bases) {
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(p) % elem == 0, "a buffer is not aligned to its element type");
    bits |= reinterpret_cast<uintptr_t>(p) / elem;
  }
  return static_cast<int>(bits & (~bits + 1));
}

/// Calls f with std::integral_constant<int, v> for the v in {1, 2, 4, 8} that is given (8 only for 16-bit types).
template <class T, class F>
void with_width(int v, F&& f) {
  if constexpr (sizeof(T) == 2) {
    if (v >= 8) return f(std::integral_constant<int, 8>{});
  }
  if (v >= 4) return f(std::integral_constant<int, 4>{});
  if (v == 2) return f(std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 1>{});
}

}  // namespace qvh
