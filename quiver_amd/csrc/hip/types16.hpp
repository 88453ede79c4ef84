// Element types of the encoder operators (fp32, fp16, bf16) and their loads and stores by whole vectors.
#pragma once

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

/// The same in global memory, aligned to T alone: the hardware takes vector accesses at any address.
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  typedef T vec __attribute__((ext_vector_type(V)));
  vec v;
};
template <class T>
struct Loose<T, 1> {
  T v[1];
};

/// Threads along an axis that a launch has to stay below.
constexpr uint64_t kGridThreads = uint64_t{1} << 32;

/// From so many bytes on, as much as the L2s hold together, what is read or written once goes past them.
constexpr uint64_t kStreamed = uint64_t{32} << 20;

/// Sixteen bytes aligned to two: a vector of smaller elements would be streamed one by one.
typedef uint32_t dwords_t __attribute__((ext_vector_type(4)));
typedef uint32_t loose_dwords_t __attribute__((ext_vector_type(4), aligned(2)));

/// STREAM: past the caches, where V elements are 16 bytes.
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void load_floats(const T* p, float (&out)[V]) {
  if constexpr (STREAM && V * sizeof(T) == 16) {
    typedef T elements __attribute__((ext_vector_type(V)));
    const dwords_t bits = __builtin_nontemporal_load(reinterpret_cast<const loose_dwords_t*>(p));
    const elements k = __builtin_bit_cast(elements, bits);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = static_cast<float>(k[i]);
  } else {
    const auto k = reinterpret_cast<const Loose<T, V>*>(p)->v;
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = static_cast<float>(k[i]);
  }
}

/// Rounds to nearest even, once.
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void store_floats(T* p, const float (&in)[V]) {
  if constexpr (STREAM && V * sizeof(T) == 16) {
    typedef T elements __attribute__((ext_vector_type(V)));
    elements k;
#pragma unroll
    for (int i = 0; i < V; ++i) k[i] = static_cast<T>(in[i]);
    __builtin_nontemporal_store(__builtin_bit_cast(dwords_t, k), reinterpret_cast<loose_dwords_t*>(p));
  } else {
    Loose<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.v[i] = static_cast<T>(in[i]);
    *reinterpret_cast<Loose<T, V>*>(p) = k;
  }
}

/// The widest access that a row of `n` elements has room for. A row is taken in ceil(n / V) pieces, the last
/// one moved back so that it ends with the row: the elements it shares with the piece before are read twice
/// and written twice with the same values, which costs less than narrow accesses of odd rows.
inline int vector_width(size_t elem, uint64_t n) {
  int v = static_cast<int>(16 / elem);
  while (static_cast<uint64_t>(v) > n) v /= 2;
  return v;
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
