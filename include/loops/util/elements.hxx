/**
 * @file elements.hxx
 * @brief Elements of 16 and 32 bits (float, _Float16, __bf16) moved as packets of V consecutive values, in accesses of up to 16
 * bytes at ANY element alignment (gfx950 takes 16-byte accesses at addresses that are only aligned to the element), and converted
 * to float for the arithmetic between.  A store rounds each value once, to nearest even.
 */
#pragma once

#include <hip/hip_runtime.h>

namespace loops {
namespace elements {

/// Values in one 16-byte access.
template <typename T>
constexpr int per_access = 16 / static_cast<int>(sizeof(T));

namespace detail {
template <typename T, int V>
struct packet {
  typedef T type __attribute__((ext_vector_type(V)));
  typedef type unaligned __attribute__((aligned(sizeof(T))));
};
}  // namespace detail

/// V values as they lie in memory; element k is `p[k]`.
template <typename T, int V>
using packet_t = typename detail::packet<T, V>::type;

/// STREAM: the lines are not expected to be read again soon.
template <int V, bool STREAM = false, typename T>
__device__ __forceinline__ packet_t<T, V> load(const T* __restrict__ p) {
  const auto* at = reinterpret_cast<const typename detail::packet<T, V>::unaligned*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(at);
  else return *at;
}

/// V floats to p, each rounded to T.
template <int V, bool STREAM = false, typename T>
__device__ __forceinline__ void store(T* __restrict__ p, const float (&in)[V]) {
  packet_t<T, V> v;
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = static_cast<T>(in[k]);
  auto* at = reinterpret_cast<typename detail::packet<T, V>::unaligned*>(p);
  if constexpr (STREAM) __builtin_nontemporal_store(v, at);
  else *at = v;
}

}  // namespace elements
}  // namespace loops
