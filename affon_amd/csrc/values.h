// Consecutive values of a type, by whole loads and stores.
#pragma once

#include <type_traits>

#include "device.h"

namespace affon {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// V (8, 4 or 1) consecutive values.
template <typename T, int V>
__device__ __forceinline__ void load_values(const uint8_t* base, int64_t at, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = T::load(base, at);
  } else if constexpr (T::bytes == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const u32x4_t raw = reinterpret_cast<const u32x4_t*>(base + at * 4)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = __uint_as_float(raw[e]);
    }
  } else {
    using raw_t = typename std::conditional<V == 8, u32x4_t, u32x2_t>::type;
    const raw_t raw = *reinterpret_cast<const raw_t*>(base + at * 2);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = __uint_as_float(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_values(uint8_t* base, int64_t at, const float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (T::bytes == 4)
      reinterpret_cast<float*>(base)[at] = v[0];
    else
      reinterpret_cast<uint16_t*>(base)[at] = f32_to_bf16_bits(v[0]);
  } else if constexpr (T::bytes == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      u32x4_t raw;
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[e] = __float_as_uint(v[4 * i + e]);
      reinterpret_cast<u32x4_t*>(base + at * 4)[i] = raw;
    }
  } else {
    using raw_t = typename std::conditional<V == 8, u32x4_t, u32x2_t>::type;
    raw_t raw;
#pragma unroll
    for (int e = 0; e < V / 2; ++e)
      raw[e] = f32_to_bf16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16;
    *reinterpret_cast<raw_t*>(base + at * 2) = raw;
  }
}

}  // namespace affon
