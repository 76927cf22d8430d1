// Device-side helpers shared by the gfx950 kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace affon {

// bf16 -> f32 widening is exact: the bf16 bits are the top half of the f32.
__device__ __forceinline__ float bf16_bits_to_f32(uint32_t h) { return __uint_as_float(h << 16); }

// f32 -> bf16 round to nearest even on the bit pattern; NaN stays a quiet NaN.
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x0040u);
  u += 0x7fffu + ((u >> 16) & 1u);
  return static_cast<uint16_t>(u >> 16);
}

// Element loads for the two floating dtypes the path accepts.
struct F32 {
  using storage = float;
  static constexpr int bytes = 4;
  __device__ __forceinline__ static float load(const uint8_t* base, int64_t index) {
    return reinterpret_cast<const float*>(base)[index];
  }
};
struct BF16 {
  using storage = uint16_t;
  static constexpr int bytes = 2;
  __device__ __forceinline__ static float load(const uint8_t* base, int64_t index) {
    return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(base)[index]);
  }
};

__device__ __forceinline__ unsigned lane_id() { return __lane_id(); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t plus_lanes(uint32_t v) {
  return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true));
}
// The sum over a whole wave's lanes up to each.
__device__ __forceinline__ uint32_t scanned(uint32_t v) {
  v = plus_lanes<0x111, 0xf>(v);  // 1, 2, 4 and 8 lanes before, of 16
  v = plus_lanes<0x112, 0xf>(v);
  v = plus_lanes<0x114, 0xf>(v);
  v = plus_lanes<0x118, 0xf>(v);
  v = plus_lanes<0x142, 0xa>(v);         // the 16 before, in every second 16
  return plus_lanes<0x143, 0xc>(v);      // the 32 before, in the upper 32
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
// v plus another lane's, among 16, for sums over 2, 4, 8 and 16 lanes, in all of them.
enum LaneStep { kNextLane = 0xB1, kNextPair = 0x4E, kOtherFour = 0x141, kOtherEight = 0x140 };
template <LaneStep STEP>
__device__ __forceinline__ float plus_lane(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(v)), STEP, 0xf, 0xf, true));
}
// A whole wave's sum of numbers below 2^56.
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
  const uint32_t low = scanned(static_cast<uint32_t>(v) & 0xffffffu), high = scanned(static_cast<uint32_t>(v >> 24));
  return (static_cast<uint64_t>(lane_of(high, 63)) << 24) + lane_of(low, 63);
}

}  // namespace affon
