// The order in which both routers (ggo_moe.cu, ggo_router.cu) rank logits.
#pragma once

#include <cstdint>

namespace ggo {

// Monotone float -> uint32 (larger float -> larger key). -0 counts as +0 and NaN as the largest, so
// that equal floats have equal keys; no float has key 0.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// The float of a key (a NaN for that of NaN).
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

}  // namespace ggo
