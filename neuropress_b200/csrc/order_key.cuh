// Total order of logits as unsigned keys, shared by the kernels that select the largest of them.
#pragma once

#include <stdint.h>

namespace npb {

// Order-preserving bits of a float: larger value, larger key; -0 counts as +0, NaN sorts last (1),
// 0 is no element at all.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 1u;
  const uint32_t b = __float_as_uint(f + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k <= 1u) return __int_as_float(0x7fc00000);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

}  // namespace npb
