// What the kernels that read or change rows of logits share.
#pragma once
#include "common.h"

namespace ninfer {

// Ascending with the order of floats, and one value for -0 and +0, as in a comparison of floats.
__device__ __forceinline__ uint32_t ordered_key(float v) {
  uint32_t b = __float_as_uint(v);
  if (b == 0x80000000u) b = 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

}  // namespace ninfer
