// Division by a number that is constant for a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bi {

// Division of numbers below 2^31 by a launch's constant: a high product, an
// addition and a shift.
struct Div {
  uint32_t d, mul, shift;
};
inline Div make_div(int64_t d) {
  uint32_t s = 0;
  while (((int64_t)1 << s) < d) s++;
  return Div{(uint32_t)d, (uint32_t)(((((uint64_t)1 << s) - (uint64_t)d) << 32) / (uint64_t)d + 1), s};
}
__device__ __forceinline__ int32_t operator/(int32_t x, const Div& v) {
  return (int32_t)((__umulhi((uint32_t)x, v.mul) + (uint32_t)x) >> v.shift);
}

}  // namespace bi
