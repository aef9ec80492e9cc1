// Division of device integers by a number that the host knows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace asc {

// x / d = x * magic >> (31 + shift) for x < 2^31, 2^shift >= d: the magic's error, below d, times x stays
// under 2^(31 + shift).
struct Divisor {
  uint32_t d, magic, shift;
  __device__ __forceinline__ uint32_t divide(uint32_t x) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(x) * magic) >> (31 + shift));
  }
};
inline Divisor divisor_of(uint32_t d) {
  Divisor r{d, 0, 0};
  while ((uint32_t{1} << r.shift) < d) ++r.shift;
  r.magic = static_cast<uint32_t>(((uint64_t{1} << (31 + r.shift)) + d - 1) / d);
  return r;
}

}  // namespace asc
