// The format of a pool held in 8 bits: codes of e4m3 with a scale of e8m0 for each
// head of every block of tokens.  value = code * 2^(byte - 127); byte 255 is NaN.
#ifndef QUANTIZED_DEVICE_H
#define QUANTIZED_DEVICE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

// The scale of a byte (2^-127 is a subnormal number).
__device__ inline float scale_of(unsigned byte) {
  const unsigned bits = byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23;
  return __builtin_bit_cast(float, bits);
}

// The least byte under which `most` (finite, not negative) is at most 448, e4m3's
// largest: with most = m 2^k, 1 <= m < 2, and 448 = 1.75 * 2^8, k - 8 where m <= 1.75
// and k - 7 elsewhere.  (Byte 0 holds everything below it.)
__device__ inline unsigned byte_for(float most) {
  const unsigned bits = __builtin_bit_cast(unsigned, most);
  const int byte = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<unsigned>(byte < 0 ? 0 : byte);
}

}  // namespace

#endif  // QUANTIZED_DEVICE_H
