// The 8-bit form of activations: a tensor is taken as one run of values in blocks of 32.  The values of a block share a
// power-of-two step 2^e and are stored as whole multiples of it:
//   e = the least integer with rint(amax 2^-e) <= 127, clamped to [-126, 121];   q = clamp(rint(x 2^-e), -127, 127)
// where amax is the largest finite |x| of the block.  A value that is not finite is stored as q = -128 and stands for NaN.
// Scaling by a power of two rounds nothing, so the only rounding is rint, off by at most half a step, amax / 127 at
// most: for a normally distributed block 0.8 % of its root mean square.  And a stored value has at most 7 significant
// bits, so bf16 holds it exactly: reading it back into the tensor cores' type costs no further rounding.
// A block takes 32 + 1 bytes.
#pragma once
#include "kernels/common.cuh"

namespace tipsk {

constexpr int kBlock8 = 32;  // values that share a step

// e of a block from the bits of its amax: amax = 1.M 2^(E - 127) needs E - 133, one more if 1.M 64 rounds to 128
// (1.M >= 127.5 / 64, M >= 0x7f0000).  Zero and subnormal values end in the lower clamp.
__device__ __forceinline__ int StepExponent(uint32_t amax_bits) {
  const int e = static_cast<int>((amax_bits + 0x10000u) >> 23) - 133;
  return e < -126 ? -126 : e > 121 ? 121 : e;
}
__device__ __forceinline__ float PowerOfTwo(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
__device__ __forceinline__ uint32_t FiniteBits(float x) {
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}
// One value as its byte; inv = 2^-e.
__device__ __forceinline__ uint32_t Quantise(float x, float inv) {
  const int q = __float2int_rn(fminf(fmaxf(x * inv, -127.f), 127.f));
  return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? static_cast<uint32_t>(q) & 0xffu : 0x80u;
}
// The same of four finite values that need no clamp, |x| inv <= 127.5: adding 1.5 * 2^23 rounds to a whole number, ties to even,
// whose two's complement stands in the sum's last byte.
__device__ __forceinline__ uint32_t Quantise4(const float* x, float inv) {
  constexpr float kRound = 12582912.f;
  const uint32_t a = __float_as_uint(fmaf(x[0], inv, kRound)), b = __float_as_uint(fmaf(x[1], inv, kRound));
  const uint32_t c = __float_as_uint(fmaf(x[2], inv, kRound)), d = __float_as_uint(fmaf(x[3], inv, kRound));
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace tipsk
