// The 8-bit blocks of blocks8.cu, for every kernel that writes or reads them.
//
// A block of 32 elements x with a = max |x| over its finite elements has the shift k = floor(log2(448 / a)), at most 127 (0 when a is 0),
// so that every |x 2^k| is at most 448 and no finite value saturates; code = e4m3(x 2^k), nearest even; NaN and +-inf become the NaN
// code and leave the rest of their block alone.  The exponent byte is 127 - k, i.e. the fp32 exponent field of 2^-k, and a code stands
// for code * 2^-k.  k is read off the bits of a (448 = 1.75 * 2^8), and the products with 2^k are exact, so the rounding to e4m3 is the
// only one: at most 2^-4 of a value that is above 2^-13 of its block's largest, and 2^-17 of the largest below that.  Where k ends at 127, in
// blocks below 2^-119, a value is off by 2^-4 of itself or by 2^-137, whichever is more.
// The products with 2^k keep subnormal numbers (mul.rn.f32 written out: the library is compiled with flush-to-zero arithmetic).
#pragma once
#include "common.cuh"

namespace blocks8 {

constexpr int kBlock = 32;

__device__ __forceinline__ float mul_keep(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// k of a block from the bits of its largest finite |x|
__device__ __forceinline__ int block_shift(uint32_t amax) {
  if (amax == 0) return 0;
  const int e = (int)(amax >> 23) - 127;
  return min(127, 8 - e - ((amax & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ float inf_to_nan(float v) {
  return (__float_as_uint(v) & 0x7fffffffu) == 0x7f800000u ? __uint_as_float(0x7fffffffu) : v;
}
// 2^-k from the exponent byte; byte 0 is the subnormal 2^-127
__device__ __forceinline__ float block_unit(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }

template <typename T>
__device__ __forceinline__ float largest();
template <>
__device__ __forceinline__ float largest<float>() { return 3.4028234663852886e38f; }
template <>
__device__ __forceinline__ float largest<__half>() { return 65504.0f; }
template <>
__device__ __forceinline__ float largest<__nv_bfloat16>() { return 3.3895313892515355e38f; }
// rounding to a code can carry the largest numbers of T past its range; NaN passes
template <typename T>
__device__ __forceinline__ float in_range(float v) {
  const float m = largest<T>();
  return v > m ? m : (v < -m ? -m : v);
}

// From this exponent byte on a code can stand for more than the largest number of T (448 * 2^(byte - 127) in bf16 and fp32 from 2^120 on, in
// fp16 from 2^8 on).
template <typename T>
__device__ __forceinline__ bool may_overflow(uint32_t byte) { return byte >= (sizeof(T) == 2 && largest<T>() < 65505.0f ? 135u : 247u); }

}    // namespace blocks8
