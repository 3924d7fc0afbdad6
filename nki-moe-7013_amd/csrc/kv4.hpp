// Entries of the 4-bit cache (head_dim 128).
//
// An entry is 128 e2m1 numbers, two a byte with the even element in the low half,
// and a power of two (a byte p for 2^(p - 127)) for every 32 of them: the block
// format that gfx950's conversions take, 68 bytes where bf16 takes 256.  The
// power is the smallest whose seventh multiple is above the block's largest
// magnitude (6 is the largest number, and up to 7 it is the nearest one), so it
// hangs on the largest element alone: its exponent, one more where its mantissa is
// 1.75 or more, less 2.  A block with an infinity or a NaN has the power 255 and
// reads as NaN.
#pragma once

#include "common.hpp"

namespace qmoe {

constexpr int KV4_ROWB = 64;    // bytes of an entry's numbers
constexpr int KV4_BLOCK = 32;   // elements that share a power
constexpr int KV4_NAN = 255;
constexpr int KV4_LOW = 7, KV4_HIGH = 252;  // powers of finite blocks: 6 * 2^125 is finite in bf16, 2^-120 / 2 normal

// The power's exponent that one element asks for (a block takes the largest),
// biased by 127 and not yet clamped.  Adding a quarter to the mantissa carries
// into the exponent from 1.75 on.
constexpr int KV4_NONFINITE = 1 << 16;
__device__ __forceinline__ int kv4_wants(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u >= 0x7f800000u ? KV4_NONFINITE : int((u + (1u << 21)) >> 23) - 2;
}
__device__ __forceinline__ int kv4_wants(double x) {
  const uint64_t u = uint64_t(__double_as_longlong(x)) & 0x7fffffffffffffffull;
  return u >= 0x7ff0000000000000ull ? KV4_NONFINITE : int((u + (1ull << 50)) >> 52) - (1023 - 127) - 2;
}
__device__ __forceinline__ int kv4_power(int wants) {
  return wants == KV4_NONFINITE ? KV4_NAN : min(max(wants, KV4_LOW), KV4_HIGH);
}

__device__ __forceinline__ float kv4_inverse(float, int power) { return __uint_as_float(uint32_t(254 - power) << 23); }
__device__ __forceinline__ double kv4_inverse(double, int power) {
  return __longlong_as_double(int64_t(1023 + 127 - power) << 52);
}

// The nearest e2m1 number of x / 2^(power - 127), ties to the even code, with x's
// sign.  The division is exact, so the result is that of the real number x.
__device__ __forceinline__ uint32_t kv4_sign(float x) { return __float_as_uint(x) >> 28 & 8u; }
__device__ __forceinline__ uint32_t kv4_sign(double x) { return uint32_t(uint64_t(__double_as_longlong(x)) >> 60) & 8u; }
template <class T>
__device__ __forceinline__ uint32_t kv4_code(T x, int power) {
  if (power == KV4_NAN) return 0;
  const T y = fabs(x) * kv4_inverse(x, power);
  const uint32_t n = uint32_t(y > T(0.25)) + uint32_t(y >= T(0.75)) + uint32_t(y > T(1.25)) + uint32_t(y >= T(1.75)) +
                     uint32_t(y > T(2.5)) + uint32_t(y >= T(3.5)) + uint32_t(y > T(5.0));
  return n | kv4_sign(x);
}

// The multiplier of a block's numbers: 2^(power - 127), NaN for 255.
__device__ __forceinline__ float kv4_scale(uint32_t power) {
  return __uint_as_float(power == KV4_NAN ? 0x7fc00000u : power << 23);
}

// Two numbers of a byte times the block's multiplier, in bf16 (exact): byte `B` of w.
template <int B>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}

}  // namespace qmoe
