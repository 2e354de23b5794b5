// The 8-bit format of activation checkpoints: a block of values shares one
// fp32 step, its largest magnitude over 127, and each value is kept as the
// nearest multiple -127..127 of it (ties to even).
//
// The code is the rounding of the quotient x * 127 / most.  Times a rounded
// reciprocal alone it would not be: half of a block's largest value, common
// in bf16, is a tie, and the product may land on either side of it.
//
// bf16: one multiply-add, x r + 1.5 * 2^23 with r = 127 / most rounded up,
// rounds the product itself to an integer.  It is off by 2^-23 of the quotient
// at most and never towards zero, and a quotient that is no tie is at least
// 2^-19 of itself away from one.  A tie has 254 x = (2 n + 1) most with odd 2 n + 1, so the
// prime 127 divides most's significand (which has 8 bits: then it is a power
// of two times 127, and r is exact) or 2 n + 1 (then 2 n + 1 = 127, the value
// is most / 2, and its tie 63.5 goes to 64, even and away from zero).
// fp16 and fp32: a significand may hold 127 times an odd number, so the
// quotient is corrected once by its residual (Markstein, 1990: with the
// correctly rounded reciprocal y of b and q near a / b, q + (a - q b) y
// rounds to the quotient), three multiply-adds in place of a division.  For
// fp16 x * 127 is exact, and the codes are those of real arithmetic as in
// bf16; for fp32 they are those of fp32 arithmetic.
//
// The kernels read and write about 3 bytes for a value and have some 20
// instructions for it before these bound them.
//
// Magnitudes near the ends of fp32 are brought to its middle by a power of
// two.  The step of the largest fp32 number is rounded towards zero: rounded
// up, 127 times it would be infinite.  A step below 2^-126 is subnormal and off
// by up to 2^-150, so what it stands for is off by up to 127 * 2^-150.  A block that holds an infinity or a NaN has a step that is not finite
// and codes of 0: all of it reads back as NaN.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace fpscan {

struct Quant8 {
  float step;       // most / 127
  float mul;        // the power of two; but for bf16, 127 times that
  float most, inv;  // the largest magnitude times the power of two, its reciprocal (bf16: 127 / most)
  uint32_t keep;    // all ones; 0: every code is 0
};

// Largest magnitudes, as the bits of absolute values compared as integers (so
// a NaN is above everything); 16-bit types two at a time.
template <typename T>
__device__ __forceinline__ uint32_t quant8_max(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) return max(a, b);
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t quant8_max(const uint4& x) {
  constexpr uint32_t m = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  return quant8_max<T>(quant8_max<T>(x.x & m, x.y & m), quant8_max<T>(x.z & m, x.w & m));
}
// The same as the bits of one fp32 magnitude.
template <typename T>
__device__ __forceinline__ uint32_t quant8_bits(uint32_t most) {
  if constexpr (sizeof(T) == 4) return most;
  const uint32_t one = max(most >> 16, most & 0xffffu);
  if constexpr (std::is_same<T, __half>::value)
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)one)));
  return one << 16;
}

// `bits`: the largest magnitude of the block, as the bits of its absolute
// value (compared as integers, a NaN is above everything).
template <typename T>
__device__ __forceinline__ Quant8 quant8_block(uint32_t bits) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  Quant8 q;
  const float most = __uint_as_float(bits);
  q.step = most / 127.f;
  if (sizeof(T) == 4 && bits == 0x7f7fffffu) q.step = __fdiv_rz(most, 127.f);
  q.keep = bits != 0 && bits < 0x7f800000u ? ~0u : 0u;
  const float up = most > 0x1p100f ? 0x1p-60f : most < 0x1p-80f ? 0x1p80f : 1.f;
  q.mul = kBf16 ? up : 127.f * up;
  q.most = q.keep ? most * up : 1.f;
  q.inv = kBf16 ? __fdiv_ru(127.f, q.most) : __frcp_rn(q.most);
  return q;
}

// Codes of four values, one byte each.
template <typename T>
__device__ __forceinline__ uint32_t quant8_codes(const Quant8& q, float a, float b, float c,
                                                 float d) {
  float x[4] = {a, b, c, d};
  uint32_t w[4];
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    if (q.mul != 1.f)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= q.mul;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // adding 1.5 * 2^23 rounds to an integer, ties to even, whose low byte
    // in two's complement is the sum's
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      w[i] = __float_as_uint(fmaf(x[i], q.inv, 12582912.f));
    } else {
      const float t = x[i] * q.mul;
      float r = t * q.inv;
      r = fmaf(fmaf(-r, q.most, t), q.inv, r);
      w[i] = __float_as_uint(r + 12582912.f);
    }
  }
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410) &
         q.keep;
}

// Value of byte j of w.
__device__ __forceinline__ float quant8_value(uint32_t w, int j, float step) {
  return (float)(int)(int8_t)(w >> (8 * j)) * step;
}

}  // namespace fpscan
