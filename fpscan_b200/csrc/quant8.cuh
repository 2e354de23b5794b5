// The 8-bit format of activation checkpoints: a block of values shares one
// fp32 step, its largest magnitude over 127, and each value is kept as the
// nearest multiple -127..127 of it (ties to even).
//
// The code is the rounding of x * 127 / most, one product and one quotient,
// each rounded as IEEE 754 says: for fp16 and bf16 the product is exact and
// the quotient can only be a tie where it is one exactly, so the codes are
// those of real arithmetic.  (x times a rounded reciprocal is not: half of
// a block's largest value, common in bf16, is a tie.)  Magnitudes near the
// ends of fp32 are brought to its middle by a power of two first.  A block
// that holds an infinity or a NaN has a step that is not finite and codes of
// 0: all of it reads back as NaN.
#pragma once

#include "common.cuh"

namespace fpscan {

struct Quant8 {
  float step, up, most;  // codes are rint(x * up * 127 / most)
};

// `bits`: the largest magnitude of the block, as the bits of its absolute
// value (compared as integers, a NaN is above everything).
__device__ __forceinline__ Quant8 quant8_block(uint32_t bits) {
  Quant8 q;
  q.most = __uint_as_float(bits);
  q.step = q.most / 127.f;
  q.up = q.most > 0x1p100f ? 0x1p-40f : q.most < 0x1p-80f ? 0x1p40f : 1.f;
  q.most *= q.up;
  return q;
}

__device__ __forceinline__ int quant8_code(const Quant8& q, float x) {
  const float r = __fdiv_rn(x * q.up * 127.f, q.most);
  // 127 may come out an ulp larger; NaN (0 / 0 of a block of zeros, too) and infinity give 0
  return fabsf(r) < 127.5f ? __float2int_rn(r) : 0;
}

__device__ __forceinline__ uint32_t quant8_pack4(int a, int b, int c, int d) {
  return (a & 0xff) | ((b & 0xff) << 8) | ((c & 0xff) << 16) | ((uint32_t)d << 24);
}

// Value of byte j of w.
__device__ __forceinline__ float quant8_value(uint32_t w, int j, float step) {
  return (float)(int)(int8_t)(w >> (8 * j)) * step;
}

}  // namespace fpscan
