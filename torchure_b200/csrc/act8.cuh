// The 8-bit format of activation checkpoints: how a block's scale and bytes follow from its largest magnitude (act8.cu has the reasons).
#pragma once

#include "common.cuh"

namespace tb {

struct ActScale {
  float inv;        // what a value is multiplied with: 127 / a, raised by 2^-20; 0 for a block that is kept as zeros
  float scale;      // what a whole number stands for: a / 127
};
__device__ __forceinline__ ActScale act_scale(float a) {
  const bool finite = a <= 3.4028235e38f;
  // 127 / a is no float for the smallest a: such blocks count as zeros, off by less than 2^-120
  const bool some = finite && a >= 7.52316385e-37f;
  // a / 127: the product with the rounded reciprocal, and what it leaves given back (Markstein's correction)
  constexpr float kPart = 1.f / 127.f;
  const float near = a * kPart;
  ActScale k;
  k.scale = finite ? (some ? fmaf(fmaf(-127.f, near, a), kPart, near) : 0.f) : __uint_as_float(0x7fffffffu);
  // (the fast division is good for divisors up to 2^126: both sides a quarter)
  k.inv = some ? __fdividef(31.75f, 0.25f * a) * 1.00000095367431640625f : 0.f;
  return k;
}
// + 1.5 2^23: the whole number, its sign included, in the low byte
__device__ __forceinline__ uint32_t act_word(float x, float inv) { return __float_as_uint(fmaf(x, inv, 12582912.f)); }
__device__ __forceinline__ uint8_t act_byte(float x, float inv) { return static_cast<uint8_t>(act_word(x, inv)); }

}  // namespace tb
