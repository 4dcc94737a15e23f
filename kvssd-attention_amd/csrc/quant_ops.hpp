// The quantiser's arithmetic, shared by the record codec and the paged append:
// groupwise scales and code words, bit for bit as quantize_tensor
// (src/kvssd/quant.py:49-65).
#pragma once

#include "common.hpp"

namespace kvssd {

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <>
__device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) {  // bfloat16 bits
  return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
}

// A word of codes, low bits first: clamp(rint(x / s32), -mid, mid - 1) + mid
// with x / s32 rounded as IEEE division does, |x| <= (mid - 1) s32 (1 + 2^-23) or
// x NaN (code 0).  Two roundings around a reciprocal stand in for the division
// (~12 instructions a value):
// * 16-bit values: q = x r, then q + (x - q s32) r, off x / s32 by at most
//   2^-46 relative before its own rounding.  The codes could then differ only
//   where x / s32 lies that close to half an ulp off some k + 0.5; with x and
//   the group's largest value in 16 bits, both quotients in question are at
//   least 2^-38 apart (checked over every such pair in float16 and bfloat16);
// * 32-bit values: q = x r is off by less than 2^-19, so that its nearest
//   integer is right unless q lies within 2^-18 of some k + 0.5; then, and for
//   scales whose reciprocal is subnormal or zero, the division itself.
// Only the division's form needs the clamp, for NaN: a NaN shows in the sums.
template <typename T, int BITS>
__device__ __forceinline__ uint32_t code_word(const float (&x)[32 / BITS], float s32) {
  constexpr int kCodes = 32 / BITS, n = kCodes / 2;
  constexpr float mid = static_cast<float>(1 << (BITS - 1));
  constexpr float radix = static_cast<float>(1 << BITS);
  float half[2];  // 16 bits at a time as an exact float sum
  bool done = false;
  if (s32 < 0x1p120f) {
    const float r0 = __builtin_amdgcn_rcpf(s32);
    const float r = __builtin_fmaf(__builtin_fmaf(-s32, r0, 1.0f), r0, r0);
    float off = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float t = 0.0f;
#pragma unroll
      for (int i = n - 1; i >= 0; --i) {
        const float v = x[k * n + i];
        float q = v * r;
        if constexpr (sizeof(T) == 2) q = __builtin_fmaf(__builtin_fmaf(-q, s32, v), r, q);
        const float c = rintf(q);  // within +-(mid - 1), or NaN, and then so is the sum
        if constexpr (sizeof(T) != 2) off = fmaxf(off, fabsf(q - c));
        t = i == n - 1 ? c : __builtin_fmaf(t, radix, c);
      }
      half[k] = t + static_cast<float>(BITS == 4 ? 0x8888 : 0xAAAA);  // mid for every code
    }
    done = half[0] == half[0] && half[1] == half[1] && (sizeof(T) == 2 || off < 0.5f - 0x1p-18f);
  }
  if (!done) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      half[k] = 0.0f;
#pragma unroll
      for (int i = n - 1; i >= 0; --i)
        half[k] = __builtin_fmaf(half[k], radix, fminf(fmaxf(rintf(x[k * n + i] / s32), -mid), mid - 1.0f) + mid);
    }
  }
  return static_cast<uint32_t>(half[0]) | (static_cast<uint32_t>(half[1]) << 16);
}

// max(amax, 1e-8) / (mid - 1), IEEE: a quotient by 7 lies at least 1/14 ulp from
// the middle of two floats, which two roundings around 1/7 resolve (checked over
// every mantissa); large values, where the remainder may not be finite, divide.
template <int BITS>
__device__ __forceinline__ float group_scale(float amax) {
  const float a = fmaxf(amax, 1e-8f);
  if constexpr (BITS == 2) return a;
  if (!(a < 0x1p120f)) return a / 7.0f;
  const float q = a * (1.0f / 7.0f);
  return __builtin_fmaf(__builtin_fmaf(-7.0f, q, a), 1.0f / 7.0f, q);
}

template <int CTRL>
__device__ __forceinline__ float max_across(float v) {
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)));
}

// largest of v over each run of `lanes` (a power of two) lanes
__device__ __forceinline__ float lanes_max(float v, int lanes) {
  if (lanes > 1) v = max_across<0xB1>(v);    // lane ^ 1
  if (lanes > 2) v = max_across<0x4E>(v);    // lane ^ 2
  if (lanes > 4) v = max_across<0x141>(v);   // the other quad of 8
  if (lanes > 8) v = max_across<0x140>(v);   // the other half of 16
  for (int m = 16; m < lanes; m <<= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

}  // namespace kvssd
