// e4m3 codes with power-of-two scales: the device helpers shared by the fp8
// linears' kernels.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace cq {

// Elements that share one scale, along k and (weights) along n.
constexpr int kFp8Block = 128;

// Bits of |v| as an unsigned integer when v is finite, else 0: the order of
// these integers is that of the magnitudes, so a block's largest finite
// magnitude is an integer maximum.
__device__ __forceinline__ uint32_t finite_magnitude(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

// Exponent e of the block scale 2^e: the least that brings the magnitude
// `amax` (its bits) to 448 = 1.75 * 2^8 or less, at least -126 so that 2^e and
// 2^-e are normal numbers; 0 for an all-zero block.
__device__ __forceinline__ int fp8_scale_exponent(uint32_t amax) {
  if (amax == 0) return 0;
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}

__device__ __forceinline__ float pow2f(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Two values, already divided by their scale, to e4m3 codes (lo in the low
// byte).  The conversion saturates at 448, so infinities are made NaN here.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  const float nan = __uint_as_float(0x7FC00000u);
  lo = fabsf(lo) == __uint_as_float(0x7F800000u) ? nan : lo;
  hi = fabsf(hi) == __uint_as_float(0x7F800000u) ? nan : hi;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float e4m3_to_float(uint8_t code) {
  __nv_fp8_e4m3 v;
  v.__x = code;
  return static_cast<float>(v);
}

// act(v) in f32 for the fp8 and expert linears' epilogues.  SiLU by the fast
// exponential and division: a few f32 ulps, far inside T's rounding step.
__device__ __forceinline__ float activate(float v, int act) {
  if (act == kActSilu) return __fdividef(v, 1.0f + __expf(-v));
  if (act == kActRelu) return v < 0.0f ? 0.0f : v;
  return v;
}

// Two f32 values rounded to T, lo in the low half.
template <int DT>
__device__ __forceinline__ uint32_t pack_t(float lo, float hi) {
  if constexpr (DT == kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

}  // namespace cq
