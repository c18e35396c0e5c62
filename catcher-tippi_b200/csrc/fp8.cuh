// e4m3 codes with power-of-two scales: the device helpers shared by the fp8
// linears' kernels.
#pragma once

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

// The same for finite values.
__device__ __forceinline__ uint32_t e4m3x2_finite(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight values as they are in memory, 16 bytes (f32: 32).
template <int T>
struct Raw8 {
  uint4 u[T == kF32 ? 2 : 1];
};

template <int T>
__device__ __forceinline__ Raw8<T> load_raw8(const void* p) {
  Raw8<T> r;
  r.u[0] = reinterpret_cast<const uint4*>(p)[0];
  if constexpr (T == kF32) r.u[1] = reinterpret_cast<const uint4*>(p)[1];
  return r;
}

template <int T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (T == kF32) {
    const uint32_t b[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(b[j]);
  } else {
    const uint32_t b[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (T == kBF16) {
        v[2 * j] = __uint_as_float(b[j] << 16);
        v[2 * j + 1] = __uint_as_float(b[j] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b[j]));
        v[2 * j] = f.x, v[2 * j + 1] = f.y;
      }
    }
  }
}

// The largest magnitude of eight values, infinities and NaN among them, as the
// bits of an f32.  16-bit magnitudes are compared two at a time as integers.
template <int T>
__device__ __forceinline__ uint32_t magnitude8(const Raw8<T>& r) {
  if constexpr (T == kF32) {
    const uint32_t b[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, b[j] & 0x7FFFFFFFu);
    return m;
  } else {
    const uint32_t m = __vmaxu2(__vmaxu2(r.u[0].x & 0x7FFF7FFFu, r.u[0].y & 0x7FFF7FFFu),
                                __vmaxu2(r.u[0].z & 0x7FFF7FFFu, r.u[0].w & 0x7FFF7FFFu));
    const uint32_t top = max(m & 0xFFFFu, m >> 16);
    if constexpr (T == kBF16) return top << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top))));
  }
}

// Eight values of one lane of 16 that hold a block of 128: the block's scale
// exponent and the lane's eight codes.  All lanes of the warp.
template <int T>
__device__ __forceinline__ uint2 quantize8(const Raw8<T>& r, int& exponent) {
  uint32_t top = magnitude8<T>(r);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  float v[8];
  widen8<T>(r, v);
  uint2 out;
  if (__any_sync(0xFFFFFFFFu, top >= 0x7F800000u)) {
    // some value of the warp is not finite: the scale comes from those that are
    top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, finite_magnitude(v[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    exponent = fp8_scale_exponent(top);
    const float inv = pow2f(-exponent);
    out.x = e4m3x2(v[0] * inv, v[1] * inv) | (e4m3x2(v[2] * inv, v[3] * inv) << 16);
    out.y = e4m3x2(v[4] * inv, v[5] * inv) | (e4m3x2(v[6] * inv, v[7] * inv) << 16);
  } else {
    exponent = fp8_scale_exponent(top);
    const float inv = pow2f(-exponent);
    out.x = e4m3x2_finite(v[0] * inv, v[1] * inv) | (e4m3x2_finite(v[2] * inv, v[3] * inv) << 16);
    out.y = e4m3x2_finite(v[4] * inv, v[5] * inv) | (e4m3x2_finite(v[6] * inv, v[7] * inv) << 16);
  }
  return out;
}

// Eight values of a row from element k on, zeros from `cols` on; aligned: the
// row can be read 16 bytes at a time.
template <int T>
__device__ __forceinline__ Raw8<T> load_row8(const void* row, int k, int cols, bool aligned) {
  constexpr int kSize = T == kF32 ? 4 : 2;
  if (aligned && k + 8 <= cols) return load_raw8<T>(reinterpret_cast<const char*>(row) + static_cast<int64_t>(k) * kSize);
  uint32_t b[8] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (k + j >= cols) continue;
    if constexpr (T == kF32) b[j] = reinterpret_cast<const uint32_t*>(row)[k + j];
    else b[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k + j]) << (16 * (j & 1));
  }
  Raw8<T> r;
  r.u[0] = make_uint4(b[0], b[1], b[2], b[3]);
  if constexpr (T == kF32) r.u[1] = make_uint4(b[4], b[5], b[6], b[7]);
  return r;
}

__device__ __forceinline__ float fast_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float fast_reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2E = 1.4426950408889634f;

// 2^(v log2 e) for SiLU, v's sigmoid being that over one more than it.  The
// exponent is cut at 62 above, where the sigmoid is 1 to the last bit; below,
// the power goes to 0 by itself, and with it the factor of v: 0 from -88 on for
// every finite v, NaN for -infinity, as the formula says.
__device__ __forceinline__ float silu_power(float v) { return fast_exp2(fminf(kLog2E * v, 62.0f)); }

// SiLU of two values, v p / (1 + p) with p = 2^(v log2 e): one reciprocal serves
// both, 1 / a = b / (a b), as an epilogue of SiLUs is bound by the
// special-function unit and by its instruction count.  a and b are at most 2^62,
// so a b stays in the range of the reciprocal.  The largest error is that of the
// rounded v log2 e: 2^-17 of the value next to v = -88, a few f32 ulps around 0,
// both far inside T's rounding step.  Powers under 2^-126 are flushed to 0, values
// under 2^-119.
__device__ __forceinline__ void silu2(float& x, float& y) {
  const float p = silu_power(x), q = silu_power(y), a = 1.0f + p, b = 1.0f + q;
  const float r = fast_reciprocal(a * b);
  x *= p * (r * b);
  y *= q * (r * a);
}

// act(v) in f32 for the few-row linear's last pass.
__device__ __forceinline__ float activate(float v, int act) {
  if (act == kActSilu) {
    const float p = silu_power(v);
    return v * (p * fast_reciprocal(1.0f + p));
  }
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

// Takes what pack_t made of lo and hi from them: 0 is left where that is not finite.
template <int DT>
__device__ __forceinline__ void take_rest_t(uint32_t packed, float& lo, float& hi) {
  float a, b;
  if constexpr (DT == kBF16) {
    a = __uint_as_float(packed << 16), b = __uint_as_float(packed & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    a = f.x, b = f.y;
  }
  lo = fabsf(a) < INFINITY ? lo - a : 0.0f;
  hi = fabsf(b) < INFINITY ? hi - b : 0.0f;
}

}  // namespace cq
