// Values in e4m3 with a power of two as scale: what the key/value cache and the
// products with 8-bit weights share.
#pragma once

#include <hip/hip_runtime.h>

#include "device_math.h"

namespace fa {

// Scale exponents. Above: the largest a finite float32 needs. Below: a
// block whose largest magnitude is under 448 * 2^-80 (4e-22) keeps the
// scale 2^-80, so that a scale times a softmax weight stays far from
// float32's subnormals in attention.
constexpr int kMinExp = -80, kMaxExp = 120;

#ifdef __HIPCC__
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// Four neighbouring values as one aligned load brings them.
template <typename T>
struct Four { using type = f32x4; };
template <>
struct Four<uint16_t> { using type = uint2; };
template <typename T>
using Raw4 = typename Four<T>::type;
template <typename T>
__device__ __forceinline__ Raw4<T> raw4(const T* p) { return *reinterpret_cast<const Raw4<T>*>(p); }
__device__ __forceinline__ f32x4 widen(f32x4 x) { return x; }
__device__ __forceinline__ f32x4 widen(uint2 w) {
  return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
               __uint_as_float(w.y & 0xFFFF0000u)};
}

// Four neighbouring values of a row, those past D as zeros. vec: the row
// starts are aligned for one load.
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int d, int D, bool vec) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (vec && d + 4 <= D) {
    r = widen(raw4(p + d));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (d + i < D) r[i] = to_f32(p[d + i]);
  }
  return r;
}

__device__ __forceinline__ void store4(float* p, int d, int D, bool vec, const f32x4& v) {
  if (vec && d + 4 <= D) {
    *reinterpret_cast<f32x4*>(p + d) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (d + i < D) p[d + i] = v[i];
  }
}
__device__ __forceinline__ uint16_t bf16_bits(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);  // to nearest, ties to even
}
__device__ __forceinline__ void store4(uint16_t* p, int d, int D, bool vec, const f32x4& v) {
  uint16_t b[4];
#pragma unroll
  for (int i = 0; i < 4; i++) b[i] = bf16_bits(v[i]);
  if (vec && d + 4 <= D) {
    *reinterpret_cast<uint2*>(p + d) = make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (d + i < D) p[d + i] = b[i];
  }
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ f32x4 unpack4(uint32_t w) {
  auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return f32x4{a[0], a[1], b[0], b[1]};
}

// The smallest e with a <= 448 * 2^e (448 = 1.75 * 2^8), from a's bits.
__device__ __forceinline__ int scale_exp(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 135 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, kMinExp), kMaxExp);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// y's magnitude joins big if it is finite; a y that is not becomes NaN.
__device__ __forceinline__ void join_max(float& y, float& big) {
  const float m = fabsf(y);
  if (m < __builtin_inff()) big = fmaxf(big, m);
  else y = __builtin_nanf("");
}
// With the largest scale, 256 * 2^120 and above would be read back as infinite.
__device__ __forceinline__ float clamp_top(float y) {
  const float top = 240.f * exp2_int(kMaxExp);
  return y > top ? top : y < -top ? -top : y;
}
#endif

}  // namespace fa
