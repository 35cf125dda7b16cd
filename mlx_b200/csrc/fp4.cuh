// Microscaled 4-bit floating point in device code: values to codes and scales, and back (formats: fp4.cu).
#pragma once
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace b200q {
namespace fp4 {

constexpr int kUnit = 16;   // consecutive values of a thread: a whole nvfp4 group, half an mxfp4 one

// Bits of the larger magnitude (fp32 bits with the sign cleared are ordered as the numbers are, infinities and NaNs last).
__device__ __forceinline__ uint32_t larger(uint32_t top, float v) { return max(top, __float_as_uint(v) & 0x7FFFFFFFu); }

// 16 values at `at` (which is 16-byte aligned: ALIGNED; else aligned to its type only), and the largest magnitude's bits.
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint32_t load_unit(const T* at, float (&v)[kUnit]) {
  uint32_t top = 0;
  if constexpr (ALIGNED) {
    uint4 raw[sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[4 * i + j] = __uint_as_float(w[j]);
          top = larger(top, v[4 * i + j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const T* e = reinterpret_cast<const T*>(&w[j]);
          v[8 * i + 2 * j] = Elem<T>::to_float(e[0]);
          v[8 * i + 2 * j + 1] = Elem<T>::to_float(e[1]);
          top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);   // two at a time, in their own bits
        }
      }
    }
    if constexpr (sizeof(T) == 2) {
      const uint32_t most = max(top & 0xFFFFu, top >> 16);
      top = __float_as_uint(Elem<T>::to_float(reinterpret_cast<const T&>(most))) & 0x7FFFFFFFu;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      v[i] = Elem<T>::to_float(at[i]);
      top = larger(top, v[i]);
    }
  }
  return top;
}

// Eight codes, lowest bits first.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// The values of two codes (the low byte's low and high half).
__device__ __forceinline__ float2 e2m1x2_value(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t e4m3(float v) {   // v >= 0; beyond 448: 448
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
  return __low2float(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float e8m0_value(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7FC00000u : (code == 0u ? 0x00400000u : code << 23));
}

// A product's sum is multiplied with the product of the two global scales; where that is no normal fp32 number, with the larger scale and
// then the smaller one, so that only a result passes fp32's range.
__device__ __forceinline__ bool one_factor(float both) { return !(both < 0x1p-126f || both > 0x1.FFFFFEp127f); }
__device__ __forceinline__ float times_scales(float v, float gx, float gw) {
  return one_factor(gx * gw) ? v * (gx * gw) : v * fmaxf(gx, gw) * fminf(gx, gw);
}

// Scale code and codes of a thread's 16 values.  MX: lanes 2i and 2i + 1 share a group; the whole warp calls.
template <bool MX>
__device__ __forceinline__ uint32_t quantize_unit(float (&v)[kUnit], uint32_t top, float G, uint32_t (&codes)[2]) {
  if constexpr (MX) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  const bool odd = top >= 0x7F800000u;
  uint32_t s;
  if constexpr (MX) {
    const int f = (int)(top >> 23) - 2;   // biased exponent; subnormal numbers count as 0
    s = f < 0 ? 0u : (uint32_t)f;
    const float inv = __uint_as_float((254u - min(s, 252u)) << 23);   // 1 / scale, exact
#pragma unroll
    for (int i = 0; i < kUnit; ++i) v[i] *= inv;
    if (odd) s = 255u;
  } else {
    s = e4m3(fminf(__fdiv_rn(__uint_as_float(top), 6.0f * G), 448.0f));
    const float d = e4m3_value(s) * G;
    if (d > 0x1p-100f && d < 0x1p100f && __uint_as_float(top) < 0x1p20f * d) {
      // Quotients rounded as a division rounds them (Markstein, 1990): with r the rounded reciprocal, q - (q d - x) r is the
      // rounded quotient once q is within one unit of it, which the first correction makes it.
      const float r = __frcp_rn(d);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) {
        float q = v[i] * r;                      // (the remainders' signs are such that -0 stays -0)
        q = fmaf(-fmaf(q, d, -v[i]), r, q);
        v[i] = fmaf(-fmaf(q, d, -v[i]), r, q);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kUnit; ++i) {
        const float q = d == 0.0f ? copysignf(0.0f, v[0]) : __fdiv_rn(v[0], d);
#pragma unroll
        for (int j = 0; j + 1 < kUnit; ++j) v[j] = v[j + 1];   // (rolled: this path is rare and long)
        v[kUnit - 1] = q;
      }
    }
    if (odd) s = 0x7Fu;
  }
  codes[0] = odd ? 0u : e2m1x8(v);
  codes[1] = odd ? 0u : e2m1x8(v + 8);
  return s;
}

}  // namespace fp4
}  // namespace b200q
