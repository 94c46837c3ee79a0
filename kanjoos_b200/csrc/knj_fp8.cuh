// knj_fp8.cuh -- the e4m3 row format: codes with one f32 scale for each group of 128 values of a row.
//   scale = most * f32(1/448), most = the group's largest magnitude;  code = e4m3(v * (1 / scale)), to nearest, ties to even
// in f32, so that any program with IEEE arithmetic forms the same bits. A group whose `most` is below 2^-100 is stored as
// zeros under a zero scale: there the scale or its inverse would leave the normal range. A group that holds a NaN or an
// infinity gets that as its scale, and every product of its row is NaN.
#pragma once

#include "knj_common.cuh"

namespace knj {

constexpr int kFp8Group = 128;

#if defined(__CUDACC__)

// maximum that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// max(a, |b|, |c|) of a >= 0 or NaN, one instruction
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// e4m3 codes of (lo, hi) in the low and high byte; magnitudes above 448 saturate, NaN stays NaN
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
struct Fp8Scale {
  float scale, inverse;
};
__device__ __forceinline__ Fp8Scale fp8_scale(float most) {
  Fp8Scale s;
  s.scale = __fmul_rn(most, 1.0f / 448.0f);
  s.inverse = __frcp_rn(s.scale);
  if (most < 0x1p-100f) s.scale = s.inverse = 0.0f;
  return s;
}

#endif

}  // namespace knj
