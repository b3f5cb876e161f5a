// e4m3 values with scales made from fp32 ones (gfx950's OCP e4m3fn conversions).
//
// A row of activations has one fp32 scale s = amax / 448, amax over its finite values, and
// the values e4m3(v / s), ties to even. A row of zeros has s = 1; amax counts as 2^-100 at
// least, so that 1 / s is finite. NaN and infinite values become NaN (e4m3fn has no
// infinity) and leave the rest of their row as it is.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_common.h"

namespace moe {

constexpr float kE4m3Max = 448.0f;
constexpr int kMostRows = (1 << 26) - 4;  // a launch has fewer than 2^32 threads, 64 a row

__device__ __forceinline__ float row_scale(float amax, float least = 0x1p-100f) {
  return amax > 0.f ? fmaxf(amax, least) / kE4m3Max : 1.0f;
}
// v, or NaN where v is not finite. A maximum with NaN is the other operand, so such values do not count
// for an amax.
__device__ __forceinline__ float finite_or_nan(float v) { return fmaf(v, 0.f, v); }
__device__ __forceinline__ float amax_with(float amax, float v) {
  return fmaxf(amax, fabsf(finite_or_nan(v)));
}
// v / s, correctly rounded, with r = 1 / s: the quotient's error is put back once, as a
// division does. bf16 values fall on the middle between two e4m3 values often enough for the
// rounding of v * r alone to show (v = 17 m, s = m). A non-finite v comes out as NaN: inf - inf
// in the remainder.
__device__ __forceinline__ float div_by(float v, float s, float r) {
  const float q = v * r;
  return fmaf(fmaf(-q, s, v), r, q);
}
// Four fp32 -> four e4m3 bytes (values within +-448 or NaN).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// q [T, n] and scale [T] of x [T, n] bf16.
hipError_t launch_quantize_rows(const uint16_t* x, int T, int n, uint8_t* q, float* scale,
                                hipStream_t s);
// add_rms.h's total and norm, with the fp32 norm in 8 bits: q [T, H] and scale [T]; norm
// [T, H] bf16 may be null.
hipError_t launch_add_rms_fp8(const uint16_t* x, const uint16_t* h, const uint16_t* w, int T, int H,
                              float eps, uint16_t* total, uint8_t* q, float* scale, uint16_t* norm,
                              hipStream_t s);

}  // namespace moe
