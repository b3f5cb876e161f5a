// Rows in 8 bits: quantize_rows and the residual add + RMSNorm that writes e4m3 rows.
//
// One wave per row, four rows per workgroup, the row held in registers between the reduction
// and the conversion, so that each byte is read and written once. Bound by memory: quantize_rows
// of 5000 x 4096 takes 10.9 us, 5.6 TB/s.
#include "fp8_rows.h"

#include "add_rms.h"

namespace moe {
namespace {

constexpr float kFloatMax = 3.402823466e+38f;

// Stores a row of HC chunks of 8 fp32 values per lane (at c * 512 + 8 lane), of which each stands for
// `times` as much (TIMES: not 1, in [1, 2)), as e4m3 with its scale.
template <int HC, bool TIMES>
__device__ __forceinline__ void store_row8(float (&v)[HC][8], float times, int n, int lane,
                                           uint8_t* q, float* scale) {
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < HC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = amax_with(amax, v[c][j]);
  amax = wave_max(amax);
  if (TIMES && amax * times > kFloatMax) {  // values that are infinite with it
    amax = 0.f;
#pragma unroll
    for (int c = 0; c < HC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (fabsf(v[c][j]) * times > kFloatMax) v[c][j] = __builtin_nanf("");
        amax = amax_with(amax, v[c][j]);
      }
    amax = wave_max(amax);
  }
  const float s = TIMES ? row_scale(amax, 0x1p-100f / times) : row_scale(amax);
  const float r = 1.0f / s;
#pragma unroll
  for (int c = 0; c < HC; ++c) {
    const int e = c * 512 + lane * 8;
    if (e >= n) break;
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = div_by(v[c][j], s, r);
    *reinterpret_cast<uint2*>(q + e) =
        make_uint2(pack_e4m3(o[0], o[1], o[2], o[3]), pack_e4m3(o[4], o[5], o[6], o[7]));
  }
  if (lane == 0) *scale = amax > 0.f ? s * times : s;
}

template <int HC>
__global__ __launch_bounds__(256) void k_quantize_rows(const uint16_t* x, int T, int n, uint8_t* q,
                                                       float* scale) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= T) return;
  uint4 in[HC];
  load_row<HC>(x + row * n, n, lane, in);
  float v[HC][8];
#pragma unroll
  for (int c = 0; c < HC; ++c) {
    const uint32_t* u = &in[c].x;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[c][2 * j] = bf_lo(u[j]), v[c][2 * j + 1] = bf_hi(u[j]);
  }
  store_row8<HC, false>(v, 1.0f, n, lane, q + row * n, scale + row);
}

// total and norm as k_add_rms. The 8-bit rows come from the fp32 norm t r (1 + w), of which only r's
// power of two is multiplied in before the division by the row's scale: t 2^e is exact and its
// product with 1 + w nearly so, while the rest of r, one factor of the whole row, goes into the scale.
// (With all of r the quotient had two more roundings: of 4096 x 2048 values 176 then fell to the other
// side of the middle between two e4m3 values than in 64 bits, 135 so.)
// 4096 x 2048 with the add and the bf16 norm: 12.5 us a call among others, 6.0 TB/s.
template <int HC>
__global__ __launch_bounds__(256) void k_add_rms_fp8(const uint16_t* x, const uint16_t* h,
                                                     const uint16_t* w, int T, int H, float eps,
                                                     uint16_t* total, uint8_t* q, float* scale,
                                                     uint16_t* norm) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= T) return;
  uint4 tot[HC], hv[HC], wv[HC];
  load_row<HC>(x + row * H, H, lane, tot);
  if (h) load_row<HC>(h + row * H, H, lane, hv);
  load_row<HC>(w, H, lane, wv);
  float v[HC][8];
  const float r = add_rms_sum<HC>(h != nullptr, H, eps, tot, hv);
  // r = two * rest, 1 <= rest < 2 (r is 0, infinite or NaN: so is two, but NaN gives infinity, and
  // infinity times the row's NaN is NaN)
  const float two = __uint_as_float(__float_as_uint(r) & 0x7f800000u);
  const float rest = __uint_as_float((__float_as_uint(r) & 0x7fffffu) | 0x3f800000u);
#pragma unroll
  for (int c = 0; c < HC; ++c) {
    const uint32_t* t = &tot[c].x;
    const uint32_t* ww = &wv[c].x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[c][2 * j] = bf_lo(t[j]) * two * (1.0f + bf_lo(ww[j]));
      v[c][2 * j + 1] = bf_hi(t[j]) * two * (1.0f + bf_hi(ww[j]));
    }
  }
  if (h) store_row<HC>(total + row * H, H, lane, tot);
  if (norm) {
#pragma unroll
    for (int c = 0; c < HC; ++c) {
      const uint32_t* t = &tot[c].x;
      uint32_t* o = &wv[c].x;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = pack_bf2_rne(bf_lo(t[j]) * r * (1.0f + bf_lo(o[j])),
                            bf_hi(t[j]) * r * (1.0f + bf_hi(o[j])));
    }
    store_row<HC>(norm + row * H, H, lane, wv);
  }
  store_row8<HC, true>(v, rest, H, lane, q + row * H, scale + row);
}

}  // namespace

hipError_t launch_quantize_rows(const uint16_t* x, int T, int n, uint8_t* q, float* scale,
                                hipStream_t s) {
  if (T <= 0) return hipSuccess;
  if (n <= 0 || n % 8 || n > 512 * kAddRmsMaxChunks || T > kMostRows) return hipErrorInvalidValue;
  const dim3 grid((T + 3) / 4), block(256);
  const int hc = (n + 511) / 512;
#define L(HC)                                                                      \
  if (hc <= HC) {                                                                  \
    hipLaunchKernelGGL((k_quantize_rows<HC>), grid, block, 0, s, x, T, n, q, scale); \
    return hipGetLastError();                                                      \
  }
  L(1) L(2) L(4) L(8) L(16)
#undef L
  return hipErrorInvalidValue;
}

hipError_t launch_add_rms_fp8(const uint16_t* x, const uint16_t* h, const uint16_t* w, int T, int H,
                              float eps, uint16_t* total, uint8_t* q, float* scale, uint16_t* norm,
                              hipStream_t s) {
  if (T <= 0) return hipSuccess;
  if (H <= 0 || H % 8 || H > 512 * kAddRmsMaxChunks || T > kMostRows) return hipErrorInvalidValue;
  const dim3 grid((T + 3) / 4), block(256);
  const int hc = (H + 511) / 512;
#define L(HC)                                                                                \
  if (hc <= HC) {                                                                            \
    hipLaunchKernelGGL((k_add_rms_fp8<HC>), grid, block, 0, s, x, h, w, T, H, eps, total, q, \
                       scale, norm);                                                         \
    return hipGetLastError();                                                                \
  }
  L(1) L(2) L(4) L(8) L(16)
#undef L
  return hipErrorInvalidValue;
}

}  // namespace moe
