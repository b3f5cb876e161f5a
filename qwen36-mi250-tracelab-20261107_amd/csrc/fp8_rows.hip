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

// Eight values as e4m3 at q, with the scale s and r = 1 / s.
__device__ __forceinline__ void store_chunk8(const float (&v)[8], float s, float r, uint8_t* q) {
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = div_by(v[j], s, r);
  *reinterpret_cast<uint2*>(q) =
      make_uint2(pack_e4m3(o[0], o[1], o[2], o[3]), pack_e4m3(o[4], o[5], o[6], o[7]));
}

// A row of HC chunks of 8 fp32 values per lane (at c * 512 + 8 lane).
template <int HC>
__device__ __forceinline__ float row_amax(const float (&v)[HC][8]) {
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < HC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = amax_with(amax, v[c][j]);
  return wave_max(amax);
}
template <int HC>
__device__ __forceinline__ void store_row8(const float (&v)[HC][8], float s, int n, int lane, uint8_t* q) {
  const float r = 1.0f / s;
#pragma unroll
  for (int c = 0; c < HC; ++c) {
    const int e = c * 512 + lane * 8;
    if (e >= n) break;
    store_chunk8(v[c], s, r, q + e);
  }
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
  const float rs = row_scale(row_amax<HC>(v));
  store_row8<HC>(v, rs, n, lane, q + row * n);
  if (lane == 0) scale[row] = rs;
}

// The 8-bit row of a norm with values that only `rest` takes past fp32 (t * two * (1 + w) is finite), which are
// infinite and so become NaN: from memory again, so that the other rows need no registers for it (with the
// values held across a branch, 175 in place of 155 at H = 4096: 22.0 us for 4096 rows with the add, 19.5 so).
__device__ __forceinline__ void add_rms_far_row(const uint16_t* x, const uint16_t* h, const uint16_t* w,
                                             int H, float two, float rest, int lane, uint8_t* q,
                                             float* scale) {
  auto values = [&](int e, float (&v)[8]) __attribute__((always_inline)) {
    for (int j = 0; j < 8; ++j) {
      float t = bf_bits2f(x[e + j]);
      if (h) t = rbf(t + bf_bits2f(h[e + j]));
      v[j] = t * two * (1.0f + bf_bits2f(w[e + j]));
      if (fabsf(v[j]) * rest > kFloatMax) v[j] = __builtin_nanf("");
    }
  };
  float amax = 0.f, v[8];
#pragma unroll 1
  for (int e = lane * 8; e < H; e += 512) {
    values(e, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = amax_with(amax, v[j]);
  }
  amax = wave_max(amax);
  const float s = row_scale(amax, 0x1p-100f / rest);
#pragma unroll 1
  for (int e = lane * 8; e < H; e += 512) {
    values(e, v);
    store_chunk8(v, s, 1.0f / s, q + e);
  }
  if (lane == 0) *scale = amax > 0.f ? s * rest : s;
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
  const float amax = row_amax<HC>(v);
  if (amax * rest > kFloatMax) {
    add_rms_far_row(x + row * H, h ? h + row * H : nullptr, w, H, two, rest, lane, q + row * H, scale + row);
    return;
  }
  const float rs = row_scale(amax, 0x1p-100f / rest);
  store_row8<HC>(v, rs, H, lane, q + row * H);
  if (lane == 0) scale[row] = amax > 0.f ? rs * rest : rs;
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
