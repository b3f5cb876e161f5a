// Products of token rows with weight rows, out[t, n] = sum_k x[t, k] w[n, k], with bf16 or
// e4m3 operands of one type, and what follows the sum in registers (an epilogue):
//
//   kRowsLinear  out = bf16(residual + mul * act(xs_t ws_n acc + bias_n))
//   kRowsGateUp  one expert's gate and up rows: a = silu(g) u in fp32, written as e4m3 in
//                groups of 32 columns with one power-of-two scale each (the group format that
//                the matrix instructions read, so the down product needs no pass of its own
//                to find a row's amax, which no tile sees whole)
//   kRowsDown    those groups times an expert's down rows: y[pair, n] = bf16(ws_n acc)
//
// The kernels see rows of bytes. A step of K is 128 bytes of a row: lane (lr, kq) of a wave
// holds the 16 bytes at 16 kq and the 16 at 64 + 16 kq of row lr, and feeds them to one
// v_mfma_f32_16x16x128_f8f6f4 (e4m3) or one v_mfma_f32_16x16x32_bf16 per half (bf16). That is the
// order of k of the first, whose scales, one of lane (lr, kq) for k = 32 kq .. 32 kq + 31, go by it; in
// the unscaled products any order would do that both operands share.
// Sums are fp32, but the e4m3 instruction brings the products of eight neighbouring k to the exponent
// of their largest and cuts, towards zero, what lies below 2^-13 of it (measured: beside 2^16, 12
// counts as 8 and 7 as 0). Only products under 2^-6 of the largest lose anything. That is the
// price of its rate, twice the bf16 instruction's.
// Weights are the A operand and tokens the B operand: lane (lr, kq) ends with four neighbouring
// outputs n = 4 kq .. 4 kq + 3 of token lr per 16 x 16 block.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fp8_rows.h"
#include "moe_common.h"

namespace moe {

enum RowsMode { kRowsLinear, kRowsGateUp, kRowsDown };
enum RowsAct { kActNone, kActRelu, kActSilu, kActGelu, kActGeluTanh };

struct RowsGemm {
  const uint8_t* x;   // token rows
  long long ldx;      // bytes from row to row, a multiple of 16
  const uint8_t* w;   // weight rows; an expert's are estride bytes apart
  long long ldw, estride;
  const float* xs;    // a scale per token row, per weight row (e4m3 only)
  const float* ws;
  int M, N;           // token rows (kRowsLinear); outputs of a token (kRowsGateUp: I)
  int Kb;             // bytes of a row, a multiple of 16
  // kRowsLinear
  const void* bias;
  const uint16_t* mul;
  const uint16_t* res;
  uint16_t* out;      // also kRowsDown's y
  int act, bias_f32;
  // experts: the sorted pairs and their tiles (route_sort.hip)
  const int* table;
  const int* order;
  int MT, topk;
  long long P;        // pairs
  uint8_t* aq;        // [P, I] e4m3, in sorted order
  uint8_t* asc;       // [ceil(I / 128)][P][4]: biased exponent of each group of 32
};

typedef int v8i_t __attribute__((ext_vector_type(8)));

// One 128-byte step of K: acc += W (a0 | a1) . X (b0 | b1).
template <int ES>
__device__ __forceinline__ f32x4_t rows_mma(uint4 a0, uint4 a1, uint4 b0, uint4 b1, f32x4_t c) {
  if (ES == 2) return mfma16x16x32(a1, b1, mfma16x16x32(a0, b0, c));
  const v8i_t a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w,
                   (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const v8i_t b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w,
                   (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}
// The same for e4m3 with token lr's values 32 kq .. 32 kq + 31 of the step times 2^(sb - 127).
__device__ __forceinline__ f32x4_t rows_mma_scaled(uint4 a0, uint4 a1, uint4 b0, uint4 b1, int sb,
                                                   f32x4_t c) {
  const v8i_t a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w,
                   (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const v8i_t b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w,
                   (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f, 0, sb);
}

// v sigmoid(t) with exp of a negative argument only: tiny results stay where exp(-t) would
// overflow.
__device__ __forceinline__ float rows_gate(float v, float t) {
  const float e = expf(-fabsf(t));
  return v * ((t < 0.f ? e : 1.0f) / (1.0f + e));
}
// gelu_tanh as v sigmoid(2 u), u = sqrt(2 / pi) (v + 0.044715 v^3), and gelu by erfc: the sums
// 1 + tanh and 1 + erf lose the digits of a negative v's small results.
__device__ __forceinline__ float rows_act(float v, int act) {
  switch (act) {
    case kActRelu:
      return v < 0.f ? 0.f : v;  // NaN stays NaN
    case kActSilu:
      return rows_gate(v, v);
    case kActGelu:
      return 0.5f * v * erfcf(v * -0.70710678118654752f);
    case kActGeluTanh:
      return rows_gate(v, 1.5957691216057308f * fmaf(0.044715f * v * v, v, v));
  }
  return v;
}

// kRowsLinear: outputs n .. n + 3 (as far as N goes) of token row m.
__device__ __forceinline__ void rows_linear_out(const RowsGemm& a, long long m, int n, f32x4_t acc) {
  if (n >= a.N) return;
  const float xs = a.xs ? a.xs[m] : 1.f;
  const long long at = m * a.N + n;
  const bool whole = a.N % 4 == 0;  // then 8-byte accesses are aligned and n + 3 < N
  uint2 mv = make_uint2(0u, 0u), rv = make_uint2(0u, 0u);
  if (whole) {
    if (a.mul) mv = *reinterpret_cast<const uint2*>(a.mul + at);
    if (a.res) rv = *reinterpret_cast<const uint2*>(a.res + at);
  }
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = n + i < a.N;
    float v = acc[i];
    if (a.ws) v *= xs * (in ? a.ws[n + i] : 0.f);
    if (a.bias && in)
      v += a.bias_f32 ? static_cast<const float*>(a.bias)[n + i]
                      : bf_bits2f(static_cast<const uint16_t*>(a.bias)[n + i]);
    v = rows_act(v, a.act);
    const uint32_t mw = i < 2 ? mv.x : mv.y, rw = i < 2 ? rv.x : rv.y;
    if (a.mul) v *= whole ? (i & 1 ? bf_hi(mw) : bf_lo(mw)) : in ? bf_bits2f(a.mul[at + i]) : 0.f;
    if (a.res) v += whole ? (i & 1 ? bf_hi(rw) : bf_lo(rw)) : in ? bf_bits2f(a.res[at + i]) : 0.f;
    o[i] = v;
  }
  const uint2 p = make_uint2(pack_bf2_rne(o[0], o[1]), pack_bf2_rne(o[2], o[3]));
  if (whole) {
    *reinterpret_cast<uint2*>(a.out + at) = p;
  } else {
    const uint32_t u[2] = {p.x, p.y};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) a.out[at + i] = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
  }
}

// kRowsGateUp: group grp (32 columns) of sorted row r, whose values the four lanes of one lr
// hold: g[h], u[h] columns 16 h + 4 kq .. + 3. Every lane of the wave calls; live: the row is
// stored. The scale 2^z is the least power of two with amax <= 448 2^z, so no value saturates;
// a non-finite value becomes NaN (v * 0 is NaN) and does not count for the amax.
__device__ __forceinline__ void rows_gate_up_out(const RowsGemm& a, bool live, long long r, int e,
                                                 float xs, int grp, int kq, const f32x4_t (&g)[2],
                                                 const f32x4_t (&u)[2]) {
  const float* sg = a.ws + (long long)e * 2 * a.N + grp * 32 + 4 * kq;
  const float* su = sg + a.N;
  float v[2][4], amax = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gv = g[h][i] * (xs * sg[16 * h + i]), uv = u[h][i] * (xs * su[16 * h + i]);
      v[h][i] = rows_gate(gv, gv) * uv;
      amax = fmaxf(amax, finite_abs(v[h][i]));
    }
  amax = fmaxf(amax, __shfl_xor(amax, 16));
  amax = fmaxf(amax, __shfl_xor(amax, 32));
  const uint32_t bits = __float_as_uint(amax);
  const int z = max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
  const float m = __uint_as_float((uint32_t)(127 - z) << 23);
  if (!live) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[h][i] = fmaf(v[h][i], 0.f, v[h][i] * m);
    *reinterpret_cast<uint32_t*>(a.aq + r * a.N + grp * 32 + 16 * h + 4 * kq) =
        pack_e4m3(v[h][0], v[h][1], v[h][2], v[h][3]);
  }
  if (kq == 0) a.asc[((grp >> 2) * a.P + r) * 4 + (grp & 3)] = (uint8_t)(z + 127);
}

// kRowsDown: outputs n .. n + 3 of pair row p.
__device__ __forceinline__ void rows_down_out(const RowsGemm& a, long long p, int e, int n,
                                              f32x4_t acc) {
  if (n >= a.N) return;  // N is a multiple of 32
  const float* s = a.ws + (long long)e * a.N + n;
  *reinterpret_cast<uint2*>(a.out + p * a.N + n) = make_uint2(
      pack_bf2_rne(acc[0] * s[0], acc[1] * s[1]), pack_bf2_rne(acc[2] * s[2], acc[3] * s[3]));
}

// es: bytes of an element. max_tiles: entries of the tile table at most (experts), built with
// rows_tile_rows rows a tile. hipErrorInvalidValue for shapes outside the contract above.
int rows_tile_rows(int T, int k, int E);
hipError_t launch_rows_gemm(RowsMode mode, int es, const RowsGemm& a, int tile_rows,
                            hipStream_t s);

}  // namespace moe
