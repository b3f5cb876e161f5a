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
  long long xbytes;   // of all token rows (kRowsGateUp)
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

// v sigmoid(t), as v / (1 + e) or v e / (1 + e) with e = exp(-|t|) <= 1, from the hardware's exp2 and
// reciprocal. e is squared from exp2(-|t| log2(e) / 2), with that argument's rounding error put back:
// so v e may be tiny where e alone would be lost (the hardware's exp2 has no subnormal results).
__device__ __forceinline__ float rows_gate(float v, float t) {
  constexpr float kHalfL2e = -0.721347520444481703680f;
  const float x = fminf(fabsf(t), 256.f);
  const float p = x * kHalfL2e;
  const float h = __builtin_amdgcn_exp2f(p) *
                  fmaf(fmaf(x, kHalfL2e, -p), 0.693147182464599609375f, 1.0f);
  const float f = t < 0.f ? h : 1.0f;
  return v * f * f * __builtin_amdgcn_rcpf(fmaf(h, h, 1.0f));
}
// The activations, by the code that they share: relu and none; silu and gelu_tanh, v sigmoid(t) with
// t = v or 2 sqrt(2 / pi) (v + 0.044715 v^3); gelu by erfc. (The sums 1 + tanh and 1 + erf would lose
// the digits of a negative v's small results.)
enum RowsActClass { kClassLinear, kClassGate, kClassErf };
__host__ __device__ inline RowsActClass rows_act_class(int act) {
  return act == kActGelu ? kClassErf : act >= kActSilu ? kClassGate : kClassLinear;
}
template <int CLASS>
__device__ __forceinline__ float rows_act(float v, int act) {
  if (CLASS == kClassErf) return 0.5f * v * erfcf(v * -0.70710678118654752f);
  if (CLASS == kClassGate) {
    const float c0 = act == kActSilu ? 1.0f : 1.5957691216057308f;
    const float c1 = act == kActSilu ? 0.0f : 1.5957691216057308f * 0.044715f;
    return rows_gate(v, v * fmaf(c1, v * v, c0));
  }
  return act == kActRelu && v < 0.f ? 0.f : v;  // NaN stays NaN
}

// kRowsLinear: C neighbouring outputs of token row m from n on (as far as N goes), whose sums are v.
// VEC: N is a multiple of C, so a row's C outputs are one aligned access.
template <int CLASS, int C, bool VEC>
__device__ __forceinline__ void rows_linear_out(const RowsGemm& a, long long m, int n, float xs,
                                                const float (&ws)[C], const float (&bias)[C],
                                                float (&v)[C]) {
  static_assert(C == 4 || C == 8, "8 or 16 bytes");
  if (n >= a.N) return;
  const long long at = m * a.N + n;
  uint16_t mv[C], rv[C];
  auto load = [&](const uint16_t* p, uint16_t (&d)[C]) __attribute__((always_inline)) {
    if (VEC) {
      if (C == 8)
        __builtin_memcpy(d, __builtin_assume_aligned(p + at, 16), 16);
      else
        __builtin_memcpy(d, __builtin_assume_aligned(p + at, 8), 8);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) d[i] = n + i < a.N ? p[at + i] : 0;
    }
  };
  if (a.mul) load(a.mul, mv);
  if (a.res) load(a.res, rv);
  if (a.ws) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] *= xs * ws[i];
  }
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += bias[i];
  }
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] = rows_act<CLASS>(v[i], a.act);
  if (a.mul) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] *= bf_bits2f(mv[i]);
  }
  if (a.res) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += bf_bits2f(rv[i]);
  }
  uint32_t o[C / 2];
#pragma unroll
  for (int i = 0; i < C; i += 2) o[i / 2] = pack_bf2_rne(v[i], v[i + 1]);
  if (VEC) {
    if (C == 8)
      st16(a.out + at, make_uint4(o[0], o[1], o[C / 2 - 2], o[C / 2 - 1]));
    else
      *reinterpret_cast<uint2*>(a.out + at) = make_uint2(o[0], o[1]);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < a.N) a.out[at + i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
  }
}
// Their weight scales and biases (zeros past N).
template <int C>
__device__ __forceinline__ void rows_linear_cols(const RowsGemm& a, int n, float (&ws)[C],
                                                 float (&bias)[C]) {
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const bool in = n + i < a.N;
    ws[i] = a.ws && in ? a.ws[n + i] : 0.f;
    bias[i] = !a.bias || !in ? 0.f
              : a.bias_f32   ? static_cast<const float*>(a.bias)[n + i]
                             : bf_bits2f(static_cast<const uint16_t*>(a.bias)[n + i]);
  }
}

// The group format's scale 2^z of a group with that amax: the least with amax <= 448 2^z, so that no
// value saturates.
__device__ __forceinline__ int group_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  return max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
}
// v / 2^z in e4m3; non-finite values become NaN (v * 0 is NaN).
__device__ __forceinline__ uint32_t pack_group4(const float (&v)[4], float m) {
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = fmaf(v[i], 0.f, v[i] * m);
  return pack_e4m3(o[0], o[1], o[2], o[3]);
}

// kRowsGateUp: C quads of four columns each of sorted row r from column n on, of which a group's
// columns lie in LANES lanes 16 apart (1 << s of them): the quads of one lane are stride columns
// apart. Every lane of the wave calls; live: the row is stored. Scales of the groups that fill
// up the last 128 columns are written as 1 (their values are read as zeros).
template <int C, int LANES, int STRIDE>
__device__ __forceinline__ void rows_gate_up_out(const RowsGemm& a, bool live, long long r, int e,
                                                 float xs, int n, const f32x4_t (&g)[C],
                                                 const f32x4_t (&u)[C]) {
  static_assert(C * 4 * LANES == 32, "one group");
  const bool in = n < a.N;  // a multiple of 32: the whole group
  const float* sg = a.ws + (long long)e * 2 * a.N + (in ? n : 0);
  const float* su = sg + a.N;
  float v[C][4], amax = 0.f;
#pragma unroll
  for (int h = 0; h < C; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gv = g[h][i] * (xs * sg[STRIDE * h + i]);
      const float uv = u[h][i] * (xs * su[STRIDE * h + i]);
      v[h][i] = rows_gate(gv, gv) * uv;
      amax = fmaxf(amax, finite_abs(v[h][i]));
    }
#pragma unroll
  for (int x = 16; x < 16 * LANES; x *= 2) amax = fmaxf(amax, __shfl_xor(amax, x));
  const int z = group_exponent(amax);
  const float m = __uint_as_float((uint32_t)(127 - z) << 23);
  if (!live) return;
  uint8_t* sc = a.asc + ((n >> 7) * a.P + r) * 4 + (n >> 5 & 3);
  if (!in) {
    *sc = 127;
    return;
  }
  uint32_t q[C];
#pragma unroll
  for (int h = 0; h < C; ++h) q[h] = pack_group4(v[h], m);
  uint8_t* out = a.aq + r * a.N + n;
  if (C == 4 && STRIDE == 4) {
    st16(out, make_uint4(q[0], q[1], q[2], q[3]));
  } else {
#pragma unroll
    for (int h = 0; h < C; ++h) *reinterpret_cast<uint32_t*>(out + STRIDE * h) = q[h];
  }
  *sc = (uint8_t)(z + 127);  // all lanes of a group the same
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
