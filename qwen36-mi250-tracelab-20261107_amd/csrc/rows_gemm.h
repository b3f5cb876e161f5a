// Products of token rows with weight rows, out[t, n] = sum_k x[t, k] w[n, k], with bf16 or
// e4m3 operands of one type, and what follows the sum in registers (an epilogue):
//
//   kRowsLinear  out = bf16(residual + mul * act(xs_t ws_n acc + bias_n))
//   kRowsGateUp  one expert's gate and up rows: a = silu(g) u in fp32, written as e4m3 in
//                groups of 32 columns with one power-of-two scale each (the group format that
//                the matrix instructions read, so the down product needs no pass of its own
//                to find a row's amax, which no tile sees whole)
//   kRowsDown    those groups times an expert's down rows: y[pair, n] = ws_n acc, in fp16 with a power
//                of two for every 32 columns
//
// The kernels see rows of bytes. A step of K is 128 bytes of a row: lane (lr, kq) of a wave
// holds the 16 bytes at 16 kq and the 16 at 64 + 16 kq of row lr, and feeds them to one
// v_mfma_f32_16x16x128_f8f6f4 (e4m3) or one v_mfma_f32_16x16x32_bf16 per half (bf16). That is the
// order of k of the first, whose scales, one of lane (lr, kq) for k = 32 kq .. 32 kq + 31, go by it; in
// the unscaled products any order would do that both operands share.
// Sums are fp32, but the e4m3 instruction brings the products of eight neighbouring k to the exponent
// of their largest and cuts, towards zero, what lies below 2^-13 of it (measured: beside 2^16, 12
// counts as 8 and 7 as 0). Only products under 2^-6 of the largest lose anything. That is the
// price of its rate, twice the bf16 instruction's: kRowsLinear's sums are off by some 2e-4 of their size, a
// tenth of the result's rounding; the experts' values between the products are rounded to e4m3 next, where
// as little puts some on the neighbouring value (4096 tokens: outputs off by 2.0e-3 of their size, 1.7e-3
// with every product kept). With few rows every product is kept (rows_mma_wide).
// Weights are the A operand and tokens the B operand: lane (lr, kq) ends with four neighbouring
// outputs n = 4 kq .. 4 kq + 3 of token lr per 16 x 16 block.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fp8_rows.h"
#include "moe_common.h"
#include "route_sort_dev.h"

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
  uint16_t* out;      // also kRowsDown's y [P, N] fp16
  int act, bias_f32;
  // experts: the sorted pairs and their tiles (route_sort.hip)
  const int* table;
  const int* order;
  int MT, topk;
  int tile0;          // the first tile of a launch (few rows)
  long long P;        // pairs
  uint8_t* aq;        // [P, I] e4m3, in sorted order
  uint8_t* asc;       // [ceil(I / 128)][P][4]: biased exponent of each group of 32
  uint8_t* yexp;      // [P, N / 32]: exponent + 128 of 32 values of y
  // a few pairs (kRowsGateUp without a table, launch_rows_pairs_down): pair p is its own sorted row
  const long long* ids;
  int E;              // experts
  const uint16_t* wts;
};

// What a layer adds to the routed sum, rounded as the block's combine rounds it: bf16(sum), then
// bf16(. + bf16(bf16(sigmoid(gate_t)) shared)), then + residual. Null: not there.
struct RowsTail {
  const uint16_t *shared, *gate, *res;  // [T, H], one per token ld_gate apart, [T, H]
  long long ld_gate;
};
__device__ __forceinline__ float rows_tail_gate(const RowsTail& t, long long row) {
  return t.shared ? rbf(sigmoidf_(bf_bits2f(t.gate[row * t.ld_gate]))) : 0.f;
}
__device__ __forceinline__ float rows_tail(const RowsTail& t, float sum, float gate, float shared,
                                           float res) {
  if (t.shared) sum = rbf(rbf(sum) + rbf(gate * shared));
  return t.res ? rbf(sum) + res : sum;
}

// Pair p's expert, ids outside [0, E) as the nearest in it: what the sort makes of them.
__device__ __forceinline__ int rows_pair_expert(const RowsGemm& a, long long p) {
  const long long v = a.ids[p];
  return (int)(v < 0 ? 0 : (v >= a.E ? a.E - 1 : v));
}

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
// The same for e4m3 with every product kept: widened to bf16, which holds e4m3 values exactly, token lr's
// times two0 and two1, the powers of two of their groups of 32 columns. Half the rate, and as many conversions
// as values: for few rows, where memory is the bound (H = 2048, I = 512, 256 experts, us a call with the e4m3
// instruction / so: 8 tokens 40.4, 40.4; 64 141.8, 141.5; 384 201.5, 199.9; linear 16 x 8192 x 8192 16.4,
// 16.5). At 32 tokens the experts' output was off by 1.9e-3 of its size, and is by 1.7e-3, the last rounding
// alone.
__device__ __forceinline__ f32x4_t rows_mma_wide(uint4 a0, uint4 a1, uint4 b0, uint4 b1, float two0,
                                                 float two1, f32x4_t c) {
  uint4 al, ah, bl, bh;
  fp8x16_to_bf16(a0, al, ah);
  fp8x16_to_bf16(b0, bl, bh, two0);
  c = mfma16x16x32(ah, bh, mfma16x16x32(al, bl, c));
  fp8x16_to_bf16(a1, al, ah);
  fp8x16_to_bf16(b1, bl, bh, two1);
  return mfma16x16x32(ah, bh, mfma16x16x32(al, bl, c));
}
// The scales of the four groups of 32 columns of a step of 128 of sorted row r; group g's, 2^(byte - 127).
__device__ __forceinline__ uint32_t rows_group_scales(const RowsGemm& a, int step, long long r) {
  return reinterpret_cast<const uint32_t*>(a.asc)[step * a.P + r];
}
__device__ __forceinline__ float rows_group_two(uint32_t scales, int g) {
  return __uint_as_float((scales >> (8 * g) & 0xffu) << 23);
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
// silu with fewer instructions, v / (1 + exp(-v)): below v = -88 the result is 0 (its size is under
// 10^-36, the least that an 8-bit group's scale can hold beside anything else).
__device__ __forceinline__ float rows_silu(float v) {
  constexpr float kL2e = -1.442695040888963407360f;
  const float x = fminf(v, 200.f);  // v kL2e may overflow, and inf - inf is NaN
  const float p = x * kL2e;
  const float e = __builtin_amdgcn_exp2f(p) * fmaf(fmaf(x, kL2e, -p), 0.693147182464599609375f, 1.0f);
  return v * __builtin_amdgcn_rcpf(1.0f + e);
}
// The activations, by the code that they share: relu and none; silu and gelu_tanh, v sigmoid(t) with
// t = v or 2 sqrt(2 / pi) (v + 0.044715 v^3); gelu by erfc. (The sums 1 + tanh and 1 + erf would lose
// the digits of a negative v's small results.)
template <int C>
__device__ __forceinline__ void rows_act(float (&v)[C], int act) {
  if (act == kActGelu) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = 0.5f * v[i] * erfcf(v[i] * -0.70710678118654752f);
  } else if (act >= kActSilu) {
    const float c0 = act == kActSilu ? 1.0f : 1.5957691216057308f;
    const float c1 = act == kActSilu ? 0.0f : 1.5957691216057308f * 0.044715f;
#pragma unroll
    for (int i = 0; i < C; ++i)  // the square may overflow, and 0 inf is NaN
      v[i] = rows_gate(v[i], v[i] * fmaf(c1, fminf(v[i] * v[i], 1e30f), c0));
  } else if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // NaN stays NaN
  }
}

// kRowsLinear: eight neighbouring outputs of a token row, whose sums times the row's scale are v,
// from their mul and residual (bf16), as bf16.
struct RowsOperands {
  uint4 mul, res;
};
template <bool WITH = true>  // whether there can be mul or residual
__device__ __forceinline__ uint4 rows_linear_value(const RowsGemm& a, const float (&ws)[8],
                                                   const float (&bias)[8], const RowsOperands& op,
                                                   float (&v)[8]) {
  if (a.ws) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= ws[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  rows_act(v, a.act);
  if (WITH && a.mul) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= i & 1 ? bf_hi((&op.mul.x)[i / 2]) : bf_lo((&op.mul.x)[i / 2]);
  }
  if (WITH && a.res) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += i & 1 ? bf_hi((&op.res.x)[i / 2]) : bf_lo((&op.res.x)[i / 2]);
  }
  return make_uint4(pack_bf2_rne(v[0], v[1]), pack_bf2_rne(v[2], v[3]), pack_bf2_rne(v[4], v[5]),
                    pack_bf2_rne(v[6], v[7]));
}
// Eight neighbouring bf16 at any element: one 16-byte access (gfx950 takes it at any address).
__device__ __forceinline__ uint4 rows_load8(const uint16_t* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// The operands and the outputs of the last columns of a row of N not a multiple of 8: `in` of eight.
__device__ __forceinline__ uint4 rows_load_tail(const uint16_t* p, int in) {
  uint32_t d[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < in) d[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
  return make_uint4(d[0], d[1], d[2], d[3]);
}
__device__ __forceinline__ void rows_linear_load(const RowsGemm& a, long long m, int n,
                                                 RowsOperands& o) {
  const long long at = m * a.N + n;
  const int in = a.N - n;
  if (a.mul) o.mul = in >= 8 ? rows_load8(a.mul + at) : rows_load_tail(a.mul + at, in);
  if (a.res) o.res = in >= 8 ? rows_load8(a.res + at) : rows_load_tail(a.res + at, in);
}
// NT: past the caches, for outputs much larger than they are.
template <bool NT>
__device__ __forceinline__ void rows_linear_store(const RowsGemm& a, long long m, int n, uint4 v) {
  typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
  uint16_t* out = a.out + m * a.N + n;
  if (n + 8 <= a.N) {
    const u32x4_any w = {v.x, v.y, v.z, v.w};
    if (NT)
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(out));
    else
      *reinterpret_cast<u32x4_any*>(out) = w;
  } else {
    const uint32_t o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (n + i < a.N) out[i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
  }
}
// Their weight scales and biases (zeros past N). The bias's type is tested at each value, so that a bf16 one
// is eight loads of 2 bytes, one after the other.
__device__ __forceinline__ void rows_linear_cols(const RowsGemm& a, int n, float (&ws)[8],
                                                 float (&bias)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
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
// kRowsGateUp: columns n .. n + 7 of sorted row r, whose sums times the token's scale are g and u and
// whose scales are sg and su; the four lanes of a group of 32 are neighbours. Every lane of the wave
// calls; live: the row is stored. The scales of groups behind the last one, whose values are read as
// zeros, are written as 1.
__device__ __forceinline__ void rows_gate_up_out(const RowsGemm& a, bool live, long long r, int n,
                                                 const float (&sg)[8], const float (&su)[8],
                                                 const float (&g)[8], const float (&u)[8]) {
  float v[8], amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = finite_or_nan(rows_silu(g[i] * sg[i]) * (u[i] * su[i]));
    amax = fmaxf(amax, fabsf(v[i]));
  }
  amax = fmaxf(amax, dppf<kDppXor1>(amax));
  amax = fmaxf(amax, dppf<kDppXor2>(amax));
  const int z = group_exponent(amax);
  const float m = __uint_as_float((uint32_t)(127 - z) << 23);
  if (!live || n >= a.N) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= m;
  *reinterpret_cast<uint2*>(a.aq + r * a.N + n) =
      make_uint2(pack_e4m3(v[0], v[1], v[2], v[3]), pack_e4m3(v[4], v[5], v[6], v[7]));
  uint8_t* sc = a.asc + ((n >> 7) * a.P + r) * 4;
  const int grp = n >> 5;
  sc[grp & 3] = (uint8_t)(z + 127);  // all lanes of a group the same
  if (grp == a.N / 32 - 1)           // the groups that fill up the last 128 columns
    for (int i = (grp & 3) + 1; i < 4; ++i) sc[i] = 127;
}
// The gate and up scales of columns n .. n + 7 of expert e.
__device__ __forceinline__ void rows_gate_up_cols(const RowsGemm& a, int e, int n, float (&sg)[8],
                                                  float (&su)[8]) {
  const float* s = a.ws + (long long)e * 2 * a.N + (n < a.N ? n : 0);  // N is a multiple of 32
#pragma unroll
  for (int i = 0; i < 8; ++i) sg[i] = s[i], su[i] = s[a.N + i];
}

// kRowsDown: outputs n .. n + 7 of pair row p, whose scales are ws, on their way to the weighted sum:
// fp16 values of a power of two 2^ex per 32 columns, ex + 128 in a byte of its own, the largest
// between 2^14 and 2^15. At bf16's size, its error (2^-11 of a value at most) does not show in the sum,
// where bf16's (2^-8) was as large as the result's own rounding. The four lanes of 32 columns are
// neighbours and all called; live: the row is stored.
__device__ __forceinline__ void rows_down_out(const RowsGemm& a, bool live, long long p, int n,
                                              const float (&ws)[8], float (&v)[8]) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] *= ws[i];
    amax = amax_with(amax, v[i]);
  }
  amax = fmaxf(amax, dppf<kDppXor1>(amax));
  amax = fmaxf(amax, dppf<kDppXor2>(amax));
  const int ex = max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -120);
  const float m = __uint_as_float((uint32_t)(127 - ex) << 23);
  if (!live || n >= a.N) return;
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    o[i / 2] = __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)(v[i] * m), (_Float16)(v[i + 1] * m)});
  st16(a.out + p * a.N + n, make_uint4(o[0], o[1], o[2], o[3]));
  a.yexp[p * (a.N / 32) + n / 32] = (uint8_t)(ex + 128);
}

// es: bytes of an element. max_tiles: entries of the tile table at most (experts), built with
// rows_tile_rows rows a tile. hipErrorInvalidValue for shapes outside the contract above.
// rows_tile_rows 0: so few pairs that each is a tile of its own (ids in place of a table).
int rows_tile_rows(int T, int H, int E, int k, int I);
hipError_t launch_rows_gemm(RowsMode mode, int es, const RowsGemm& a, int tile_rows,
                            hipStream_t s);
// kRowsDown and the weighted sum for tile_rows 0: out [T, N] = bf16(sum_j wts_tj ws acc) and the tail.
hipError_t launch_rows_pairs_down(const RowsGemm& a, const RowsTail& tail, int T, hipStream_t s);
// out [T, H] = bf16(sum_j w_tj y_tj) and the tail, for y as kRowsDown writes it.
hipError_t launch_rows_combine(const uint16_t* y, const uint8_t* yexp, const uint16_t* w,
                               const RowsTail& tail, int T, int H, int k, uint16_t* out,
                               hipStream_t s);

}  // namespace moe
