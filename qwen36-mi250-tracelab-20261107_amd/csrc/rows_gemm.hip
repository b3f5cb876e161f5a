// Kernels of rows_gemm.h.
#include "rows_gemm.h"

namespace moe {
namespace {

// The tile of weight block column blockIdx.x and tile blockIdx.y.
struct RowsTile {
  int e;
  long long r0, r1;  // token rows (kRowsLinear) or sorted pairs
};
template <int MODE>
__device__ __forceinline__ bool rows_tile(const RowsGemm& a, int tile, int tile_rows, RowsTile& t) {
  if (MODE == kRowsLinear) {
    t.e = 0;
    t.r0 = (long long)tile * tile_rows;
    t.r1 = min(t.r0 + tile_rows, (long long)a.M);
    return t.r0 < a.M;
  }
  if (tile >= a.table[3 * a.MT]) return false;
  t.e = a.table[tile];
  t.r0 = a.table[a.MT + tile];
  t.r1 = min((long long)a.table[2 * a.MT + tile], t.r0 + tile_rows);
  return true;
}

// Few token rows: 16 NB weight rows times 16 MB token rows a workgroup, K split over its W
// waves, operands straight from memory into the matrix instructions; the waves' sums meet in
// LDS in a fixed order. Bound by the stream of weights.
template <int ES, int MODE, int NB, int MB, int W>
__global__ __launch_bounds__(W * 64) void k_rows_few(RowsGemm a) {
  __shared__ f32x4_t red[W][NB * MB][64];
  RowsTile t;
  if (!rows_tile<MODE>(a, blockIdx.y, 16 * MB, t)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, kq = lane >> 4;
  const uint8_t* wp[NB];
  const uint8_t* xp[MB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    long long n;
    if (MODE == kRowsGateUp)  // a group's gate rows, then its up rows
      n = blockIdx.x * 32 + (b & 1) * 16 + lr + (b >> 1) * a.N;
    else
      n = min((int)(blockIdx.x * NB + b) * 16 + lr, a.N - 1);
    wp[b] = a.w + t.e * a.estride + n * a.ldw;
  }
  long long row[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const long long r = min(t.r0 + m * 16 + lr, t.r1 - 1);
    row[m] = MODE == kRowsGateUp ? a.order[r] / a.topk : r;
    xp[m] = a.x + row[m] * a.ldx;
  }
  f32x4_t acc[NB][MB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[b][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int nch = (a.Kb + 127) / 128;
  const int c0 = (int)((long long)nch * wave / W), c1 = (int)((long long)nch * (wave + 1) / W);
  for (int c = c0; c < c1; ++c) {
    // past the row's end: its last 16 bytes again, the token's as zeros
    const int k0 = c * 128 + kq * 16, k1 = k0 + 64;
    const int o0 = min(k0, a.Kb - 16), o1 = min(k1, a.Kb - 16);
    uint4 xv[MB][2];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      xv[m][0] = ld16(xp[m] + o0);
      xv[m][1] = ld16(xp[m] + o1);
      if (k0 >= a.Kb) xv[m][0] = make_uint4(0u, 0u, 0u, 0u);
      if (k1 >= a.Kb) xv[m][1] = make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint4 w0 = ld16_stream(wp[b] + o0), w1 = ld16_stream(wp[b] + o1);
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        if (MODE == kRowsDown) {
          const int sb = c * 128 + kq * 32 < a.Kb ? a.asc[(c * a.P + row[m]) * 4 + kq] : 127;
          acc[b][m] = rows_mma_scaled(w0, w1, xv[m][0], xv[m][1], sb, acc[b][m]);
        } else {
          acc[b][m] = rows_mma<ES>(w0, w1, xv[m][0], xv[m][1], acc[b][m]);
        }
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int m = 0; m < MB; ++m) red[wave][b * MB + m][lane] = acc[b][m];
  __syncthreads();
  auto sum = [&](int b, int m) {
    f32x4_t s = red[0][b * MB + m][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += red[w][b * MB + m][lane];
    return s;
  };
  if (MODE == kRowsGateUp) {
    for (int m = wave; m < MB; m += W) {
      const long long r = t.r0 + m * 16 + lr;
      const f32x4_t g[2] = {sum(0, m), sum(1, m)}, u[2] = {sum(2, m), sum(3, m)};
      const float xs = a.xs[a.order[min(r, t.r1 - 1)] / a.topk];
      rows_gate_up_out(a, r < t.r1, r, t.e, xs, blockIdx.x, kq, g, u);
    }
  } else {
    for (int i = wave; i < NB * MB; i += W) {
      const int b = i / MB, m = i - b * MB;
      const long long r = t.r0 + m * 16 + lr;
      const f32x4_t v = sum(b, m);
      const int n = (blockIdx.x * NB + b) * 16 + 4 * kq;
      if (r >= t.r1) continue;
      if (MODE == kRowsLinear)
        rows_linear_out(a, r, n, v);
      else
        rows_down_out(a, a.order[r], t.e, n, v);
    }
  }
}

template <int ES, int MODE, int MB>
hipError_t launch_few(const RowsGemm& a, hipStream_t s) {
  constexpr int NB = MODE == kRowsGateUp ? 4 : 2, W = 4;
  const long long cols = MODE == kRowsGateUp ? a.N / 32 : (a.N + 16 * NB - 1) / (16 * NB);
  const long long tiles = MODE == kRowsLinear ? (a.M + 16 * MB - 1) / (16 * MB) : a.MT;
  if (tiles <= 0 || cols <= 0) return hipSuccess;
  if (tiles > 65535 || cols > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_rows_few<ES, MODE, NB, MB, W>), dim3((unsigned)cols, (unsigned)tiles),
                     dim3(W * 64), 0, s, a);
  return hipGetLastError();
}

}  // namespace

int rows_tile_rows(int T, int k, int E) { return (long long)T * k > 16LL * E ? 64 : 16; }

hipError_t launch_rows_gemm(RowsMode mode, int es, const RowsGemm& a, int tile_rows,
                            hipStream_t s) {
  if (a.Kb < 16 || a.Kb % 16 || a.N < 1) return hipErrorInvalidValue;
  if (mode == kRowsLinear) {
    if (es == 2) return a.M <= 16 ? launch_few<2, kRowsLinear, 1>(a, s) : launch_few<2, kRowsLinear, 4>(a, s);
    return a.M <= 16 ? launch_few<1, kRowsLinear, 1>(a, s) : launch_few<1, kRowsLinear, 4>(a, s);
  }
  if (es != 1 || a.N % 32) return hipErrorInvalidValue;
  if (mode == kRowsGateUp)
    return tile_rows == 16 ? launch_few<1, kRowsGateUp, 1>(a, s) : launch_few<1, kRowsGateUp, 4>(a, s);
  return tile_rows == 16 ? launch_few<1, kRowsDown, 1>(a, s) : launch_few<1, kRowsDown, 4>(a, s);
}

}  // namespace moe
