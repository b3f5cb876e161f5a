// Kernels of rows_gemm.h.
#include <mutex>
#include <type_traits>

#include "lds_dma.h"
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
template <int ES, int MODE, int NB, int MB, int W, int CLASS>
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
          const int sb = a.asc[(c * a.P + row[m]) * 4 + kq];
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
  if constexpr (MODE == kRowsGateUp) {
    for (int m = wave; m < MB; m += W) {
      const long long r = t.r0 + m * 16 + lr;
      const f32x4_t g[2] = {sum(0, m), sum(1, m)}, u[2] = {sum(2, m), sum(3, m)};
      const float xs = a.xs[a.order[min(r, t.r1 - 1)] / a.topk];
      rows_gate_up_out<2, 4, 16>(a, r < t.r1, r, t.e, xs, blockIdx.x * 32 + 4 * kq, g, u);
      // the scales behind the last group
      const int grp = blockIdx.x + 1 + kq;
      if (blockIdx.x + 1 == gridDim.x && blockIdx.x % 4 + 1 + kq < 4 && r < t.r1)
        a.asc[((grp >> 2) * a.P + r) * 4 + (grp & 3)] = 127;
    }
  } else {
    for (int i = wave; i < NB * MB; i += W) {
      const int b = i / MB, m = i - b * MB;
      const long long r = t.r0 + m * 16 + lr;
      const f32x4_t v = sum(b, m);
      const int n = (blockIdx.x * NB + b) * 16 + 4 * kq;
      if (r >= t.r1) continue;
      if (MODE == kRowsLinear) {
        float ws[4], bias[4], o[4] = {v[0], v[1], v[2], v[3]};
        rows_linear_cols(a, n, ws, bias);
        const float xs = a.xs ? a.xs[r] : 1.f;
        if (a.N % 4 == 0)
          rows_linear_out<CLASS, 4, true>(a, r, n, xs, ws, bias, o);
        else
          rows_linear_out<CLASS, 4, false>(a, r, n, xs, ws, bias, o);
      } else {
        rows_down_out(a, a.order[r], t.e, n, v);
      }
    }
  }
}

// Many token rows: 32 NA weight rows times 32 NB token rows a workgroup of four waves, both operands
// staged in LDS. Wave (wm, wn) owns 16 NA weight rows and every other 16-row token block: 16 x 16
// blocks acc[NA][NB], so each fragment read from LDS feeds NA or NB matrix instructions (at NA = NB = 8
// the reads of a step take half the time of its products; with 64 x 128 blocks, three quarters).
//
// Staging. A step of K (128 bytes of a row) is loaded memory -> LDS by DMA, eight rows (1 KiB) a load
// of a wave, into rings of SA weight and SB token stages: step d + SA of the weights and d + SB of the
// tokens are requested once step d has been read. Row r's 16-byte unit u is kept at unit u ^ key(r),
// so that the eight lanes that LDS serves at a time read eight different units. Rows past the tile's
// last one and bytes past a row's end lie outside the load's buffer and come as zeros.
//
// Order of the weight rows: row 4 q + i of block b is the wave's output 4 NA q + 4 b + i, so a lane
// ends with 4 NA neighbouring outputs (2 NA gate and 2 NA up ones, half a group of 32) of each token
// and stores them in 16-byte pieces.
//
// A step's products go in four quarters (weight half, token half): (0, 0), (0, 1), (1, 1), (1, 0), each
// reading from LDS, between its matrix instructions, the half that the next one needs; the last two
// read the next step's first halves, the tokens' into the registers that held half 1. One barrier a
// step, after the second quarter: the step has been read by all, and the next one has arrived.
struct Frag {
  u32x4v v[2];
};
template <int ES, bool SC>
__device__ __forceinline__ f32x4_t tile_mma(const Frag& w, const Frag& t, uint32_t sb, f32x4_t c) {
  const uint4 w0 = __builtin_bit_cast(uint4, w.v[0]), w1 = __builtin_bit_cast(uint4, w.v[1]);
  const uint4 t0 = __builtin_bit_cast(uint4, t.v[0]), t1 = __builtin_bit_cast(uint4, t.v[1]);
  return SC ? rows_mma_scaled(w0, w1, t0, t1, (int)sb, c) : rows_mma<ES>(w0, w1, t0, t1, c);
}
__device__ __forceinline__ u32x4v lds_read16(uint32_t addr) {
  u32x4v r;
  asm volatile("ds_read_b128 %0, %1" : "=v"(r) : "v"(addr));
  return r;
}
__device__ __forceinline__ uint32_t lds_read4(uint32_t addr) {
  uint32_t r;
  asm volatile("ds_read_b32 %0, %1" : "=v"(r) : "v"(addr));
  return r;
}
__device__ __forceinline__ void dma4_buffer(__amdgpu_buffer_rsrc_t buf, void* lds, uint32_t voff,
                                            uint32_t soff) {
  typedef __attribute__((address_space(3))) void lds_void;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_void*)lds, 4, voff, soff, 0, 0);
}

template <int MODE, int NA, int NB>
struct TileShape {
  static constexpr int kWRows = 32 * NA, kTRows = 32 * NB;
  static constexpr int kSA = 3, kSB = 2;
  static constexpr bool kScaled = MODE == kRowsDown;
  static constexpr int kAStage = kWRows * 128;
  static constexpr int kBStage = kTRows * 128 + (kScaled ? kTRows * 4 : 0);
  static constexpr int kLds = kSA * kAStage + kSB * kBStage;
  static constexpr int kOut = MODE == kRowsGateUp ? kWRows / 2 : kWRows;  // outputs per workgroup
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

template <int ES, int MODE, int NA, int NB, int CLASS, bool VEC>
__global__ __launch_bounds__(256, 1) void k_rows_tile(RowsGemm a, int ncol, int ntile) {
  using S = TileShape<MODE, NA, NB>;
  constexpr bool SC = S::kScaled;
  constexpr int HA = NA / 2, HB = NB / 2;
  constexpr int LA = S::kWRows / 32, LB = S::kTRows / 32;  // loads of a wave and step
  extern __shared__ uint4 smem[];
  // Workgroup id % 8 is its XCD. Experts: the ncol workgroups of one tile on one XCD, so they share its
  // token rows in that L2. Linear: each XCD walks its own part of the output in columns of four tiles
  // of token rows, whose workgroups share both operands.
  int tile, col;
  {
    const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
    if (MODE == kRowsLinear) {
      const int all = ncol * ntile, per = (all + 7) / 8;
      const int pos = xcd * per + j;
      if (j >= per || pos >= all) return;
      const int g = pos / (4 * ncol), in = pos - g * 4 * ncol;
      const int high = min(4, ntile - 4 * g);
      col = in / high;
      tile = 4 * g + in - col * high;
    } else {
      tile = (j / ncol) * 8 + xcd;
      col = j - (j / ncol) * ncol;
    }
  }
  RowsTile t;
  if (!rows_tile<MODE>(a, tile, S::kTRows, t)) return;
  const int ntok = (int)(t.r1 - t.r0);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int lr = lane & 15, kq = lane >> 4;
  char* lds = reinterpret_cast<char*>(smem);

  // ---- DMA: the wave's load i fills LDS rows (wave + 4 i) 8 .. + 7, lane l unit l & 7 of row l >> 3
  constexpr uint32_t kNowhere = 0x80000000u;  // past the end of any of the buffers
  constexpr int SPAN = MODE == kRowsGateUp ? 2 * NA : 4 * NA;
  const int grow = lane >> 3, row0 = wave * 8 + grow;
  const int n0 = col * S::kOut;
  const uint32_t ldw = (uint32_t)a.ldw, ldx = (uint32_t)a.ldx;
  const int wrows = MODE == kRowsGateUp ? 2 * a.N - n0 : min(S::kWRows, a.N - n0);
  // (a load's uniform offset never passes its buffer's end, its lanes' own offsets may)
  const uint32_t wbytes = (uint32_t)(wrows - 1) * ldw + a.Kb;
  const __amdgpu_buffer_rsrc_t wbuf = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w + t.e * a.estride + (long long)n0 * a.ldw), 0, wbytes, 0x00020000);
  uint32_t wunit[2], woff[2];  // by load parity (the key of row0 + 32)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + 32 * i, key = (r & 3) | (((r / SPAN) & 1) << 2);
    wunit[i] = ((lane & 7) ^ key) * 16;
    woff[i] = row0 * ldw + wunit[i];
  }
  const uint8_t* xbase = MODE == kRowsGateUp ? a.x : a.x + t.r0 * a.ldx;
  const uint32_t xbytes = MODE == kRowsGateUp ? (uint32_t)a.xbytes : (uint32_t)(ntok - 1) * ldx + a.Kb;
  const __amdgpu_buffer_rsrc_t xbuf =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(xbase), 0, xbytes, 0x00020000);
  const uint32_t tunit = ((lane & 7) ^ grow) * 16;
  uint32_t toff[MODE == kRowsGateUp ? LB : 1];
  if (MODE == kRowsGateUp) {
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int r = row0 + 32 * i;
      toff[i] = r < ntok ? (uint32_t)(a.order[t.r0 + r] / a.topk) * ldx + tunit : kNowhere;
    }
  } else {
    toff[0] = row0 * ldx + tunit;
  }
  const __amdgpu_buffer_rsrc_t sbuf = __builtin_amdgcn_make_buffer_rsrc(
      SC ? a.asc + t.r0 * 4 : nullptr, 0,
      SC ? (uint32_t)(((a.Kb + 127) / 128 - 1) * a.P * 4 + ntok * 4) : 0, 0x00020000);
  const int nd = (a.Kb + 127) / 128;
  const bool ragged = a.Kb % 128 != 0;
  auto issue_a = [&](int d) __attribute__((always_inline)) {
    char* st = lds + (d % S::kSA) * S::kAStage;
    const uint32_t k0 = d * 128;
    const bool last = ragged && d == nd - 1;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      uint32_t soff = k0;
      if (MODE == kRowsGateUp)  // LDS rows: per wm 8 NA gate rows, then their up rows
        soff += (uint32_t)(((i / (NA / 4)) & 1) * a.N + (i / (NA / 2)) * 8 * NA +
                           (i % (NA / 4)) * 32) * ldw;
      else
        soff += 32u * i * ldw;
      const bool past = last && k0 + wunit[i & 1] >= (uint32_t)a.Kb;
      const bool in = soff - k0 < wbytes;  // else all of its rows are past the last one
      dma16_buffer(wbuf, st + (wave + 4 * i) * 1024, past || !in ? kNowhere : woff[i & 1], in ? soff : 0);
    }
  };
  auto issue_b = [&](int d) __attribute__((always_inline)) {
    char* st = lds + S::kSA * S::kAStage + (d % S::kSB) * S::kBStage;
    const uint32_t k0 = d * 128;
    const bool past = ragged && d == nd - 1 && k0 + tunit >= (uint32_t)a.Kb;
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const uint32_t v = MODE == kRowsGateUp ? toff[i] : toff[0];
      const bool in = MODE == kRowsGateUp || 32 * i < ntok;
      const uint32_t soff = MODE == kRowsGateUp ? k0 : in ? k0 + 32u * i * ldx : 0;
      dma16_buffer(xbuf, st + (wave + 4 * i) * 1024, past || !in ? kNowhere : v, soff);
    }
    if (SC && wave < S::kTRows / 64)  // a dword of four groups' scales per row
      dma4_buffer(sbuf, st + S::kTRows * 128 + wave * 256,
                  wave * 64 + lane < ntok ? (wave * 64 + lane) * 4 : kNowhere,
                  (uint32_t)(d * a.P * 4));
  };

  // ---- fragment addresses
  const uint32_t lbase = lds_addr(lds);
  uint32_t aaddr, baddr;
  {
    const int r = wm * 16 * NA + (lr >> 2) * SPAN + (lr & 3);  // block b: + 4 b rows
    const int key = (r & 3) | (((r / SPAN) & 1) << 2);
    aaddr = lbase + r * 128 + (kq ^ key) * 16;
    baddr = lbase + S::kSA * S::kAStage + (wn * 16 + lr) * 128 + (kq ^ (lr & 7)) * 16;
  }
  const uint32_t saddr = lbase + S::kSA * S::kAStage + S::kTRows * 128 + (wn * 16 + lr) * 4;
  // weight block b: gate blocks first (kRowsGateUp), then the up blocks 8 NA rows on
  auto read_a = [&](int d, int b, Frag& f) __attribute__((always_inline)) {
    const uint32_t at = aaddr + (d % S::kSA) * S::kAStage +
                        (MODE == kRowsGateUp && b >= HA ? 8 * NA + 4 * (b - HA) : 4 * b) * 128;
    f.v[0] = lds_read16(at);
    f.v[1] = lds_read16(at ^ 64);
  };
  auto read_b = [&](int d, int b, Frag& f, uint32_t& sc) __attribute__((always_inline)) {
    const uint32_t st = (d % S::kSB) * S::kBStage;
    const uint32_t at = baddr + st + b * 32 * 128;
    f.v[0] = lds_read16(at);
    f.v[1] = lds_read16(at ^ 64);
    if (SC) sc = lds_read4(saddr + st + b * 32 * 4);
  };

  f32x4_t acc[NA][NB];
#pragma unroll
  for (int x = 0; x < NA; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int nblk = (ntok + 15) / 16;
  const int nb = __builtin_amdgcn_readfirstlane(min(NB, (nblk - wn + 1) / 2));  // blocks with tokens

  Frag a0[HA], a1[HA], bx[HB], by[HB];
  uint32_t sx[HB] = {}, sy[HB] = {};
  auto ready_a = [&](Frag (&f)[HA]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HA; ++i) after_wait(f[i].v[0]), after_wait(f[i].v[1]);
  };
  auto ready_b = [&](Frag (&f)[HB], uint32_t (&sc)[HB]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      after_wait(f[i].v[0]), after_wait(f[i].v[1]);
      if (SC) {
        asm volatile("" : "+v"(sc[i]));
        sc[i] >>= 8 * kq;
      }
    }
  };
  // One quarter: weight half x, token half y; work(i) is called after token block i's products.
  auto quarter = [&](const Frag (&w)[HA], const Frag (&tk)[HB], const uint32_t (&sc)[HB], auto xh, auto yh,
                     auto work) __attribute__((always_inline)) {
    constexpr int X = decltype(xh)::value, Y = decltype(yh)::value;
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      if (Y * HB + i < nb) {
#pragma unroll
        for (int j = 0; j < HA; ++j)
          acc[X * HA + j][Y * HB + i] =
              tile_mma<ES, SC>(w[j], tk[i], sc[i], acc[X * HA + j][Y * HB + i]);
      }
      __builtin_amdgcn_sched_barrier(0);
      work(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const std::integral_constant<int, 0> c0{};
  const std::integral_constant<int, 1> c1{};
  // Step d with its tokens' half 0 in p; half 1 goes to q, and the next step's half 0 after it.
  auto step = [&](int d, Frag (&p)[HB], uint32_t (&sp)[HB], Frag (&q)[HB], uint32_t (&sq)[HB])
                  __attribute__((always_inline)) {
    quarter(a0, p, sp, c0, c0, [&](int i) __attribute__((always_inline)) { read_b(d, HB + i, q[i], sq[i]); });
    lds_frags_ready();
    ready_b(q, sq);
    quarter(a0, q, sq, c0, c1, [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = i * HA / HB; j < (i + 1) * HA / HB; ++j) read_a(d, HA + j, a1[j]);
    });
    lds_frags_ready();
    ready_a(a1);
    wait_loads(d + 2 < nd ? LA : 0);
    __builtin_amdgcn_s_barrier();
    if (d + 2 < nd) issue_b(d + 2);
    if (d + 3 < nd) issue_a(d + 3);
    quarter(a1, q, sq, c1, c1, [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = i * HA / HB; j < (i + 1) * HA / HB; ++j) read_a(d + 1, j, a0[j]);
    });
    quarter(a1, p, sp, c1, c0, [&](int i) __attribute__((always_inline)) { read_b(d + 1, i, q[i], sq[i]); });
    lds_frags_ready();
    ready_a(a0);
    ready_b(q, sq);
  };
  issue_a(0);
  issue_b(0);
  if (nd > 1) issue_a(1);
  if (nd > 1) issue_b(1);
  if (nd > 2) issue_a(2);
  const int lb = LB + (SC && wave < S::kTRows / 64 ? 1 : 0);
  wait_loads((LA + lb) * (nd > 1) + LA * (nd > 2));
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int j = 0; j < HA; ++j) read_a(0, j, a0[j]);
#pragma unroll
  for (int i = 0; i < HB; ++i) read_b(0, i, bx[i], sx[i]);
  lds_frags_ready();
  ready_a(a0);
  ready_b(bx, sx);
  for (int d = 0; d < nd; d += 2) {
    step(d, bx, sx, by, sy);
    if (d + 1 >= nd) break;
    step(d + 1, by, sy, bx, sx);
  }

  // ---- epilogue
  const int ncols = n0 + wm * (S::kOut / 2) + kq * SPAN;  // the lane's first output
  if constexpr (MODE == kRowsLinear) {
    float xs[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) xs[b] = a.xs ? a.xs[min(t.r0 + (2 * b + wn) * 16 + lr, t.r1 - 1)] : 1.f;
#pragma unroll
    for (int x = 0; x < NA; x += 2) {
      float ws[8], bias[8];
      rows_linear_cols(a, ncols + 4 * x, ws, bias);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const long long r = t.r0 + (2 * b + wn) * 16 + lr;
        __builtin_amdgcn_sched_barrier(0);  // one unit's values live at a time
        if (r >= t.r1) continue;
        const f32x4_t u = acc[x][b], w = acc[x + 1][b];
        float o[8] = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
        rows_linear_out<CLASS, 8, VEC>(a, r, ncols + 4 * x, xs[b], ws, bias, o);
      }
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b >= nb) break;
      const long long r = t.r0 + (2 * b + wn) * 16 + lr;
      const bool live = r < t.r1;
      if constexpr (MODE == kRowsGateUp) {
        f32x4_t g[HA], u[HA];
#pragma unroll
        for (int x = 0; x < HA; ++x) g[x] = acc[x][b], u[x] = acc[HA + x][b];
        const float xs = a.xs[a.order[min(r, t.r1 - 1)] / a.topk];
        rows_gate_up_out<HA, 32 / SPAN, 4>(a, live, r, t.e, xs, ncols, g, u);
      } else if (live) {
        const long long p = a.order[r];
#pragma unroll
        for (int x = 0; x < NA; ++x) rows_down_out(a, p, t.e, ncols + 4 * x, acc[x][b]);
      }
    }
  }
}

template <int ES, int MODE, int MB, int CLASS = 0>
hipError_t launch_few(const RowsGemm& a, hipStream_t s) {
  constexpr int NB = MODE == kRowsGateUp ? 4 : 2, W = 4;
  const long long cols = MODE == kRowsGateUp ? a.N / 32 : (a.N + 16 * NB - 1) / (16 * NB);
  const long long tiles = MODE == kRowsLinear ? (a.M + 16 * MB - 1) / (16 * MB) : a.MT;
  if (tiles <= 0 || cols <= 0) return hipSuccess;
  if (tiles > 65535 || cols > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_rows_few<ES, MODE, NB, MB, W, CLASS>), dim3((unsigned)cols, (unsigned)tiles),
                     dim3(W * 64), 0, s, a);
  return hipGetLastError();
}

// A kernel's dynamic LDS above the default limit, allowed once per device.
template <int ES, int MODE, int NA, int NB, int CLASS, bool VEC>
hipError_t allow_tile_lds() {
  static std::mutex mu;
  static uint64_t done = 0;  // bit d: device d
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (done >> dev & 1) return hipSuccess;
  err = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_rows_tile<ES, MODE, NA, NB, CLASS, VEC>),
                            hipFuncAttributeMaxDynamicSharedMemorySize,
                            TileShape<MODE, NA, NB>::kLds);
  if (err == hipSuccess) done |= uint64_t(1) << dev;
  return err;
}

template <int ES, int MODE, int NA, int NB, int CLASS = 0, bool VEC = true>
hipError_t launch_tile(const RowsGemm& a, hipStream_t s) {
  using S = TileShape<MODE, NA, NB>;
  const long long ncol = (a.N + S::kOut - 1) / S::kOut;
  const long long ntile = MODE == kRowsLinear ? (a.M + S::kTRows - 1) / S::kTRows : a.MT;
  if (ntile <= 0) return hipSuccess;
  const long long grid = MODE == kRowsLinear ? (ncol * ntile + 7) / 8 * 8 : (ntile + 7) / 8 * 8 * ncol;
  if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
  hipError_t err = allow_tile_lds<ES, MODE, NA, NB, CLASS, VEC>();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((k_rows_tile<ES, MODE, NA, NB, CLASS, VEC>), dim3((unsigned)grid), dim3(256), S::kLds, s, a,
                     (int)ncol, (int)ntile);
  return hipGetLastError();
}

// The tile kernel's byte offsets into a tile's rows, an expert's weights, all token rows (gathered) and
// the scales are 32-bit, below its kNowhere.
bool tile_fits(RowsMode mode, const RowsGemm& a) {
  const long long most = 1LL << 31;
  if (256 * a.ldw >= most || 256 * a.ldx >= most) return false;
  if (mode == kRowsGateUp) return 2LL * a.N * a.ldw < most && a.xbytes < most;
  if (mode == kRowsDown) return (a.Kb + 127) / 128 * a.P * 4 < most;
  return true;
}

template <int ES, int CLASS>
hipError_t launch_linear(const RowsGemm& a, int c, bool vec, hipStream_t s) {
  if (c == 256) return launch_tile<ES, kRowsLinear, 8, 8, CLASS, true>(a, s);
  if (c == 128)
    return vec ? launch_tile<ES, kRowsLinear, 4, 4, CLASS, true>(a, s)
               : launch_tile<ES, kRowsLinear, 4, 4, CLASS, false>(a, s);
  if (c == 64)
    return vec ? launch_tile<ES, kRowsLinear, 2, 2, CLASS, true>(a, s)
               : launch_tile<ES, kRowsLinear, 2, 2, CLASS, false>(a, s);
  return c ? launch_few<ES, kRowsLinear, 4, CLASS>(a, s) : launch_few<ES, kRowsLinear, 1, CLASS>(a, s);
}

}  // namespace

int rows_tile_rows(int T, int k, int E) {
  const long long P = (long long)T * k;
  const char* e = getenv("ROWS_TILE");
  if (e) return atoi(e);
  return P > 32LL * E ? 192 : P > 16LL * E ? 64 : 16;
}

hipError_t launch_rows_gemm(RowsMode mode, int es, const RowsGemm& a, int tile_rows,
                            hipStream_t s) {
  if (a.Kb < 16 || a.Kb % 16 || a.N < 1) return hipErrorInvalidValue;
  if (mode == kRowsLinear) {
    const char* e = getenv("ROWS_LIN");
    int c = e ? atoi(e) : a.M <= 16 ? 0 : a.M <= 64 ? 1 : 256;
    if (!e && c == 256) {
      auto n = [&](long long b) { return ((a.M + b - 1) / b) * ((a.N + b - 1) / b); };
      c = n(256) >= 200 ? 256 : n(128) >= 128 ? 128 : 64;
    }
    if (!tile_fits(mode, a) && c > 1) c = 1;
    const bool vec = a.N % 8 == 0;
    if (c == 256 && !vec) c = 128;
    switch (rows_act_class(a.act)) {
#define L(CLASS) \
  case CLASS: return es == 2 ? launch_linear<2, CLASS>(a, c, vec, s) : launch_linear<1, CLASS>(a, c, vec, s);
      L(kClassLinear) L(kClassGate) L(kClassErf)
#undef L
    }
  }
  if (es != 1 || a.N % 32) return hipErrorInvalidValue;
  if (mode == kRowsGateUp) {
    if (tile_rows == 192) return tile_fits(mode, a) ? launch_tile<1, kRowsGateUp, 8, 6>(a, s) : hipErrorInvalidValue;
    return tile_rows == 16 ? launch_few<1, kRowsGateUp, 1>(a, s) : launch_few<1, kRowsGateUp, 4>(a, s);
  }
  if (tile_rows == 192) return tile_fits(mode, a) ? launch_tile<1, kRowsDown, 8, 6>(a, s) : hipErrorInvalidValue;
  return tile_rows == 16 ? launch_few<1, kRowsDown, 1>(a, s) : launch_few<1, kRowsDown, 4>(a, s);
}

}  // namespace moe
