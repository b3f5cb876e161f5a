// Kernels of rows_gemm.h.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "lds_dma.h"
#include "rows_gemm.h"

namespace moe {
namespace {

// A tile's expert and rows.
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
  if (MODE == kRowsGateUp && a.ids) {
    t.e = rows_pair_expert(a, tile);
    t.r0 = tile;
    t.r1 = tile + 1;
    return true;
  }
  if (tile >= a.table[3 * a.MT]) return false;
  t.e = a.table[tile];
  t.r0 = a.table[a.MT + tile];
  t.r1 = min((long long)a.table[2 * a.MT + tile], t.r0 + tile_rows);
  return true;
}

// Few token rows: 16 NB weight rows times 16 MB token rows a workgroup, K split over its W
// waves, operands straight from memory into the matrix instructions, the loads of U steps (2 NB U KiB
// of weights a wave) together; the waves' sums meet in LDS in a fixed order. Bound by the stream of
// weights (32 tokens of 256 experts, H = 2048, I = 512: gate_up 5.0 TB/s, down 4.9), for one token
// by its latency (2048 x 2048 bf16 5.4 us).
template <int ES, int MODE, int NB, int MB, int W, int U>
__global__ __launch_bounds__(W * 64) void k_rows_few(RowsGemm a) {
  // linear of 17 to 32 e4m3 rows has products enough to notice (17 x 4096 x 16384: 16.9 us, wide 18.7)
  constexpr bool WIDE = ES == 1 && !(MODE == kRowsLinear && MB > 1);
  __shared__ f32x4_t red[W][NB * MB][64];
  RowsTile t;
  if (!rows_tile<MODE>(a, a.tile0 + blockIdx.y, 16 * MB, t)) return;
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
  auto token = [&](long long r) __attribute__((always_inline)) {
    return MODE != kRowsGateUp ? r : (a.ids ? r : (long long)a.order[r]) / a.topk;
  };
  long long row[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const long long r = min(t.r0 + m * 16 + lr, t.r1 - 1);
    row[m] = r;
    xp[m] = a.x + token(r) * a.ldx;
  }
  // The epilogue's thread: eight neighbouring outputs of a token row. What it needs beside the sums
  // is requested here, so that it does not wait for memory at the end; a bf16 bias, whose values are loaded one
  // after the other, and the ragged end of mul and residual are waited for here, in front of the weights (16 x
  // 2048 x 8192 e4m3 7.5 us with a bf16 bias, 6.4 with an fp32 one or none).
  constexpr int PER = MODE == kRowsGateUp ? 4 : 2 * NB;  // threads of a row
  static_assert(16 * MB * PER <= W * 64, "a thread each");
  const int tid = threadIdx.x, erow = tid / PER, ec = tid - erow * PER;
  const long long er = t.r0 + erow, err = min(er, t.r1 - 1);
  const int en = (MODE == kRowsGateUp ? blockIdx.x * 32 : blockIdx.x * NB * 16) + ec * 8;
  const bool mine = erow < 16 * MB && (MODE != kRowsLinear || (er < t.r1 && en < a.N));
  float ews[8], eother[8], exs = 1.f;
  RowsOperands eop;
  long long pair = 0;
  if (mine) {
    if constexpr (MODE == kRowsGateUp) {
      rows_gate_up_cols(a, t.e, en, ews, eother);
      exs = a.xs[token(err)];
    } else if constexpr (MODE == kRowsLinear) {
      rows_linear_cols(a, en, ews, eother);
      rows_linear_load(a, er, en, eop);
      if (a.xs) exs = a.xs[er];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) ews[j] = a.ws[(long long)t.e * a.N + min(en, a.N - 8) + j];
      pair = a.order[err];
    }
  }
  f32x4_t acc[NB][MB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[b][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int nch = (a.Kb + 127) / 128;
  const int c0 = (int)((long long)nch * wave / W), c1 = (int)((long long)nch * (wave + 1) / W);
  for (int c = c0; c < c1; c += U) {
    uint4 wv[U][NB][2], xv[U][MB][2];
    uint32_t sv[U][MB];
#pragma unroll
    for (int s = 0; s < U; ++s) {
      // past the wave's part or the row's end: bytes there again, below made zeros
      const int k0 = (c + s) * 128 + kq * 16, k1 = k0 + 64;
      const int o0 = min(k0, a.Kb - 16), o1 = min(k1, a.Kb - 16);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        wv[s][b][0] = ld16_stream(wp[b] + o0);
        wv[s][b][1] = ld16_stream(wp[b] + o1);
      }
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        xv[s][m][0] = ld16(xp[m] + o0);
        xv[s][m][1] = ld16(xp[m] + o1);
        if (MODE == kRowsDown) sv[s][m] = rows_group_scales(a, min(c + s, nch - 1), row[m]);
      }
    }
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int k0 = (c + s) * 128 + kq * 16, k1 = k0 + 64;
      const int end = c + s < c1 ? a.Kb : 0;
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        if (k0 >= end) xv[s][m][0] = make_uint4(0u, 0u, 0u, 0u);
        if (k1 >= end) xv[s][m][1] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (ES == 2) {  // whose weights may be infinite, and zero times that is NaN
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          if (k0 >= end) wv[s][b][0] = make_uint4(0u, 0u, 0u, 0u);
          if (k1 >= end) wv[s][b][1] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m)
          if constexpr (MODE == kRowsDown)
            acc[b][m] = rows_mma_wide(wv[s][b][0], wv[s][b][1], xv[s][m][0], xv[s][m][1],
                                      rows_group_two(sv[s][m], kq >> 1),
                                      rows_group_two(sv[s][m], 2 + (kq >> 1)), acc[b][m]);
          else if constexpr (WIDE)
            acc[b][m] = rows_mma_wide(wv[s][b][0], wv[s][b][1], xv[s][m][0], xv[s][m][1], 1.f, 1.f, acc[b][m]);
          else
            acc[b][m] = rows_mma<ES>(wv[s][b][0], wv[s][b][1], xv[s][m][0], xv[s][m][1], acc[b][m]);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int m = 0; m < MB; ++m) red[wave][m * NB + b][lane] = acc[b][m];
  __syncthreads();
  if (!mine) return;  // (whole waves, or for kRowsLinear threads that share nothing)
  // quads (b, 2 h) and (b, 2 h + 1) of token row (m, lr) lie 16 lanes apart
  auto sum = [&](int b, float (&v)[8]) __attribute__((always_inline)) {
    const int l = (erow & 15) + (ec & 1) * 32, at = (erow >> 4) * NB + b;
    f32x4_t s0 = red[0][at][l], s1 = red[0][at][l + 16];
#pragma unroll
    for (int w = 1; w < W; ++w) s0 += red[w][at][l], s1 += red[w][at][l + 16];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = s0[j], v[4 + j] = s1[j];
  };
  float v[8];
  sum(ec >> 1, v);
  if constexpr (MODE == kRowsGateUp) {
    float u[8];
    sum(2 + (ec >> 1), u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= exs, u[j] *= exs;
    rows_gate_up_out(a, er < t.r1, er, en, ews, eother, v, u);
  } else if constexpr (MODE == kRowsLinear) {
    if (a.xs) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= exs;
    }
    rows_linear_store<false>(a, er, en, rows_linear_value(a, ews, eother, eop, v));
  } else {
    rows_down_out(a, er < t.r1, pair, en, ews, v);
  }
}

// Many token rows: 16 NA kWM weight rows times 32 NB token rows a workgroup of W = 2 kWM waves, both
// operands staged in LDS. Wave (wm, wn) owns 16 NA weight rows and every other 16-row token block:
// 16 x 16 blocks acc[NA][NB], so each fragment read from LDS feeds NA or NB matrix instructions (at NA =
// NB = 8 the reads of a step take half the time of its products; with 64 x 128 blocks, three quarters).
// Linear's larger tiles: four waves, a SIMD's whole register file each, since the products are the bound (8192^2, K =
// 2048 bf16 270 us, 273 with eight waves; K = 4096 e4m3 220 and 229). The experts' larger tiles wait for
// memory and take long in their epilogue: eight waves, which wait in turns (4096 tokens as below 299 ->
// 276 us).
//
// Staging. A step of K (128 bytes of a row) is loaded memory -> LDS by DMA, eight rows (1 KiB) a load
// of a wave, into rings of SA weight and SB token stages: step d + SA of the weights and d + SB of the
// tokens are requested once step d has been read. Row r's 16-byte unit u is kept at unit u ^ key(r),
// so that the eight lanes that LDS serves at a time read eight different units. Rows past the tile's
// last one and bytes past a row's end lie outside the load's buffer and come as zeros.
//
// Order of the weight rows: row 4 q + i of block b is the wave's output 4 NA q + 4 b + i, so a lane
// ends with 4 NA neighbouring outputs (or 2 NA gate and 2 NA up ones) of each token
// and stores them in 16-byte pieces.
//
// A larger tile's step: its products go in four quarters (weight half, token half): (0, 0), (0, 1), (1, 1), (1, 0). Between
// its matrix instructions, which leave three of four issue slots free, each reads from LDS, early, the
// half that the next one needs; the last two read the next step's first halves, the tokens' into the
// registers that held half 1. Two barriers a step. After the first quarter the step's tokens have been
// read by all: their stage is loaded during the second. After the third, its weights have: theirs is
// loaded during the fourth. Behind the first the next step's weights have arrived, behind the second
// its tokens: either has a step and a half. (With one barrier, after the second quarter, the tokens
// had one step, less than L2 takes where there are 192 rows. With the loads issued together after it
// and the reads after each block's products, a step of 256 x 256 took 4400 cycles; its products
// take 2048.)
//
// A workgroup walks over tiles, as many workgroups as the chip holds. The next tile's first steps
// are requested before the present one's epilogue, which needs only the last weight stage of LDS, so
// that memory is not idle during it. In front of them the epilogue's scales, bias and first operands are
// waited for.
struct Frag {
  u32x4v v[2];
};
// acc += w . t for one step (bf16: for its half H), in place: as asm, because the compiler, given 256
// sums, moves some of them between registers around every product. It does not see these writes,
// so the sums are read only behind mma_done.
template <int ES, bool SC, int H>
__device__ __forceinline__ void tile_mma(const Frag& w, const Frag& t, uint32_t sb, f32x4_t& acc) {
  if constexpr (ES == 2) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(w.v[H]), "v"(t.v[H]));
  } else {
    typedef unsigned u32x8v __attribute__((ext_vector_type(8)));
    const u32x8v w8 = __builtin_shufflevector(w.v[0], w.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    const u32x8v t8 = __builtin_shufflevector(t.v[0], t.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (SC) {
      const uint32_t one = 0x7f;
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
                   : "+a"(acc) : "v"(w8), "v"(t8), "v"(one), "v"(sb));
    } else {
      asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+a"(acc) : "v"(w8), "v"(t8));
    }
  }
}
__device__ __forceinline__ void tie(uint4& v) {
  asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
}
// (also as asm: the compiler would read all sums of a tile ahead of the loop that stores them, into
// registers that are not there)
__device__ __forceinline__ void lds_write_scaled_sums(uint32_t addr, const f32x4_t& acc, float s) {
  f32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(f) : "a"(acc[i]));
    v[i] = f * s;
  }
  asm volatile("ds_write_b128 %0, %1" : : "v"(addr), "v"(v) : "memory");
}
__device__ __forceinline__ void lds_write_sums(uint32_t addr, const f32x4_t& acc) {
  asm volatile("ds_write_b128 %0, %1" : : "v"(addr), "a"(acc) : "memory");
}
// The last product's passes, before anything else reads the sums.
template <int NA, int NB>
__device__ __forceinline__ void mma_done(f32x4_t (&acc)[NA][NB]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int x = 0; x < NA; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y) asm volatile("" : "+a"(acc[x][y]));
}
template <int OFF>
__device__ __forceinline__ uint32_t lds_read4(uint32_t addr) {
  uint32_t r;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(OFF));
  return r;
}
template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (N > 0) {
    static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}
__device__ __forceinline__ void dma4_buffer(__amdgpu_buffer_rsrc_t buf, void* lds, uint32_t voff,
                                            uint32_t soff) {
  typedef __attribute__((address_space(3))) void lds_void;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_void*)lds, 4, voff, soff, 0, 0);
}

template <int MODE, int NA, int NB, int W>
struct TileShape {
  static constexpr int kWM = W / 2;  // waves side by side along the weight rows
  static constexpr int kWRows = 16 * NA * kWM, kTRows = 32 * NB;
  // Small tiles, whose fragments of a step fit in registers twice. Four stages where they fit (256 x 2048 x
  // 8192 bf16 by 128 x 64: 15.6 us with three, 14.5 with four; by 64 x 64, which share a CU, six take 20).
  static constexpr bool kFlat = W * NA * NB <= 32;
  static constexpr int kSA = kFlat && NA == 2 ? 4 : 3, kSB = kFlat ? kSA : 2;
  static constexpr bool kScaled = MODE == kRowsDown;
  static constexpr int kAStage = kWRows * 128;
  static constexpr int kBStage = kTRows * 128 + (kScaled ? kTRows * 4 : 0);
  static constexpr int kMetas = kSA * kAStage + kSB * kBStage;  // kRowsDown: the rows' pairs
  static constexpr int kLds = kMetas + (kScaled ? kTRows * 4 : 0);
  static constexpr int kOut = MODE == kRowsGateUp ? kWRows / 2 : kWRows;  // outputs per workgroup
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

template <int ES, int MODE, int NA, int NB, int W>
__global__ __launch_bounds__(64 * W, 1) void k_rows_tile(RowsGemm a, int ncol, int ntile) {
  using S = TileShape<MODE, NA, NB, W>;
  constexpr bool SC = S::kScaled, FLAT = S::kFlat;
  constexpr int HA = NA / 2, HB = NB / 2;
  constexpr int LA = S::kWRows / (8 * W), LB = S::kTRows / (8 * W);  // loads of a wave and step
  extern __shared__ uint4 smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % S::kWM, wn = wave / S::kWM;
  const int lr = lane & 15, kq = lane >> 4;
  char* lds = reinterpret_cast<char*>(smem);

  struct Tile {
    int e, r0, ntok, n0;  // expert, first token row (or sorted pair), rows, first output
  };
  // Tile `id`, id % 8 being this workgroup's XCD. Experts: the ncol tiles of the same rows on one XCD,
  // so they share them in that L2. Linear: each XCD walks its own part of the output in columns of
  // four tiles of token rows, whose workgroups share both operands.
  auto tile_of = [&](int id, Tile& t) __attribute__((always_inline)) {
    int tile, col;
    const int xcd = id & 7, j = id >> 3;
    if (MODE == kRowsLinear) {
      const int all = ncol * ntile, per = (all + 7) / 8;
      const int pos = xcd * per + j;
      if (j >= per || pos >= all) return false;
      const int g = pos / (4 * ncol), in = pos - g * 4 * ncol;
      const int high = min(4, ntile - 4 * g);
      col = in / high;
      tile = 4 * g + in - col * high;
    } else {
      tile = (j / ncol) * 8 + xcd;
      col = j - (j / ncol) * ncol;
    }
    RowsTile r;
    if (!rows_tile<MODE>(a, tile, S::kTRows, r)) return false;
    t.e = r.e, t.r0 = (int)r.r0, t.ntok = (int)(r.r1 - r.r0), t.n0 = col * S::kOut;
    return true;
  };
  int id = blockIdx.x;
  Tile cur, next;
  if (!tile_of(id, cur)) return;

  // ---- DMA: the wave's load i fills LDS rows (wave + W i) 8 .. + 7, lane l unit l & 7 of row l >> 3
  constexpr uint32_t kNowhere = 0x80000000u;  // past the end of any of the buffers
  constexpr int SPAN = MODE == kRowsGateUp ? 2 * NA : 4 * NA;
  // kRowsGateUp's LDS rows: per wm 8 NA gate rows, then their up rows; UP: both in one load of the waves
  constexpr bool UP = MODE == kRowsGateUp && W > NA;
  static_assert(!UP || W == 2 * NA, "the waves' load is a wm's rows");
  const int grow = lane >> 3, row0 = wave * 8 + grow;
  const uint32_t ldw = (uint32_t)a.ldw, ldx = (uint32_t)a.ldx;
  uint32_t wunit[2], woff[2];  // by load parity (the key of row0 + 8 W)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + 8 * W * i, key = (r & 3) | (((r / SPAN) & 1) << 2);
    wunit[i] = ((lane & 7) ^ key) * 16;
    woff[i] = (UP ? row0 % (8 * NA) : row0) * ldw + wunit[i];
  }
  const uint32_t tunit = ((lane & 7) ^ grow) * 16;
  // (the last wave's scale load, past the stage's rows, repeats the one before)
  const int srow = min(wave, S::kTRows / 64 - 1) * 64;
  const int nd = (a.Kb + 127) / 128;
  // Where a tile's loads come from. A load's uniform offset never passes its buffer's end: the rows of a
  // group past the last row are those of the first group again.
  __amdgpu_buffer_rsrc_t wbuf, xbuf, sbuf;
  uint32_t wrow[LA], xrow[LB], toff[MODE == kRowsGateUp ? LB : 1], soff;
  int rot = 0;
  auto set_sources = [&](const Tile& t) __attribute__((always_inline)) {
    if (MODE != kRowsLinear && ldw % 4096 == 0)
      rot = (int)__umulhi((uint32_t)t.e * 2654435769u, (uint32_t)nd);
    const int wrows = MODE == kRowsGateUp ? 2 * a.N - t.n0 : min(S::kWRows, a.N - t.n0);
    wbuf = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.w + t.e * a.estride + (long long)t.n0 * a.ldw), 0,
        (uint32_t)(wrows - 1) * ldw + a.Kb, 0x00020000);
    const uint8_t* xbase = MODE == kRowsGateUp ? a.x : a.x + t.r0 * a.ldx;
    const uint32_t xbytes =
        MODE == kRowsGateUp ? (uint32_t)a.xbytes : (uint32_t)(t.ntok - 1) * ldx + a.Kb;
    xbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(xbase), 0, xbytes, 0x00020000);
    sbuf = __builtin_amdgcn_make_buffer_rsrc(
        SC ? a.asc + (long long)t.r0 * 4 : nullptr, 0,
        SC ? (uint32_t)((nd - 1) * a.P * 4 + t.ntok * 4) : 0, 0x00020000);
    soff = srow + lane < t.ntok ? (srow + lane) * 4 : kNowhere;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      constexpr int Q = MODE == kRowsGateUp && !UP ? NA / W : 1;
      const uint32_t r = UP                    ? (uint32_t)(wave / NA * a.N + i * 8 * NA)
                         : MODE == kRowsGateUp ? (uint32_t)((i / Q & 1) * a.N + i / (2 * Q) * 8 * NA + i % Q * 8 * W)
                                               : 8u * W * i;
      wrow[i] = __builtin_amdgcn_readfirstlane((int)r < wrows ? r * ldw : 0);
    }
#pragma unroll
    for (int i = 0; i < LB; ++i)
      xrow[i] =
          __builtin_amdgcn_readfirstlane(MODE != kRowsGateUp && 8 * W * i < t.ntok ? 8u * W * i * ldx : 0);
    if constexpr (MODE == kRowsGateUp) {
#pragma unroll
      for (int i = 0; i < LB; ++i) {
        const int tok = a.order[t.r0 + min(row0 + 8 * W * i, t.ntok - 1)] / a.topk;
        toff[i] = row0 + 8 * W * i < t.ntok ? (uint32_t)tok * ldx + tunit : kNowhere;
      }
    } else {
      toff[0] = row0 * ldx + tunit;
    }
  };
  // The loads of step d; past the last one, of nothing, so that every step has the same loads in
  // flight. All of it is selects and sums: a branch among the products would cost more than they do.
  struct Step {
    uint32_t k0, stage;  // byte of K, LDS offset of the stage
    uint32_t off[2];     // kNowhere for the lanes past the row's end, else 0
  };
  auto byte_of = [&](int d) __attribute__((always_inline)) {
    const int at = MODE == kRowsLinear ? d : d + rot;
    return (uint32_t)min(MODE == kRowsLinear || at < nd ? at : at - nd, nd - 1) * 128;
  };
  auto past = [&](int d, uint32_t k0, uint32_t unit) __attribute__((always_inline)) {
    if (MODE == kRowsLinear) return (uint32_t)d * 128 + unit < (uint32_t)a.Kb ? 0u : kNowhere;
    return d < nd && k0 + unit < (uint32_t)a.Kb ? 0u : kNowhere;
  };
  auto step_a = [&](int d, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t k0 = byte_of(d);
    return Step{k0, stage, {past(d, k0, wunit[0]), past(d, k0, wunit[1])}};
  };
  auto step_b = [&](int d, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t k0 = byte_of(d);
    return Step{k0, stage, {past(d, k0, tunit), d < nd ? 0u : kNowhere}};
  };
  auto load_a = [&](const Step& st, auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    dma16_buffer(wbuf, lds + st.stage + (wave + W * i) * 1024, woff[i & 1] | st.off[i & 1],
                 st.k0 + wrow[i]);
  };
  auto load_b = [&](const Step& st, auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i == LB)  // a dword of four groups' scales per row
      dma4_buffer(sbuf, lds + st.stage + S::kTRows * 128 + srow * 4, soff | st.off[1],
                  (st.k0 >> 7) * (uint32_t)(a.P * 4));
    else
      dma16_buffer(xbuf, lds + st.stage + (wave + W * i) * 1024,
                   toff[MODE == kRowsGateUp ? i : 0] | st.off[0], st.k0 + xrow[i]);
  };
  constexpr int NLB = LB + (SC ? 1 : 0);
  constexpr int kB0 = S::kSA * S::kAStage;  // the token ring
  // The first steps' loads, each step's weights and then its tokens; what goes to the last weight stage, which
  // the epilogue uses, is requested at the tile's start (last_loads).
  auto first_loads = [&]() __attribute__((always_inline)) {
    static_for<S::kSA - 1>([&](auto dc) __attribute__((always_inline)) {
      constexpr int d = decltype(dc)::value;
      static_for<LA>([&](auto k) __attribute__((always_inline)) { load_a(step_a(d, d * S::kAStage), k); });
      static_for<NLB>([&](auto k)
                          __attribute__((always_inline)) { load_b(step_b(d, kB0 + d * S::kBStage), k); });
    });
  };
  auto last_loads = [&]() __attribute__((always_inline)) {
    constexpr int d = S::kSA - 1;
    static_for<LA>([&](auto k) __attribute__((always_inline)) { load_a(step_a(d, d * S::kAStage), k); });
    if constexpr (FLAT)
      static_for<NLB>([&](auto k)
                          __attribute__((always_inline)) { load_b(step_b(d, kB0 + d * S::kBStage), k); });
  };

  // ---- fragments
  const uint32_t lbase = lds_addr(lds);
  uint32_t aaddr, baddr;
  {
    const int r = wm * 16 * NA + (lr >> 2) * SPAN + (lr & 3);  // block b: + 4 b rows
    const int key = (r & 3) | (((r / SPAN) & 1) << 2);
    aaddr = lbase + r * 128 + (kq ^ key) * 16;
    baddr = lbase + (wn * 16 + lr) * 128 + (kq ^ (lr & 7)) * 16;
  }
  const uint32_t saddr = lbase + S::kTRows * 128 + (wn * 16 + lr) * 4;
  // weight block b: gate blocks first (kRowsGateUp), then the up blocks 8 NA rows on
  auto read_a = [&](uint32_t at, auto bc, Frag& f) __attribute__((always_inline)) {
    constexpr int b = decltype(bc)::value;
    constexpr int off = (MODE == kRowsGateUp && b >= HA ? 8 * NA + 4 * (b - HA) : 4 * b) * 128;
    f.v[0] = lds_read_frag<off>(at);
    f.v[1] = lds_read_frag<off>(at ^ 64);
  };
  auto read_b = [&](uint32_t stage, auto bc, Frag& f, uint32_t& sc) __attribute__((always_inline)) {
    constexpr int b = decltype(bc)::value;
    f.v[0] = lds_read_frag<b * 32 * 128>(baddr + stage);
    f.v[1] = lds_read_frag<b * 32 * 128>((baddr + stage) ^ 64);
    if constexpr (SC) sc = lds_read4<b * 32 * 4>(saddr + stage);
  };

  f32x4_t acc[NA][NB];
  constexpr int FA = FLAT ? NA : HA, FB = FLAT ? NB : HB;
  Frag a0[FA], a1[FA], bx[FB], by[FB];
  uint32_t sx[FB] = {}, sy[FB] = {};
  auto ready_a = [&](Frag (&f)[FA]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FA; ++i) after_wait(f[i].v[0]), after_wait(f[i].v[1]);
  };
  auto ready_b = [&](Frag (&f)[FB], uint32_t (&sc)[FB]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FB; ++i) {
      after_wait(f[i].v[0]), after_wait(f[i].v[1]);
      if (SC) {
        asm volatile("" : "+v"(sc[i]));
        sc[i] >>= 8 * kq;
      }
    }
    // Two wait states between the last shift and a product that reads it: the compiler keeps them for
    // products of its own, not for asm. The ties hold the shifts in front of the wait.
    if (SC) {
#pragma unroll
      for (int i = 0; i < FB; ++i) asm volatile("" : "+v"(sc[i]));
      asm volatile("s_nop 1");
    }
  };
  // One quarter: weight half x, token half y. After its product p (bf16: all first halves, then all
  // second ones, so that no product waits for the one before), what falls due: read k of NR at
  // product RS k, load k of NL at product (k PROD) / NL (one later where there is room).
  constexpr int PROD = HA * HB * ES;
  auto quarter = [&](const Frag (&w)[FA], const Frag (&tk)[FB], const uint32_t (&sc)[FB], auto xh, auto yh,
                     auto nr, auto read, auto nl, auto load) __attribute__((always_inline)) {
    constexpr int X = decltype(xh)::value, Y = decltype(yh)::value;
    constexpr int NR = decltype(nr)::value, NL = decltype(nl)::value;
    constexpr int RS = PROD / 2 / NR > 0 ? PROD / 2 / NR : 1;
    constexpr int LO = NL > 0 && PROD / (NL > 0 ? NL : 1) > 1 ? 1 : 0;
    static_for<PROD>([&](auto prod) __attribute__((always_inline)) {
      constexpr int p = decltype(prod)::value, H = p / (HA * HB), i = p / HA % HB, j = p % HA;
      tile_mma<ES, SC, H>(w[j], tk[i], sc[i], acc[X * HA + j][Y * HB + i]);
      __builtin_amdgcn_sched_barrier(0);
      static_for<NR>([&](auto k) __attribute__((always_inline)) {
        constexpr int due = decltype(k)::value * RS;
        if constexpr ((due < PROD ? due : PROD - 1) == p) read(k);
      });
      static_for<NL>([&](auto k) __attribute__((always_inline)) {
        if constexpr (decltype(k)::value * PROD / NL + LO == p) load(k);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  using std::integral_constant;
  const integral_constant<int, 0> c0{};
  const integral_constant<int, 1> c1{};
  const integral_constant<int, HA> cha{};
  const integral_constant<int, HB> chb{};
  const auto none = [](auto) {};
  // Ring offsets: the stages of this step and the next ones.
  uint32_t ra[S::kSA], rb[S::kSB];
  auto turn = [](auto& r) __attribute__((always_inline)) {
    constexpr int n = sizeof(r) / sizeof(r[0]);
    const uint32_t first = r[0];
#pragma unroll
    for (int i = 0; i + 1 < n; ++i) r[i] = r[i + 1];
    r[n - 1] = first;
  };
  // Step d with its tokens' half 0 in p; half 1 goes to q, and the next step's half 0 after it.
  auto step = [&](int d, Frag (&p)[FB], uint32_t (&sp)[FB], Frag (&q)[FB], uint32_t (&sq)[FB])
                  __attribute__((always_inline)) {
    if constexpr (!FLAT) {
      const uint32_t at = aaddr + ra[0], at1 = aaddr + ra[1];
      quarter(a0, p, sp, c0, c0, chb, [&](auto k) __attribute__((always_inline)) {
        constexpr int K = decltype(k)::value;
        read_b(rb[0], integral_constant<int, HB + K>{}, q[K], sq[K]);
      }, c0, none);
      lds_frags_ready();
      ready_b(q, sq);
      wait_loads(LA + NLB);  // in flight: step d + 1's tokens, step d + 2's weights
      __builtin_amdgcn_s_barrier();
      const Step nb = step_b(d + S::kSB, rb[0]), na = step_a(d + S::kSA, ra[0]);
      quarter(a0, q, sq, c0, c1, cha, [&](auto k) __attribute__((always_inline)) {
        constexpr int K = decltype(k)::value;
        read_a(at, integral_constant<int, HA + K>{}, a1[K]);
      }, integral_constant<int, NLB>{}, [&](auto k) __attribute__((always_inline)) { load_b(nb, k); });
      lds_frags_ready();
      ready_a(a1);
      quarter(a1, q, sq, c1, c1, cha, [&](auto k) __attribute__((always_inline)) {
        read_a(at1, k, a0[decltype(k)::value]);
      }, c0, none);
      lds_frags_ready();
      ready_a(a0);
      wait_loads(LA + NLB);  // in flight: step d + 2's weights and tokens
      __builtin_amdgcn_s_barrier();
      quarter(a1, p, sp, c1, c0, chb, [&](auto k) __attribute__((always_inline)) {
        constexpr int K = decltype(k)::value;
        read_b(rb[1], k, q[K], sq[K]);
      }, integral_constant<int, LA>{}, [&](auto k) __attribute__((always_inline)) { load_a(na, k); });
      lds_frags_ready();
      ready_b(q, sq);
      turn(ra), turn(rb);
    }
  };

  // A small tile's step: its fragments are in registers (w, tk), the next step's are read to others
  // during its products, and what is a ring's length on is loaded to the stages that it was read from.
  // One barrier and one wait for LDS; in quarters there are four, with a product or two between them
  // (64 x 2048 x 2048 bf16 11.2 us in quarters, 9.6 so; 128 x 64 blocks a wave and larger hide theirs).
  auto flat_step = [&](int d, const Frag (&w)[FA], const Frag (&tk)[FB], const uint32_t (&sc)[FB],
                       Frag (&wn)[FA], Frag (&tn)[FB], uint32_t (&sn)[FB])
                       __attribute__((always_inline)) {
    if constexpr (FLAT) {
      wait_loads((S::kSA - 2) * (LA + NLB));  // step d + 1 has arrived
      __builtin_amdgcn_s_barrier();
      const Step nb = step_b(d + S::kSB, rb[0]), na = step_a(d + S::kSA, ra[0]);
      const uint32_t at = aaddr + ra[1];
      constexpr int ALL = NA * NB * ES, NL = LA + NLB;
      static_for<ALL>([&](auto prod) __attribute__((always_inline)) {
        constexpr int p = decltype(prod)::value, H = p / (NA * NB), i = p / NA % NB, j = p % NA;
        tile_mma<ES, SC, H>(w[j], tk[i], sc[i], acc[j][i]);
        __builtin_amdgcn_sched_barrier(0);
        static_for<NA + NB>([&](auto kc) __attribute__((always_inline)) {
          constexpr int k = decltype(kc)::value;
          if constexpr ((k < ALL ? k : ALL - 1) == p) {
            if constexpr (k < NB)
              read_b(rb[1], kc, tn[k], sn[k]);
            else
              read_a(at, integral_constant<int, k - NB>{}, wn[k - NB]);
          }
        });
        static_for<NL>([&](auto kc) __attribute__((always_inline)) {
          constexpr int k = decltype(kc)::value;
          if constexpr (k * ALL / NL == p) {
            if constexpr (k < LA)
              load_a(na, kc);
            else
              load_b(nb, integral_constant<int, k - LA>{});
          }
        });
        __builtin_amdgcn_sched_barrier(0);
      });
      lds_frags_ready();
      ready_a(wn);
      ready_b(tn, sn);
      turn(ra), turn(rb);
    }
  };

  // ---- epilogue: a token block (16 rows) of a wave at a time through its part of a weight stage, so that
  // one small loop serves all of the sums (unrolled over the registers it was 80 KB of instructions,
  // which took longer to fetch than a tile of K = 1024 to multiply) and a row's outputs are stored
  // together. Unit u of row r lies at unit u ^ (r & 7), so that eight rows differ in banks.
  constexpr int PER = (MODE == kRowsGateUp ? NA : 2 * NA);  // lanes of a row, eight outputs each
  constexpr int RPI = 64 / PER;
  static_assert(PER >= 4 && 64 % PER == 0 && 16 % (64 / PER) == 0, "whole turns in a token block");
  constexpr int UE = 16 / RPI;  // rows of a lane in a token block
  constexpr int kRow = 16 * NA * 4;
  static_assert(W * 16 * kRow == S::kAStage, "the waves' parts");
  const uint32_t part = lbase + (S::kSA - 1) * S::kAStage + wave * 16 * kRow;
  const int c = lane % PER, rsub = lane / PER;
  float ws[8], other[8], xs[NB];  // column scales, and the up scales or the bias; row scales
  auto scales = [&](const Tile& t) __attribute__((always_inline)) {
    const int n = t.n0 + wm * (S::kOut / S::kWM) + c * 8;
    if constexpr (MODE == kRowsGateUp) {
      rows_gate_up_cols(a, t.e, n, ws, other);
    } else if constexpr (MODE == kRowsLinear) {
      rows_linear_cols(a, n, ws, other);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) ws[i] = a.ws[(long long)t.e * a.N + min(n + i, a.N - 1)];
      const int pair = a.order[t.r0 + min(tid, t.ntok - 1)];
      if (tid < S::kTRows)
        asm volatile("ds_write_b32 %0, %1" : : "v"(lbase + S::kMetas + tid * 4), "v"(pair) : "memory");
    }
    if constexpr (ES == 1 && MODE != kRowsDown) {
      int row[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) row[b] = t.r0 + min((2 * b + wn) * 16 + lr, t.ntok - 1);
      if constexpr (MODE == kRowsGateUp) {
#pragma unroll
        for (int b = 0; b < NB; ++b) row[b] = a.order[row[b]];
#pragma unroll
        for (int b = 0; b < NB; ++b) row[b] /= a.topk;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) xs[b] = a.xs[row[b]];
    }
  };
  auto stage = [&](auto bc) __attribute__((always_inline)) {
    constexpr int b = decltype(bc)::value;
    const uint32_t row = part + lr * kRow, key = lr & 7;
#pragma unroll
    for (int x = 0; x < NA; ++x) {
      const int unit = MODE == kRowsGateUp && x >= HA ? 2 * NA + kq * (SPAN / 4) + x - HA
                                                      : kq * (SPAN / 4) + x;
      const uint32_t at = row + ((unit ^ key) * 16);
      if constexpr (ES == 1 && MODE != kRowsDown) {
        lds_write_scaled_sums(at, acc[x][b], xs[b]);
      } else {
        lds_write_sums(at, acc[x][b]);
      }
    }
  };
  // mul and residual of a token block. They are requested two blocks ahead and before the stores of the
  // block then at hand, because loads and stores complete in order: a load behind the stores would wait
  // for them, and with it everything. For the same reason there is no branch here (behind one the
  // compiler waits for all in flight): what is not there reads 16 bytes of a weight row.
  struct Ops {
    RowsOperands row[UE];
  };
  const uint16_t* idle = reinterpret_cast<const uint16_t*>(a.w);
  auto row_of = [&](int b, int i) __attribute__((always_inline)) {  // in the tile
    return (2 * b + wn) * 16 + rsub + i * RPI;
  };
  auto fetch = [&](const Tile& t, int b, Ops& o) __attribute__((always_inline)) {
    const int n = t.n0 + wm * (S::kOut / S::kWM) + c * 8;
#pragma unroll
    for (int i = 0; i < UE; ++i) {
      const int row = row_of(b, i);
      const bool there = row < t.ntok && n + 8 <= a.N;
      const long long at = (long long)(t.r0 + row) * a.N + n;
      o.row[i].mul = rows_load8(a.mul && there ? a.mul + at : idle);
      o.row[i].res = rows_load8(a.res && there ? a.res + at : idle);
    }
  };
  // Token block b of the nb. LDS is accessed by asm: around accesses of its own the compiler would wait
  // for the DMA loads, as which it counts the stores here too.
  auto finish = [&](auto with, const Tile& t, int b, int nb, Ops& o) __attribute__((always_inline)) {
    constexpr bool WITH = decltype(with)::value;
    const int n = t.n0 + wm * (S::kOut / S::kWM) + c * 8;
    static_for<NB>([&](auto k) __attribute__((always_inline)) {
      if (b == decltype(k)::value) stage(k);
    });
    u32x4v raw[UE][MODE == kRowsGateUp ? 4 : 2];
    uint32_t mv[UE];
#pragma unroll
    for (int i = 0; i < UE; ++i) {
      const int r = rsub + i * RPI;
      const uint32_t at = part + r * kRow + ((2 * c) ^ (r & 7)) * 16;
      raw[i][0] = lds_read_frag<0>(at);
      raw[i][1] = lds_read_frag<0>(at ^ 16);
      if constexpr (MODE == kRowsGateUp) {
        raw[i][2] = lds_read_frag<32 * NA>(at);
        raw[i][3] = lds_read_frag<32 * NA>(at ^ 16);
      }
      if constexpr (SC) mv[i] = lds_read4<0>(lbase + S::kMetas + row_of(b, i) * 4);
    }
    lds_frags_ready();
#pragma unroll
    for (int i = 0; i < UE; ++i) {
      if (SC) asm volatile("" : "+v"(mv[i]));
#pragma unroll
      for (u32x4v& f : raw[i]) after_wait(f);
    }
    uint4 w[UE];
#pragma unroll
    for (int i = 0; i < UE; ++i) {
      const bool live = row_of(b, i) < t.ntok;
      const long long r = t.r0 + row_of(b, i);
      float v[8], u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __uint_as_float(raw[i][j / 4][j % 4]);
        if constexpr (MODE == kRowsGateUp) u[j] = __uint_as_float(raw[i][2 + j / 4][j % 4]);
      }
      if constexpr (MODE == kRowsGateUp) {
        rows_gate_up_out(a, live, r, n, ws, other, v, u);
      } else if constexpr (MODE == kRowsDown) {
        rows_down_out(a, live, mv[i], n, ws, v);
      } else {
        RowsOperands op;
        if (WITH) {
          op = o.row[i];
          if (live && n < a.N && n + 8 > a.N) rows_linear_load(a, r, n, op);
        }
        w[i] = rows_linear_value<WITH>(a, ws, other, op, v);
      }
    }
    if constexpr (MODE == kRowsLinear) {
      if (WITH) fetch(t, min(b + 2, nb - 1), o);
#pragma unroll
      for (int i = 0; i < UE; ++i)
        if (row_of(b, i) < t.ntok && n < a.N)
          rows_linear_store<NA == 8>(a, t.r0 + row_of(b, i), n, w[i]);
    }
  };

  set_sources(cur);
  first_loads();
  for (;;) {
    last_loads();
#pragma unroll
    for (int i = 0; i < S::kSA; ++i) ra[i] = i * S::kAStage;
#pragma unroll
    for (int i = 0; i < S::kSB; ++i) rb[i] = kB0 + i * S::kBStage;
#pragma unroll
    for (int x = 0; x < NA; ++x)
#pragma unroll
      for (int y = 0; y < NB; ++y) acc[x][y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    wait_loads((S::kSB - 1) * (LA + NLB) + (FLAT ? 0 : LA));  // step 0 has arrived
    __builtin_amdgcn_s_barrier();
    static_for<FA>([&](auto k) __attribute__((always_inline)) { read_a(aaddr, k, a0[decltype(k)::value]); });
    static_for<FB>([&](auto k) __attribute__((always_inline)) {
      constexpr int K = decltype(k)::value;
      read_b(kB0, k, bx[K], sx[K]);
    });
    lds_frags_ready();
    ready_a(a0);
    ready_b(bx, sx);
    for (int d = 0; d < nd; d += 2) {
      if constexpr (FLAT) {
        flat_step(d, a0, bx, sx, a1, by, sy);
        flat_step(d + 1, a1, by, sy, a0, bx, sx);
      } else {
        step(d, bx, sx, by, sy);
        step(d + 1, by, sy, bx, sx);  // of zeros if nd is odd
      }
    }
    wait_loads(0);
    mma_done(acc);
    // What the epilogue reads is here before the next tile's loads are requested: behind them it would
    // wait for them.
    const int nb =
        __builtin_amdgcn_readfirstlane(min(NB, ((cur.ntok + 15) / 16 - wn + 1) / 2));  // blocks with rows
    Ops s0, s1;
    const bool with = MODE == kRowsLinear && (a.mul || a.res) && nb > 0;
    if (with) {
      fetch(cur, 0, s0);
      fetch(cur, min(1, nb - 1), s1);
    }
    id += gridDim.x;
    const bool more = tile_of(id, next);
    scales(cur);
    if (more) set_sources(next);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(ws[i]), "+v"(other[i]));
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (ES == 1 && MODE != kRowsDown) asm volatile("" : "+v"(xs[b]));
    if (with) {
#pragma unroll
      for (int i = 0; i < UE; ++i) {
        tie(s0.row[i].mul), tie(s0.row[i].res);
        tie(s1.row[i].mul), tie(s1.row[i].res);
      }
    }
    __builtin_amdgcn_s_barrier();  // the stages have been read by all
    if (more) first_loads();
    if (with) {
#pragma unroll 1
      for (int b = 0; b < nb; b += 2) {
        finish(std::true_type{}, cur, b, nb, s0);
        finish(std::true_type{}, cur, b + 1, nb, s1);  // (of no live rows if nb is odd)
      }
    } else {
#pragma unroll 1
      for (int b = 0; b < nb; ++b) finish(std::false_type{}, cur, b, nb, s0);
    }
    if (!more) return;
    __builtin_amdgcn_s_barrier();  // the last weight stage is free
    cur = next;
  }
}

// The down product of a few pairs and their weighted sum: 16 outputs of one token a workgroup, a wave
// a pair.
constexpr int kPairWaves = 8;
__global__ __launch_bounds__(kPairWaves * 64) void k_rows_pairs_down(RowsGemm a,
                                                                    RowsTail tail) {
  __shared__ float part[kPairWaves][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16;  // N is a multiple of 32
  const int nch = (a.Kb + 127) / 128;
  float total[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = wave; j < a.topk; j += kPairWaves) {
    const long long p = (long long)blockIdx.y * a.topk + j;
    const long long e = rows_pair_expert(a, p);
    const uint8_t* wp = a.w + e * a.estride + (n0 + lr) * a.ldw;
    const uint8_t* xp = a.x + p * a.ldx;  // every column of the product is the pair's row
    const float w = bf_bits2f(a.wts[p]);
    const float* sd = a.ws + e * a.N + n0 + 4 * kq;
    float sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sw[i] = sd[i];
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;
    for (int c = 0; c < nch; c += U) {
      uint4 wv[U][2], xv[U][2];
      uint32_t sv[U];
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const int k0 = (c + s) * 128 + kq * 16;
        const int o0 = min(k0, a.Kb - 16), o1 = min(k0 + 64, a.Kb - 16);
        wv[s][0] = ld16_stream(wp + o0), wv[s][1] = ld16_stream(wp + o1);
        xv[s][0] = ld16(xp + o0), xv[s][1] = ld16(xp + o1);
        sv[s] = rows_group_scales(a, min(c + s, nch - 1), p);
      }
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const int k0 = (c + s) * 128 + kq * 16;
        if (k0 >= a.Kb) xv[s][0] = make_uint4(0u, 0u, 0u, 0u);
        if (k0 + 64 >= a.Kb) xv[s][1] = make_uint4(0u, 0u, 0u, 0u);
        acc = rows_mma_wide(wv[s][0], wv[s][1], xv[s][0], xv[s][1], rows_group_two(sv[s], kq >> 1),
                            rows_group_two(sv[s], 2 + (kq >> 1)), acc);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) total[i] = fmaf(w, acc[i] * sw[i], total[i]);
  }
  if (lr == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][4 * kq + i] = total[i];
  }
  const int n = threadIdx.x;
  const long long at = (long long)blockIdx.y * a.N + n0 + (n & 15);
  const float gate = rows_tail_gate(tail, blockIdx.y);
  const float shared = tail.shared ? bf_bits2f(tail.shared[at]) : 0.f;
  const float res = tail.res ? bf_bits2f(tail.res[at]) : 0.f;
  __syncthreads();
  if (n >= 16) return;
  float s = part[0][n];
#pragma unroll
  for (int w = 1; w < kPairWaves; ++w) s += part[w][n];
  a.out[at] = f2bf_bits(rows_tail(tail, s, gate, shared, res));
}

// Eight outputs a thread, the pairs' values of eight pairs requested together. Bound by memory.
__global__ __launch_bounds__(256) void k_rows_combine(const uint16_t* y, const uint8_t* yexp,
                                                      const uint16_t* w, RowsTail tail, int T, int H,
                                                      int k, uint16_t* out) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int per = H / 8;
  const long long t = i / per;
  if (t >= T) return;
  const int c = (int)(i - t * per) * 8;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  const uint4 sh = tail.shared ? ld16_stream(tail.shared + t * H + c) : none;
  const uint4 rs = tail.res ? ld16_stream(tail.res + t * H + c) : none;
  const float gate = rows_tail_gate(tail, t);
  float acc[8] = {};
  for (int j0 = 0; j0 < k; j0 += 8) {
    uint4 v[8];
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long p = t * k + min(j0 + j, k - 1);
      v[j] = ld16_stream(y + p * H + c);
      m[j] = bf_bits2f(w[p]) * __uint_as_float((uint32_t)(yexp[p * (H / 32) + c / 32] - 1) << 23);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j0 + j >= k) break;
      const uint32_t u[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        const f16x2_t h = __builtin_bit_cast(f16x2_t, u[x]);
        acc[2 * x] = fmaf((float)h[0], m[j], acc[2 * x]);
        acc[2 * x + 1] = fmaf((float)h[1], m[j], acc[2 * x + 1]);
      }
    }
  }
  const uint32_t su[4] = {sh.x, sh.y, sh.z, sh.w}, ru[4] = {rs.x, rs.y, rs.z, rs.w};
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    acc[2 * x] = rows_tail(tail, acc[2 * x], gate, bf_lo(su[x]), bf_lo(ru[x]));
    acc[2 * x + 1] = rows_tail(tail, acc[2 * x + 1], gate, bf_hi(su[x]), bf_hi(ru[x]));
  }
  st16(out + t * H + c, make_uint4(pack_bf2_rne(acc[0], acc[1]), pack_bf2_rne(acc[2], acc[3]),
                                   pack_bf2_rne(acc[4], acc[5]), pack_bf2_rne(acc[6], acc[7])));
}

template <int ES, int MODE, int NB, int MB, int W, int U>
hipError_t launch_few(const RowsGemm& a, hipStream_t s) {
  const long long cols = MODE == kRowsGateUp ? a.N / 32 : (a.N + 16 * NB - 1) / (16 * NB);
  const long long tiles = MODE == kRowsLinear     ? (a.M + 16 * MB - 1) / (16 * MB)
                          : a.ids && !a.table ? a.P
                                              : a.MT;
  if (cols * W * 64 > 0xffffffffLL || tiles > 0x7fffffffLL) return hipErrorInvalidValue;
  constexpr long long kGridY = 65535;
  for (long long i = 0; i < tiles; i += kGridY) {
    RowsGemm part = a;
    part.tile0 = (int)i;
    hipLaunchKernelGGL((k_rows_few<ES, MODE, NB, MB, W, U>),
                       dim3((unsigned)cols, (unsigned)std::min(tiles - i, kGridY)), dim3(W * 64), 0, s,
                       part);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

// A kernel's dynamic LDS above the default limit, allowed once per device.
template <int ES, int MODE, int NA, int NB, int W>
hipError_t allow_tile_lds() {
  static std::mutex mu;
  static uint64_t done = 0;  // bit d: device d
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (done >> dev & 1) return hipSuccess;
  err = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_rows_tile<ES, MODE, NA, NB, W>),
                            hipFuncAttributeMaxDynamicSharedMemorySize,
                            TileShape<MODE, NA, NB, W>::kLds);
  if (err == hipSuccess) done |= uint64_t(1) << dev;
  return err;
}

// Workgroups of the tile kernel that the device holds at once, by their LDS.
int resident(int lds) {
  static std::atomic<int> cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cus[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 8)
      n = 256;
    cus[dev].store(n, std::memory_order_relaxed);
  }
  return n / 8 * 8 * (160 * 1024 / lds);
}

template <int ES, int MODE, int NA, int NB, int W = 4>
hipError_t launch_tile(const RowsGemm& a, hipStream_t s) {
  using S = TileShape<MODE, NA, NB, W>;
  const long long ncol = (a.N + S::kOut - 1) / S::kOut;
  const long long ntile = MODE == kRowsLinear ? (a.M + S::kTRows - 1) / S::kTRows : a.MT;
  if (ntile <= 0) return hipSuccess;
  const long long tiles = MODE == kRowsLinear ? (ncol * ntile + 7) / 8 * 8 : (ntile + 7) / 8 * 8 * ncol;
  if (tiles > 0x3fffffffLL) return hipErrorInvalidValue;
  hipError_t err = allow_tile_lds<ES, MODE, NA, NB, W>();
  if (err != hipSuccess) return err;
  const long long grid = std::min<long long>(tiles, resident(S::kLds));
  hipLaunchKernelGGL((k_rows_tile<ES, MODE, NA, NB, W>), dim3((unsigned)grid), dim3(64 * W), S::kLds, s, a,
                     (int)ncol, (int)ntile);
  return hipGetLastError();
}

// The tile kernel's byte offsets into a tile's rows, an expert's weights, all token rows (gathered) and
// the scales are 32-bit, below its kNowhere.
bool tile_fits(RowsMode mode, const RowsGemm& a) {
  const long long most = 1LL << 31;
  if (256 * a.ldw >= most || 256 * a.ldx >= most) return false;
  if (mode == kRowsLinear) return 512LL * a.N < most;
  if (mode == kRowsGateUp) return 2LL * a.N * a.ldw < most && a.xbytes < most;
  return (a.Kb + 127) / 128 * a.P * 4 < most;
}

// Up to 16 token rows one block of them, up to 32 two (K = 2048, kernel us at M = 32: N = 2048 bf16 6.8
// as two workgroups of one block each, 10.1 as one of two, 10.9 by the 64 x 64 tile; N = 8192 e4m3 9.0,
// 7.2, 8.4; at M = 64 that tile takes 8.9, two blocks 11.3). Of weight rows, 16 a workgroup up to
// N = 4096, so that there are enough workgroups (one token, N = 2048 bf16: 5.5 us, 7.1 with 32), above
// it 32, whose token loads are half (16 tokens, N = 8192 e4m3: 8.3, 9.1 with 16).
//
// Above that the tile that takes the least time by its turns (us of K = 2048 bf16): 256 squared, a CU each,
// 54 a turn; 128 squared, 17.5, two on a CU; 128 weight rows by 64 token rows, a CU each, 12; 64 squared, 7.3,
// several on a CU. (64 / 128 by 64 / 128 / 256 squared: 200 x 2048 10.1, 12.5, -, -; 1111 x 1537 16.7, 14.4,
// 17.5, -; 256 x 8192 17.1, 14.5, -, -; 2048 x 2048 30.7, -, 21.2, 48; 1024 x 8192 -, -, 38.8, 50.4; 2048 x
// 8192 -, -, 71.2, 58.7.) The times of e4m3 and of other K lie alike, so that these four serve them too: e4m3
// 200 x 2048 7.6, 9.0, 11.8, 29.8; 1111 x 1537 10.4, 10.0, 13.4, 33.8; 256 x 8192 10.7, 10.3, 12.7, 31; 2048 x
// 2048 19.6, 17.8, 14.3, 31.4; 1024 x 8192 37.6, 32.7, 22.9, 32.2; 2048 x 8192 65.4, 61.5, 39.5, 36.3. Of 44
// sizes of either type, K = 512 to 8192, the tile chosen takes at most 1.09 of the best's time (8192 x 8192 x
// 512 e4m3: 77 us by 256 squared, 70 by 128).
template <int ES>
hipError_t launch_linear(const RowsGemm& a, hipStream_t s) {
  const bool fits = tile_fits(kRowsLinear, a);
  if (a.M <= 32 || !fits) {
    if (a.N > 4096 && a.M > 16) return launch_few<ES, kRowsLinear, 2, 2, 8, 2>(a, s);
    return a.N > 4096 ? launch_few<ES, kRowsLinear, 2, 1, 8, 2>(a, s)
                      : launch_few<ES, kRowsLinear, 1, 1, 8, 4>(a, s);
  }
  auto turns = [&](long long n, long long m) {
    return (double)(((a.M + m - 1) / m) * ((a.N + n - 1) / n)) / 256;
  };
  const double c64 = 7.3 * std::max(1.0, turns(64, 64)), c12864 = 12 * std::ceil(turns(128, 64)),
               c128 = 17.5 * std::max(1.0, turns(128, 128)), c256 = 54 * std::ceil(turns(256, 256));
  const double least = std::min(std::min(c64, c12864), std::min(c128, c256));
  if (c256 == least) return launch_tile<ES, kRowsLinear, 8, 8>(a, s);
  if (c128 == least) return launch_tile<ES, kRowsLinear, 4, 4>(a, s);
  if (c12864 == least) return launch_tile<ES, kRowsLinear, 2, 2, 8>(a, s);
  return launch_tile<ES, kRowsLinear, 2, 2>(a, s);
}

}  // namespace

// Up to 16 pairs, or one for every four experts, no tiles: few share an expert, and there is nothing to
// sort (us, H = 2048, I = 512, 256 experts, each pair by itself / tiles of 16: 32 pairs 25, 34; 64 41,
// 50; 128 75, 74; 16 experts of H = 4096, I = 1024: 32 pairs 79, 48). Else by the pairs r of an expert on
// average (256 experts as above, tiles of 16 / 64 / 128 / 192 pairs: r = 4 162, 172, 182, 191; r = 16 252,
// 191, 199, 208; r = 32 396, 201, 202, 214; r = 64 668, 253, 225, 240; r = 128 1187, 391, 307, 277). Tiles
// of 128 and 192 take a CU each and 128 outputs of gate_up: where these are under half a chip of
// workgroups, the next smaller tile (8 experts, r = 512: 70, 62 with 128, 59 with 192 for 96 workgroups;
// r = 256: 48, 47, 52).
int rows_tile_rows(int T, int H, int E, int k, int I) {
  const long long P = (long long)T * k;
  if (P <= std::max(16, E / 4)) return 0;
  RowsGemm gu{}, dn{};
  gu.N = I, gu.ldw = gu.ldx = H, gu.xbytes = (long long)T * H;
  dn.Kb = I, dn.ldw = dn.ldx = I, dn.P = P;
  if (P <= 12LL * E || !tile_fits(kRowsGateUp, gu) || !tile_fits(kRowsDown, dn)) return 16;
  auto workgroups = [&](long long rows) {
    return (P + E * rows - 1) / (E * rows) * E * ((I + 127) / 128);
  };
  if (P <= 48LL * E) return 64;
  if (P > 96LL * E && workgroups(192) >= 128) return 192;
  return workgroups(128) >= 128 ? 128 : 64;
}

hipError_t launch_rows_pairs_down(const RowsGemm& a, const RowsTail& tail, int T, hipStream_t s) {
  if (T <= 0) return hipSuccess;
  if (T > 65535 || a.N % 32 || a.Kb < 16 || a.Kb % 16) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k_rows_pairs_down, dim3(a.N / 16, T), dim3(kPairWaves * 64), 0, s, a, tail);
  return hipGetLastError();
}

hipError_t launch_rows_combine(const uint16_t* y, const uint8_t* yexp, const uint16_t* w,
                               const RowsTail& tail, int T, int H, int k, uint16_t* out,
                               hipStream_t s) {
  if (T <= 0) return hipSuccess;
  const long long grid = ((long long)T * (H / 8) + 255) / 256;
  if (H % 32 || grid * 256 > 0xffffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k_rows_combine, dim3((unsigned)grid), dim3(256), 0, s, y, yexp, w, tail, T, H, k,
                     out);
  return hipGetLastError();
}

hipError_t launch_rows_gemm(RowsMode mode, int es, const RowsGemm& a, int tile_rows,
                            hipStream_t s) {
  if (a.Kb < 16 || a.Kb % 16 || a.N < 1) return hipErrorInvalidValue;
  if (mode == kRowsLinear) return es == 2 ? launch_linear<2>(a, s) : launch_linear<1>(a, s);
  if (es != 1 || a.N % 32) return hipErrorInvalidValue;
  if (tile_rows > 16 && !tile_fits(mode, a)) return hipErrorInvalidValue;
  if (mode == kRowsGateUp) {
    switch (tile_rows) {
      case 64: return launch_tile<1, kRowsGateUp, 4, 2>(a, s);
      case 128: return launch_tile<1, kRowsGateUp, 4, 4, 8>(a, s);
      case 192: return launch_tile<1, kRowsGateUp, 4, 6, 8>(a, s);
      default: return launch_few<1, kRowsGateUp, 4, 1, 4, 1>(a, s);
    }
  }
  switch (tile_rows) {
    case 64: return launch_tile<1, kRowsDown, 4, 2>(a, s);
    case 128: return launch_tile<1, kRowsDown, 4, 4, 8>(a, s);
    case 192: return launch_tile<1, kRowsDown, 4, 6, 8>(a, s);
    default: return launch_few<1, kRowsDown, 2, 1, 4, 1>(a, s);
  }
}

}  // namespace moe
