// Products of microscaled rows (mx.h) with 4-bit weights on the scaled matrix instructions:
//
//   y[m, n] = sum_b 2^(sx[m, b] + sw[n, b] - 254) sum_{i in b} qx[m, i] qw[n, i]  (+ bias[n])
//
// plain, gated (silu of the first half of W's rows times the second) and over experts'
// segments (moe_tiles.h).  A lane of v_mfma_scale_f32_16x16x128_f8f6f4 has a row's block of 32
// values, 16 bytes of 4-bit codes, and its scale, so codes go from memory to LDS to the matrix
// unit as they are.  6-bit codes of x make exact products as well, in as many cycles (with values
// from registers 6.8 PFLOP/s where 4 bits have 7.3: the clock falls further); 8-bit ones would
// not: next to 4-bit numbers the unit adds their products up in too few bits (1024 inputs: 4e-6
// to 1.3e-5 of the result off, 6 and 4 bits 3e-8).
//
// Tiles of BM x BN, 256 inputs at a time: rows of 128 bytes, whole cache lines, loaded straight
// to LDS, and the scales of two such tiles at a time (K is taken in pairs of tiles).  Of a tile's
// eight blocks a lane of quarter q takes the blocks 2q and 2q + 1 in two products, whose scale
// bytes are neighbours: one read of two bytes serves both.  Which tile and how many parts of K:
// mx_plan; few rows have mx_few.hip.

#include <algorithm>

#include "mx_product.h"
#include "mx_wide.h"

namespace {

using mx::f32x4_t;
using mx::i32x2_t;
using mx::i32x4_t;
using mx::i32x8_t;

DEVINLINE float gate(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// Tiles of few rows: WM x WN waves, SLOTS whole tiles in LDS, each asked for SLOTS - 1 ahead.
// Bound by the bytes of W.  Where one tile has all rows (ONCE), they are read past the caches (57344 x
// 8192, 61 rows: 50 us kept in them, 46 so; 512 rows, where tiles share W: 37 kept, 42 not).  There a
// loop over all of K begins at another pair of tiles from column to column, as workgroups at the
// same one ask for the same part of every row at a time (us, at the same | turned: 57344 x 8192,
// 61 rows of 6 bits 52.9 | 47.3, 17 rows 50.0 | 48.5; 8 experts of 4096 x 14336, 50 rows of 6 bits
// each 61.1 | 56.1; 4 of 8200 x 8192, 13 rows of 6 bits 46.2 | 42.2; 28672 x 4096, 64 rows 19.1 |
// 19.5).  A part of K does not: parts are apart already (10240 x 8192 in two, 61 rows 22.7 | 23.5;
// 8192 x 28672 in four 36.2 | 35.7).
//
// Scales are what costs most to load: a row's are in a line of their own, and 8 bytes of it a tile,
// 32 lines a load, took as long as the codes (59 us there).  So two tiles' come together, 16
// bytes a row and lane, to a place of their own beside the slots.
template <int BM_, int BN_, int WM, int WN, int SLOTS, int XBITS, bool ONCE>
struct Narrow {
  static constexpr int BM = BM_, BN = BN_, kWN = WN;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  static constexpr int kTM = BM / WM / 16, kTN = BN / WN / 16;
  static constexpr int kX0 = BM * 128, kX1 = XBITS == 6 ? BM * 64 : 0;
  static constexpr int kAtW = kX0 + kX1, kSlot = kAtW + BN * 128;
  // scales of two tiles, 16 bytes a row, in as many places as no load meets a read in
  static constexpr int kPairs = (SLOTS + 2) / 2, kWsRows = (BN + 63) / 64 * 64;
  static constexpr int kAtScales = SLOTS * kSlot, kPair = (64 + kWsRows) * 16;
  static constexpr int kSpare = kAtScales + kPairs * kPair, kLds = kSpare + 1024;
  // loads of a wave: 8 rows of 128 bytes, 16 of 64, 64 of 16
  static constexpr int each(int loads) { return (loads + kWaves - 1) / kWaves; }
  static constexpr int kX0Loads = BM / 8, kXLoads = kX0Loads + kX1 / 1024, kWLoads = BN / 8;
  static constexpr int kScaleLoads = 1 + kWsRows / 64;
  static constexpr int kXEach = each(kXLoads), kWEach = each(kWLoads), kScaleEach = each(kScaleLoads);
  static constexpr int kLoads = kXEach + kWEach;
  static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && BM <= 64, "whole tiles");
  static_assert(kLds <= 160 * 1024 && (SLOTS - 1) * kLoads + SLOTS / 2 * kScaleEach < 64, "LDS, vmcnt");

  // as Wide::run
  template <typename XRow, typename WRow>
  static DEVINLINE void run(f32x4_t (&acc)[kTM][kTN], char* lds, const mx::Operands& p, XRow x_row,
                            WRow w_row) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4, wm = wave / WN, wn = wave % WN;
    unsigned x_off[kXEach], w_off[kWEach], s_off[kScaleEach];
    int w_chunk[kWEach];
#pragma unroll
    for (int i = 0; i < kXEach; ++i) {
      const int l = i * kWaves + wave;
      if (l < kX0Loads || kX1 == 0) {
        const int r = min(l * 8 + lane / 8, BM - 1);
        x_off[i] = x_row(r) * (unsigned)(p.pitch / 2) + mx::block_at((lane % 8) ^ (r / 2 % 8)) * 16;
      } else {
        const int r = min((l - kX0Loads) * 16 + lane / 4, BM - 1);
        x_off[i] = x_row(r) * (unsigned)(p.pitch / 4) + ((lane % 4) ^ (r / 4 % 4)) * 16;
      }
    }
#pragma unroll
    for (int i = 0; i < kWEach; ++i) {
      const int r = min((i * kWaves + wave) * 8 + lane / 8, BN - 1);
      w_off[i] = w_row(r) * (unsigned)p.k_bytes;
      w_chunk[i] = mx::block_at((lane % 8) ^ (r / 2 % 8)) * 16;
    }
#pragma unroll
    for (int i = 0; i < kScaleEach; ++i) {
      const int l = i * kWaves + wave, r = (l - 1) * 64 + lane;
      s_off[i] = (l == 0 ? x_row(min(lane, BM - 1)) : w_row(min(r, BN - 1))) * (unsigned)(p.pitch / 32);
    }

    const int n = p.tiles;
    // Past the last tile, and of waves without a load of their own: loads of nothing, so that
    // the counts stay what they are (one of the same again would wait for the first).  W's rows
    // end with K, its last tiles perhaps inside or past it: lanes past the end load the row's
    // last piece, which meets zeros of x and of the scales (both have rows of whole pairs).
    int pair_in = kAtScales;
    auto load = [&](auto even, int tile, char* slot) __attribute__((always_inline)) {
      const unsigned size = __builtin_amdgcn_readfirstlane(tile < n ? -1 : 0);
      const int turned = ONCE ? tile + p.turn : tile;
      const int t = p.first + (turned < n ? turned : turned - n);
      if constexpr (decltype(even)::value) {
#pragma unroll
        for (int i = 0; i < kScaleEach; ++i) {
          const int l = i * kWaves + wave;
          const bool one = l < kScaleLoads;
          block_gemm::load_lds(lds + (one ? pair_in + l * 1024 : kSpare),
                               block_gemm::resource(mx::either(l == 0, p.xs, p.ws), one ? size : 0), s_off[i],
                               t * 8);
        }
        pair_in = pair_in == kAtScales + (kPairs - 1) * kPair ? kAtScales : pair_in + kPair;
      }
#pragma unroll
      for (int i = 0; i < kXEach; ++i) {
        const int l = i * kWaves + wave;
        const bool one = kXLoads % kWaves == 0 || l < kXLoads, first = kX1 == 0 || l < kX0Loads;
        block_gemm::load_lds(one ? slot + l * 1024 : lds + kSpare,
                             block_gemm::resource(mx::either(first, p.x0, p.x1), one ? size : 0), x_off[i],
                             first ? t * 128 : t * 64);
      }
#pragma unroll
      for (int i = 0; i < kWEach; ++i) {
        const int l = i * kWaves + wave;
        const bool one = kWLoads % kWaves == 0 || l < kWLoads;
        block_gemm::load_lds<ONCE ? 2 : 0>(one ? slot + kAtW + l * 1024 : lds + kSpare,
                                           block_gemm::resource(p.w, one ? size : 0),
                                           w_off[i] + min(t * 128 + w_chunk[i], p.k_bytes - 16), 0);
      }
    };

    const int sw = col / 2 % 8;
    const int x_at = (wm * kTM * 16 + col) * 128, w_at = kAtW + (wn * kTN * 16 + col) * 128;
    const int x1_at = kX0 + (wm * kTM * 16 + col) * 64 + quad % 2 * 8;
    const int xs_at = (wm * kTM * 16 + col) * 16 + quad * 2;
    const int ws_at = (64 + wn * kTN * 16 + col) * 16 + quad * 2;
    constexpr std::true_type kEven{};
    constexpr std::false_type kOdd{};

#pragma unroll
    for (int s = 0; s < SLOTS - 1; ++s) {
      if (s % 2 == 0) load(kEven, s, lds + s * kSlot);
      else load(kOdd, s, lds + s * kSlot);
    }
    int at = 0, pair = kAtScales;
    auto turn = [&](auto even, int t) __attribute__((always_inline)) {
      constexpr bool EVEN = decltype(even)::value;
      // behind this tile's loads: those of SLOTS - 2 tiles, with the scales of the even ones
      constexpr int kScales = (EVEN ? (SLOTS - 2) / 2 : (SLOTS - 1) / 2) * kScaleEach;
      block_gemm::wait_loads_and_reads<(SLOTS - 2) * kLoads + kScales>();
      block_gemm::meet();
      const char* slot = lds + at * kSlot;
      load(std::integral_constant<bool, EVEN == (SLOTS % 2 == 1)>{}, t + SLOTS - 1,
           lds + (at == 0 ? SLOTS - 1 : at - 1) * kSlot);
      const char* scales = lds + pair + (EVEN ? 0 : 8);
      int sx[kTM], sq[kTN];
#pragma unroll
      for (int i = 0; i < kTM; ++i)
        sx[i] = *reinterpret_cast<const unsigned short*>(scales + xs_at + i * 256);
#pragma unroll
      for (int j = 0; j < kTN; ++j)
        sq[j] = *reinterpret_cast<const unsigned short*>(scales + ws_at + j * 256);
      auto step = [&](auto which) __attribute__((always_inline)) {
        constexpr int J = decltype(which)::value;
        const int chunk = ((4 * J + quad) ^ sw) * 16;
        const int chunk1 = ((2 * J + quad / 2) ^ (col / 4)) * 16;
        i32x8_t fx[kTM], fw[kTN];
#pragma unroll
        for (int j = 0; j < kTN; ++j) {
          const i32x4_t v = *reinterpret_cast<const i32x4_t*>(slot + w_at + j * 2048 + chunk);
          fw[j] = __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
        }
#pragma unroll
        for (int i = 0; i < kTM; ++i) {
          const i32x4_t v = *reinterpret_cast<const i32x4_t*>(slot + x_at + i * 2048 + chunk);
          if constexpr (XBITS == 6) {
            const i32x2_t u = *reinterpret_cast<const i32x2_t*>(slot + x1_at + chunk1 + i * 1024);
            fx[i] = __builtin_shufflevector(v, __builtin_shufflevector(u, u, 0, 1, -1, -1), 0, 1, 2,
                                            3, 4, 5, -1, -1);
          } else {
            fx[i] = __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
          }
        }
#pragma unroll
        for (int i = 0; i < kTM; ++i)
#pragma unroll
          for (int j = 0; j < kTN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                fw[j], fx[i], acc[i][j], 4, XBITS == 6 ? 2 : 4, J, sq[j], J, sx[i]);
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
      if (++at == SLOTS) at = 0;
      if (!EVEN) pair = pair == kAtScales + (kPairs - 1) * kPair ? kAtScales : pair + kPair;
    };
    for (int t = 0; t < n; t += 2) {
      turn(kEven, t);
      turn(kOdd, t + 1);
    }
    block_gemm::wait_loads<0>();   // (loads of nothing still write LDS)
  }
};

template <typename CORE, bool GATED, bool GROUPED>
DEVINLINE void tile(const MxProduct& p, char* lds) {
  constexpr int BM = CORE::BM, TM = CORE::kTM, TN = CORE::kTN;
  constexpr int OUT = GATED ? TN / 2 : TN;                       // output tiles of a wave
  constexpr int COLS = GATED ? CORE::BN / 2 : CORE::BN;          // outputs of a tile
  static_assert(!GATED || TN % 2 == 0, "a gate and what it gates in one lane");

  // the tile and the part of K
  const int n_tiles = (p.N + COLS - 1) / COLS;
  int row0, rows, n0, expert = 0, part;
  if constexpr (GROUPED) {
    const int tiles = moe::count_chunks(p.segs, BM) * n_tiles, all = tiles * p.parts;
    const int per_xcd = (all + 7) / 8, slot = blockIdx.x / 8, id = blockIdx.x % 8 * per_xcd + slot;
    if (slot >= per_xcd || id >= all) return;
    part = id / tiles;
    const moe::Tile at = moe::tile_of(p.segs, BM, n_tiles, id - part * tiles);
    row0 = at.row0, rows = min(at.rows, p.M - row0), n0 = at.n * COLS, expert = at.expert;
    if (row0 < 0 || rows <= 0) return;   // (segments that are none)
  } else {
    // an XCD's workgroups are neighbours: groups of eight columns, row by row
    const int m_tiles = (p.M + BM - 1) / BM, tiles = m_tiles * n_tiles, all = tiles * p.parts;
    const int per_xcd = (all + 7) / 8, slot = blockIdx.x / 8, id = blockIdx.x % 8 * per_xcd + slot;
    if (slot >= per_xcd || id >= all) return;
    part = id / tiles;
    const int t = id - part * tiles, group = t / (8 * m_tiles), left = min(8, n_tiles - group * 8);
    const int in = t - group * 8 * m_tiles;
    row0 = in / left * BM, n0 = (group * 8 + in % left) * COLS;
    rows = min(BM, p.M - row0);
  }

  // Rows past the last are the last one, whose results nobody stores.  Places in rows are
  // relative to the tile's first, of 32 bits in bytes (checked by the host).
  const bool listed = GROUPED && p.segs.rows != nullptr;
  const long x_base = listed ? 0 : row0, w_base = (long)expert * (GATED ? 2 : 1) * p.N + n0;
  const int n_left = p.N - n0, xs_pitch = p.pitch / 32;
  const int tiles_of_k = min(p.pitch / mx::kTile - part * p.depth, p.depth);
  const mx::Operands from{p.x0 + x_base * (p.pitch / 2),
                          p.x1 == nullptr ? nullptr : p.x1 + x_base * (p.pitch / 4),
                          p.xs + x_base * xs_pitch, p.w + w_base * (p.K / 2),
                          p.ws + w_base * xs_pitch, p.pitch, p.K / 2, part * p.depth,
                          tiles_of_k, p.parts == 1 ? n0 / COLS * 2 % tiles_of_k : 0};
  // acc[i][j][r]: row i * 16 + col of x, row j * 16 + quad * 4 + r of the wave's of W
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4, wm = wave / CORE::kWN, wn = wave % CORE::kWN;
  f32x4_t acc[TM][TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    f32x4_t first{};
    if (!GATED && !GROUPED && p.bias != nullptr && part == 0) {   // sums begin with the bias
#pragma unroll
      for (int r = 0; r < 4; ++r)
        first[r] = mx::get(p.bias, p.type, min(n0 + (wn * OUT + j) * 16 + quad * 4 + r, p.N - 1));
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i][j] = first;
  }
  CORE::run(
      acc, lds, from,
      [&](int r) -> unsigned {
        const int at = min(r, rows - 1);
        return listed ? min((unsigned)p.segs.rows[row0 + at], (unsigned)p.tokens - 1) : at;
      },
      [&](int r) -> unsigned {   // a wave's rows: its gates, then what they gate
        const int w = r / (TN * 16), j = r / 16 % TN;
        return min(w * OUT * 16 + j % OUT * 16 + r % 16, n_left - 1) + (j >= OUT ? p.N : 0);
      });

  const int cols = (p.N + 3) / 4 * 4;   // of a row of a part, or of half of it
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = (wm * TM + i) * 16 + col;
    if (m < rows) {
      const long row = row0 + m;
#pragma unroll
      for (int j = 0; j < OUT; ++j) {
        const int n1 = n0 + (wn * OUT + j) * 16 + quad * 4;
        if (n1 < p.N) {
          if (p.part != nullptr) {
            float* to = p.part + ((long)part * p.M + row) * ((GATED ? 2 : 1) * cols) + n1;
            *reinterpret_cast<f32x4_t*>(to) = acc[i][j];
            if (GATED) *reinterpret_cast<f32x4_t*>(to + cols) = acc[i][OUT + j];
          } else {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              v[r] = GATED ? gate(acc[i][j][r], acc[i][GATED ? OUT + j : j][r]) : acc[i][j][r];
            // (whole fours apart: a branch of the wave instead of one of lanes, 1 % of 256 x 256 tiles)
            if (p.N % 4 == 0) mx::put4(p.y, p.type, row * p.N + n1, v, 4);
            else mx::put4(p.y, p.type, row * p.N + n1, v, p.N - n1);
          }
        }
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, int SLOTS, int OCC, int XBITS, bool ONCE, bool GATED,
          bool GROUPED>
__global__ __launch_bounds__(WM * WN * 64, OCC) void mx_narrow_kernel(const MxProduct p) {
  using Core = Narrow<BM, BN, WM, WN, SLOTS, XBITS, ONCE>;
  __shared__ __align__(16) char lds[Core::kLds];
  tile<Core, GATED, GROUPED>(p, lds);
}

template <int BM, int BN, int WM, int WN, int SLOTS, int OCC, int XBITS, bool GATED, bool GROUPED>
__global__ __launch_bounds__(WM * WN * 64, OCC) void mx_wide_kernel(const MxProduct p) {
  using Core = mx::Wide<BM, BN, WM, WN, SLOTS, XBITS>;
  __shared__ __align__(16) char lds[Core::kLds];
  tile<Core, GATED, GROUPED>(p, lds);
}

// Sums of the parts, and the gate.  Four outputs a thread.
template <bool GATED>
__global__ __launch_bounds__(256) void mx_merge_kernel(const MxProduct p, const long rows) {
  const int quads = (p.N + 3) / 4, cols = quads * 4, width = (GATED ? 2 : 1) * cols;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * quads) return;
  const long row = i / quads;
  const int n1 = (int)(i % quads) * 4;
  if (p.segs.off != nullptr && row >= p.segs.off[p.segs.experts]) return;
  f32x4_t a{}, b{};
  for (int q = 0; q < p.parts; ++q) {
    const float* from = p.part + ((long)q * p.M + row) * width + n1;
    a += *reinterpret_cast<const f32x4_t*>(from);
    if (GATED) b += *reinterpret_cast<const f32x4_t*>(from + cols);
  }
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = GATED ? gate(a[r], b[r]) : a[r];
  mx::put4(p.y, p.type, row * p.N + n1, v, p.N - n1);
}

enum Form { kOnce, kNarrow, kWide };

template <Form FORM, int BM, int BN, int WM, int WN, int SLOTS, int OCC, int XBITS, bool GATED,
          bool GROUPED>
constexpr auto tile_kernel() {
  if constexpr (FORM == kWide)
    return mx_wide_kernel<BM, BN, WM, WN, SLOTS, OCC, XBITS, GATED, GROUPED>;
  else
    return mx_narrow_kernel<BM, BN, WM, WN, SLOTS, OCC, XBITS, FORM == kOnce, GATED, GROUPED>;
}

template <Form FORM, int BM, int BN, int WM, int WN, int SLOTS, int OCC, int XBITS>
void launch_tile(const MxProduct& p, bool gated, hipStream_t stream) {
  const int cols = gated ? BN / 2 : BN, n_tiles = (p.N + cols - 1) / cols;
  auto go = [&](auto kernel, long tiles) {
    const long blocks = (tiles * p.parts + 7) / 8 * 8;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(WM * WN * 64), 0, stream, p);
  };
  if (p.segs.off != nullptr) {
    const long tiles = moe::max_blocks(p.M, p.segs.experts, BM, n_tiles);
    if (gated) go(tile_kernel<FORM, BM, BN, WM, WN, SLOTS, OCC, XBITS, true, true>(), tiles);
    else go(tile_kernel<FORM, BM, BN, WM, WN, SLOTS, OCC, XBITS, false, true>(), tiles);
  } else {
    const long tiles = (long)((p.M + BM - 1) / BM) * n_tiles;
    if (gated) go(tile_kernel<FORM, BM, BN, WM, WN, SLOTS, OCC, XBITS, true, false>(), tiles);
    else go(tile_kernel<FORM, BM, BN, WM, WN, SLOTS, OCC, XBITS, false, false>(), tiles);
  }
}

template <int XBITS>
void launch_product(const MxProduct& p, const MxPlan& plan, bool once, bool gated, hipStream_t stream) {
  constexpr bool FOUR = XBITS == 4;
  switch (plan.bm * 1000 + plan.bn) {
    case 16128: return launch_tile<kOnce, 16, 128, 1, 4, 3, 2, XBITS>(p, gated, stream);
    case 32128: return launch_tile<kOnce, 32, 128, 1, 4, 3, 2, XBITS>(p, gated, stream);
    case 64128:
      if (once) return launch_tile<kOnce, 64, 128, 1, 4, 3, 2, XBITS>(p, gated, stream);
      return launch_tile<kNarrow, 64, 128, 1, 4, 3, 2, XBITS>(p, gated, stream);
    case 64224: return launch_tile<kOnce, 64, 224, 1, 7, 3, 2, XBITS>(p, gated, stream);
    case 64256: return launch_tile<kOnce, 64, 256, 1, 8, 3, 2, XBITS>(p, gated, stream);
    case 128128: return launch_tile<kWide, 128, 128, 2, 2, FOUR ? 4 : 3, 2, XBITS>(p, gated, stream);
    case 128256: return launch_tile<kWide, 128, 256, 2, 2, FOUR ? 5 : 4, 1, XBITS>(p, gated, stream);
    default: return launch_tile<kWide, 256, 256, 2, 2, FOUR ? 4 : 3, 1, XBITS>(p, gated, stream);
  }
}

}  // namespace

// What a product is made by.
MxPlan mx_plan(long rows, int N, int K, int experts, int x_bits, bool gated, bool x_aligned) {
  const long each = experts > 0 ? (rows + experts - 1) / experts : rows, groups = std::max(experts, 1);
  const int cols = gated ? 2 * N : N, depth = (K + mx::kTile - 1) / mx::kTile;
  if (each <= 64) {
    const int bm = each <= 16 ? 16 : each <= 32 ? 32 : 64;
    if ((x_aligned || bm > 16) && mx_few_fits(rows, bm, N, K, experts, x_bits, gated))
      return MxPlan{true, bm == 16, bm, 0, 1};
    // Tiles of 64 rows and 224 or 256 columns where they fill three quarters of the chip, the ones
    // that leave the busiest CU the fewest rows of W (us, 61 rows of 6 bits, 128 | 224 | 256 columns:
    // 57344 x 8192 58 | 46 | 48, 28672 x 8192 29 | 35 | 38); else K is cut until each CU has a
    // tile (8192 x 8192 in 2 | 4 | 8 parts 16 | 12 | 16, 28672 x 8192 in 1 | 2 29 | 34).
    MxPlan plan{false, false, bm, 128, 1};
    auto tiles_of = [&](int bn) { return (long)((cols + bn - 1) / bn) * groups; };
    if (bm == 64) {
      auto busiest = [&](int bn) { return (tiles_of(bn) + 255) / 256 * bn; };
      const int wide = busiest(224) < busiest(256) ? 224 : 256;
      if (tiles_of(wide) >= 192) plan.bn = wide;
    }
    while (plan.parts < 16 && tiles_of(plan.bn) * plan.parts * 2 <= 256 && depth >= plan.parts * 4)
      plan.parts *= 2;
    return plan;
  }
  // The least of what they take: rounds of the chip, each tiles of K at a time measured in a round
  // of many (of one: less) and what a tile takes beside, and the merge of parts.  us, 4 | 6 bits
  struct Form {
    int bm, bn, per_cu[2];
    float step[2], alone[2], tile;
  };
  static constexpr Form forms[] = {
      {64, 128, {2, 1}, {0.82f, 0.58f}, {0.47f, 0.55f}, 3.f},
      {128, 128, {2, 2}, {1.20f, 1.47f}, {0.58f, 0.70f}, 4.f},
      {128, 256, {1, 1}, {1.10f, 1.18f}, {0.88f, 0.92f}, 5.f},
      {256, 256, {1, 1}, {1.85f, 2.10f}, {1.30f, 1.50f}, 6.f},
  };
  MxPlan best{};
  float least = 1e30f;
  for (const Form& f : forms) {
    // (of an expert's last chunk half is taken to be there)
    const long chunks = experts > 0 ? rows / f.bm + (experts + 1) / 2 : (rows + f.bm - 1) / f.bm;
    const long tiles = chunks * ((cols + f.bn - 1) / f.bn);
    for (int parts = 1; parts <= 8 && (parts == 1 || parts * 2 <= depth); parts *= 2) {
      const int b = x_bits == 6;
      const long at_once = 256L * f.per_cu[b], blocks = tiles * parts, rounds = (blocks + at_once - 1) / at_once;
      const int steps = (depth + parts * 2 - 1) / (parts * 2) * 2;
      const float step = blocks <= at_once / 2 ? f.alone[b] : f.step[b];
      const float bytes = 4.f * parts * rows * cols;   // of parts, written and read
      const float time = rounds * (steps * step + f.tile) +
                         (parts > 1 ? 3.5f + bytes * (1 / 6e6f + 1 / 8e6f) : 0.f);
      if (time < least) {
        least = time;
        best = MxPlan{false, false, f.bm, f.bn, parts};
      }
    }
  }
  return best;
}

long mx_product_scratch(const MxPlan& plan, long rows, int N, bool gated) {
  return plan.parts > 1 ? plan.parts * rows * ((N + 3) / 4 * 4) * (gated ? 2 : 1) : 0;
}

void launch_mx_product(const MxPlan& plan, MxProduct p, int x_bits, bool gated, hipStream_t stream) {
  if (plan.few) {
    launch_mx_few(p, plan.bm, x_bits, gated, stream);
    return;
  }
  // parts are pairs of tiles, which have their scales together
  const int depth = p.pitch / mx::kTile;
  p.depth = (depth + plan.parts * 2 - 1) / (plan.parts * 2) * 2;
  p.parts = (depth + p.depth - 1) / p.depth;
  const bool once = p.segs.off == nullptr ? p.M <= plan.bm : p.M <= (long)plan.bm * p.segs.experts;
  if (x_bits == 4) launch_product<4>(p, plan, once, gated, stream);
  else launch_product<6>(p, plan, once, gated, stream);
  if (plan.parts > 1) {
    const long quads = (long)p.M * ((p.N + 3) / 4);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((quads + 255) / 256), dim3(256), 0, stream, p, (long)p.M);
    };
    if (gated) go(mx_merge_kernel<true>);
    else go(mx_merge_kernel<false>);
  }
}
