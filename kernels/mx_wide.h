// The main loop of large products of microscaled rows (mx_gemm.hip): BM x BN tiles by four
// waves, one a SIMD, of up to 128 x 128 each, whose sums fill all accumulation registers.
//
// A tile of 256 inputs is 128 bytes a row, whole cache lines, and what counts is to have
// enough of them on their way without a pause of the matrix unit:
//  - Memory comes in slots of half of the rows of x and of W, SLOTS of them in LDS, each
//    asked for SLOTS - 1 half tiles ahead.  A half tile is half of the rows of x times all of
//    W, one half after the other; W's halves take turns in order from tile to tile (x0 w0,
//    x1 w1 | x0 w1, x1 w0), so that each quarter of the products reads one half of an operand
//    into the registers of one that is done with.
//  - Scales come two tiles' at a time, 16 bytes a row and lane, a round of two tiles ahead (8 bytes
//    of a tile, two lanes a row, held up the codes: 128 x 128 tiles took 351 us instead of 278 for the
//    product below, 256 x 256 ones 171 instead of 155 of zeros).
//  - One barrier a half tile.  Reads and loads stand between the products in source order.
// The accumulation registers are named in the products themselves (multiply0 below).
//
// 8192 rows, 14336 to 4096: 205 us of 4 bits, 4.7 PFLOP/s, and 237 of 6; whole tiles in two slots
// by eight waves 290.  Bound by stalls first: the matrix unit is busy for 57 % of the cycles (6
// bits 50 %), with zeros, which the clock does not fall so for, 55 % (177 us); from registers it
// is for 93 %.  The chip's power is behind the rest: the clock is 1.87 GHz with values and 2.26
// with zeros (from registers 1.89, 7.3 PFLOP/s, and 2.39, 9.6).  In a program of its own, all of
// zeros, the loop took 155 us, without loads 134, without reads of LDS or barriers no less.
// Products of 32 x 32 are no faster with zeros and slower with values (6.5 PFLOP/s).
#pragma once

#include <type_traits>

#include "block_gemm.h"
#include "mx_round.h"

namespace mx {

using block_gemm::f32x4_t;

// What a workgroup multiplies: the first of its rows' codes and scales, and how many tiles
// of 256 inputs, from tile `first` on: an even number, from an even one.
struct Operands {
  const unsigned char *x0, *x1, *xs, *w, *ws;
  int pitch;     // of x and of scales: inputs of a row, whole pairs of tiles
  int k_bytes;   // of a row of W
  int first, tiles;
  int turn;      // the tile (even) that a loop which may begin anywhere begins with
};

// One of two places (of values: of an operand's fields the compiler would choose by address, which
// puts the operands into memory)
DEVINLINE const unsigned char* either(bool first, const unsigned char* a, const unsigned char* b) {
  return first ? a : b;
}

template <int BM_, int BN_, int WM, int WN, int SLOTS, int XBITS>
struct Wide {
  static constexpr int BM = BM_, BN = BN_, kWN = WN;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  static constexpr int kTM = BM / WM / 16, kTN = BN / WN / 16;   // 16 x 16 tiles of a wave
  static constexpr int kHM = kTM / 2, kHN = kTN / 2;             // of half of its rows
  static constexpr int kX0 = BM / 2 * 128, kX1 = XBITS == 6 ? BM / 2 * 64 : 0;
  static constexpr int kAtW = kX0 + kX1, kSlot = kAtW + BN / 2 * 128;
  // scales of two tiles, 16 bytes a row, in two places; and a place that nobody reads
  static constexpr int kAtScales = SLOTS * kSlot, kPair = (BM + BN) * 16;
  static constexpr int kSpare = kAtScales + 2 * kPair;
  static constexpr int each(int loads) { return (loads + kWaves - 1) / kWaves; }
  static constexpr int kX0Loads = BM / 16, kX1Loads = kX1 / 1024, kWLoads = BN / 16;
  static constexpr int kX0Each = each(kX0Loads), kX1Each = each(kX1Loads), kWEach = each(kWLoads);
  static constexpr int kLoads = kX0Each + kX1Each + kWEach;   // a wave's
  static constexpr int kScaleLoads = (BM + BN) / 64, kScaleEach = each(kScaleLoads);
  static constexpr int kLds = kSpare + (kScaleLoads % kWaves ? 1024 : 0);
  static_assert(kTM % 2 == 0 && kTN % 2 == 0, "halves");
  static_assert(kX0Loads % kWaves == 0 && kX1Loads % kWaves == 0 && kWLoads % kWaves == 0 &&
                    BM % 64 == 0 && BN % 64 == 0, "a load a wave");
  static_assert(kLds <= 160 * 1024 && (SLOTS - 1) * kLoads + kScaleEach < 64 && SLOTS <= 5,
                "LDS of a CU, vmcnt, the scales' turn");

  using X = typename std::conditional<XBITS == 6, i32x6_t, i32x4_t>::type;

  // A sum stays in its accumulation registers: all 256 are in use, and the compiler's own
  // choice copies some of them in every turn.  Written out, a product is no matrix instruction
  // to the compiler, which adds no wait states: a form is sound only if between the products
  // sums are neither copied nor spilled and fragments and scales come from LDS alone, and if
  // `settle` is the first to follow the last product.  tests/test_mx_products.py looks for that
  // in the built code.  0, 1: which of a row's two blocks, and which byte of its scales.
  static DEVINLINE void multiply0(f32x4_t& acc, const i32x4_t& w, const X& x, int ws, int xs) {
    if constexpr (XBITS == 6)
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[0,0,0] "
                   "op_sel_hi:[0,0,0] cbsz:4 blgp:2" : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
    else
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[0,0,0] "
                   "op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
  }
  static DEVINLINE void multiply1(f32x4_t& acc, const i32x4_t& w, const X& x, int ws, int xs) {
    if constexpr (XBITS == 6)
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] "
                   "op_sel_hi:[0,0,0] cbsz:4 blgp:2" : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
    else
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] "
                   "op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
  }
  // 18 wait states at most lie between a product and what reads its sum without the matrix
  // unit.  They are taken in the loop, behind the last product of the last turn: on the way out
  // of it the compiler copies sums.  One block, since a branch of its own would be moved there too.
  static DEVINLINE void settle(int turn, int turns) {
    asm volatile("s_cmp_lt_i32 %0, %1\n\ts_cbranch_scc1 1f\n\ts_nop 15\n\ts_nop 7\n1:"
                 ::"s"(turn), "s"(turns) : "scc");
    __builtin_amdgcn_sched_barrier(0);
  }
  // (the compiler would spill some of 256 that it takes to be wanted elsewhere)
  static DEVINLINE void keep(f32x4_t (&acc)[kTM][kTN]) {
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j = 0; j < kTN; ++j) asm volatile("" : "+a"(acc[i][j]));
  }

  // acc[i][j][r]: row i * 16 + lane % 16 of the wave's of x, row j * 16 + lane / 16 * 4 + r of
  // W.  x_row, w_row: where a row of the tile lies, in rows from the operands' first.
  template <typename XRow, typename WRow>
  static DEVINLINE void run(f32x4_t (&acc)[kTM][kTN], char* lds, const Operands& p, XRow x_row,
                            WRow w_row) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    auto load_of = [&](int i) { return i * kWaves + wave; };
    // a slot's rows are half of every wave's
    auto x_of = [&](int r, int h) {
      return x_row(r / (kHM * 16) * (kTM * 16) + h * (kHM * 16) + r % (kHM * 16));
    };
    auto w_of = [&](int r, int h) {
      return w_row(r / (kHN * 16) * (kTN * 16) + h * (kHN * 16) + r % (kHN * 16));
    };
    unsigned x_off[2][kX0Each], x1_off[2][kX1Each + 1], w_off[2][kWEach], s_off[kScaleEach];
    int w_chunk[kWEach];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < kX0Each; ++i) {
        const int r = load_of(i) * 8 + lane / 8;
        x_off[h][i] =
            x_of(r, h) * (unsigned)(p.pitch / 2) + block_at((lane % 8) ^ (r / 2 % 8)) * 16;
      }
#pragma unroll
      for (int i = 0; i < kX1Each; ++i) {
        const int r = load_of(i) * 16 + lane / 4;
        x1_off[h][i] = x_of(r, h) * (unsigned)(p.pitch / 4) + ((lane % 4) ^ (r / 4 % 4)) * 16;
      }
#pragma unroll
      for (int i = 0; i < kWEach; ++i) {
        const int r = load_of(i) * 8 + lane / 8;
        w_off[h][i] = w_of(r, h) * (unsigned)p.k_bytes;
        w_chunk[i] = block_at((lane % 8) ^ (r / 2 % 8)) * 16;
      }
    }
#pragma unroll
    for (int i = 0; i < kScaleEach; ++i) {
      const int r = load_of(i) * 64 + lane;
      s_off[i] = (r < BM ? x_row(r) : w_row(min(r - BM, BN - 1))) * (unsigned)(p.pitch / 32);
    }
    // Past the last tile: loads of nothing, so that the counts stay what they are.  W's rows
    // end with K, its last tiles perhaps inside or past it: lanes past the end load the row's
    // last piece, which meets zeros of x and of the scales (both have rows of whole pairs).
    const int n = p.tiles;
    auto size = [&](int tile) {
      return (unsigned)__builtin_amdgcn_readfirstlane(tile < n ? -1 : 0);
    };
    // load q of half hx of x and hw of W of a tile
    auto load = [&](int q, char* slot, int hx, int hw, int tile, unsigned bytes) {
      const int t = p.first + tile;
      if (q < kX0Each) {
        block_gemm::load_lds(slot + load_of(q) * 1024, block_gemm::resource(p.x0, bytes),
                             x_off[hx][q < kX0Each ? q : 0], t * 128);
        return;
      }
      q -= kX0Each;
      if (q < kWEach) {
        const int i = q < kWEach ? q : 0;
        block_gemm::load_lds(slot + kAtW + load_of(i) * 1024,
                             block_gemm::resource(p.w, bytes),
                             w_off[hw][i] + min(t * 128 + w_chunk[i], p.k_bytes - 16), 0);
        return;
      }
      q -= kWEach;
      block_gemm::load_lds(slot + kX0 + load_of(q) * 1024, block_gemm::resource(p.x1, bytes),
                           x1_off[hx][q < kX1Each ? q : 0], t * 64);
    };
    // load q of the scales of a tile and the next one
    auto load_scales = [&](int q, char* to, int tile, unsigned bytes) {
      const int l = load_of(q);
      const bool one = kScaleLoads % kWaves == 0 || l < kScaleLoads;
      block_gemm::load_lds(one ? to + l * 1024 : lds + kSpare,
                           block_gemm::resource(either(l < BM / 64, p.xs, p.ws), one ? bytes : 0), s_off[q],
                           (p.first + tile) * 8);
    };
    const int sw = col / 2 % 8, c0 = (quad ^ sw) * 16, c1 = ((4 + quad) ^ sw) * 16;
    const int x_at = (wm * kHM * 16 + col) * 128, w_at = kAtW + (wn * kHN * 16 + col) * 128;
    const int x1_at = kX0 + (wm * kHM * 16 + col) * 64 + quad % 2 * 8;
    const int d0 = (quad / 2 ^ (col / 4)) * 16, d1 = ((2 + quad / 2) ^ (col / 4)) * 16;
    const int xs_at = (wm * kTM * 16 + col) * 16 + quad * 2;
    const int ws_at = (BM + wn * kTN * 16 + col) * 16 + quad * 2;
    // a half's fragments and scales; read q of kReadsX or kReadsW
    struct HalfX { X f[2 * kHM]; int s[kHM]; };
    struct HalfW { i32x4_t f[2 * kHN]; int s[kHN]; };
    constexpr int kReadsX = 3 * kHM, kReadsW = 3 * kHN;
    // (scales: of which tile of two and which half)
    auto read_x = [&](HalfX& to, const char* slot, const char* scales, int tile, int h, int q) {
      if (q < kHM) {
        to.s[q] = *reinterpret_cast<const unsigned short*>(scales + xs_at + tile * 8 +
                                                           (h * kHM + q) * 256);
        return;
      }
      q -= kHM;
      const int i = q % kHM, ks = q / kHM;
      const i32x4_t v = *reinterpret_cast<const i32x4_t*>(slot + x_at + (ks ? c1 : c0) + i * 2048);
      if constexpr (XBITS == 6) {
        const i32x2_t u = *reinterpret_cast<const i32x2_t*>(slot + x1_at + (ks ? d1 : d0) + i * 1024);
        to.f[q] = __builtin_shufflevector(v, __builtin_shufflevector(u, u, 0, 1, -1, -1), 0, 1, 2, 3,
                                          4, 5);
      } else {
        to.f[q] = v;
      }
    };
    auto read_w = [&](HalfW& to, const char* slot, const char* scales, int tile, int h, int q) {
      if (q < kHN)
        to.s[q] = *reinterpret_cast<const unsigned short*>(scales + ws_at + tile * 8 +
                                                           (h * kHN + q) * 256);
      else
        to.f[q - kHN] = *reinterpret_cast<const i32x4_t*>(
            slot + w_at + ((q - kHN) / kHN ? c1 : c0) + (q - kHN) % kHN * 2048);
    };

    // The order of the halves, two tiles in a round: x0 w0, x1 w1 | x0 w1, x1 w0.  Their scales
    // come a round ahead, the second round's here behind the slots as later ones' come behind a
    // round's.
    char* scales = lds + kAtScales;
    char* scales_next = scales + kPair;
#pragma unroll
    for (int q = 0; q < kScaleEach; ++q) load_scales(q, scales, 0, size(0));
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
      for (int q = 0; q < kLoads; ++q)
        load(q, lds + s * kSlot, s % 2, (s + 1) / 2 % 2, s / 2, size(s / 2));
#pragma unroll
    for (int q = 0; q < kScaleEach; ++q) load_scales(q, scales_next, 2, size(2));
    block_gemm::wait_loads<(SLOTS - 1) * kLoads + kScaleEach>();
    block_gemm::meet();
    HalfX fx0, fx1;
    HalfW fw0, fw1;
#pragma unroll
    for (int q = 0; q < kReadsX; ++q) read_x(fx0, lds, scales, 0, 0, q);
#pragma unroll
    for (int q = 0; q < kReadsW; ++q) read_w(fw0, lds, scales, 0, 0, q);
    // (told apart from 16 bits: the compiler would carry those round the loop and widen them
    // again right ahead of the products)
#pragma unroll
    for (int i = 0; i < kHM; ++i) asm volatile("" : "+v"(fx0.s[i]));
#pragma unroll
    for (int j = 0; j < kHN; ++j) asm volatile("" : "+v"(fw0.s[j]));

    int at = 0, next = 1;    // places of the slot that has been read and of the next one
    // A quarter of a tile's products, the reads of a half and half of the loads in between
    auto quarter = [&](int i0, int j0, HalfX& fx, HalfW& fw, int reads, auto read, int first,
                       int last, auto ask) {
      constexpr int kProducts = 2 * kHM * kHN;
#pragma unroll
      for (int q = 0; q < kProducts; ++q) {
        const int ks = q / (kHM * kHN), i = q / kHN % kHM, jj = q % kHN;
        const int j = i % 2 ? kHN - 1 - jj : jj;
#pragma unroll
        for (int r = 0; r < reads; ++r)   // in the first half of the products, if they fit
          if (r * (2 * reads > kProducts ? kProducts : kProducts / 2) / reads == q) read(r);
        const int each = kProducts / (last - first);
#pragma unroll
        for (int l = first; l < last; ++l)
          if (min((l - first) * kProducts / (last - first) + each / 2 + 1, kProducts - 1) == q)
            ask(l);
        if (ks == 0) multiply0(acc[i0 + i][j0 + j], fw.f[j], fx.f[i], fw.s[j], fx.s[i]);
        else multiply1(acc[i0 + i][j0 + j], fw.f[kHN + j], fx.f[kHM + i], fw.s[j], fx.s[i]);
        if (q % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
    };
    // what begins a half of a tile, H of a round's four: the slot before has been read by all, the
    // next is there.  Behind it SLOTS - 2 slots were asked for, with scales at the end of a round.
    auto begin = [&](auto half) {
      constexpr int H = decltype(half)::value;
      block_gemm::wait_loads_and_reads<(SLOTS - 2) * kLoads + (H < SLOTS - 2 ? kScaleEach : 0)>();
      block_gemm::meet();
    };
    auto advance = [&] {
      at = next;
      if (++next == SLOTS) next = 0;
    };
    for (int t = 0; t < n; t += 2) {
      {
        // even tile: x0 w0, x0 w1 (reading w1, x1), x1 w1, x1 w0 (reading x0', w1')
        begin(std::integral_constant<int, 0>{});
        char* here = lds + at * kSlot;
        const char* there = lds + next * kSlot;
        const int tile = t + SLOTS / 2;
        const unsigned bytes = size(tile);
        auto ask0 = [&](int p) { load(p, here, SLOTS % 2, (SLOTS + 1) / 2 % 2, tile, bytes); };
        quarter(0, 0, fx0, fw0, kReadsW, [&](int q) { read_w(fw1, there, scales, 0, 1, q); }, 0,
                kLoads / 2, ask0);
        quarter(0, kHN, fx0, fw1, kReadsX, [&](int q) { read_x(fx1, there, scales, 0, 1, q); },
                kLoads / 2, kLoads, ask0);
        advance();
        begin(std::integral_constant<int, 1>{});
        char* here1 = lds + at * kSlot;
        const char* there1 = lds + next * kSlot;
        const int tile1 = t + (SLOTS + 1) / 2;
        const unsigned bytes1 = size(tile1);
        auto ask1 = [&](int p) {
          load(p, here1, (SLOTS + 1) % 2, (SLOTS + 2) / 2 % 2, tile1, bytes1);
        };
        quarter(kHM, kHN, fx1, fw1, kReadsX, [&](int q) { read_x(fx0, there1, scales, 1, 0, q); },
                0, kLoads / 2, ask1);
        quarter(kHM, 0, fx1, fw0, kReadsW, [&](int q) { read_w(fw1, there1, scales, 1, 1, q); },
                kLoads / 2, kLoads, ask1);
        advance();
      }
      {
        // odd tile: x0 w1, x0 w0 (reading w0, x1), x1 w0, x1 w1 (reading x0', w0')
        begin(std::integral_constant<int, 2>{});
        char* here = lds + at * kSlot;
        const char* there = lds + next * kSlot;
        const int tile = t + 1 + SLOTS / 2;
        const unsigned bytes = size(tile);
        auto ask0 = [&](int p) { load(p, here, SLOTS % 2, (SLOTS + 3) / 2 % 2, tile, bytes); };
        quarter(0, kHN, fx0, fw1, kReadsW, [&](int q) { read_w(fw0, there, scales, 1, 0, q); }, 0,
                kLoads / 2, ask0);
        quarter(0, 0, fx0, fw0, kReadsX, [&](int q) { read_x(fx1, there, scales, 1, 1, q); },
                kLoads / 2, kLoads, ask0);
        advance();
        begin(std::integral_constant<int, 3>{});
        char* here1 = lds + at * kSlot;
        const char* there1 = lds + next * kSlot;
        const int tile1 = t + 1 + (SLOTS + 1) / 2;
        const unsigned bytes1 = size(tile1);
        const unsigned bytes2 = size(t + 4);
        auto ask1 = [&](int p) {
          if (p < kLoads) load(p, here1, (SLOTS + 1) % 2, (SLOTS + 4) / 2 % 2, tile1, bytes1);
          else load_scales(p - kLoads, scales, t + 4, bytes2);   // (nobody reads these any more)
        };
        quarter(kHM, 0, fx1, fw0, kReadsX, [&](int q) { read_x(fx0, there1, scales_next, 0, 0, q); },
                0, (kLoads + kScaleEach) / 2, ask1);
        quarter(kHM, kHN, fx1, fw1, kReadsW,
                [&](int q) { read_w(fw0, there1, scales_next, 0, 0, q); },
                (kLoads + kScaleEach) / 2, kLoads + kScaleEach, ask1);
        char* const read = scales;
        scales = scales_next;
        scales_next = read;
        __builtin_amdgcn_sched_barrier(0);
        settle(t + 2, n);
        advance();
      }
    }
    block_gemm::wait_loads<0>();
    keep(acc);
  }
};

}  // namespace mx
