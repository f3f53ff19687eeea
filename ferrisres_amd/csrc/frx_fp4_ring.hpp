// frx_fp4_ring.hpp — the 4-bit product for many tokens, software-pipelined.
//
// A tile of BM tokens x BN weight rows on WM x WN waves of 16 FM x 16 FN, over NS stages of 256
// columns in LDS: rows of 128 bytes, filled with 16-byte LDS DMA whose pieces are XOR-swizzled
// by row as in the 8-bit engine, and 16 bytes of scales a row for two stages. Of a stage's 8
// blocks lane group g takes 2g in its first product and 2g + 1 in its second, so that both
// scales are one 16-bit read, the byte selected by the instruction. Columns past K are read
// past the buffer's end, which is a zero.
//
// A stage is two halves of FM x FN products. The first
// half's products run while the second half's operands are read, and the second half's while
// the next stage's first operands are: so a stage is free for the DMA of a later one when its
// second half begins, behind the stage's only barrier. Reads, DMA and products are fenced
// into small groups: left to itself the compiler issues a half's reads in one burst, which
// holds up every wave's products (8192^3 393 us against 325).
//
// Bound by what the L2s deliver, then by power (the products alone reach 6.6 PFLOP/s on
// random codes, 9.6 on zeros). So a row's scales arrive 16 bytes at a time, for two stages: 8
// bytes a stage ask the caches for as many lines as all codes do (without products and
// scales 8192^3 217 us, with them 272; in all 339 against 301). Measured and not kept:
// workgroups that begin at different columns, as rows of 2048 or 4096 bytes have the same
// column in the same channel of an L2 (8192 x 8448 x 8192 339 -> 317, but 2048 x 4096 x
// 11008 64.5 -> 71); wave tiles of 128 x 128 (8192^3 325 -> 348).
#pragma once
#include "frx_fp4.hpp"

namespace frx {

template <int WM, int WN, int FM_, int FN_, int NS_>
struct Fp4Ring {
  static constexpr int FM = FM_, FN = FN_, WAVES = WM * WN, NT = WAVES * 64;
  static constexpr int TM = FM * 16, TN = FN * 16, BM = WM * TM, BN = WN * TN;
  static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // 1 KB load instructions of a wave and stage
  static constexpr int SA = BM / 64, SB = BN / 64, SPW = (SA + SB + WAVES - 1) / WAVES;  // and of scales for two
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && BM % 64 == 0 && BN % 64 == 0, "whole instructions");
  static constexpr int DATA = (BM + BN) * 32, SCALES = (SA + SB) * 256;  // dwords of a stage; of two stages' scales
  static constexpr int NS = NS_;
  static constexpr int LDS_BYTES = (NS * DATA + 2 * SCALES) * 4;
  static_assert(LDS_BYTES <= 160 << 10, "stages");

  // Load instruction i of a wave covers 8 rows (64 of scales): a lane's offset in them (two, as
  // the swizzle of neighbouring groups of 8 rows differs; others for a step that K ends in) and,
  // in the scalar offset, the group's first row, clamped to the last group that has a valid
  // row. Rows past the valid ones are past the buffer's end.
  struct Ctx {
    __amdgpu_buffer_rsrc_t ra, rb, rsa, rsb;
    uint32_t av[2], bv[2], at[2], bt[2], sv;
    uint32_t lda8, ldb8, sld64, a_last, b_last, s_a_last, s_b_last;
    int wave, last;  // last: K's last step
    int t, t1;       // the step that is loaded next, and the item's end
  };
  struct Step {
    uint32_t *data, *scales;
    int t;
    uint32_t av[2], bv[2];
  };
  // The next step, g-th of all, into stage `stage`. A step past its item's last one is zeros.
  __device__ __forceinline__ static Step step(uint32_t *lds, const Ctx &c, int stage, int g) {
    Step s;
    s.data = lds + stage;
    s.scales = lds + NS * DATA + ((g >> 1) & 1) * SCALES;
    s.t = c.t;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s.av[h] = c.t >= c.t1 ? FP4_OUTSIDE : c.t < c.last ? c.av[h] : c.at[h];
      s.bv[h] = c.t >= c.t1 ? FP4_OUTSIDE : c.t < c.last ? c.bv[h] : c.bt[h];
    }
    return s;
  }
  static constexpr int CODES = LA + LB;
  __device__ __forceinline__ static void load(int i, const Ctx &c, const Step &s) {
    const uint32_t k0 = 128u * (uint32_t)s.t;
    if (i < LA) {
      lds_load16(c.ra, s.data + (c.wave * LA + i) * 256, s.av[i & 1], min((uint32_t)(c.wave * LA + i) * c.lda8, c.a_last) + k0);
    } else {
      const int j = i - LA;
      lds_load16(c.rb, s.data + BM * 32 + (c.wave * LB + j) * 256, s.bv[j & 1],
                 min((uint32_t)(c.wave * LB + j) * c.ldb8, c.b_last) + k0);
    }
  }
  // The scales of an even step and the one behind it.
  __device__ __forceinline__ static void load_scales(const Ctx &c, const Step &s) {
#pragma unroll
    for (int i = 0; i < SPW; i++) {
      const int j = min(c.wave * SPW + i, SA + SB - 1);  // (the last one by several waves)
      const uint32_t k0 = 8u * (uint32_t)s.t;
      if (j < SA) lds_load16(c.rsa, s.scales + j * 256, c.sv, min((uint32_t)j * c.sld64, c.s_a_last) + k0);
      else lds_load16(c.rsb, s.scales + j * 256, c.sv, min((uint32_t)(j - SA) * c.sld64, c.s_b_last) + k0);
    }
  }

  // Waits for this wave's LDS reads and for all but its last N loads.
  template <int N>
  __device__ __forceinline__ static void wait_all_but() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4));
  }

  // The workgroup's items (tiles, or slices of K of tiles) one after the other, through one ring:
  // the next item's first steps are on their way while one's last are multiplied and its
  // sums stored. items.at(i, o): operands of the i-th, false behind the last; items.take(i, t0,
  // t1): the steps of the i-th, whose sums items.store(acc) takes; items.span: steps of an item,
  // even, as the scales come in pairs (an item's last step may be zeros). !MANY: one item.
  template <bool MANY, typename Items>
  __device__ static void run(uint32_t *lds, Items &items) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    Fp4Operands o;
    int item = 0, loading = 0;
    if (!items.at(0, o)) return;
    Ctx c;
    c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c.last = (o.K + 255) / 256 - 1;
    const int wm = c.wave % WM, wn = c.wave / WM, left = o.K - 256 * c.last;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int pa = (lane & 7) ^ xswz(((c.wave * LA + h) & 1) * 8 + (lane >> 3));
      const int pb = (lane & 7) ^ xswz(((c.wave * LB + h) & 1) * 8 + (lane >> 3));
      c.av[h] = (uint32_t)(lane >> 3) * o.lda + 16 * pa;
      c.bv[h] = (uint32_t)(lane >> 3) * o.ldb + 16 * pb;
      c.at[h] = 32 * pa < left ? c.av[h] : FP4_OUTSIDE;
      c.bt[h] = 32 * pb < left ? c.bv[h] : FP4_OUTSIDE;
    }
    c.sv = (uint32_t)lane * o.s_ld;
    c.lda8 = 8 * o.lda;
    c.ldb8 = 8 * o.ldb;
    c.sld64 = 64 * o.s_ld;
    const auto begin = [&](const Fp4Operands &q) {
      c.a_last = (uint32_t)((q.a_rows - 1) >> 3) * c.lda8;
      c.b_last = (uint32_t)((q.b_rows - 1) >> 3) * c.ldb8;
      c.s_a_last = (uint32_t)((q.a_rows - 1) >> 6) * c.sld64;
      c.s_b_last = (uint32_t)((q.b_rows - 1) >> 6) * c.sld64;
      c.ra = buffer_rsrc(q.a, (uint32_t)(q.a_rows - 1) * q.lda + (uint32_t)q.K / 2);
      c.rb = buffer_rsrc(q.b, (uint32_t)(q.b_rows - 1) * q.ldb + (uint32_t)q.K / 2);
      c.rsa = buffer_rsrc(q.sa, (uint32_t)(q.a_rows - 1) * q.s_ld + fp4_scale_bytes((uint32_t)q.K));
      c.rsb = buffer_rsrc(q.sb, (uint32_t)(q.b_rows - 1) * q.s_ld + fp4_scale_bytes((uint32_t)q.K));
      c.t = q.t0;
      c.t1 = q.t1;
    };
    begin(o);
    const int span = items.span;
    int to_load = span;
    const auto loaded = [&]() {  // one more step is
      c.t++;
      if (MANY && --to_load == 0) {
        to_load = span;
        Fp4Operands q;
        if (items.at(++loading, q)) begin(q);
        else c.t = c.t1 = 0;  // zeros, and scales that do not matter
      }
    };
    f32x4 acc[FN][FM];
#pragma unroll
    for (int fn = 0; fn < FN; fn++)
#pragma unroll
      for (int fm = 0; fm < FM; fm++) acc[fn][fm] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const int xo = (wm * TM + l16) * 32, wo = (BM + wn * TN + l16) * 32;  // dwords of a stage
    const int p0 = ((2 * g) ^ xswz(l16)) * 4, p1 = ((2 * g + 1) ^ xswz(l16)) * 4;
    const int so = (wm * TM + l16) * 8 + g, bo = (BM + wn * TN + l16) * 8 + g;  // 16-bit words of the scales
    const auto op = [](const uint32_t *st, int at) { return *reinterpret_cast<const u32x4 *>(st + at); };
    const auto scale = [](const uint32_t *sc, int t, int at) {
      return (uint32_t)reinterpret_cast<const uint16_t *>(sc)[at + (t & 1) * 4];
    };
    const uint32_t keep = (64 * g < left ? 0xFFu : 0) | (64 * g + 32 < left ? 0xFF00u : 0);

    // (steps behind the last item are loaded as well: the waits go by the number of loads)
#pragma unroll
    for (int i = 0; i < NS; i++) {
      const Step s = step(lds, c, i * DATA, i);
      if (i % 2 == 0) load_scales(c, s);
#pragma unroll
      for (int j = 0; j < CODES; j++) load(j, c, s);
      loaded();
    }
    wait_vmcnt<(NS - 1) * CODES + (NS == 3 ? SPW : 0)>();
    barrier_nofence();
    u32x4 w[2][FN], x[2][FM];
    uint32_t sw[FN], sx[FM], swn[FN], sxn[FM];
    {
      const uint32_t *sc = lds + NS * DATA;
#pragma unroll
      for (int f = 0; f < FN; f++) {
        w[0][f] = op(lds, wo + f * 512 + p0);
        sw[f] = scale(sc, 0, bo + f * 128);
      }
#pragma unroll
      for (int f = 0; f < FM; f++) {
        x[0][f] = op(lds, xo + f * 512 + p0);
        sx[f] = scale(sc, 0, so + f * 128);
      }
    }
    int here = 0, t, t1, to_do = span;
    items.take(0, t, t1);
    for (int n = 0;; n++) {
      uint32_t *cur = lds + here;
      const int stage = here;
      here = here == (NS - 1) * DATA ? 0 : here + DATA;
      uint32_t *nxt = lds + here;
      if (t >= c.last || t >= t1) {  // scales past a row's blocks, whatever they are: none that is a NaN
        const uint32_t mask = t >= t1 ? 0 : keep;
#pragma unroll
        for (int f = 0; f < FN; f++) sw[f] &= mask;
#pragma unroll
        for (int f = 0; f < FM; f++) sx[f] &= mask;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int fm = 0; fm < FM; fm++) {
        x[1][fm] = op(cur, xo + fm * 512 + p1);
#pragma unroll
        for (int f = fm * FN / FM; f < (fm + 1) * FN / FM; f++) w[1][f] = op(cur, wo + f * 512 + p1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int fn = 0; fn < FN; fn++) fp4_mul<0>(acc[fn][fm], w[0][fn], sw[fn], x[0][fm], sx[fm]);
        __builtin_amdgcn_sched_barrier(0);
      }
      // every wave is done with this stage, the next one has landed; in flight behind it NS - 2 steps
      // (and an item's stores: waited for with the loads before them)
      const bool even = ((n + NS) & 1) == 0;  // the step that is loaded now
      if (NS == 2) wait_all_but<0>();
      else if (even) wait_all_but<(NS - 2) * CODES>();  // (the step before, an odd one)
      else wait_all_but<(NS - 2) * CODES + SPW>();
      barrier_nofence();
      __builtin_amdgcn_sched_barrier(0);
      const Step s = step(lds, c, stage, n + NS);
      const uint32_t *sc = lds + NS * DATA + (((n + 1) >> 1) & 1) * SCALES;
      if (even) load_scales(c, s);
#pragma unroll
      for (int fm = 0; fm < FM; fm++) {
        x[0][fm] = op(nxt, xo + fm * 512 + p0);
        sxn[fm] = scale(sc, n + 1, so + fm * 128);
#pragma unroll
        for (int f = fm * FN / FM; f < (fm + 1) * FN / FM; f++) {
          w[0][f] = op(nxt, wo + f * 512 + p0);
          swn[f] = scale(sc, n + 1, bo + f * 128);
        }
#pragma unroll
        for (int j = fm * CODES / FM; j < (fm + 1) * CODES / FM; j++) load(j, c, s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int fn = 0; fn < FN; fn++) fp4_mul<1>(acc[fn][fm], w[1][fn], sw[fn], x[1][fm], sx[fm]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int f = 0; f < FN; f++) sw[f] = swn[f];
#pragma unroll
      for (int f = 0; f < FM; f++) sx[f] = sxn[f];
      loaded();
      t++;
      if (MANY ? --to_do == 0 : t >= t1) {
        items.store(acc);
        if (!MANY || !items.take(++item, t, t1)) break;
        to_do = span;
#pragma unroll
        for (int fn = 0; fn < FN; fn++)
#pragma unroll
          for (int fm = 0; fm < FM; fm++) acc[fn][fm] = (f32x4){0.f, 0.f, 0.f, 0.f};
      }
    }
    wait_vmcnt<0>();  // nothing is in flight into LDS any more
  }

  // A piece is 16 bytes of a row a lane: 16 columns of f32 or 32 of bf16 over the 4 lane groups, so that a
  // store writes 16 rows of 64 bytes (bf16 as it comes off the accumulators, 32: gradients of 16 x 128
  // rows, 5632 x 2048, 148 -> 122 us, 8192 x 2048 x 8192 135 -> 113, 2048 x 4096 x 11008 73 -> 70). Of two pieces of
  // f32 lanes 8 apart exchange one each: 8 rows of 128 bytes (8192 x 2048 x 8192 161 -> 128, 11008 x
  // 2016 x 4096 94 -> 90; of bf16 122 -> 131, 113 -> 111).
  template <typename YT>
  __device__ __forceinline__ static void store(const f32x4 (&acc)[FN][FM], YT *y, size_t ldy, int m_rows, int n_rows) {
    constexpr int W = 16 / sizeof(YT), NP = FN * 4 / W;  // values of a lane; whole pieces
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int EXCHANGED = sizeof(YT) == 4 ? NP & ~1 : 0;
    const int l16 = lane & 15, g = lane >> 4, hi = l16 >> 3;
    const int m0 = (wave % WM) * TM, n0 = (wave / WM) * TN;
    const auto piece = [&](int j, int fm) {
      if constexpr (sizeof(YT) == 4) return __builtin_bit_cast(u32x4, acc[j][fm]);
      else return fp4_join8(acc[2 * j][fm], acc[2 * j + 1][fm]);
    };
    const auto put = [&](const u32x4 &v, int m, int n) {
      if (m >= m_rows || n >= n_rows) return;
      YT *d = y + (size_t)m * ldy + n;
      if (n + W <= n_rows) {
        *reinterpret_cast<u32x4_u *>(d) = v;
      } else {
#pragma unroll
        for (int e = 0; e < W; e++)
          if (n + e < n_rows) {
            if constexpr (sizeof(YT) == 4) d[e] = __uint_as_float(v[e]);
            else d[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
          }
      }
    };
#pragma unroll
    for (int fm = 0; fm < FM; fm++) {
      const int m = m0 + fm * 16;
#pragma unroll
      for (int j = 0; j < EXCHANGED; j += 2) {
        const u32x4 p = piece(j, fm), q = piece(j + 1, fm);
        u32x4 lo, up;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(hi ? p[i] : q[i]), 0x128, 0xF, 0xF, true);
          lo[i] = hi ? other : p[i];
          up[i] = hi ? q[i] : other;
        }
        const int n = n0 + (j + hi) * 4 * W + W * g;
        put(lo, m + (l16 & 7), n);
        put(up, m + 8 + (l16 & 7), n);
      }
#pragma unroll
      for (int j = EXCHANGED; j < NP; j++) put(piece(j, fm), m + l16, n0 + j * 4 * W + W * g);
      if constexpr (sizeof(YT) == 2 && (FN & 1)) {
        const int n = n0 + (FN - 1) * 16 + 4 * g;
        if (m + l16 < m_rows && n < n_rows)
          fp4_store4(y + (size_t)(m + l16) * ldy + n, acc[FN - 1][fm], (uint32_t)(n_rows - n));
      }
    }
  }
};

}  // namespace frx
