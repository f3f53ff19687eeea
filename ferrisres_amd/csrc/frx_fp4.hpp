// frx_fp4.hpp — MFMA tile engine of the 4-bit floating-point linears.
//
// y[m][n] = sum over blocks b of 32 columns of 2^(sa[m][b] + sb[n][b] - 254) sum_{k in b} a b.
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands as codes and both scales, and adds
// to the fp32 accumulator. Products of two codes are multiples of 1/4 up to 36, so a
// block's sum is exact, and blocks are added in fp32 one after the other (measured with
// planted operands: beside a 1 a block of 2^-23 is kept, and a half of the last bit rounds to
// even, as does an addition of its own): nothing is cut as with 8-bit operands. A scale of
// 255 makes a NaN of every product, of zeros too; scales that add up to less than any f32
// number's exponent are right as well.
//
// A lane (row l16, group g) gives 32 codes of one row and one scale byte, so a lane's codes
// are one block. A stage in LDS holds 256 columns: rows of 128 bytes, filled with 16-byte
// LDS DMA whose pieces are XOR-swizzled by row as in the 8-bit engine, and 8 bytes of scales
// a row. Of the stage's 8 blocks group g takes 2g in its first product and 2g + 1 in its
// second, so that both scales are one 16-bit read, the byte selected by the instruction.
// Columns past K are read past the buffer's end, which is a zero.
#pragma once
#include "frx_fp4_codes.hpp"
#include "frx_fp8.hpp"

namespace frx {

// The operands of one output tile: first rows of both sides and of their scales.
struct Fp4Operands {
  const uint8_t *a, *b, *sa, *sb;
  uint32_t lda, ldb, s_ld;  // bytes between rows
  int a_rows, b_rows;       // valid rows in the tile
  int K;
  int t0, t1;               // steps of 256 columns
};

constexpr uint32_t FP4_OUTSIDE = 0x60000000u;  // past every buffer: 256 rows of at most 2^22 bytes

// acc += w x over 128 columns: byte S of the scales.
template <int S>
__device__ __forceinline__ void fp4_mul(f32x4 &acc, const u32x4 &w, uint32_t sw, const u32x4 &x, uint32_t sx) {
  const i32x8 a = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const i32x8 b = {(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, S, (int)sw, S, (int)sx);
}

// BM tokens x BN weight rows, WM x WN waves.
template <int BM_, int BN_, int WM, int WN>
struct Fp4Tile {
  static constexpr int BM = BM_, BN = BN_;
  static constexpr int WAVES = WM * WN, NT = WAVES * 64;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // 1 KB load instructions per wave
  static constexpr int SA = BM / 32, SB = BN / 32;                // 256-byte scale instructions
  static constexpr int SPW = (SA + SB + WAVES - 1) / WAVES;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && BM % 32 == 0 && BN % 32 == 0, "whole instructions");
  static constexpr int DATA = (BM + BN) * 32;  // dwords
  static constexpr int STAGE = DATA + SPW * WAVES * 64;
  static constexpr int LDS_BYTES = 2 * STAGE * 4;

  struct Ctx {
    __amdgpu_buffer_rsrc_t ra, rb, rsa, rsb;
    uint32_t a[LA], b[LB], s[SPW];  // a lane's offsets in the first step
    int pa[LA], pb[LB];             // and its pieces of 32 columns in a step
    int wave, lane, K;
  };

  __device__ __forceinline__ static void issue(uint32_t *stage, const Ctx &c, int t) {
    const uint32_t k0 = 128u * (uint32_t)t;
    const int left = c.K - 256 * t;  // columns from here on
#pragma unroll
    for (int i = 0; i < LA; i++)
      lds_load16(c.ra, stage + (c.wave * LA + i) * 256, 32 * c.pa[i] < left ? c.a[i] : FP4_OUTSIDE, k0);
#pragma unroll
    for (int i = 0; i < LB; i++)
      lds_load16(c.rb, stage + BM * 32 + (c.wave * LB + i) * 256, 32 * c.pb[i] < left ? c.b[i] : FP4_OUTSIDE, k0);
#pragma unroll
    for (int i = 0; i < SPW; i++) {
      const int s = c.wave * SPW + i;  // uniform
      uint32_t *d = stage + DATA + s * 64;
      const uint32_t v = 128 * (c.lane & 1) < left ? c.s[i] : FP4_OUTSIDE;
      if (s < SA) lds_load4(c.rsa, d, v, 8u * (uint32_t)t);
      else lds_load4(c.rsb, d, v, 8u * (uint32_t)t);
    }
  }

  __device__ static void run(uint32_t *lds, const Fp4Operands &o, f32x4 (&acc)[FN][FM]) {
    Ctx c;
    c.lane = threadIdx.x & 63;
    c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c.K = o.K;
    const int lane = c.lane, wm = c.wave % WM, wn = c.wave / WM, l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < LA; i++) {
      const int r = (c.wave * LA + i) * 8 + (lane >> 3);
      c.pa[i] = (lane & 7) ^ xswz(r);
      c.a[i] = (uint32_t)min(r, o.a_rows - 1) * o.lda + 16 * c.pa[i];
    }
#pragma unroll
    for (int i = 0; i < LB; i++) {
      const int r = (c.wave * LB + i) * 8 + (lane >> 3);
      c.pb[i] = (lane & 7) ^ xswz(r);
      c.b[i] = (uint32_t)min(r, o.b_rows - 1) * o.ldb + 16 * c.pb[i];
    }
#pragma unroll
    for (int i = 0; i < SPW; i++) {
      const int s = c.wave * SPW + i;
      const int r = s < SA ? min(s * 32 + (lane >> 1), o.a_rows - 1) : min((s - SA) * 32 + (lane >> 1), o.b_rows - 1);
      c.s[i] = (uint32_t)r * o.s_ld + 4 * (lane & 1);
    }
    const uint32_t row = (uint32_t)o.K / 2;
    c.ra = buffer_rsrc(o.a, (uint32_t)(o.a_rows - 1) * o.lda + row);
    c.rb = buffer_rsrc(o.b, (uint32_t)(o.b_rows - 1) * o.ldb + row);
    c.rsa = buffer_rsrc(o.sa, (uint32_t)o.a_rows * o.s_ld);
    c.rsb = buffer_rsrc(o.sb, (uint32_t)o.b_rows * o.s_ld);
#pragma unroll
    for (int fn = 0; fn < FN; fn++)
#pragma unroll
      for (int fm = 0; fm < FM; fm++) acc[fn][fm] = (f32x4){0.f, 0.f, 0.f, 0.f};

    if (o.t0 < o.t1) issue(lds, c, o.t0);
    for (int t = o.t0; t < o.t1; t++) {
      uint32_t *cur = lds + ((t - o.t0) & 1) * STAGE;
      wait_vmcnt<0>();  // this step's loads have landed
      __syncthreads();  // for every wave, and the other stage's last reads are done
      if (t + 1 < o.t1) issue(lds + ((t + 1 - o.t0) & 1) * STAGE, c, t + 1);
      const uint16_t *sc = reinterpret_cast<const uint16_t *>(cur + DATA);
      uint32_t sw[FN], sx[FM];
#pragma unroll
      for (int fn = 0; fn < FN; fn++) sw[fn] = sc[(BM + wn * TN + fn * 16 + l16) * 4 + g];
#pragma unroll
      for (int fm = 0; fm < FM; fm++) sx[fm] = sc[(wm * TM + fm * 16 + l16) * 4 + g];
      if (c.K - 256 * t < 256) {  // a row's scales past its blocks, whatever they are: none that is a NaN
        const int left = c.K - 256 * t;
        const uint32_t keep = (64 * g < left ? 0xFFu : 0) | (64 * g + 32 < left ? 0xFF00u : 0);
#pragma unroll
        for (int fn = 0; fn < FN; fn++) sw[fn] &= keep;
#pragma unroll
        for (int fm = 0; fm < FM; fm++) sx[fm] &= keep;
      }
      const auto op = [&](int r, int s) {
        return *reinterpret_cast<const u32x4 *>(cur + r * 32 + (((2 * g + s) ^ xswz(r)) * 4));
      };
      const auto half = [&](auto which) {
        constexpr int S = decltype(which)::value;
        u32x4 w[FN];
#pragma unroll
        for (int fn = 0; fn < FN; fn++) w[fn] = op(BM + wn * TN + fn * 16 + l16, S);
#pragma unroll
        for (int fm = 0; fm < FM; fm++) {
          const u32x4 x = op(wm * TM + fm * 16 + l16, S);
#pragma unroll
          for (int fn = 0; fn < FN; fn++) fp4_mul<S>(acc[fn][fm], w[fn], sw[fn], x, sx[fm]);
        }
      };
      half(std::integral_constant<int, 0>{});
      half(std::integral_constant<int, 1>{});
    }
  }

  template <typename YT>
  __device__ __forceinline__ static void store(const f32x4 (&acc)[FN][FM], YT *y, size_t ldy, int m_rows, int n_rows,
                                               bool vec) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    fp8_store<FN, FM>(acc, y, ldy, (wave % WM) * TM + (lane & 15), (wave / WM) * TN + 4 * (lane >> 4), m_rows, n_rows,
                      vec);
  }
};

}  // namespace frx
