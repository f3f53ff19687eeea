// frx_fp8.hpp — MFMA tile engine of the 8-bit floating-point linears.
//
// y[m][n] = sum_b sa[m][b] sb[n / br][b] sum_{k in b} a[m][k] b[n][k], blocks b of
// 128 columns. A block's product starts from zero and is added to the fp32
// accumulator times the two scales, 4 VALU fused multiply-adds per 16 x 16
// tile. Weight rows are the instruction's rows and tokens its columns: a lane
// then holds four consecutive n of one token, so a block's scale is one number
// per lane and token fragment (b_rows = 128).
//
// Two pipes:
//  - bf16 (WIDE), for every output unless the caller asks otherwise: the codes widened to
//    bf16 (exact, one conversion per two codes) into four v_mfma_f32_16x16x32_bf16,
//    whose products are exact and whose sums are fp32.
//  - 8-bit, for bf16 outputs under FRX_FP8_SUMS_PIPE: v_mfma_f32_16x16x128_f8f6f4, which
//    covers exactly one block at twice the rate (4356 TFLOP/s in a loop of nothing else).
//    It adds groups of 8 products cut to multiples of 2^-13 of the group's largest power
//    of two (measured: beside a product of 2^8 one of 2^-5 is kept and one of 2^-6 is
//    dropped; across groups the sum is fp32): at most 2^-10 of a group's magnitudes,
//    1.5e-5 of the result on normal values, which turns the bf16 rounding of 1 in 130
//    values. So it is a choice of the caller's.
//
// Data movement. Rows of 128 bytes go global -> LDS with 16-byte LDS DMA
// (buffer_load ... lds), the scales of the step with 4-byte DMA behind them, so
// every wave issues the same number of loads per stage. 16-byte pieces are
// XOR-swizzled by row on the source side, which spreads an operand read (16
// rows at one piece) over all banks. Rows past the tile's valid rows are
// clamped to the last one (their results are not stored). K's last step reads
// past K into the next row (nothing past the buffer's end, which is the last
// row's K) and clears those pieces of both sides, so that no NaN there meets
// a zero.
#pragma once
#include "frx_gemm2.hpp"
#include "frx_internal.hpp"

namespace frx {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// A block's two scales, of the lane's token and of the wave's weight rows, as one factor
// of its product. Where their product would leave the normal f32 numbers (gradients of
// 1e-30 and less) and lose bits that y has, the bf16 pipe gets the token's codes as f =
// 2^-64 of themselves, which is exact, and the factor is 2^64 as large. What goes by the
// weights' scale is made once a block, so that a token adds a comparison and two
// selections, made a fragment ahead of their use (2048 x 4096 x 11008 157.2 us, 154.5
// with the plain product; where they are used 161).
struct Fp8Block {
  float s, s64;  // the scale; 2^64 of it, finite, so that a scale of 0 stays one
  float low;     // tokens' scales below this have a product below 2^-100
  __device__ __forceinline__ explicit Fp8Block(float v = 0.f)
      : s(v), s64(__builtin_amdgcn_fmed3f(v * 0x1p64f, -3.402823466e38f, 3.402823466e38f)),
        low(__builtin_fabsf(__builtin_amdgcn_rcpf(v) * 0x1p-100f)) {}
};
struct Fp8Factor {
  float s, f;
};
// A scale per weight row (BR1) multiplies the token's share of a product by itself, and the
// 8-bit pipe, which keeps fewer bits anyway, takes the product of the two scales as it is.
template <bool WIDE, bool BR1>
__device__ __forceinline__ Fp8Factor fp8_factor(float sa, const Fp8Block &b) {
  if constexpr (BR1) return {sa, 1.0f};
  if constexpr (!WIDE) return {sa * b.s, 1.0f};
  const bool small = __builtin_fabsf(sa) < b.low;
  return {sa * (small ? b.s64 : b.s), small ? 0x1p-64f : 1.0f};
}

// The 32 codes of a lane, times a power of two, as 32 bf16 values: x[2j], x[2j + 1] of
// dword d / 2.
struct Fp8Wide {
  u32x4 v[4];
};
template <bool E5M2>
__device__ __forceinline__ Fp8Wide fp8_widen(const i32x8 &c, float f) {
  Fp8Wide r;
#pragma unroll
  for (int d = 0; d < 8; d++) {
    uint32_t lo, hi;
    if constexpr (E5M2) {
      lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((uint32_t)c[d], f, false));
      hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((uint32_t)c[d], f, true));
    } else {
      lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)c[d], f, false));
      hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)c[d], f, true));
    }
    r.v[d >> 1][(d & 1) * 2] = lo;
    r.v[d >> 1][(d & 1) * 2 + 1] = hi;
  }
  return r;
}

// One operand in the form its pipe takes (the bf16 pipe: times a power of two f), and
// the 16 x 16 product of weight rows w and tokens x over one block. WIDE: the bf16 pipe.
template <bool WIDE>
struct Fp8Pipe {
  using Op = i32x8;
  template <bool E5M2>
  __device__ __forceinline__ static Op op(const i32x8 &c, float = 1.0f) { return c; }
  template <bool E5M2>
  __device__ __forceinline__ static f32x4 mul(const Op &w, const Op &x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, E5M2 ? 1 : 0, 0, 0,
                                                            0, 0);
  }
};
template <>
struct Fp8Pipe<true> {
  using Op = Fp8Wide;
  template <bool E5M2>
  __device__ __forceinline__ static Op op(const i32x8 &c, float f = 1.0f) { return fp8_widen<E5M2>(c, f); }
  template <bool E5M2>
  __device__ __forceinline__ static f32x4 mul(const Op &w, const Op &x) {
    f32x4 p = mfma16(w.v[0], x.v[0], (f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int i = 1; i < 4; i++) p = mfma16(w.v[i], x.v[i], p);
    return p;
  }
};

// The operands of one output tile: first rows of both sides and their valid
// rows, scales of those rows (row strides in floats).
struct Fp8Operands {
  const uint8_t *a, *b;
  const float *sa, *sb;  // of the tile's first token; of the block that holds its first weight row
  uint32_t lda, ldb, sa_ld, sb_ld;
  int a_rows, b_rows;    // valid rows in the tile
  int b_first;           // first weight row, modulo br
  int K;                 // columns (bytes) of a row
  int kb0, kb1;          // blocks of 128 to sum over
};

// Zeros in a stage's rows from column K on (k0: the stage's first column).
__device__ __forceinline__ void fp8_clear_tail(uint32_t *rows, int n, int k0, int K, int nt) {
  for (int i = threadIdx.x; i < n * 8; i += nt)
    if (k0 + 16 * (i & 7) >= K)
      *reinterpret_cast<u32x4 *>(rows + (i >> 3) * 32 + ((i & 7) ^ xswz(i >> 3)) * 4) = (u32x4){0, 0, 0, 0};
}

// The results of a lane, FN x FM fragments from (token m0, weight row n0) of the
// tile on. y: the tile's first element, row stride ldy. vec: quads of y are
// aligned to their size.
template <int FN, int FM, typename YT>
__device__ __forceinline__ void fp8_store(const f32x4 (&acc)[FN][FM], YT *y, size_t ldy, int m0, int n0, int m_rows,
                                          int n_rows, bool vec) {
#pragma unroll
  for (int fm = 0; fm < FM; fm++) {
    const int m = m0 + fm * 16;
    if (m >= m_rows) continue;
#pragma unroll
    for (int fn = 0; fn < FN; fn++) {
      const int n = n0 + fn * 16;
      if (n >= n_rows) continue;
      YT *d = y + (size_t)m * ldy + n;
      const f32x4 v = acc[fn][fm];
      if constexpr (sizeof(YT) == 4) {
        if (vec && n + 4 <= n_rows) *reinterpret_cast<f32x4 *>(d) = v;
        else
          for (int e = 0; e < 4 && n + e < n_rows; e++) d[e] = v[e];
      } else {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = bf16_rne_nb(v[e]);
        if (vec && n + 4 <= n_rows) *reinterpret_cast<u32x2 *>(d) = (u32x2){h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
        else
          for (int e = 0; e < 4 && n + e < n_rows; e++) d[e] = (uint16_t)h[e];
      }
    }
  }
}

// BM tokens x BN weight rows, WM x WN waves, BR1: a scale per weight row, WIDE:
// the bf16 pipe.
template <int BM_, int BN_, int WM, int WN, bool E5M2, bool BR1, bool WIDE>
struct Fp8Tile {
  static constexpr int BM = BM_, BN = BN_;
  using Pipe = Fp8Pipe<WIDE>;
  static constexpr int WAVES = WM * WN, NT = WAVES * 64;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // 1 KB load instructions per wave
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "loads split evenly over the waves");
  static_assert(TN <= 128 && 128 % TN == 0, "a wave's weight rows lie in one block of 128");
  static constexpr int SIA = (BM + 63) / 64, SIB = (BN + 63) / 64;  // scale load instructions
  static constexpr int SPW = (SIA + SIB + WAVES - 1) / WAVES;
  static constexpr int DATA = (BM + BN) * 32;  // dwords
  static constexpr int STAGE = DATA + SPW * WAVES * 64;
  static constexpr int LDS_BYTES = 2 * STAGE * 4;

  struct Offsets {
    uint32_t a[LA], b[LB], s[SPW];
  };

  __device__ __forceinline__ static void issue(uint32_t *stage, const Fp8Operands &o, const Offsets &f,
                                               __amdgpu_buffer_rsrc_t ra, __amdgpu_buffer_rsrc_t rb,
                                               __amdgpu_buffer_rsrc_t rsa, __amdgpu_buffer_rsrc_t rsb, int kb,
                                               int wave) {
    const uint32_t k0 = 128u * (uint32_t)kb;
#pragma unroll
    for (int i = 0; i < LA; i++) lds_load16(ra, stage + (wave * LA + i) * 256, f.a[i], k0);
#pragma unroll
    for (int i = 0; i < LB; i++) lds_load16(rb, stage + BM * 32 + (wave * LB + i) * 256, f.b[i], k0);
#pragma unroll
    for (int i = 0; i < SPW; i++) {
      const int s = wave * SPW + i;  // uniform
      uint32_t *d = stage + DATA + s * 64;
      if (s < SIA) lds_load4(rsa, d, f.s[i], 4u * (uint32_t)kb);
      else lds_load4(rsb, d, f.s[i], 4u * (uint32_t)kb);
    }
  }

  __device__ __forceinline__ static i32x8 operand(const uint32_t *rows, int r, int g) {
    const u32x4 lo = *reinterpret_cast<const u32x4 *>(rows + r * 32 + (((2 * g) ^ xswz(r)) * 4));
    const u32x4 hi = *reinterpret_cast<const u32x4 *>(rows + r * 32 + (((2 * g + 1) ^ xswz(r)) * 4));
    return (i32x8){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  }

  __device__ static void run(uint32_t *lds, const Fp8Operands &o, f32x4 (&acc)[FN][FM]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM, l16 = lane & 15, g = lane >> 4;
    Offsets f;
#pragma unroll
    for (int i = 0; i < LA; i++) {
      const int r = (wave * LA + i) * 8 + (lane >> 3);
      f.a[i] = (uint32_t)min(r, o.a_rows - 1) * o.lda + 16 * ((lane & 7) ^ xswz(r));
    }
#pragma unroll
    for (int i = 0; i < LB; i++) {
      const int r = (wave * LB + i) * 8 + (lane >> 3);
      f.b[i] = (uint32_t)min(r, o.b_rows - 1) * o.ldb + 16 * ((lane & 7) ^ xswz(r));
    }
#pragma unroll
    for (int i = 0; i < SPW; i++) {
      const int s = wave * SPW + i;
      if (s < SIA) {
        f.s[i] = (uint32_t)min(s * 64 + lane, o.a_rows - 1) * o.sa_ld * 4;
      } else {
        const int r = min((s - SIA) * 64 + lane, o.b_rows - 1);  // (past the last instruction: the last row again)
        f.s[i] = (uint32_t)(BR1 ? r : (o.b_first + r) >> 7) * o.sb_ld * 4;
      }
    }
    const __amdgpu_buffer_rsrc_t ra = buffer_rsrc(o.a, (uint32_t)(o.a_rows - 1) * o.lda + o.K);
    const __amdgpu_buffer_rsrc_t rb = buffer_rsrc(o.b, (uint32_t)(o.b_rows - 1) * o.ldb + o.K);
    const uint32_t kbs = (uint32_t)(o.K + 127) >> 7;
    const __amdgpu_buffer_rsrc_t rsa = buffer_rsrc(o.sa, ((uint32_t)(o.a_rows - 1) * o.sa_ld + kbs) * 4);
    const __amdgpu_buffer_rsrc_t rsb =
        buffer_rsrc(o.sb, ((uint32_t)(BR1 ? o.b_rows - 1 : (o.b_first + o.b_rows - 1) >> 7) * o.sb_ld + kbs) * 4);
#pragma unroll
    for (int fn = 0; fn < FN; fn++)
#pragma unroll
      for (int fm = 0; fm < FM; fm++) acc[fn][fm] = (f32x4){0.f, 0.f, 0.f, 0.f};

    if (o.kb0 < o.kb1) issue(lds, o, f, ra, rb, rsa, rsb, o.kb0, wave);
    for (int kb = o.kb0; kb < o.kb1; kb++) {
      uint32_t *cur = lds + ((kb - o.kb0) & 1) * STAGE;
      wait_vmcnt<0>();  // this step's loads have landed
      __syncthreads();  // for every wave, and the other stage's last reads are done
      if (kb + 1 < o.kb1) issue(lds + ((kb + 1 - o.kb0) & 1) * STAGE, o, f, ra, rb, rsa, rsb, kb + 1, wave);
      if (kb * 128 + 128 > o.K) {
        fp8_clear_tail(cur, BM + BN, kb * 128, o.K, NT);
        __syncthreads();
      }
      const float *sc = reinterpret_cast<const float *>(cur + DATA);
      typename Pipe::Op w[FN];
      f32x4 sw[FN];
#pragma unroll
      for (int fn = 0; fn < FN; fn++) {
        w[fn] = Pipe::template op<false>(operand(cur + BM * 32, wn * TN + fn * 16 + l16, g));
        if (BR1) sw[fn] = *reinterpret_cast<const f32x4 *>(sc + SIA * 64 + wn * TN + fn * 16 + 4 * g);
      }
      const Fp8Block sblk(BR1 ? 0.f : sc[SIA * 64 + wn * TN]);
      // one token fragment's products are issued between the multiply-adds of
      // the one before, so that neither waits for the other; the next
      // fragment's codes are on their way from LDS meanwhile
      i32x8 xc = operand(cur, wm * TM + l16, g);
      Fp8Factor xf = fp8_factor<WIDE, BR1>(sc[wm * TM + l16], sblk);
      float sn = 0.f, s[2] = {0.f, 0.f};
      f32x4 p[2][FN];
#pragma unroll
      for (int fm = 0; fm <= FM; fm++) {
        typename Pipe::Op x;
        if (fm < FM) {
          x = Pipe::template op<E5M2>(xc, xf.f);
          s[fm & 1] = xf.s;
          if (fm + 1 < FM) {
            xc = operand(cur, wm * TM + (fm + 1) * 16 + l16, g);
            sn = sc[wm * TM + (fm + 1) * 16 + l16];
          }
        }
#pragma unroll
        for (int fn = 0; fn < FN; fn++) {
          if (fm < FM) p[fm & 1][fn] = Pipe::template mul<E5M2>(w[fn], x);
          if (fm > 0) {
            const float q = s[(fm - 1) & 1];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              if (BR1) acc[fn][fm - 1][e] += p[(fm - 1) & 1][fn][e] * q * sw[fn][e];
              else acc[fn][fm - 1][e] += p[(fm - 1) & 1][fn][e] * q;
            }
          }
        }
        if (fm + 1 < FM) xf = fp8_factor<WIDE, BR1>(sn, sblk);
        if (fm > 0 && fm < FM) {
          __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
          for (int fn = 0; fn < FN; fn++) {
            __builtin_amdgcn_sched_group_barrier(0x008, WIDE ? 4 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, BR1 ? 8 : 4, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
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
