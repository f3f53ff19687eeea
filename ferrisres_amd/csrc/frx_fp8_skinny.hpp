// frx_fp8_skinny.hpp — the 8-bit product for up to 64 tokens, or a few groups of 64.
//
// Bound by the weights' bytes: each is read once, straight into registers (a
// lane of an MFMA operand holds 32 codes of one row: two 16-byte loads, 64
// bytes of each of 16 rows an instruction), no LDS on the way. A workgroup
// owns 16 * RT weight rows; its 8 waves take slices of K (blocks of 128, whole
// slices in order) and the slices' sums meet in LDS, added in order. Tokens
// past M repeat the last one (same addresses, so no traffic).
//
// What costs beside the weights are the address lookups of the tokens' codes
// and scales (16 lines an instruction, as many as the weights': 16 tokens of
// 4096 columns 17.1 us against 12.5 when every lane reads one token's), so
// the scales of four blocks are one load, and a workgroup takes as many row
// tiles as leave each compute unit one workgroup (fp8_plan). us, 1 / 16 tokens,
// graph replays over cold weights: 2048 x 2048 4.2 / 4.9, 4096 x 4096 7.2 / 7.6,
// 11008 x 4096 11.7 / 12.5 (3.8 / 3.6 TB/s; a large copy moves 4.7), 13824 x 5120
// 18.9 at 16. Loads of 2 or 4 blocks ahead of the products were slower (16
// tokens of 11008 x 4096 14.6 / 14.8), as were 4 or 16 waves. Above 16 tokens a
// wave holds two or four token tiles (TT) against the same weights.
//
// XT uint8_t: a's codes with scales. Else up to FP8_ACT_MAX_M f32 or bf16
// tokens, whose codes and scales the workgroup makes in LDS while its first
// weights are on their way: the quantiser's operations on the quantiser's
// blocks, so the result equals the two calls' bit for bit.
#pragma once
#include "frx_fp8.hpp"
#include "frx_fp8_codes.hpp"

namespace frx {

struct Fp8Skinny {
  const void *a;   // codes, or activations, of the first token
  const float *sa;
  const uint8_t *b;  // of weight row 0
  const float *sb;
  void *y;         // of the first token
  size_t lda;      // elements of a
  size_t ldb;
  uint32_t M, K, N;  // M: 1 to 16 * TT
  int vec;         // activations: rows 16-byte aligned
};

constexpr int FP8_SK_WAVES = 8;

// Dynamic LDS of a workgroup: the slices' sums; behind them the codes and
// scales that it makes of activations.
__host__ __device__ constexpr size_t fp8_skinny_red_bytes(int tiles) { return (size_t)FP8_SK_WAVES * tiles * 64 * 16; }
__host__ __device__ constexpr size_t fp8_skinny_act_bytes(uint32_t M, uint32_t K) {
  return (size_t)M * K + (size_t)M * ((K + 127) >> 7) * 4;
}

// 32 codes of one row from block kb on: pieces g and g + 4 of the block's 8,
// the row's last piece where K ends before.
__device__ __forceinline__ void fp8_row_load(const uint8_t *row, int k0, int K, int g, u32x4 &lo, u32x4 &hi) {
  const int last = K - 16;
  lo = *reinterpret_cast<const u32x4 *>(row + min(k0 + 16 * g, last));
  hi = *reinterpret_cast<const u32x4 *>(row + min(k0 + 64 + 16 * g, last));
}

__device__ __forceinline__ i32x8 fp8_join(const u32x4 &lo, const u32x4 &hi) {
  return (i32x8){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// Codes [M][K] and, behind them, scales [M][blocks] of the activations: 16
// lanes a block, 8 values a lane, as fp8_rows_kernel.
template <typename XT>
__device__ __forceinline__ void fp8_skinny_quantize(const Fp8Skinny &p, uint8_t *codes, float *scales) {
  const int K = (int)p.K, kbs = (K + 127) >> 7;
  const int l = threadIdx.x & 15;
  for (int b = threadIdx.x >> 4; b < (int)p.M * kbs; b += FP8_SK_WAVES * 4) {
    const int m = b / kbs, k = (b - m * kbs) * 128 + 8 * l;
    const XT *src = static_cast<const XT *>(p.a) + (size_t)m * p.lda + k;
    float v[8];
    if (p.vec && k + 8 <= K) {
      ld8v(src, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = k + i < K ? ld1(src + i) : 0.0f;
    }
    u32x2 c;
    const float s = fp8_block_codes<false>(v, c);
    if (k < K) *reinterpret_cast<u32x2 *>(codes + (size_t)m * K + k) = c;  // K % 16 == 0: whole groups of 8
    if (l == 0) scales[b] = s;
  }
}

// On the bf16 pipe whatever the output: the 8-bit one would save 3% (bf16 y, 64 tokens of
// 4096 x 4096 14.5 us against 15.0).
template <int RT, int TT, bool E5M2, bool BR1, typename XT, typename YT>
__device__ __forceinline__ void fp8_skinny(const Fp8Skinny &p, uint32_t n0, f32x4 *red) {
  constexpr bool CODES = sizeof(XT) == 1;
  using Pipe = Fp8Pipe<true>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int K = (int)p.K, kbs = (K + 127) >> 7;
  const int per = (kbs + FP8_SK_WAVES - 1) / FP8_SK_WAVES;
  const int kb0 = wave * per, kb1 = min(kb0 + per, kbs);
  uint8_t *codes = reinterpret_cast<uint8_t *>(red) + fp8_skinny_red_bytes(RT * TT);
  float *scales = reinterpret_cast<float *>(codes + (size_t)p.M * K);
  const uint8_t *xrow[TT];
  const float *sx[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) {
    const uint32_t tok = min((uint32_t)(16 * t + l16), p.M - 1);
    xrow[t] = CODES ? static_cast<const uint8_t *>(p.a) + (size_t)tok * p.lda : codes + (size_t)tok * K;
    sx[t] = (CODES ? p.sa : scales) + (size_t)tok * kbs;
  }
  const uint8_t *wrow[RT];
  const float *srow[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) {
    wrow[r] = p.b + (size_t)min(n0 + 16 * r + l16, p.N - 1) * p.ldb;
    if (BR1) srow[r] = p.sb + (size_t)(n0 + 16 * r + 4 * g) * kbs;
  }
  // the row tiles' scales, uniform: three tiles may run over a block's end
  constexpr int NB = BR1 ? 0 : 128 % (16 * RT) == 0 ? 1 : RT;
  const float *sblk[RT];
#pragma unroll
  for (int r = 0; r < NB; r++) sblk[r] = p.sb + (size_t)(min(n0 + 16 * r, p.N - 1) >> 7) * kbs;
  f32x4 acc[RT][TT];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < TT; t++) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 wlo[RT], whi[RT];
  if constexpr (!CODES) {
    // a wave without blocks loads the last one's weights and drops them
#pragma unroll
    for (int r = 0; r < RT; r++) fp8_row_load(wrow[r], min(kb0, kbs - 1) * 128, K, g, wlo[r], whi[r]);
    fp8_skinny_quantize<XT>(p, codes, scales);
    __syncthreads();
  }
  float s4[TT] = {};  // scales of four blocks: lane (token, g) has the g-th's
  for (int kb = kb0; kb < kb1; kb++) {
    if (CODES || kb > kb0) {
#pragma unroll
      for (int r = 0; r < RT; r++) fp8_row_load(wrow[r], kb * 128, K, g, wlo[r], whi[r]);
    }
    Fp8Block sb[RT];
#pragma unroll
    for (int r = 0; r < NB; r++) sb[r] = Fp8Block(sblk[r][kb]);
    typename Pipe::Op x[TT];
    float s[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
      u32x4 xlo, xhi;
      fp8_row_load(xrow[t], kb * 128, K, g, xlo, xhi);
      if constexpr (CODES) {
        const int j = (kb - kb0) & 3;
        if (j == 0) s4[t] = sx[t][min(kb + g, kb1 - 1)];
        s[t] = __shfl(s4[t], 16 * j + l16);
      } else {
        s[t] = sx[t][kb];
      }
      if (kb * 128 + 128 > K) {  // pieces past K: zeros on the token side
        if (kb * 128 + 16 * g >= K) xlo = (u32x4){0, 0, 0, 0};
        if (kb * 128 + 64 + 16 * g >= K) xhi = (u32x4){0, 0, 0, 0};
      }
      float f = 1.0f;
      if (NB == 1) {
        const Fp8Factor xf = fp8_factor<true, BR1>(s[t], sb[0]);
        s[t] = xf.s;
        f = xf.f;
      }
      x[t] = Pipe::template op<E5M2>(fp8_join(xlo, xhi), f);
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const auto w = Pipe::template op<false>(fp8_join(wlo[r], whi[r]));
      float sw[4];
      if (BR1)
#pragma unroll
        for (int e = 0; e < 4; e++) sw[e] = n0 + 16 * r + 4 * g + e < p.N ? srow[r][(size_t)e * kbs + kb] : 0.f;
#pragma unroll
      for (int t = 0; t < TT; t++) {
        const f32x4 q = Pipe::template mul<E5M2>(w, x[t]);
        if constexpr (BR1) {
#pragma unroll
          for (int e = 0; e < 4; e++) acc[r][t][e] += q[e] * s[t] * sw[e];
        } else if constexpr (NB == 1) {
#pragma unroll
          for (int e = 0; e < 4; e++) acc[r][t][e] += q[e] * s[t];
        } else {  // blocks of their own: the factor's power of two goes to the product
          const Fp8Factor xf = fp8_factor<true, BR1>(s[t], sb[r]);
#pragma unroll
          for (int e = 0; e < 4; e++) acc[r][t][e] += q[e] * xf.f * xf.s;
        }
      }
    }
  }
  // the slices, in order
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < TT; t++) red[(wave * RT * TT + r * TT + t) * 64 + lane] = acc[r][t];
  __syncthreads();
  static_assert(RT * TT <= FP8_SK_WAVES, "a wave each for the tiles");
  if (wave >= RT * TT) return;
  f32x4 v = red[wave * 64 + lane];
#pragma unroll
  for (int w = 1; w < FP8_SK_WAVES; w++) v += red[(w * RT * TT + wave) * 64 + lane];
  const uint32_t n = n0 + 16 * (wave / TT) + 4 * g, m = 16 * (wave % TT) + l16;
  if (m >= p.M || n >= p.N) return;
  YT *d = static_cast<YT *>(p.y) + (size_t)m * p.N + n;
  const bool vec = ((reinterpret_cast<uintptr_t>(p.y) & (4 * sizeof(YT) - 1)) | (p.N & 3)) == 0;
  if constexpr (sizeof(YT) == 4) {
    if (vec) *reinterpret_cast<f32x4 *>(d) = v;
    else
      for (uint32_t e = 0; e < 4 && n + e < p.N; e++) d[e] = v[e];
  } else {
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = bf16_rne_nb(v[e]);
    if (vec) *reinterpret_cast<u32x2 *>(d) = (u32x2){h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
    else
      for (uint32_t e = 0; e < 4 && n + e < p.N; e++) d[e] = (uint16_t)h[e];
  }
}

}  // namespace frx
