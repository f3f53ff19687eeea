// frx_fp4_skinny.hpp — the 4-bit product for up to 32 tokens.
//
// Bound by the weights' bytes: each is read once, straight into registers (a lane of an
// MFMA operand holds one block of 32 codes of one row, 16 bytes: an instruction reads 64
// bytes of each of 16 rows). A workgroup owns 16 * RT weight rows; its 8 waves take slices
// of K (steps of 128, whole slices in order) and the slices' sums meet in LDS, added in
// order. Tokens past M repeat the last one (same addresses, so no traffic).
//
// XT uint8_t: a's codes with scales. Else up to FP4_ACT_MAX_M f32 or bf16 tokens, whose
// codes and scales the workgroup makes in LDS while its first weights are on their way:
// the quantiser's operations on the quantiser's blocks, so the result equals the two
// calls' bit for bit.
#pragma once
#include "frx_fp4.hpp"

namespace frx {

struct Fp4Skinny {
  const void *a;          // codes, or activations, of the first token
  const uint8_t *sa;
  const uint8_t *b, *sb;  // of weight row 0
  void *y;                // of the first token
  size_t lda;             // bytes of codes, elements of activations
  size_t ldb;
  uint32_t M, K, N;       // M: 1 to 16 * TT
  int vec;                // activations: rows 16-byte aligned
};

constexpr int FP4_SK_WAVES = 8;

// Dynamic LDS of a workgroup: the slices' sums; behind them the codes and scales that it
// makes of activations.
__host__ __device__ constexpr size_t fp4_skinny_red_bytes(int tiles) { return (size_t)FP4_SK_WAVES * tiles * 64 * 16; }
__host__ __device__ constexpr size_t fp4_skinny_act_bytes(uint32_t M, uint32_t K) {
  return (size_t)M * (K / 2 + fp4_scale_bytes(K));
}

template <typename XT>
__device__ __forceinline__ void fp4_skinny_quantize(const Fp4Skinny &p, uint8_t *codes, uint32_t *scales) {
  const int K = (int)p.K, kbs = (K + 127) >> 7;
  const int l = threadIdx.x & 15;
  for (int b = threadIdx.x >> 4; b < (int)p.M * kbs; b += FP4_SK_WAVES * 4) {
    const int m = b / kbs, k = (b - m * kbs) * 128 + 8 * l;
    const XT *src = static_cast<const XT *>(p.a) + (size_t)m * p.lda + k;
    float v[8];
    if (p.vec && k + 8 <= K) {
      ld8v(src, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = k + i < K ? ld1(src + i) : 0.0f;
    }
    uint32_t s;
    const uint32_t c = fp4_block_codes(v, s);
    if (k < K) *reinterpret_cast<uint32_t *>(codes + ((size_t)m * K + k) / 2) = c;
    if (l == 0) scales[b] = s;
  }
}

template <int RT, int TT, typename XT, typename YT>
__device__ __forceinline__ void fp4_skinny(const Fp4Skinny &p, uint32_t n0, f32x4 *red) {
  constexpr bool CODES = sizeof(XT) == 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int K = (int)p.K, kbs = (K + 127) >> 7;
  const int per = (kbs + FP4_SK_WAVES - 1) / FP4_SK_WAVES;
  const int kb0 = min(wave * per, kbs), kb1 = min(kb0 + per, kbs);
  uint8_t *codes = reinterpret_cast<uint8_t *>(red) + fp4_skinny_red_bytes(RT * TT);
  uint32_t *scales = reinterpret_cast<uint32_t *>(codes + (size_t)p.M * K / 2);
  const uint8_t *xrow[TT];
  const uint32_t *sx[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) {
    const uint32_t tok = min((uint32_t)(16 * t + l16), p.M - 1);
    xrow[t] = CODES ? static_cast<const uint8_t *>(p.a) + (size_t)tok * p.lda : codes + (size_t)tok * K / 2;
    sx[t] = (CODES ? reinterpret_cast<const uint32_t *>(p.sa) : scales) + (size_t)tok * kbs;
  }
  const uint8_t *wrow[RT];
  const uint32_t *sw[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const size_t n = min(n0 + 16 * r + l16, p.N - 1);
    wrow[r] = p.b + n * p.ldb;
    sw[r] = reinterpret_cast<const uint32_t *>(p.sb) + n * kbs;
  }
  // the row's last block where K ends before
  const auto at = [&](int kb) { return min(kb * 64 + 16 * g, K / 2 - 16); };
  f32x4 acc[RT][TT];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < TT; t++) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 w[RT];
  uint32_t ws[RT];
  if constexpr (!CODES) {
    // a wave without steps loads the last one's weights and drops them
#pragma unroll
    for (int r = 0; r < RT; r++) {
      w[r] = *reinterpret_cast<const u32x4 *>(wrow[r] + at(min(kb0, kbs - 1)));
      ws[r] = sw[r][min(kb0, kbs - 1)];
    }
    fp4_skinny_quantize<XT>(p, codes, scales);
    __syncthreads();
  }
  for (int kb = kb0; kb < kb1; kb++) {
    if (CODES || kb > kb0) {
#pragma unroll
      for (int r = 0; r < RT; r++) {
        w[r] = *reinterpret_cast<const u32x4 *>(wrow[r] + at(kb));
        ws[r] = sw[r][kb];
      }
    }
    const bool inside = kb * 128 + 32 * g < K;  // past K: zeros on both sides, no scale that is a NaN
    u32x4 x[TT];
    uint32_t xs[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
      x[t] = *reinterpret_cast<const u32x4 *>(xrow[t] + at(kb));
      xs[t] = inside ? sx[t][kb] >> (8 * g) : 0;
      if (!inside) x[t] = (u32x4){0, 0, 0, 0};
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const uint32_t s = inside ? ws[r] >> (8 * g) : 0;
#pragma unroll
      for (int t = 0; t < TT; t++) fp4_mul<0>(acc[r][t], w[r], s, x[t], xs[t]);
    }
  }
  // the slices, in order
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < TT; t++) red[(wave * RT * TT + r * TT + t) * 64 + lane] = acc[r][t];
  __syncthreads();
  static_assert(RT * TT <= FP4_SK_WAVES, "a wave each for the tiles");
  if (wave >= RT * TT) return;
  f32x4 v = red[wave * 64 + lane];
#pragma unroll
  for (int i = 1; i < FP4_SK_WAVES; i++) v += red[(i * RT * TT + wave) * 64 + lane];
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
