// frx_fp4_skinny.hpp — the 4-bit product for up to 32 tokens.
//
// Bound by the weights' bytes: each is read once, straight into registers (a lane of an
// MFMA operand holds one block of 32 codes of one row, 16 bytes: an instruction reads 64
// bytes of each of 16 rows). A workgroup owns 16 * RT weight rows; its 8 waves take slices
// of K (steps of 128, whole slices in order) and the slices' sums meet in LDS, added in
// order. Four steps of a wave are on their way at once, their scales as one load of 16 bytes;
// whatever is not to be read (rows past N, tokens past M, steps of another wave) is past its
// buffer's end, which costs no traffic and is a zero. us: 16 x 4096 x 11008 7.6 (a step at a
// time 10.7; its bytes 4.7), 1 x 4096 x 11008 6.9, 32 x 4096 x 11008 9.2 (64 x 64 tiles 9.4), 16 x
// 2048 x 5632 4.3, 16 x 4096 x 32000 16.0.
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
};

constexpr int FP4_SK_WAVES = 8;
constexpr int FP4_SK_DEPTH = 4;  // steps of a wave on their way (their scales are one load)

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
    if (k + 8 <= K) {
      ld8u(src, v);
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
  constexpr int D = FP4_SK_DEPTH;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int K = (int)p.K, kbs = (K + 127) >> 7;
  const int per = (kbs + FP4_SK_WAVES - 1) / FP4_SK_WAVES;
  const int kb0 = min(wave * per, kbs), kb1 = min(kb0 + per, kbs);
  uint8_t *codes = reinterpret_cast<uint8_t *>(red) + fp4_skinny_red_bytes(RT * TT);
  uint32_t *scales = reinterpret_cast<uint32_t *>(codes + (size_t)p.M * K / 2);
  const uint32_t ldb = (uint32_t)p.ldb, lda = (uint32_t)p.lda, s_ld = 4u * (uint32_t)kbs;
  const uint32_t rows = min(16u * RT, p.N - n0);
  const __amdgpu_buffer_rsrc_t rb = buffer_rsrc(p.b + (size_t)n0 * p.ldb, (rows - 1) * ldb + (uint32_t)K / 2);
  const __amdgpu_buffer_rsrc_t rsb = buffer_rsrc(p.sb + (size_t)n0 * s_ld, rows * s_ld);
  const __amdgpu_buffer_rsrc_t ra = buffer_rsrc(p.a, CODES ? (p.M - 1) * lda + (uint32_t)K / 2 : 0);
  const __amdgpu_buffer_rsrc_t rsa = buffer_rsrc(p.sa, CODES ? p.M * s_ld : 0);
  const uint32_t bv = (uint32_t)l16 * ldb + 16 * g, av = (uint32_t)l16 * lda + 16 * g, sv = (uint32_t)l16 * s_ld;
  f32x4 acc[RT][TT];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < TT; t++) acc[r][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 w[D][RT], x[D][TT], ws[RT], xs[TT], wsn[RT], xsn[TT];
  const auto inside = [&](int kb) { return kb < kb1 && kb * 128 + 32 * g < K; };
  const auto load_scales = [&](int kb, u32x4(&sw)[RT], u32x4(&sx)[TT]) {
#pragma unroll
    for (int r = 0; r < RT; r++)
      sw[r] = __builtin_amdgcn_raw_buffer_load_b128(rsb, sv, 16 * r * s_ld + 4 * kb, 0);
    if constexpr (CODES) {
#pragma unroll
      for (int t = 0; t < TT; t++)
        sx[t] = __builtin_amdgcn_raw_buffer_load_b128(rsa, sv, 16 * t * s_ld + 4 * kb, 0);
    }
  };
  // a step that is not this wave's, or a block past K: zeros
  const auto load = [&](int kb, u32x4(&wd)[RT], u32x4(&xd)[TT]) {
    const bool in = inside(kb);
#pragma unroll
    for (int r = 0; r < RT; r++)
      wd[r] = __builtin_amdgcn_raw_buffer_load_b128(rb, in ? bv : FP4_OUTSIDE, 16 * r * ldb + 64 * kb, 0);
    if constexpr (CODES) {
#pragma unroll
      for (int t = 0; t < TT; t++)
        xd[t] = __builtin_amdgcn_raw_buffer_load_b128(ra, in ? av : FP4_OUTSIDE, 16 * t * lda + 64 * kb, 0);
    }
  };
  // last: steps that are not this wave's have no scale that is a NaN either
  const auto mul = [&](int kb, int u, bool last) {
    const bool in = !last || inside(kb + u);
    uint32_t sx[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
      if constexpr (CODES) {
        sx[t] = xs[t][u];
      } else {
        const int m = min(16 * t + l16, (int)p.M - 1), k = in ? kb + u : 0, gk = in ? g : 0;
        x[u][t] = *reinterpret_cast<const u32x4 *>(codes + (size_t)m * (K / 2) + 64 * k + 16 * gk);
        sx[t] = scales[m * kbs + k];
      }
      sx[t] = in ? sx[t] >> (8 * g) : 0;
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const uint32_t sw = in ? ws[r][u] >> (8 * g) : 0;
#pragma unroll
      for (int t = 0; t < TT; t++) fp4_mul<0>(acc[r][t], w[u][r], sw, x[u][t], sx[t]);
    }
  };
  load_scales(kb0, ws, xs);
#pragma unroll
  for (int u = 0; u < D; u++) load(kb0 + u, w[u], x[u]);
  if constexpr (!CODES) {
    fp4_skinny_quantize<XT>(p, codes, scales);
    barrier_lds();  // (the weights stay on their way)
  }
  int kb = kb0;
  for (; kb + D < kb1; kb += D) {
    load_scales(kb + D, wsn, xsn);
#pragma unroll
    for (int u = 0; u < D; u++) {
      mul(kb, u, false);
      load(kb + D + u, w[u], x[u]);
    }
#pragma unroll
    for (int r = 0; r < RT; r++) ws[r] = wsn[r];
#pragma unroll
    for (int t = 0; t < TT; t++) xs[t] = xsn[t];
  }
#pragma unroll
  for (int u = 0; u < D; u++) mul(kb, u, true);
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
  fp4_store4(static_cast<YT *>(p.y) + (size_t)m * p.N + n, v, p.N - n);
}

}  // namespace frx
