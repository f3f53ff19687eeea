// frx_fp8.hip — launches of the 8-bit floating-point linears (engine: frx_fp8.hpp).
#include "frx_fp8_skinny.hpp"
#include "frx_fp8_ring.hpp"
#include "frx_tiles.hpp"

namespace frx {

namespace {

// Dense product. parts != 0: slice blockIdx.z of K into fp32 part z.
struct DenseArgs {
  const uint8_t *a, *b;
  const float *sa, *sb;
  void *y;
  float *part;
  size_t lda, ldb;
  uint32_t M, K, N;
  int per;  // per: blocks of 128 in a slice
};

template <bool BR1>
__device__ __forceinline__ void fill_operands(Fp8Operands &o, const uint8_t *a, size_t lda, const float *sa,
                                              const uint8_t *b, size_t ldb, const float *sb, uint32_t m0, uint32_t mr,
                                              uint32_t n0, uint32_t nr, uint32_t K) {
  const uint32_t kbs = (K + 127) >> 7;
  o.a = a + (size_t)m0 * lda;
  o.b = b + (size_t)n0 * ldb;
  o.sa = sa + (size_t)m0 * kbs;
  o.sb = sb + (size_t)(BR1 ? n0 : n0 >> 7) * kbs;
  o.lda = (uint32_t)lda;
  o.ldb = (uint32_t)ldb;
  o.sa_ld = o.sb_ld = kbs;
  o.a_rows = (int)mr;
  o.b_rows = (int)nr;
  o.b_first = (int)(n0 & 127);
  o.K = (int)K;
}

template <typename Tile, bool BR1, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp8_dense_kernel(const DenseArgs p) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr int BM = Tile::BM, BN = Tile::BN;
  uint32_t mt, nt;
  xcd_tile<8>(blockIdx.x, (p.M + BM - 1) / BM, (p.N + BN - 1) / BN, mt, nt);
  const uint32_t m0 = mt * BM, n0 = nt * BN;
  Fp8Operands o;
  fill_operands<BR1>(o, p.a, p.lda, p.sa, p.b, p.ldb, p.sb, m0, min((uint32_t)BM, p.M - m0), n0,
                     min((uint32_t)BN, p.N - n0), p.K);
  const int kbs = (int)((p.K + 127) >> 7);
  o.kb0 = p.part ? (int)blockIdx.z * p.per : 0;
  o.kb1 = p.part ? min(o.kb0 + p.per, kbs) : kbs;
  f32x4 acc[Tile::FN][Tile::FM];
  Tile::run(lds, o, acc);
  const size_t at = (size_t)m0 * p.N + n0;
  if (p.part) Tile::template store<float>(acc, p.part + (size_t)blockIdx.z * p.M * p.N + at, p.N, o.a_rows, o.b_rows, (p.N & 3) == 0);
  else Tile::template store<YT>(acc, (YT *)p.y + at, p.N, o.a_rows, o.b_rows, quads<YT>(p.y, p.N));
}

// Rows sorted by expert: blockIdx.x runs over the tiles of all experts (each
// expert's rows in tiles of their own; workgroups past the last tile end).
struct GroupArgs {
  const uint8_t *a;
  const float *sa;
  void *y;
  const uint32_t *offsets;
  size_t lda, ldb;
  uint32_t R, K, N;
  int E;
  const uint8_t *b[FP8_MAXE];
  const float *sb[FP8_MAXE];
};

// mts: tiles of rows there may be. An XCD's run of tiles goes down the rows
// first: the tiles of an expert's rows share its weights in that L2.
template <typename Tile, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp8_grouped_kernel(const GroupArgs p, uint32_t mts) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr int BM = Tile::BM, BN = Tile::BN;
  uint32_t mt, nt;
  xcd_tile<0x40000000>(blockIdx.x, mts, (p.N + BN - 1) / BN, mt, nt);
  uint32_t m0, end;
  const int e = expert_tile<BM>(p.offsets, p.E, p.R, mt, m0, end);
  if (e < 0) return;
  const uint32_t n0 = nt * BN;
  Fp8Operands o;
  fill_operands<false>(o, p.a, p.lda, p.sa, p.b[e], p.ldb, p.sb[e], m0, min((uint32_t)BM, end - m0), n0,
                       min((uint32_t)BN, p.N - n0), p.K);
  o.kb0 = 0;
  o.kb1 = (int)((p.K + 127) >> 7);
  f32x4 acc[Tile::FN][Tile::FM];
  Tile::run(lds, o, acc);
  Tile::template store<YT>(acc, (YT *)p.y + (size_t)m0 * p.N + n0, p.N, o.a_rows, o.b_rows, quads<YT>(p.y, p.N));
}

// blockIdx.y: the group of 16 * TT tokens.
template <int RT, int TT, bool E5M2, bool BR1, typename XT, typename YT>
__global__ __launch_bounds__(FP8_SK_WAVES * 64) void fp8_skinny_kernel(Fp8Skinny p) {
  extern __shared__ __align__(16) uint32_t lds[];
  if constexpr (TT == 4) {
    const uint32_t m0 = blockIdx.y * 64;
    p.a = static_cast<const XT *>(p.a) + m0 * p.lda;
    p.sa += (size_t)m0 * ((p.K + 127) >> 7);
    p.y = static_cast<YT *>(p.y) + (size_t)m0 * p.N;
    p.M = min(64u, p.M - m0);
  }
  fp8_skinny<RT, TT, E5M2, BR1, XT, YT>(p, blockIdx.x * 16 * RT, reinterpret_cast<f32x4 *>(lds));
}

// Sorted rows in tiles of 16 (decode batches: a few rows of each expert).
template <int RT, bool E5M2, typename YT>
__global__ __launch_bounds__(FP8_SK_WAVES * 64) void fp8_skinny_grouped_kernel(const GroupArgs p) {
  extern __shared__ __align__(16) uint32_t lds[];
  const uint32_t nts = (p.N + 16 * RT - 1) / (16 * RT);
  const uint32_t mt = blockIdx.x / nts, nt = blockIdx.x - mt * nts;
  uint32_t m0, end;
  const int e = expert_tile<16>(p.offsets, p.E, p.R, mt, m0, end);
  if (e < 0) return;
  const uint32_t kbs = (p.K + 127) >> 7;
  const Fp8Skinny q = {p.a + (size_t)m0 * p.lda, p.sa + (size_t)m0 * kbs, p.b[e], p.sb[e],
                       static_cast<YT *>(p.y) + (size_t)m0 * p.N, p.lda, p.ldb, min(16u, end - m0), p.K, p.N, 0};
  fp8_skinny<RT, 1, E5M2, false, uint8_t, YT>(q, nt * 16 * RT, reinterpret_cast<f32x4 *>(lds));
}

// Weight gradients: expert blockIdx.y sums over the blocks of its rows. Here
// the engine's tokens are dw's rows (dy's columns) and its weight rows x's
// columns.
struct GradArgs {
  const uint8_t *a, *b;
  const float *sa, *sb;
  const uint32_t *offsets;
  size_t lda, ldb;
  uint32_t R, N, K;
  void *dw[FP8_MAXE];
};

template <typename Tile, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp8_grad_kernel(const GradArgs p) {
  constexpr int BM = Tile::BM, BN = Tile::BN;
  extern __shared__ __align__(16) uint32_t lds[];
  const uint32_t mts = (p.N + BM - 1) / BM;
  const uint32_t nt = blockIdx.x / mts, mt = blockIdx.x - nt * mts;
  const uint32_t m0 = mt * BM, n0 = nt * BN;
  const int e = blockIdx.y;
  uint32_t first, end;
  expert_rows(p.offsets, e, p.R, first, end);
  Fp8Operands o;
  fill_operands<true>(o, p.a, p.lda, p.sa, p.b, p.ldb, p.sb, m0, min((uint32_t)BM, p.N - m0), n0,
                                    min((uint32_t)BN, p.K - n0), p.R);
  o.kb0 = (int)(first >> 7);
  o.kb1 = (int)((end + 127) >> 7);
  f32x4 acc[Tile::FN][Tile::FM];
  Tile::run(lds, o, acc);
  const size_t at = (size_t)m0 * p.K + n0;
  YT *dw = static_cast<YT *>(p.dw[e]);
  Tile::template store<YT>(acc, dw + at, p.K, o.a_rows, o.b_rows, quads<YT>(dw, p.K));
}

template <typename K, typename A>
hipError_t go(K kernel, int lds, std::atomic<uint64_t> &done, dim3 grid, int nt, hipStream_t stream, const A &args) {
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel), lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, grid, dim3(nt), lds, stream, args);
  return hipGetLastError();
}

template <typename Tile, bool BR1, typename YT>
hipError_t dense_go(const DenseArgs &p, int S, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const size_t tiles = (size_t)((p.M + Tile::BM - 1) / Tile::BM) * ((p.N + Tile::BN - 1) / Tile::BN);
  if (tiles * Tile::NT > 0xFFFFFFFFu) return hipErrorInvalidValue;
  return go(fp8_dense_kernel<Tile, BR1, YT>, Tile::LDS_BYTES, done, dim3((unsigned)tiles, 1, S), Tile::NT, stream, p);
}

template <bool E5M2, bool BR1, bool WIDE, typename YT>
hipError_t dense_tile(int tile, const DenseArgs &p, int S, hipStream_t stream) {
  if constexpr (!(BR1 && WIDE))
    if (tile == FP8_T_RING4) return dense_go<Fp8Ring<4, E5M2, BR1, WIDE>, BR1, YT>(p, S, stream);
  if constexpr (!BR1)
    if (tile == FP8_T_RING6) return dense_go<Fp8Ring<6, E5M2, BR1, WIDE>, BR1, YT>(p, S, stream);
  if constexpr (!BR1 && !WIDE)
    if (tile == FP8_T_RING8) return dense_go<Fp8Ring<8, E5M2, BR1, WIDE>, BR1, YT>(p, S, stream);
  return dense_go<Fp8Tile<128, 128, 2, 2, E5M2, BR1, WIDE>, BR1, YT>(p, S, stream);
}

template <int RT, int TT, bool E5M2, bool BR1, typename XT, typename YT>
hipError_t skinny_rt(const Fp8Skinny &p, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  constexpr size_t red = fp8_skinny_red_bytes(RT * TT);
  const auto kernel = fp8_skinny_kernel<RT, TT, E5M2, BR1, XT, YT>;
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel),
                                  (int)(red + (sizeof(XT) == 1 ? 0 : FP8_ACT_MAX_BYTES)), done);
  if (e != hipSuccess) return e;
  const size_t lds = red + (sizeof(XT) == 1 ? 0 : fp8_skinny_act_bytes(p.M, p.K));
  hipLaunchKernelGGL(kernel, dim3((p.N + 16 * RT - 1) / (16 * RT), (p.M + 16 * TT - 1) / (16 * TT)),
                     dim3(FP8_SK_WAVES * 64), lds, stream, p);
  return hipGetLastError();
}

template <int TT, bool E5M2, bool BR1, typename XT, typename YT>
hipError_t skinny_go(int rt, const Fp8Skinny &p, hipStream_t stream) {
  if constexpr (TT <= 2) {
    if (rt == 4) return skinny_rt<4, TT, E5M2, BR1, XT, YT>(p, stream);
    if (rt == 3) return skinny_rt<3, TT, E5M2, BR1, XT, YT>(p, stream);
  }
  if (rt == 2) return skinny_rt<2, TT, E5M2, BR1, XT, YT>(p, stream);
  return skinny_rt<1, TT, E5M2, BR1, XT, YT>(p, stream);
}

template <bool E5M2, bool BR1, typename YT>
hipError_t skinny_tt(int rt, const Fp8Skinny &p, hipStream_t stream) {
  if (p.M > 32) return skinny_go<4, E5M2, BR1, uint8_t, YT>(rt, p, stream);
  return p.M > 16 ? skinny_go<2, E5M2, BR1, uint8_t, YT>(rt, p, stream) : skinny_go<1, E5M2, BR1, uint8_t, YT>(rt, p, stream);
}

template <typename YT>
hipError_t skinny_any(int e5m2, int b_rows, int rt, const Fp8Skinny &p, hipStream_t stream) {
  if (b_rows == 1) return e5m2 ? skinny_tt<true, true, YT>(rt, p, stream) : skinny_tt<false, true, YT>(rt, p, stream);
  return e5m2 ? skinny_tt<true, false, YT>(rt, p, stream) : skinny_tt<false, false, YT>(rt, p, stream);
}

template <bool WIDE, typename YT>
hipError_t dense_any(int e5m2, int b_rows, int tile, const DenseArgs &p, int S, hipStream_t stream) {
  if (b_rows == 1)
    return e5m2 ? dense_tile<true, true, WIDE, YT>(tile, p, S, stream) : dense_tile<false, true, WIDE, YT>(tile, p, S, stream);
  return e5m2 ? dense_tile<true, false, WIDE, YT>(tile, p, S, stream) : dense_tile<false, false, WIDE, YT>(tile, p, S, stream);
}

template <typename Tile, typename YT>
hipError_t grouped_go(const GroupArgs &p, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const size_t mts = (size_t)(p.R + Tile::BM - 1) / Tile::BM + p.E, tiles = mts * ((p.N + Tile::BN - 1) / Tile::BN);
  if (tiles * Tile::NT > 0xFFFFFFFFu) return hipErrorInvalidValue;
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(fp8_grouped_kernel<Tile, YT>), Tile::LDS_BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((fp8_grouped_kernel<Tile, YT>), dim3((unsigned)tiles), dim3(Tile::NT), Tile::LDS_BYTES, stream, p,
                     (uint32_t)mts);
  return hipGetLastError();
}

template <bool E5M2, typename YT>
hipError_t grouped_any(const GroupArgs &p, int tile, hipStream_t stream) {
  if (tile == FP8_T_SKINNY) {
    const dim3 grid((unsigned)(((p.R + 15) / 16 + p.E) * ((p.N + 15) / 16))), block(FP8_SK_WAVES * 64);
    hipLaunchKernelGGL((fp8_skinny_grouped_kernel<1, E5M2, YT>), grid, block, (int)fp8_skinny_red_bytes(1), stream, p);
    return hipGetLastError();
  }
  if constexpr (!E5M2 && sizeof(YT) == 2) {
    if (tile == FP8_T_RING8) return grouped_go<Fp8Ring<8, E5M2, false, false>, YT>(p, stream);
    if (tile == FP8_T_RING4) return grouped_go<Fp8Ring<4, E5M2, false, false>, YT>(p, stream);
  }
  return grouped_go<Fp8Tile<64, 128, 2, 2, E5M2, false, true>, YT>(p, stream);
}

template <bool E5M2, bool WIDE, typename YT>
hipError_t grad_go(const GradArgs &p, int E, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  using Tile = Fp8Tile<128, 128, 2, 2, E5M2, true, WIDE>;
  const size_t tiles = (size_t)((p.N + Tile::BM - 1) / Tile::BM) * ((p.K + Tile::BN - 1) / Tile::BN);
  if (tiles * Tile::NT > 0xFFFFFFFFu) return hipErrorInvalidValue;
  return go(fp8_grad_kernel<Tile, YT>, Tile::LDS_BYTES, done, dim3((unsigned)tiles, (unsigned)E), Tile::NT, stream, p);
}

}  // namespace

size_t fp8_part_bytes(uint32_t M, uint32_t N, const Fp8Plan &p) { return p.S > 1 ? (size_t)p.S * M * N * 4 : 0; }

hipError_t launch_fp8_linear(const uint8_t *a, size_t lda, int e5m2, const float *sa, const uint8_t *b, size_t ldb,
                             const float *sb, int b_rows, void *y, int yt_bf16, int pipe8, uint32_t M, uint32_t K,
                             uint32_t N, const Fp8Plan &plan, float *part, hipStream_t stream) {
  if (plan.tile == FP8_T_SKINNY) {
    const Fp8Skinny p = {a, sa, b, sb, y, lda, ldb, M, K, N, 0};
    return yt_bf16 ? skinny_any<uint16_t>(e5m2, b_rows, plan.per, p, stream)
                   : skinny_any<float>(e5m2, b_rows, plan.per, p, stream);
  }
  const DenseArgs p = {a, b, sa, sb, y, plan.S > 1 ? part : nullptr, lda, ldb, M, K, N, plan.per};
  const hipError_t e = !yt_bf16 ? dense_any<true, float>(e5m2, b_rows, plan.tile, p, plan.S, stream)
                       : pipe8  ? dense_any<false, uint16_t>(e5m2, b_rows, plan.tile, p, plan.S, stream)
                                : dense_any<true, uint16_t>(e5m2, b_rows, plan.tile, p, plan.S, stream);
  if (e != hipSuccess || plan.S == 1) return e;
  const size_t n = (size_t)M * N;
  const dim3 grid((unsigned)((n + 1023) / 1024));
  if (yt_bf16) hipLaunchKernelGGL(join_parts_kernel<uint16_t>, grid, dim3(256), 0, stream, part, plan.S, n, (uint16_t *)y);
  else hipLaunchKernelGGL(join_parts_kernel<float>, grid, dim3(256), 0, stream, part, plan.S, n, (float *)y);
  return hipGetLastError();
}

bool fp8_act_fits(uint32_t M, uint32_t K) {
  return M <= FP8_ACT_MAX_M && fp8_skinny_act_bytes(M, K) <= FP8_ACT_MAX_BYTES;
}

hipError_t launch_fp8_linear_act(const void *x, int xt_bf16, const uint8_t *b, size_t ldb, const float *sb, void *y,
                                 int yt_bf16, uint32_t M, uint32_t K, uint32_t N, const Fp8Plan &plan,
                                 hipStream_t stream) {
  const int vec = ((reinterpret_cast<uintptr_t>(x) | (size_t)K * (xt_bf16 ? 2 : 4)) & 15) == 0;
  const Fp8Skinny p = {x, nullptr, b, sb, y, K, ldb, M, K, N, vec};
  if (xt_bf16)
    return yt_bf16 ? skinny_go<1, false, false, uint16_t, uint16_t>(plan.per, p, stream)
                   : skinny_go<1, false, false, uint16_t, float>(plan.per, p, stream);
  return yt_bf16 ? skinny_go<1, false, false, float, uint16_t>(plan.per, p, stream)
                 : skinny_go<1, false, false, float, float>(plan.per, p, stream);
}

hipError_t launch_fp8_grouped(const uint8_t *a, size_t lda, int e5m2, const float *sa, const uint8_t *const *b,
                              size_t ldb, const float *const *sb, const uint32_t *offsets, int E, void *y,
                              int yt_bf16, int pipe8, uint32_t R, uint32_t K, uint32_t N, int cus, hipStream_t stream) {
  GroupArgs p = {a, sa, y, offsets, lda, ldb, R, K, N, E, {}, {}};
  for (int e = 0; e < E; e++) {
    p.b[e] = b[e];
    p.sb[e] = sb[e];
  }
  const int tile = fp8_grouped_tile(R, N, (uint32_t)E, pipe8 && !e5m2, cus);
  if (yt_bf16) return e5m2 ? grouped_any<true, uint16_t>(p, tile, stream) : grouped_any<false, uint16_t>(p, tile, stream);
  return e5m2 ? grouped_any<true, float>(p, tile, stream) : grouped_any<false, float>(p, tile, stream);
}

hipError_t launch_fp8_grad_weight(const uint8_t *a, size_t lda, int e5m2, const float *sa, const uint8_t *b,
                                  size_t ldb, const float *sb, const uint32_t *offsets, int E, void *const *dw,
                                  int yt_bf16, int pipe8, uint32_t R, uint32_t N, uint32_t K, hipStream_t stream) {
  GradArgs p = {a, b, sa, sb, offsets, lda, ldb, R, N, K, {}};
  for (int e = 0; e < E; e++) p.dw[e] = dw[e];
  if (!yt_bf16) return e5m2 ? grad_go<true, true, float>(p, E, stream) : grad_go<false, true, float>(p, E, stream);
  if (pipe8) return e5m2 ? grad_go<true, false, uint16_t>(p, E, stream) : grad_go<false, false, uint16_t>(p, E, stream);
  return e5m2 ? grad_go<true, true, uint16_t>(p, E, stream) : grad_go<false, true, uint16_t>(p, E, stream);
}

}  // namespace frx
