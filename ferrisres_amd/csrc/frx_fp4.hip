// frx_fp4.hip — launches of the 4-bit floating-point linears (engines: frx_fp4_ring.hpp,
// frx_fp4_skinny.hpp).
#include "frx_fp4_ring.hpp"
#include "frx_fp4_skinny.hpp"
#include "frx_internal.hpp"
#include "frx_tiles.hpp"

namespace frx {

namespace {

// Dense product. part != 0: slice blockIdx.z of K into fp32 part z.
struct DenseArgs {
  const uint8_t *a, *b, *sa, *sb;
  void *y;
  float *part;
  size_t lda, ldb;
  uint32_t M, K, N;
  int per;  // steps of 256 columns in a slice
};

__device__ __forceinline__ void fill_operands(Fp4Operands &o, const uint8_t *a, size_t lda, const uint8_t *sa,
                                              const uint8_t *b, size_t ldb, const uint8_t *sb, uint32_t m0,
                                              uint32_t mr, uint32_t n0, uint32_t nr, uint32_t K) {
  o.s_ld = fp4_scale_bytes(K);
  o.a = a + (size_t)m0 * lda;
  o.b = b + (size_t)n0 * ldb;
  o.sa = sa + (size_t)m0 * o.s_ld;
  o.sb = sb + (size_t)n0 * o.s_ld;
  o.lda = (uint32_t)lda;
  o.ldb = (uint32_t)ldb;
  o.a_rows = (int)mr;
  o.b_rows = (int)nr;
  o.K = (int)K;
}

template <typename Tile, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp4_dense_kernel(const DenseArgs p) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr int BM = Tile::BM, BN = Tile::BN;
  uint32_t mt, nt;
  xcd_tile<8>(blockIdx.x, (p.M + BM - 1) / BM, (p.N + BN - 1) / BN, mt, nt);
  const uint32_t m0 = mt * BM, n0 = nt * BN;
  Fp4Operands o;
  fill_operands(o, p.a, p.lda, p.sa, p.b, p.ldb, p.sb, m0, min((uint32_t)BM, p.M - m0), n0, min((uint32_t)BN, p.N - n0),
                p.K);
  const int steps = (int)((p.K + 255) >> 8);
  o.t0 = p.part ? (int)blockIdx.z * p.per : 0;
  o.t1 = p.part ? min(o.t0 + p.per, steps) : steps;
  f32x4 acc[Tile::FN][Tile::FM];
  Tile::run(lds, o, acc);
  const size_t at = (size_t)m0 * p.N + n0;
  if (p.part)
    Tile::template store<float>(acc, p.part + (size_t)blockIdx.z * p.M * p.N + at, p.N, o.a_rows, o.b_rows,
                                (p.N & 3) == 0);
  else Tile::template store<YT>(acc, (YT *)p.y + at, p.N, o.a_rows, o.b_rows, quads<YT>(p.y, p.N));
}

// Rows sorted by expert: blockIdx.x runs over the tiles of all experts (each expert's
// rows in tiles of their own; workgroups past the last tile end).
struct GroupArgs {
  const uint8_t *a, *sa;
  void *y;
  const uint32_t *offsets;
  size_t lda, ldb;
  uint32_t R, K, N;
  int E;
  const uint8_t *b[FP8_MAXE], *sb[FP8_MAXE];
};

// mts: tiles of rows there may be. An XCD's run of tiles goes down the rows first: the
// tiles of an expert's rows share its weights in that L2.
template <typename Tile, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp4_grouped_kernel(const GroupArgs p, uint32_t mts) {
  extern __shared__ __align__(16) uint32_t lds[];
  constexpr int BM = Tile::BM, BN = Tile::BN;
  uint32_t mt, nt;
  xcd_tile<0x40000000>(blockIdx.x, mts, (p.N + BN - 1) / BN, mt, nt);
  uint32_t m0, end;
  const int e = expert_tile<BM>(p.offsets, p.E, p.R, mt, m0, end);
  if (e < 0) return;
  const uint32_t n0 = nt * BN;
  Fp4Operands o;
  fill_operands(o, p.a, p.lda, p.sa, p.b[e], p.ldb, p.sb[e], m0, min((uint32_t)BM, end - m0), n0,
                min((uint32_t)BN, p.N - n0), p.K);
  o.t0 = 0;
  o.t1 = (int)((p.K + 255) >> 8);
  f32x4 acc[Tile::FN][Tile::FM];
  Tile::run(lds, o, acc);
  Tile::template store<YT>(acc, (YT *)p.y + (size_t)m0 * p.N + n0, p.N, o.a_rows, o.b_rows, quads<YT>(p.y, p.N));
}

template <int RT, int TT, typename XT, typename YT>
__global__ __launch_bounds__(FP4_SK_WAVES * 64) void fp4_skinny_kernel(const Fp4Skinny p) {
  extern __shared__ __align__(16) uint32_t lds[];
  fp4_skinny<RT, TT, XT, YT>(p, blockIdx.x * 16 * RT, reinterpret_cast<f32x4 *>(lds));
}

template <typename Tile, typename YT>
hipError_t dense_go(const DenseArgs &p, int S, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const size_t tiles = (size_t)((p.M + Tile::BM - 1) / Tile::BM) * ((p.N + Tile::BN - 1) / Tile::BN);
  if (tiles * Tile::NT > 0xFFFFFFFFu) return hipErrorInvalidValue;
  const auto kernel = fp4_dense_kernel<Tile, YT>;
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel), Tile::LDS_BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, 1, S), dim3(Tile::NT), Tile::LDS_BYTES, stream, p);
  return hipGetLastError();
}

// tokens x weight rows
using Tile64x64 = Fp4Ring<2, 2, 2, 2, 3>;
using Tile64x128 = Fp4Ring<2, 2, 2, 4, 3>;
using Tile128x192 = Fp4Ring<2, 4, 4, 3, 3>;
using Tile128x256 = Fp4Ring<2, 4, 4, 4, 3>;
using Tile192x256 = Fp4Ring<2, 4, 6, 4, 2>;
using Tile256x256 = Fp4Ring<2, 4, 8, 4, 2>;
static_assert(3 * Tile64x64::LDS_BYTES <= 160 << 10, "three workgroups to a compute unit");
static_assert(2 * Tile64x128::LDS_BYTES <= 160 << 10, "two workgroups to a compute unit");

template <typename YT>
hipError_t dense_tile(int tile, const DenseArgs &p, int S, hipStream_t stream) {
  switch (tile) {
    case FP4_T_256X256: return dense_go<Tile256x256, YT>(p, S, stream);
    case FP4_T_192X256: return dense_go<Tile192x256, YT>(p, S, stream);
    case FP4_T_128X256: return dense_go<Tile128x256, YT>(p, S, stream);
    case FP4_T_128X192: return dense_go<Tile128x192, YT>(p, S, stream);
    case FP4_T_64X128: return dense_go<Tile64x128, YT>(p, S, stream);
    default: return dense_go<Tile64x64, YT>(p, S, stream);
  }
}

template <int RT, int TT, typename XT, typename YT>
hipError_t skinny_rt(const Fp4Skinny &p, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  constexpr size_t red = fp4_skinny_red_bytes(RT * TT);
  const auto kernel = fp4_skinny_kernel<RT, TT, XT, YT>;
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel),
                                  (int)(red + (sizeof(XT) == 1 ? 0 : FP4_ACT_MAX_BYTES)), done);
  if (e != hipSuccess) return e;
  const size_t lds = red + (sizeof(XT) == 1 ? 0 : fp4_skinny_act_bytes(p.M, p.K));
  hipLaunchKernelGGL(kernel, dim3((p.N + 16 * RT - 1) / (16 * RT)), dim3(FP4_SK_WAVES * 64), lds, stream, p);
  return hipGetLastError();
}

template <int TT, typename XT, typename YT>
hipError_t skinny_go(int rt, const Fp4Skinny &p, hipStream_t stream) {
  if (rt == 4) return skinny_rt<4, TT, XT, YT>(p, stream);
  if (rt == 3) return skinny_rt<3, TT, XT, YT>(p, stream);
  if (rt == 2) return skinny_rt<2, TT, XT, YT>(p, stream);
  return skinny_rt<1, TT, XT, YT>(p, stream);
}

template <typename YT>
hipError_t skinny_any(int rt, const Fp4Skinny &p, hipStream_t stream) {
  return p.M > 16 ? skinny_go<2, uint8_t, YT>(rt, p, stream) : skinny_go<1, uint8_t, YT>(rt, p, stream);
}

template <typename Tile, typename YT>
hipError_t grouped_go(const GroupArgs &p, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const size_t mts = (size_t)(p.R + Tile::BM - 1) / Tile::BM + p.E, tiles = mts * ((p.N + Tile::BN - 1) / Tile::BN);
  if (tiles * Tile::NT > 0xFFFFFFFFu) return hipErrorInvalidValue;
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(fp4_grouped_kernel<Tile, YT>), Tile::LDS_BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((fp4_grouped_kernel<Tile, YT>), dim3((unsigned)tiles), dim3(Tile::NT), Tile::LDS_BYTES, stream, p,
                     (uint32_t)mts);
  return hipGetLastError();
}

template <typename YT>
hipError_t grouped_any(const GroupArgs &p, int tile, hipStream_t stream) {
  switch (tile) {
    case FP4_T_256X256: return grouped_go<Tile256x256, YT>(p, stream);
    case FP4_T_128X256: return grouped_go<Tile128x256, YT>(p, stream);
    case FP4_T_64X128: return grouped_go<Tile64x128, YT>(p, stream);
    default: return grouped_go<Tile64x64, YT>(p, stream);
  }
}

}  // namespace

hipError_t launch_fp4_linear(const uint8_t *a, size_t lda, const uint8_t *sa, const uint8_t *b, size_t ldb,
                             const uint8_t *sb, void *y, int yt_bf16, uint32_t M, uint32_t K, uint32_t N,
                             const Fp4Plan &plan, float *part, hipStream_t stream) {
  if (plan.tile == FP4_T_SKINNY) {
    const Fp4Skinny p = {a, sa, b, sb, y, lda, ldb, M, K, N, 0};
    return yt_bf16 ? skinny_any<uint16_t>(plan.per, p, stream) : skinny_any<float>(plan.per, p, stream);
  }
  const DenseArgs p = {a, b, sa, sb, y, plan.S > 1 ? part : nullptr, lda, ldb, M, K, N, plan.per};
  const hipError_t e = yt_bf16 ? dense_tile<uint16_t>(plan.tile, p, plan.S, stream) : dense_tile<float>(plan.tile, p, plan.S, stream);
  if (e != hipSuccess || plan.S == 1) return e;
  const size_t n = (size_t)M * N;
  const dim3 grid((unsigned)((n + 1023) / 1024));
  if (yt_bf16) hipLaunchKernelGGL(join_parts_kernel<uint16_t>, grid, dim3(256), 0, stream, part, plan.S, n, (uint16_t *)y);
  else hipLaunchKernelGGL(join_parts_kernel<float>, grid, dim3(256), 0, stream, part, plan.S, n, (float *)y);
  return hipGetLastError();
}

bool fp4_act_fits(uint32_t M, uint32_t K) {
  return M <= FP4_ACT_MAX_M && fp4_skinny_act_bytes(M, K) <= FP4_ACT_MAX_BYTES;
}

hipError_t launch_fp4_linear_act(const void *x, int xt_bf16, const uint8_t *b, size_t ldb, const uint8_t *sb, void *y,
                                 int yt_bf16, uint32_t M, uint32_t K, uint32_t N, const Fp4Plan &plan,
                                 hipStream_t stream) {
  const int vec = ((reinterpret_cast<uintptr_t>(x) | (size_t)K * (xt_bf16 ? 2 : 4)) & 15) == 0;
  const Fp4Skinny p = {x, nullptr, b, sb, y, K, ldb, M, K, N, vec};
  if (xt_bf16)
    return yt_bf16 ? skinny_go<1, uint16_t, uint16_t>(plan.per, p, stream) : skinny_go<1, uint16_t, float>(plan.per, p, stream);
  return yt_bf16 ? skinny_go<1, float, uint16_t>(plan.per, p, stream) : skinny_go<1, float, float>(plan.per, p, stream);
}

hipError_t launch_fp4_grouped(const uint8_t *a, size_t lda, const uint8_t *sa, const uint8_t *const *b, size_t ldb,
                              const uint8_t *const *sb, const uint32_t *offsets, int E, void *y, int yt_bf16,
                              uint32_t R, uint32_t K, uint32_t N, int cus, hipStream_t stream) {
  GroupArgs p = {a, sa, y, offsets, lda, ldb, R, K, N, E, {}, {}};
  for (int e = 0; e < E; e++) {
    p.b[e] = b[e];
    p.sb[e] = sb[e];
  }
  const int tile = fp4_grouped_tile(R, K, N, (uint32_t)E, cus);
  return yt_bf16 ? grouped_any<uint16_t>(p, tile, stream) : grouped_any<float>(p, tile, stream);
}

}  // namespace frx
