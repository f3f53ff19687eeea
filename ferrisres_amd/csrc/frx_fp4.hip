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

// A workgroup's tile.
template <typename Tile, typename YT>
struct DenseItem {
  const DenseArgs &p;
  uint32_t m0, n0, mr, nr;
  int span, t0, t1;
  __device__ __forceinline__ DenseItem(const DenseArgs &args) : p(args) {
    uint32_t mt, nt;
    xcd_tile<8>(blockIdx.x, (p.M + Tile::BM - 1) / Tile::BM, (p.N + Tile::BN - 1) / Tile::BN, mt, nt);
    m0 = mt * Tile::BM;
    n0 = nt * Tile::BN;
    mr = min((uint32_t)Tile::BM, p.M - m0);
    nr = min((uint32_t)Tile::BN, p.N - n0);
    const int steps = (int)((p.K + 255) >> 8);
    t0 = p.part ? (int)blockIdx.z * p.per : 0;
    t1 = p.part ? min(t0 + p.per, steps) : steps;
    span = t1 - t0;
  }
  __device__ __forceinline__ bool at(int, Fp4Operands &o) const {
    fill_operands(o, p.a, p.lda, p.sa, p.b, p.ldb, p.sb, m0, mr, n0, nr, p.K);
    o.t0 = t0;
    o.t1 = t1;
    return true;
  }
  __device__ __forceinline__ bool take(int, int &from, int &to) const {
    from = t0;
    to = t1;
    return true;
  }
  template <typename Acc>
  __device__ __forceinline__ void store(const Acc &acc) const {
    const size_t at = (size_t)m0 * p.N + n0;
    if (p.part)
      Tile::template store<float>(acc, p.part + (size_t)blockIdx.z * p.M * p.N + at, p.N, (int)mr, (int)nr);
    else Tile::template store<YT>(acc, (YT *)p.y + at, p.N, (int)mr, (int)nr);
  }
};

template <typename Tile, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp4_dense_kernel(const DenseArgs p) {
  extern __shared__ __align__(16) uint32_t lds[];
  DenseItem<Tile, YT> item(p);
  Tile::template run<false>(lds, item);
}

// Rows sorted by expert, each expert's in tiles of their own.
struct GroupArgs {
  const uint8_t *a, *sa;
  void *y;
  const uint32_t *offsets;
  size_t lda, ldb;
  uint32_t R, K, N;
  int E;
  const uint8_t *b[FP8_MAXE], *sb[FP8_MAXE];
};

// A workgroup's tiles: every gridDim.x-th of all. An XCD's run of them goes down the rows
// first: the tiles of an expert's rows share its weights in that L2.
template <typename Tile, typename YT>
struct GroupItems {
  const GroupArgs &p;
  const ExpertTiles<Tile::BM> rows;
  const uint32_t mts, nts;
  const int steps, span;
  uint32_t m0, end, n0;  // of the tile whose sums come next
  __device__ __forceinline__ GroupItems(const GroupArgs &args)
      : p(args), rows(p.offsets, p.E, p.R), mts(rows.total()), nts((p.N + Tile::BN - 1) / Tile::BN),
        steps((int)((p.K + 255) >> 8)), span((steps + 1) & ~1) {}
  __device__ __forceinline__ int where(int i, uint32_t &first, uint32_t &last, uint32_t &col) const {
    const uint32_t at = blockIdx.x + (uint32_t)i * gridDim.x;
    if (at >= mts * nts) return -1;
    uint32_t mt, nt;
    xcd_tile<0x40000000>(at, mts, nts, mt, nt);
    col = nt * Tile::BN;
    return rows.find(mt, first, last);
  }
  __device__ __forceinline__ bool at(int i, Fp4Operands &o) const {
    uint32_t first, last, col;
    const int e = where(i, first, last, col);
    if (e < 0) return false;
    fill_operands(o, p.a, p.lda, p.sa, p.b[e], p.ldb, p.sb[e], first, min((uint32_t)Tile::BM, last - first), col,
                  min((uint32_t)Tile::BN, p.N - col), p.K);
    o.t0 = 0;
    o.t1 = steps;
    return true;
  }
  __device__ __forceinline__ bool take(int i, int &from, int &to) {
    from = 0;
    to = steps;
    return where(i, m0, end, n0) >= 0;
  }
  template <typename Acc>
  __device__ __forceinline__ void store(const Acc &acc) const {
    Tile::template store<YT>(acc, (YT *)p.y + (size_t)m0 * p.N + n0, p.N, (int)min((uint32_t)Tile::BM, end - m0),
                             (int)min((uint32_t)Tile::BN, p.N - n0));
  }
};

// MANY: as many workgroups as are resident at once take tiles in turn. Rows of 16 experts, 2048 x
// 5632, 1024 rows of uneven experts 37.6 -> 32.8 us, 2048 rows 45.3 -> 41.7, 64 rows in four
// experts 12.1 -> 10.2. Not for 256 x 256, which then spills 76 registers (a dense 4096^3 43 -> 164
// us), nor for the dense product, whose prologue looks up no expert (1024 x 4096 x 4096 20.0 -> 21.1,
// 1999 x 11008 x 4096 58 -> 68).
template <typename Tile, typename YT, bool MANY>
__global__ __launch_bounds__(Tile::NT, 2) void fp4_grouped_kernel(const GroupArgs p) {
  extern __shared__ __align__(16) uint32_t lds[];
  GroupItems<Tile, YT> items(p);
  Tile::template run<MANY>(lds, items);
}

// Weight gradients: expert blockIdx.y's sums over its rows, whose columns of the codes begin at
// a multiple of 128 (so codes and scales begin at whole 64 and 4 bytes). Here the engine's tokens are
// dw's rows (dy's columns) and its weight rows x's columns. Bound by writing dw where experts have few
// rows: 16 x 128 rows, 5632 x 2048, f32 166 us (738 MB, 4.4 TB/s), bf16 122; 8 x 1024 rows, 2048 x 5632
// 142 and 104. Tiles in turn gained nothing (128 x 256 176 us, 256 x 256 spills).
struct GradArgs {
  const uint8_t *a, *b, *sa, *sb;
  const uint32_t *offsets;
  size_t lda, ldb;
  uint32_t R, N, K;
  void *dw[FP8_MAXE];
};

template <typename Tile, typename YT>
struct GradItem {
  const GradArgs &p;
  uint32_t m0, n0, mr, nr, first, len;
  int span;
  __device__ __forceinline__ GradItem(const GradArgs &args) : p(args) {
    uint32_t mt, nt, end;
    xcd_tile<8>(blockIdx.x, (p.N + Tile::BM - 1) / Tile::BM, (p.K + Tile::BN - 1) / Tile::BN, mt, nt);
    m0 = mt * Tile::BM;
    n0 = nt * Tile::BN;
    mr = min((uint32_t)Tile::BM, p.N - m0);
    nr = min((uint32_t)Tile::BN, p.K - n0);
    expert_rows(p.offsets, blockIdx.y, p.R, first, end);
    len = end > first ? (end - (first & ~127u)) & ~31u : 0;
    first &= ~127u;
    span = (int)((len + 255) >> 8);
  }
  __device__ __forceinline__ bool at(int, Fp4Operands &o) const {
    o.s_ld = fp4_scale_bytes(p.R);
    o.a = p.a + (size_t)m0 * p.lda + first / 2;
    o.b = p.b + (size_t)n0 * p.ldb + first / 2;
    o.sa = p.sa + (size_t)m0 * o.s_ld + first / 32;
    o.sb = p.sb + (size_t)n0 * o.s_ld + first / 32;
    o.lda = (uint32_t)p.lda;
    o.ldb = (uint32_t)p.ldb;
    o.a_rows = (int)mr;
    o.b_rows = (int)nr;
    o.K = (int)len;
    o.t0 = 0;
    o.t1 = span;
    return true;
  }
  __device__ __forceinline__ bool take(int, int &from, int &to) const {
    from = 0;
    to = span;
    return true;
  }
  template <typename Acc>
  __device__ __forceinline__ void store(const Acc &acc) const {
    Tile::template store<YT>(acc, static_cast<YT *>(p.dw[blockIdx.y]) + (size_t)m0 * p.K + n0, p.K, (int)mr, (int)nr);
  }
};

template <typename Tile, typename YT>
__global__ __launch_bounds__(Tile::NT, 2) void fp4_grad_kernel(const GradArgs p) {
  extern __shared__ __align__(16) uint32_t lds[];
  GradItem<Tile, YT> item(p);
  Tile::template run<false>(lds, item);
}

template <int RT, int TT, typename XT, typename YT>
__global__ __launch_bounds__(FP4_SK_WAVES * 64) void fp4_skinny_kernel(const Fp4Skinny p) {
  extern __shared__ __align__(16) uint32_t lds[];
  fp4_skinny<RT, TT, XT, YT>(p, blockIdx.x * 16 * RT, reinterpret_cast<f32x4 *>(lds));
}

// Workgroups for so many tiles: as many as are resident at once, a multiple of the XCDs.
template <typename Tile>
unsigned resident(size_t tiles, int cus) {
  const size_t most = max(8, (160 << 10) / Tile::LDS_BYTES * cus & ~7);
  return (unsigned)min(tiles, most);
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
  constexpr size_t most = FP4_ACT_MAX_VALUES / 2 + FP4_ACT_MAX_VALUES / 32 + 4 * FP4_ACT_MAX_M;  // fp4_skinny_act_bytes
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel), (int)(red + (sizeof(XT) == 1 ? 0 : most)), done);
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

template <typename Tile, typename YT, bool MANY>
hipError_t grouped_go(const GroupArgs &p, int cus, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const size_t mts = (size_t)(p.R + Tile::BM - 1) / Tile::BM + p.E, tiles = mts * ((p.N + Tile::BN - 1) / Tile::BN);
  if ((MANY ? tiles : tiles * Tile::NT) > 0xF0000000u) return hipErrorInvalidValue;  // (counted in 32 bits)
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(fp4_grouped_kernel<Tile, YT, MANY>), Tile::LDS_BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((fp4_grouped_kernel<Tile, YT, MANY>), dim3(MANY ? resident<Tile>(tiles, cus) : (unsigned)tiles), dim3(Tile::NT), Tile::LDS_BYTES,
                     stream, p);
  return hipGetLastError();
}

template <typename YT>
hipError_t grouped_any(const GroupArgs &p, int tile, int cus, hipStream_t stream) {
  switch (tile) {
    case FP4_T_256X256: return grouped_go<Tile256x256, YT, false>(p, cus, stream);
    case FP4_T_128X256: return grouped_go<Tile128x256, YT, true>(p, cus, stream);
    case FP4_T_64X128: return grouped_go<Tile64x128, YT, true>(p, cus, stream);
    default: return grouped_go<Tile64x64, YT, true>(p, cus, stream);
  }
}

template <typename Tile, typename YT>
hipError_t grad_go(const GradArgs &p, int E, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const size_t tiles = (size_t)((p.N + Tile::BM - 1) / Tile::BM) * ((p.K + Tile::BN - 1) / Tile::BN);
  if (tiles * Tile::NT > 0xFFFFFFFFu) return hipErrorInvalidValue;
  const auto kernel = fp4_grad_kernel<Tile, YT>;
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel), Tile::LDS_BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, E), dim3(Tile::NT), Tile::LDS_BYTES, stream, p);
  return hipGetLastError();
}

template <typename YT>
hipError_t grad_any(const GradArgs &p, int tile, int E, hipStream_t stream) {
  if (tile == FP4_T_256X256) return grad_go<Tile256x256, YT>(p, E, stream);
  return tile == FP4_T_128X256 ? grad_go<Tile128x256, YT>(p, E, stream) : grad_go<Tile64x128, YT>(p, E, stream);
}

}  // namespace

hipError_t launch_fp4_linear(const uint8_t *a, size_t lda, const uint8_t *sa, const uint8_t *b, size_t ldb,
                             const uint8_t *sb, void *y, int yt_bf16, uint32_t M, uint32_t K, uint32_t N,
                             const Fp4Plan &plan, float *part, hipStream_t stream) {
  if (plan.tile == FP4_T_SKINNY) {
    const Fp4Skinny p = {a, sa, b, sb, y, lda, ldb, M, K, N};
    return yt_bf16 ? skinny_any<uint16_t>(plan.per, p, stream) : skinny_any<float>(plan.per, p, stream);
  }
  const DenseArgs p = {a, b, sa, sb, y, plan.S > 1 ? part : nullptr, lda, ldb, M, K, N, plan.per};
  const hipError_t e = yt_bf16 ? dense_tile<uint16_t>(plan.tile, p, plan.S, stream)
                                  : dense_tile<float>(plan.tile, p, plan.S, stream);
  if (e != hipSuccess || plan.S == 1) return e;
  const size_t n = (size_t)M * N;
  const dim3 grid((unsigned)((n + 1023) / 1024));
  if (yt_bf16) hipLaunchKernelGGL(join_parts_kernel<uint16_t>, grid, dim3(256), 0, stream, part, plan.S, n, (uint16_t *)y);
  else hipLaunchKernelGGL(join_parts_kernel<float>, grid, dim3(256), 0, stream, part, plan.S, n, (float *)y);
  return hipGetLastError();
}

bool fp4_act_fits(uint32_t M, uint32_t K) {
  return M <= FP4_ACT_MAX_M && (uint64_t)M * K <= FP4_ACT_MAX_VALUES;
}

hipError_t launch_fp4_linear_act(const void *x, int xt_bf16, const uint8_t *b, size_t ldb, const uint8_t *sb, void *y,
                                 int yt_bf16, uint32_t M, uint32_t K, uint32_t N, const Fp4Plan &plan,
                                 hipStream_t stream) {
  const Fp4Skinny p = {x, nullptr, b, sb, y, K, ldb, M, K, N};
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
  return yt_bf16 ? grouped_any<uint16_t>(p, tile, cus, stream) : grouped_any<float>(p, tile, cus, stream);
}

hipError_t launch_fp4_grad_weight(const uint8_t *a, size_t lda, const uint8_t *sa, const uint8_t *b, size_t ldb,
                                  const uint8_t *sb, const uint32_t *offsets, int E, void *const *dw, int yt_bf16,
                                  uint32_t R, uint32_t N, uint32_t K, int cus, hipStream_t stream) {
  GradArgs p = {a, b, sa, sb, offsets, lda, ldb, R, N, K, {}};
  for (int e = 0; e < E; e++) p.dw[e] = dw[e];
  const int tile = fp4_grad_tile(R, N, K, (uint32_t)E, cus);
  return yt_bf16 ? grad_any<uint16_t>(p, tile, E, stream) : grad_any<float>(p, tile, E, stream);
}

}  // namespace frx
