// frx_tiles.hpp — what the 8-bit and the 4-bit products share around their tile engines:
// which tile a workgroup takes, whose rows it holds, and the join of K slices.
#pragma once
#include "frx_device.hpp"

namespace frx {

// Whether rows of n elements from y on are whole aligned quads.
template <typename YT>
__device__ __forceinline__ bool quads(const void *y, uint32_t n) {
  return ((reinterpret_cast<uintptr_t>(y) & (4 * sizeof(YT) - 1)) | (n & 3)) == 0;
}

// The tile of workgroup `bid` of mts x nts. Hardware deals workgroups out to the
// 8 XCDs in turn; each XCD gets a contiguous run of tiles, ordered by groups of
// GM tiles of tokens, within a group down the tokens first, so that the tiles
// an XCD works on at a time share rows of both sides in its L2.
template <int GM>
__device__ __forceinline__ void xcd_tile(uint32_t bid, uint32_t mts, uint32_t nts, uint32_t &mt, uint32_t &nt) {
  const uint32_t total = mts * nts, q = total / 8, r = total % 8, xcd = bid % 8, i = bid / 8;
  const uint32_t lin = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + i;
  const uint32_t rows = min((uint32_t)GM, mts);  // (GM * nts may pass 32 bits)
  const uint32_t group = lin / (rows * nts), rest = lin - group * (rows * nts);
  const uint32_t gm = min(rows, mts - group * rows);
  nt = rest / gm;
  mt = group * rows + rest - nt * gm;
}

// Expert e's rows [first, end), kept inside the R rows there are.
__device__ __forceinline__ void expert_rows(const uint32_t *offsets, int e, uint32_t R, uint32_t &first,
                                            uint32_t &end) {
  first = min(offsets[e], R);
  end = max(min(offsets[e + 1], R), first);
}

// Every expert's rows cut into tiles of BM. Lane e holds expert e's; the expert of a tile is
// the first whose running count passes it.
template <int BM>
struct ExpertTiles {
  uint32_t first, last, before, upto;
  __device__ __forceinline__ ExpertTiles(const uint32_t *offsets, int E, uint32_t R) {
    const int lane = threadIdx.x & 63;
    first = last = 0;
    if (lane < E) expert_rows(offsets, lane, R, first, last);
    const uint32_t tiles = (last - first + BM - 1) / BM;
    upto = tiles;
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t v = (uint32_t)__shfl_up((int)upto, s);
      if (lane >= s) upto += v;
    }
    before = upto - tiles;
  }
  __device__ __forceinline__ uint32_t total() const { return (uint32_t)__builtin_amdgcn_readlane((int)upto, 63); }
  // Tile mt's expert, its first row and its expert's last + 1; -1 past the last tile.
  __device__ __forceinline__ int find(uint32_t mt, uint32_t &m0, uint32_t &end) const {
    const unsigned long long past = __ballot(upto > mt);
    if (past == 0) return -1;
    const int e = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
    m0 = (uint32_t)__builtin_amdgcn_readlane((int)first, e) + (mt - (uint32_t)__builtin_amdgcn_readlane((int)before, e)) * BM;
    end = (uint32_t)__builtin_amdgcn_readlane((int)last, e);
    return e;
  }
};

template <int BM>
__device__ __forceinline__ int expert_tile(const uint32_t *offsets, int E, uint32_t R, uint32_t mt, uint32_t &m0,
                                           uint32_t &end) {
  return ExpertTiles<BM>(offsets, E, R).find(mt, m0, end);
}

// y = the parts added in order, four values a thread (n of them, parts n apart).
template <typename YT>
static __global__ __launch_bounds__(256) void join_parts_kernel(const float *__restrict__ part, int S, size_t n,
                                                       YT *__restrict__ y) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  if (((n & 3) | (reinterpret_cast<uintptr_t>(y) & (4 * sizeof(YT) - 1))) == 0) {
    f32x4 v = *reinterpret_cast<const f32x4 *>(part + i);
    for (int s = 1; s < S; s++) v += *reinterpret_cast<const f32x4 *>(part + (size_t)s * n + i);
    if constexpr (sizeof(YT) == 4) {
      *reinterpret_cast<f32x4 *>(y + i) = v;
    } else {
      *reinterpret_cast<u32x2 *>(y + i) = (u32x2){bf16_rne_nb(v[0]) | (bf16_rne_nb(v[1]) << 16),
                                                 bf16_rne_nb(v[2]) | (bf16_rne_nb(v[3]) << 16)};
    }
    return;
  }
  for (size_t k = i; k < n && k < i + 4; k++) {
    float v = part[k];
    for (int s = 1; s < S; s++) v += part[(size_t)s * n + k];
    if constexpr (sizeof(YT) == 4) y[k] = v;
    else y[k] = (uint16_t)bf16_rne_nb(v);
  }
}

}  // namespace frx
