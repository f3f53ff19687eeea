// frx_policy.hpp — host-side rules: the sizes of the context workspaces, the
// kernels of the decode FFN and those of the 8-bit linears, kept free of HIP so
// that a CPU build can check them.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <cmath>

namespace frx {

// Size to allocate when a workspace of `have` bytes must hold `need`:
// at least 1.5x the old size (rounded to 256 bytes), so that a run of rising
// requests makes O(log(max / first)) allocations and the buffers it retires
// sum to less than twice the final size.
inline size_t grow_bytes(size_t have, size_t need) {
  const size_t a = (need + 255) & ~(size_t)255;
  if (need <= have) return have;
  const size_t g = have + have / 2;
  const size_t b = (g + 255) & ~(size_t)255;
  return b > a ? b : a;
}

// ---- the FFN of 1-16 tokens: gate and up over K columns and N rows each, then
// the down projection (times are of the whole FFN, hidden / intermediate) -------

// bf16 tokens from which gate and up leave the kernel with operand loads for the
// staged one (gemv_xs_kernel), 8 where it is not ahead from 5 or 6. Writing h as
// planes (the FFN): over 2048 to 4096 columns past 4096 rows (4096 / 14336, 5 / 7
// tokens 25.9 / 27.4 us with operand loads, 24.4 / 23.7 staged; 2560 / 8192 15.9 / 16.7
// and 15.4 / 15.6; over fewer rows the FFN is level). Writing fp32 h
// (frx_ternary_glu): past 8192 rows, and below where the columns fill its waves'
// quads (2816 / 12288 8.1 / 8.5 and 7.6 / 7.6, 4096 / 5632 7.6 / 7.9 and 7.1 / 7.1; but
// 3328 / 5632 6.4 / 6.6 and 7.0 / 6.9, 2432 / 5632 5.8 / 6.0 and 6.9 / 6.9). Below 2048
// columns a workgroup's few quads leave its waves idle (FFN 1024 / 2048, 5 tokens
// 8.8 against 9.3). Above 4096 its x outweighs its rows (FFN 5120 / 4096, 5 / 7 tokens
// 16.1 / 14.0 against 17.1 / 14.6, 5120 / 13824 28.3 / 30.5 against 29.8 / 30.2) but
// where the FFN gives each unit two tiles of them (5120 / 5632, 5 / 6 / 7 tokens 17.9 /
// 18.5 / 18.9 against 18.0 / 17.9 / 17.9, 5120 / 8192 20.0 / 20.7 / 21.2 against 20.2 /
// 20.6 / 20.5). fp32 h leaves the operand loads there only where rows that are no
// multiple of 16 bytes narrow them (5 / 7 tokens: 4432 / 5632 11.3 / 12.3 against 9.6 /
// 9.5, 5136 / 8192 12.6 / 14.6 against 10.0 / 10.1; 4416 / 5632 7.8 / 8.7 against 9.5 /
// 9.5, 5120 / 5632 8.8 / 9.8 against 9.7 / 9.7).
constexpr int glu_staged_min_tokens(int K, int N, bool planes) {
  if (K < 2048) return 8;
  if (K > 4096 && (N <= 4096 || N > 8192)) return 8;
  if (K > 4096) return planes ? 6 : K % 64 != 0 ? 5 : 8;
  if (planes) return N > 4096 ? 5 : 8;
  return N > 8192 || (K > 3840 && N > 4096) ? 5 : 8;
}

// Whether one f32 token takes the staged kernel: not over more than 4096
// columns (5120 / 13824 31.8 us with the 16-row tiles, 35.9 staged) nor, where
// short rows make a workgroup's start its time, over more than 4096 rows (1024 /
// 5632 8.7 and 9.7, 1024 / 13824 12.1 and 13.7; but 1024 / 4096 7.7 and 7.6, 3072 /
// 11008 18.0 and 16.6).
constexpr bool glu_staged_one_f32(int K, int N) { return K <= 4096 && (K > 2048 || N <= 4096); }

// Most 16-row tiles of both matrices in a workgroup of the staged kernel (its
// weight registers allow 4 up to 4096 columns, 2 up to 8192, 1 above). bf16 x:
// not so many that the fullest compute unit gets more of them, and where three
// do not hold a unit's rows, two workgroups of two on it (their loads overlap)
// before one of four. 5 / 16 tokens: 5120 / 11008, one tile 24.9 / 28.3 us, two
// (344 workgroups, four tiles on the units that have two) 29.4 / 31.3; 5120 / 5632
// 18.4 / 20.5 against 18.0 / 20.3; 4096 / 13824, two 21.7 / 24.8, four 22.1 / 25.6;
// 4096 / 11008, two 20.8 / 23.9, three 19.3 / 22.2. f32 x has one workgroup per
// unit anyway (LDS) and keeps the most tiles (2048 / 13824, 5 tokens 17.5 us with
// four, 20.2 with two).
constexpr int glu_staged_tiles(int K, int N, bool bf16, int cus) {
  if (K > 8192) return 1;
  if (K > 4096) {
    const int one = ((N + 15) / 16 + cus - 1) / cus, two = 2 * (((N + 31) / 32 + cus - 1) / cus);
    return bf16 && two > one ? 1 : 2;
  }
  return bf16 && N > 48 * cus ? 2 : 4;
}

// Intermediate from which the down projection of `tokens` is split over K. Up to
// 8 tokens, whose planes share the 16 columns (whole rows / split: 4096 / 5632, 5 / 8
// tokens 18.3 / 15.9 and 14.9 / 15.1 us; 2048 / 5632 16.5 / 14.0 and 13.1 / 13.3),
// and above over H output rows whose 16-row tiles are few or past one round of
// the compute units (12 / 16 tokens: 1024 / 5632 14.1 / 14.5 and 12.8 / 13.6, 5120 /
// 5632 20.4 / 20.8 and 19.4 / 20.3; but 3072 / 5632 16.2 / 16.6 and 17.3 / 18.4, 4096 /
// 5632 16.3 / 16.9 and 16.3 / 17.0, 2048 / 5632 14.5 / 14.8 and 14.4 / 15.0).
constexpr int ffn_down_split_min(int tokens, int H, int cus) {
  return tokens <= 8 || H < 2048 || H > 16 * cus ? 4097 : 8192;
}

// ---- the staged kernel over one matrix, 2-16 tokens ----------------------------

// Most 16-row tiles of a workgroup, by its weight registers (planes: 2 for f32 x).
constexpr int linear_staged_tiles(int K, int planes) {
  return planes == 1 ? (K <= 8192 ? 4 : 2) : K <= 4096 ? 4 : K <= 8192 ? 2 : 1;
}

// Rounds of workgroups, one to a compute unit, over `tiles` 16-row tiles: a
// workgroup per unit while it holds them, else as many as hold them.
constexpr int staged_rounds(int tiles, int tmax, int cus) {
  return tiles <= tmax * cus ? 1 : ((tiles + tmax - 1) / tmax + cus - 1) / cus;
}

// Whether one launch over the tiles of a group's matrices takes fewer rounds
// than a launch for each: above 8192 columns a workgroup holds two tiles, and
// two launches of one round are ahead of one of two (5 / 16 bf16 tokens, us, apart /
// one launch: 5504 and 2752 rows of 9216 15.4 / 15.9 and 16.9 / 17.3, 8192 and
// 4096 rows of 11008 17.6 / 18.5 and 18.9 / 19.3; but 3 x 5440 of 11008 30.3 / 31.5
// and 21.0 / 21.4, 2 x 4096 of 11008 15.0 / 15.4 and 10.2 / 10.6).
constexpr bool group_fewer_rounds(int count, const int *n, int K, int planes, int cus) {
  const int tmax = linear_staged_tiles(K, planes);
  int tiles = 0, apart = 0;
  for (int i = 0; i < count; i++) {
    tiles += (n[i] + 15) / 16;
    apart += staged_rounds((n[i] + 15) / 16, tmax, cus);
  }
  return staged_rounds(tiles, tmax, cus) < apart;
}

// ---- the 8-bit floating-point linears --------------------------------------------

enum { FP8_T_SKINNY = 0, FP8_T_128 = 1, FP8_T_RING8 = 2, FP8_T_RING6 = 3, FP8_T_RING4 = 4, FP8_T_64 = 5 };
struct Fp8Plan {
  int tile;     // FP8_T_*
  int S, per;   // K slices, blocks of 128 in each (FP8_T_SKINNY: 1, 16-row tiles of a workgroup)
};

// Tiles of many tokens: height x width, workgroups resident at once on a
// compute unit, and what a step of 128 columns takes (ns, all of them resident;
// 8192^3, 2048 x 4096 x 11008 and 4096^3). On the 8-bit pipe a taller tile costs
// less per product, and a smaller one pays where the taller would leave units
// idle (us, 256 / 192 / 128 / 128 x 128: 8192^3 374 / 432 / 517 / 570, 2048 x 4096 x
// 11008 105 / 88 / 110 / 126, 2048 x 4096 x 4096 53 / 43 / 37 / 49, 4096^3 53 / 78 / 76 /
// 90). Long products run into the card's power: 8192^3 takes 350 us on zeros
// (3140 TFLOP/s) and 460 on normal values; a library's product with one scale for
// all takes 257 and 348. On the bf16 pipe widening the operands bounds them all
// (8192^3 931 / 952 / 998 us for 192 / 128 / 128 x 128, 2048 x 4096 x 11008 158 / 175 /
// 174, 2048 x 4096 x 4096 80 / 61 / 63, 4096^3 158 / 119 / 119).
struct Fp8TileCost {
  int tile, bm, bn, wgs, ns;
};
constexpr Fp8TileCost kFp8Narrow[] = {{FP8_T_RING8, 256, 256, 1, 1460}, {FP8_T_RING6, 192, 256, 1, 1130},
                                {FP8_T_RING4, 128, 256, 1, 1010}, {FP8_T_128, 128, 128, 2, 1110}};
constexpr Fp8TileCost kFp8Wide[] = {{FP8_T_RING6, 192, 256, 1, 2600}, {FP8_T_RING4, 128, 256, 1, 1800},
                              {FP8_T_128, 128, 128, 2, 1870}};
// A scale per weight row (weight gradients): sixteen more multiplies a product,
// taller tiles run out of registers; on the bf16 pipe 128 x 256 takes 2200.
constexpr Fp8TileCost kFp8NarrowRows[] = {{FP8_T_RING4, 128, 256, 1, 1010}, {FP8_T_128, 128, 128, 2, 1110}};
constexpr Fp8TileCost kFp8WideRows[] = {{FP8_T_128, 128, 128, 2, 2150}};

// pipe8: the 8-bit pipe may sum (bf16 outputs under FRX_FP8_SUMS_PIPE), here and below.
inline Fp8Plan fp8_plan(uint32_t M, uint32_t K, uint32_t N, int b_rows, int pipe8, int cus) {
  // Few tokens: no join, no tile of 128 mostly empty. Up to 32 always (us, against the tiles, which split K here, on
  // the bf16 pipe / on the 8-bit one: 32 tokens, K x N 1024^2 4.3 / 10.5 / 9.6, 4096^2 10.4 / 17.6 / 14.7, 4096 x 11008
  // 16.5 / 22.4 / 17.4, 11008 x 4096 22.2 / 27.9 / 20.1), up to 64 while two row tiles a workgroup cover N and the waves'
  // slices of K are short, since every workgroup reads all tokens (64 tokens, 1024^2 5.9 / 11.9 / 10.8, 4096^2 14.9 /
  // 21.1 / 17.5, 4096 x 8192 18.7 / 22.7 / 18.9, f32 2048 x 5632 11.0 / 19.5; 40 tokens f32 5120^2 20.5 / 21.4; but 64 tokens
  // 8192 x 4096 26.2 / 24.7, 11008 x 4096 33.1 / 29.9 / 22.4), more in groups of 64 while two rounds of workgroups hold
  // them and K is short for that (128 tokens, 2048^2 8.6 / 18.6 / 14.6, 4096 x 2048 13.3 / 21.2 / 17.5, 2048 x 4096 14.1 /
  // 21.0 / 16.6; 256 tokens, 2048^2 14.0 / 20.2 / 16.9, f32 2048 x 1024 8.6 / 18.4; 512 tokens, 1024^2 9.4 / 17.9 / 13.3; but
  // 128 tokens 4096^2 23.2 / 24.9 / 22.6, 256 tokens 5120 x 2048 28.9 / 26.1 / 21.1). The 8-bit pipe's tiles set the lines;
  // beside the bf16 pipe's they could lie at 52 blocks of a slice (6656 x 4096 21.8 / 23.9) and 64 of a round.
  const int steps = (int)((K + 127) / 128), most = M <= 32 ? 4 : 2;  // row tiles a workgroup
  const size_t rounds64 = ((size_t)((M + 63) / 64) * ((N + 15) / 16) + cus - 1) / cus;
  if (M <= 32 || (M <= 64 && N <= 32u * cus && steps <= 40) || (rounds64 <= 2 && rounds64 * steps <= 40)) {
    // the fewest rounds of row tiles on the fullest compute unit; of equals the most tiles a workgroup
    const uint32_t tiles = (N + 15) / 16;
    int best = 1;
    uint32_t least = ~0u;
    for (int rt = 1; rt <= most; rt++) {
      const uint32_t wgs = (tiles + rt - 1) / rt, rounds = (wgs + cus - 1) / cus * rt;
      if (rounds <= least) {
        least = rounds;
        best = rt;
      }
    }
    return {FP8_T_SKINNY, 1, best};
  }
  const Fp8TileCost *costs = b_rows == 1 ? (pipe8 ? kFp8NarrowRows : kFp8WideRows) : pipe8 ? kFp8Narrow : kFp8Wide;
  const int count = b_rows == 1 ? (pipe8 ? 2 : 1) : pipe8 ? 4 : 3;
  Fp8Plan plan = {FP8_T_128, 1, steps};
  double least = 1e30;
  for (int t = 0; t < count; t++) {
    const Fp8TileCost &c = costs[t];
    const double tiles = (double)((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    // a K slice more: fewer steps, but every part is written and read (4 bytes a value at
    // about 4 TB/s) and the parts joined by another launch (4 us)
    for (int S = 1; S <= 8 && S <= steps; S++) {
      const int per = (steps + S - 1) / S;
      if ((S - 1) * per >= steps) continue;  // an empty slice
      const double rounds = std::ceil(tiles * S / ((double)c.wgs * cus));
      const double ns = rounds * per * c.ns + (S > 1 ? 4000.0 + (double)S * M * N * 8 / 4000 : 0.0);
      if (ns < least) {
        least = ns;
        plan = {c.tile, S, per};
      }
    }
  }
  return plan;
}

// The tile of the experts' products. On the bf16 pipe 64 x 128: widening bounds every tile
// alike. bf16 rows of e4m3 codes that the caller lets the 8-bit pipe sum go there from 256
// rows an expert on (R / E: the groups' lengths are not known here), where the products
// bound, in tiles of 128 or 256 x 256, priced for groups of equal length with half a tile
// of remainder; below, the weights' bytes bound and it would gain little. us, K -> N, bf16
// pipe 64 x 128 / 8-bit 64 x 128 / 128 x 256 / 256 x 256:
//   8 experts   128 rows 2048 -> 5632    44 /  42 /  45 /  33
//               256 rows 2048 -> 5632     - /  59 /  49 /  66
//               384 rows 2048 -> 5632    92 /  77 /  72 /  72
//              1024 rows 2048 -> 5632   218 / 173 / 143 / 143
//   16 experts   64 rows 5632 -> 2048    62 /  61 /  55 /  61
//                64 rows 2048 -> 5632     - /  54 /  52 /  63
//   16 experts of 64 rows padded to 128, 5632 -> 2048    64 / 62 / 61 / 67
// Other tiles of the bf16 pipe (128 x 128 / 128 x 256): 8 x 128 rows 53 / 66, 8 x 1024
// 205 / 205, 16 x 64 padded to 128 87 / 77.
inline double fp8_grouped_cost(uint32_t R, uint32_t N, uint32_t E, uint32_t bm, uint32_t bn, double ns, int cus) {
  const double tiles = E * ((double)R / E / bm + 0.5) * ((N + bn - 1) / bn);
  return ns * std::ceil(tiles / cus);
}

// Experts' rows: tiles of 16 where R / E is small (us, 8 experts, 16-row tiles / 64 x 128: 2
// rows 5632 -> 2048 19.4 / 40.1, 2048 -> 5632 20.7 / 21.2, 1024^2 5.1 / 8.2; 8 rows 22.5 / 40.1,
// 24.2 / 21.3, 5.4 / 8.1) and the launch holds its workgroups of 512 (less than 2^32
// work-items).
inline int fp8_grouped_tile(uint32_t R, uint32_t N, uint32_t E, int pipe8, int cus) {
  if (R <= 8 * E && ((size_t)(R + 15) / 16 + E) * ((N + 15) / 16) < (size_t)1 << 23) return FP8_T_SKINNY;
  if (!pipe8 || R < 256 * E) return FP8_T_64;
  return fp8_grouped_cost(R, N, E, 256, 256, 1460, cus) < fp8_grouped_cost(R, N, E, 128, 256, 1010, cus) ? FP8_T_RING8
                                                                                                        : FP8_T_RING4;
}

}  // namespace frx
