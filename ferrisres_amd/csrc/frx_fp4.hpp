// frx_fp4.hpp — what the products of the 4-bit floating-point linears share.
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
// are one block.
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

// ---- stores of y, and a barrier ----------------------------------------------------

// Four sums of a row of y, from d on (any element), of which `left` are the row's. One store at
// any address: with an odd N single values cost 2048 x 4096 x 11010 94 us instead of 71.
typedef uint64_t __attribute__((aligned(2))) u64_u;
__device__ __forceinline__ void fp4_store4(float *d, const f32x4 &v, uint32_t left) {
  if (left >= 4) *reinterpret_cast<u32x4_u *>(d) = __builtin_bit_cast(u32x4, v);
  else
    for (uint32_t e = 0; e < left; e++) d[e] = v[e];
}
__device__ __forceinline__ void fp4_store4(uint16_t *d, const f32x4 &v, uint32_t left) {
  uint32_t h[4];
#pragma unroll
  for (int e = 0; e < 4; e++) h[e] = bf16_rne_nb(v[e]);
  if (left >= 4) *reinterpret_cast<u64_u *>(d) = (uint64_t)(h[2] | (h[3] << 16)) << 32 | (h[0] | (h[1] << 16));
  else
    for (uint32_t e = 0; e < left; e++) d[e] = (uint16_t)h[e];
}

// Two pieces of 16 sums of a row that 4 lane groups hold, 4 of each a group, as bf16: group g gets the 8
// from 8 g on, which lie behind one another in y.
__device__ __forceinline__ u32x4 fp4_join8(const f32x4 &v, const f32x4 &w) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t p = bf16_rne_nb(v[2 * i]) | (bf16_rne_nb(v[2 * i + 1]) << 16);
    const uint32_t q = bf16_rne_nb(w[2 * i]) | (bf16_rne_nb(w[2 * i + 1]) << 16);
    const auto a = __builtin_amdgcn_permlane32_swap(p, q, false, false);        // groups 2, 3 of p with 0, 1 of q
    const auto b = __builtin_amdgcn_permlane16_swap(a[0], a[1], false, false);  // groups 1, 3 with 0, 2
    o[i] = b[0];
    o[2 + i] = b[1];
  }
  return o;
}

// A barrier that waits for this wave's LDS accesses alone: __syncthreads() would wait for the
// weights on their way too.
__device__ __forceinline__ void barrier_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace frx
