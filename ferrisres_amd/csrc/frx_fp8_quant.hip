// frx_fp8_quant.hip — codes and scales of the 8-bit floating-point linears.
//
// A block of 128 values (1 x 128 along a row, 128 x 1 along a column, or a
// 128 x 128 tile) shares one scale:
//   s = max(amax * f32(1 / top), 2^-126)   inv = f32(1 / s)   code = rne8(x * inv)
// each one f32 rounding. 2^-126 keeps inv finite for blocks of zeros and of
// denormals. x * inv exceeds top by at most a few f32 steps, which round to
// top. amax is the unsigned maximum of the magnitude bits: a NaN orders above
// infinity and infinity above every number, so either becomes the scale.
//
// Bound by memory: 2 or 4 bytes in and 1 out per value, about 4 VALU ops per
// value (mask, max, multiply, half a conversion). us: rows of 2048 x 5632 bf16
// 8.8 (3.9 TB/s; a large copy moves 4.7), columns of 1999 x 11008 bf16 22.7 (2.9 TB/s),
// tiles of 4096 x 11008 f32 46.8 (4.8 TB/s), their codes transposed right after,
// from the cache, 34.3.
#include "frx_fp8_codes.hpp"
#include "frx_internal.hpp"

namespace frx {

namespace {

// 1 x 128 blocks: 16 lanes a block, 8 values a lane (a wave reads 1 KB of
// bf16, 2 KB of f32 in a row of x); the 16 lanes agree on amax with four
// exchanges inside their row of lanes. VEC: x rows 16-byte aligned.
template <typename XT, bool E5M2, bool VEC>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const XT *__restrict__ x, uint32_t M, uint32_t K, size_t ldx,
                                                       uint32_t kb, uint8_t *__restrict__ q, size_t ldq,
                                                       float *__restrict__ scale) {
  const size_t blk = ((size_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (blk >= (size_t)M * kb) return;
  const uint32_t m = (uint32_t)(blk / kb), b = (uint32_t)(blk - (size_t)m * kb);
  const uint32_t k = b * 128 + (threadIdx.x & 15) * 8;
  const XT *src = x + (size_t)m * ldx + k;
  float v[8];
  if (VEC && k + 8 <= K) {
    ld8v(src, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = k + i < K ? ld1(src + i) : 0.0f;
  }
  u32x2 c;
  const float s = fp8_block_codes<E5M2>(v, c);
  if (k < ((K + 15) & ~15u)) {
    // a value past K has no code of its block, whatever its scale
    *reinterpret_cast<u32x2 *>(q + (size_t)m * ldq + k) = fp8_keep(c, k < K ? min(8u, K - k) : 0);
  }
  if ((threadIdx.x & 15) == 0) scale[blk] = s;
}

// A 128 x 128 tile of x per workgroup of 256: thread (wave w, lane group h of
// 16, lane c of it) holds rows 32w + 8h .. + 7 of columns 8c .. 8c + 7, read 16
// bytes of bf16 (32 of f32) a row. Codes that keep x's order go straight to q
// (128 bytes of a row from 16 lanes); transposed ones through LDS, a column's
// 8 rows as 8 bytes, in chunks XOR-swizzled by column / 8 so that the 16 lanes
// of a group hit different banks.
//   COLS: a scale per column (its 128 rows), q transposed
//   TILES, TILES_T: one scale
template <typename XT, bool E5M2, int BLOCKS, bool VEC>
__global__ __launch_bounds__(256) void fp8_tile_kernel(const XT *__restrict__ x, uint32_t M, uint32_t K, size_t ldx,
                                                       uint8_t *__restrict__ q, size_t ldq,
                                                       float *__restrict__ scale) {
  constexpr bool T = BLOCKS != FRXQ_TILES;
  __shared__ __align__(16) u32x2 st[T ? 128 * 16 : 1];
  __shared__ uint32_t red[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 4, c = lane & 15;
  const uint32_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  const uint32_t mt = blockIdx.x / kb, kt = blockIdx.x - mt * kb;
  const uint32_t k = kt * 128 + 8 * c, m0 = mt * 128 + 32 * wave + 8 * h;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const XT *src = x + (size_t)(m0 + i) * ldx + k;
    if (m0 + i < M && VEC && k + 8 <= K) {
      ld8v(src, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[i][j] = m0 + i < M && k + j < K ? ld1(src + j) : 0.0f;
    }
  }
  uint32_t mx[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    mx[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) mx[j] = max(mx[j], __float_as_uint(v[i][j]) & FP8_MAG);
  }
  float s[8], inv[8];
  if constexpr (BLOCKS == FRXQ_COLS) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      mx[j] = max(mx[j], (uint32_t)__shfl_xor((int)mx[j], 16));
      mx[j] = max(mx[j], (uint32_t)__shfl_xor((int)mx[j], 32));
      if (h == 0) red[wave][8 * c + j] = mx[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) {
      s[j] = fp8_scale<E5M2>(max(max(red[0][8 * c + j], red[1][8 * c + j]), max(red[2][8 * c + j], red[3][8 * c + j])));
      inv[j] = 1.0f / s[j];
    }
    if (threadIdx.x < 16)
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (k + j < K) scale[(size_t)(k + j) * mb + mt] = s[j];
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, mx[j]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if (lane == 0) red[wave][0] = m;
    __syncthreads();
    s[0] = fp8_scale<E5M2>(max(max(red[0][0], red[1][0]), max(red[2][0], red[3][0])));
    inv[0] = 1.0f / s[0];
#pragma unroll
    for (int j = 1; j < 8; j++) inv[j] = inv[0];
    if (threadIdx.x == 0) scale[BLOCKS == FRXQ_TILES ? (size_t)mt * kb + kt : (size_t)kt * mb + mt] = s[0];
  }
  // a place past M or K holds a zero, but a scale that is no number would make
  // it a NaN: bytes of such places are cleared
  if constexpr (!T) {
    const uint32_t n = k < K ? min(8u, K - k) : 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (m0 + i >= M || k >= ((K + 15) & ~15u)) continue;
      u32x2 w;
      w.x = fp8_pack4<E5M2>(v[i][0] * inv[0], v[i][1] * inv[1], v[i][2] * inv[2], v[i][3] * inv[3]);
      w.y = fp8_pack4<E5M2>(v[i][4] * inv[4], v[i][5] * inv[5], v[i][6] * inv[6], v[i][7] * inv[7]);
      *reinterpret_cast<u32x2 *>(q + (size_t)(m0 + i) * ldq + k) = fp8_keep(w, n);
    }
  } else {
    const uint32_t n = m0 < M ? min(8u, M - m0) : 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      u32x2 w;
      w.x = fp8_pack4<E5M2>(v[0][j] * inv[j], v[1][j] * inv[j], v[2][j] * inv[j], v[3][j] * inv[j]);
      w.y = fp8_pack4<E5M2>(v[4][j] * inv[j], v[5][j] * inv[j], v[6][j] * inv[j], v[7][j] * inv[j]);
      st[(8 * c + j) * 16 + ((4 * wave + h) ^ c)] = fp8_keep(w, n);
    }
    __syncthreads();
    // rows of q: 8 lanes of 16 bytes (two chunks, exchanged where the swizzle is odd) each
    const uint32_t r0 = kt * 128, c0 = mt * 128, qcols = (M + 15) & ~15u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t r = (threadIdx.x >> 3) + 32 * i, p = threadIdx.x & 7, z = r >> 3;
      const u32x4 w = *reinterpret_cast<const u32x4 *>(&st[r * 16 + ((2 * p) ^ (z & ~1u))]);
      if (r0 + r < K && c0 + 16 * p < qcols)
        *reinterpret_cast<u32x4 *>(q + (size_t)(r0 + r) * ldq + c0 + 16 * p) =
            z & 1 ? (u32x4){w.z, w.w, w.x, w.y} : w;
    }
  }
}

template <typename XT, bool E5M2>
hipError_t quantize_t(const XT *x, uint32_t M, uint32_t K, size_t ldx, int blocks, uint8_t *q, size_t ldq,
                      float *scale, hipStream_t stream) {
  const uint32_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | (ldx * sizeof(XT))) & 15) == 0;
  if (blocks == FRXQ_ROWS) {
    const size_t wgs = ((size_t)M * kb + 15) / 16;
    if (wgs > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const auto fn = vec ? fp8_rows_kernel<XT, E5M2, true> : fp8_rows_kernel<XT, E5M2, false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)wgs), dim3(256), 0, stream, x, M, K, ldx, kb, q, ldq, scale);
    return hipGetLastError();
  }
  using Fn = void (*)(const XT *, uint32_t, uint32_t, size_t, uint8_t *, size_t, float *);
  Fn fn;
  if (blocks == FRXQ_COLS) fn = vec ? fp8_tile_kernel<XT, E5M2, FRXQ_COLS, true> : fp8_tile_kernel<XT, E5M2, FRXQ_COLS, false>;
  else if (blocks == FRXQ_TILES)
    fn = vec ? fp8_tile_kernel<XT, E5M2, FRXQ_TILES, true> : fp8_tile_kernel<XT, E5M2, FRXQ_TILES, false>;
  else fn = vec ? fp8_tile_kernel<XT, E5M2, FRXQ_TILES_T, true> : fp8_tile_kernel<XT, E5M2, FRXQ_TILES_T, false>;
  if ((size_t)kb * mb > 0x7FFFFFFFu) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fn, dim3(kb * mb), dim3(256), 0, stream, x, M, K, ldx, q, ldq, scale);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_quantize(const void *x, int xt_bf16, uint32_t M, uint32_t K, size_t ldx, int blocks, int e5m2,
                               uint8_t *q, size_t ldq, float *scale, hipStream_t stream) {
  if (xt_bf16) {
    const uint16_t *p = static_cast<const uint16_t *>(x);
    return e5m2 ? quantize_t<uint16_t, true>(p, M, K, ldx, blocks, q, ldq, scale, stream)
                : quantize_t<uint16_t, false>(p, M, K, ldx, blocks, q, ldq, scale, stream);
  }
  const float *p = static_cast<const float *>(x);
  return e5m2 ? quantize_t<float, true>(p, M, K, ldx, blocks, q, ldq, scale, stream)
              : quantize_t<float, false>(p, M, K, ldx, blocks, q, ldq, scale, stream);
}

}  // namespace frx
