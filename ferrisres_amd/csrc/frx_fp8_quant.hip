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
// value (mask, max, multiply, half a conversion).
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
    if (k + 8 > K) {
      const uint32_t n = k < K ? K - k : 0;
      c.x &= n >= 4 ? ~0u : (1u << (8 * n)) - 1;
      c.y &= n <= 4 ? 0u : (1u << (8 * (n - 4))) - 1;
    }
    *reinterpret_cast<u32x2 *>(q + (size_t)m * ldq + k) = c;
  }
  if ((threadIdx.x & 15) == 0) scale[blk] = s;
}

// A 128 x 128 tile of x per workgroup of 256: thread (wave w, lane l) holds
// rows 32w .. 32w + 31 of columns 2l and 2l + 1. The codes go through LDS so
// that whole 128-byte rows of q are written.
//   COLS: a scale per column (its 128 rows), q transposed
//   TILES, TILES_T: one scale
template <typename XT, bool E5M2, int BLOCKS, bool VEC>
__global__ __launch_bounds__(256) void fp8_tile_kernel(const XT *__restrict__ x, uint32_t M, uint32_t K, size_t ldx,
                                                       uint8_t *__restrict__ q, size_t ldq,
                                                       float *__restrict__ scale) {
  constexpr bool T = BLOCKS != FRXQ_TILES;
  constexpr int PITCH = 128 + 16;  // bytes of a staged row
  __shared__ __align__(16) uint8_t st[128 * PITCH];
  __shared__ uint32_t red[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  const uint32_t mt = blockIdx.x / kb, kt = blockIdx.x - mt * kb;
  const uint32_t k = kt * 128 + 2 * lane, m0 = mt * 128 + 32 * wave;
  float v[32][2];
#pragma unroll
  for (int i = 0; i < 32; i++) {
    const uint32_t m = m0 + i;
    v[i][0] = v[i][1] = 0.0f;
    if (m < M) {
      const XT *src = x + (size_t)m * ldx + k;
      if (VEC && k + 2 <= K) {
        if constexpr (sizeof(XT) == 2) {
          const uint32_t p = *reinterpret_cast<const uint32_t *>(src);
          v[i][0] = __uint_as_float(p << 16);
          v[i][1] = __uint_as_float(p & 0xFFFF0000u);
        } else {
          const float2 p = *reinterpret_cast<const float2 *>(src);
          v[i][0] = p.x;
          v[i][1] = p.y;
        }
      } else {
        if (k < K) v[i][0] = ld1(src);
        if (k + 1 < K) v[i][1] = ld1(src + 1);
      }
    }
  }
  uint32_t mx[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 32; i++)
#pragma unroll
    for (int c = 0; c < 2; c++) mx[c] = max(mx[c], __float_as_uint(v[i][c]) & FP8_MAG);
  if constexpr (BLOCKS == FRXQ_COLS) {
    red[wave][2 * lane] = mx[0];
    red[wave][2 * lane + 1] = mx[1];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
      for (int w = 0; w < 4; w++) mx[c] = max(mx[c], red[w][2 * lane + c]);
  } else {
    uint32_t m = max(mx[0], mx[1]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if (lane == 0) red[wave][0] = m;
    __syncthreads();
    m = max(max(red[0][0], red[1][0]), max(red[2][0], red[3][0]));
    mx[0] = mx[1] = m;
  }
  float s[2], inv[2];
#pragma unroll
  for (int c = 0; c < 2; c++) {
    s[c] = fp8_scale<E5M2>(mx[c]);
    inv[c] = 1.0f / s[c];
  }
  if constexpr (BLOCKS == FRXQ_COLS) {
    if (wave == 0) {
      if (k < K) scale[(size_t)k * mb + mt] = s[0];
      if (k + 1 < K) scale[(size_t)(k + 1) * mb + mt] = s[1];
    }
  } else if (threadIdx.x == 0) {
    scale[BLOCKS == FRXQ_TILES ? (size_t)mt * kb + kt : (size_t)kt * mb + mt] = s[0];
  }
  // a place past M or K holds a zero, but a scale that is no number would make it a NaN
  const uint32_t rows = m0 < M ? min(32u, M - m0) : 0;
  if constexpr (T) {
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        uint32_t w = fp8_pack4<E5M2>(v[i][c] * inv[c], v[i + 1][c] * inv[c], v[i + 2][c] * inv[c],
                                     v[i + 3][c] * inv[c]);
        if (rows < (uint32_t)i + 4) w &= rows <= (uint32_t)i ? 0u : (1u << (8 * (rows - i))) - 1;
        *reinterpret_cast<uint32_t *>(st + (2 * lane + c) * PITCH + 32 * wave + i) = w;
      }
  } else {
    const uint32_t keep = k + 1 < K ? 0xFFFFu : k < K ? 0xFFu : 0u;
#pragma unroll
    for (int i = 0; i < 32; i++)
      *reinterpret_cast<uint16_t *>(st + (32 * wave + i) * PITCH + 2 * lane) =
          (uint16_t)(fp8_pack4<E5M2>(v[i][0] * inv[0], v[i][1] * inv[1], 0.f, 0.f) & keep);
  }
  __syncthreads();
  // rows of q: 8 lanes of 16 bytes each
  const uint32_t qrows = T ? K : M, qcols = ((T ? M : K) + 15) & ~15u;
  const uint32_t r0 = (T ? kt : mt) * 128, c0 = (T ? mt : kt) * 128;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t r = (threadIdx.x >> 3) + 32 * i, c = (threadIdx.x & 7) * 16;
    if (r0 + r < qrows && c0 + c < qcols)
      *reinterpret_cast<u32x4 *>(q + (size_t)(r0 + r) * ldq + c0 + c) =
          *reinterpret_cast<const u32x4 *>(st + r * PITCH + c);
  }
}

template <typename XT, bool E5M2>
hipError_t quantize_t(const XT *x, uint32_t M, uint32_t K, size_t ldx, int blocks, uint8_t *q, size_t ldq,
                      float *scale, hipStream_t stream) {
  const uint32_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  if (blocks == FRXQ_ROWS) {
    const bool vec = ((reinterpret_cast<uintptr_t>(x) | (ldx * sizeof(XT))) & 15) == 0;
    const size_t wgs = ((size_t)M * kb + 15) / 16;
    if (wgs > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const auto fn = vec ? fp8_rows_kernel<XT, E5M2, true> : fp8_rows_kernel<XT, E5M2, false>;
    hipLaunchKernelGGL(fn, dim3((unsigned)wgs), dim3(256), 0, stream, x, M, K, ldx, kb, q, ldq, scale);
    return hipGetLastError();
  }
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | (ldx * sizeof(XT))) & (2 * sizeof(XT) - 1)) == 0;
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
