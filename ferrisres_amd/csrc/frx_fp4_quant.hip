// frx_fp4_quant.hip — codes and scales of the 4-bit floating-point linears, and back.
//
// Formulas: frx_fp4_codes.hpp. Bound by memory: 2 or 4 bytes in and 17/32 out a value (the
// way back the other way round), about 3 VALU operations a value. 11008 x 4096: f32 along the
// rows 36.0 us (5.7 TB/s), along the columns 44.9, back 44.7; bf16 24.6, 29.5, 25.4. 2048 x 4096
// bf16 6.3, 7.4, 5.6. Loads and stores of 16 bytes at any element's address: 2458 x 12829 f32 along
// the columns and back 38.6 + 37.7 (by single values 144 in all). Tried and no faster: two pieces of a row a thread, tiles of 256 x 64 along
// the columns (whole lines of codes), divisions in 32 bits.
#include "frx_fp4_codes.hpp"
#include "frx_internal.hpp"

namespace frx {

namespace {

// Blocks along the rows: 16 lanes hold 128 columns, 8 values a lane, and write 64 bytes of
// codes and a dword of scales. A block past K has zero codes and the smallest scale.
template <typename XT>
__global__ __launch_bounds__(256) void fp4_rows_kernel(const XT *__restrict__ x, uint32_t M, uint32_t K, size_t ldx,
                                                       uint32_t kb, uint8_t *__restrict__ q, size_t ldq,
                                                       uint32_t *__restrict__ scale) {
  const size_t blk = ((size_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (blk >= (size_t)M * kb) return;
  const uint32_t m = (uint32_t)(blk / kb), b = (uint32_t)(blk - (size_t)m * kb);
  const uint32_t k = b * 128 + (threadIdx.x & 15) * 8;
  const XT *src = x + (size_t)m * ldx + k;
  float v[8];
  if (k + 8 <= K) {
    ld8u(src, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = k + i < K ? ld1(src + i) : 0.0f;
  }
  uint32_t s;
  const uint32_t c = fp4_block_codes(v, s);
  if (k < ((K + 31) & ~31u)) *reinterpret_cast<uint32_t *>(q + (size_t)m * ldq + (k >> 1)) = c;
  if ((threadIdx.x & 15) == 0) scale[blk] = s;
}

// Blocks along the columns, codes transposed: a 128 x 128 tile of x per workgroup of 256.
// Thread (wave w, lane group h of 16, lane c of it) holds rows 32w + 8h .. + 7 of columns
// 8c .. 8c + 7, so a wave holds whole blocks. A column's 8 rows are a dword of codes; 16
// of them, swizzled by column / 8, make its 64 bytes in LDS.
template <typename XT>
__global__ __launch_bounds__(256) void fp4_cols_kernel(const XT *__restrict__ x, uint32_t M, uint32_t K, size_t ldx,
                                                       uint8_t *__restrict__ q, size_t ldq,
                                                       uint32_t *__restrict__ scale) {
  __shared__ __align__(16) uint32_t st[128 * 16];
  __shared__ uint32_t sc[128];  // a column's scales, a byte from each wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 4, c = lane & 15;
  const uint32_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  const uint32_t mt = blockIdx.x / kb, kt = blockIdx.x - mt * kb;
  const uint32_t k = kt * 128 + 8 * c, m0 = mt * 128 + 32 * wave + 8 * h;
  float v[8][8];  // [column][row]
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const XT *src = x + (size_t)(m0 + i) * ldx + k;
    float r[8];
    if (m0 + i < M && k + 8 <= K) {
      ld8u(src, r);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) r[j] = m0 + i < M && k + j < K ? ld1(src + j) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j][i] = r[j];
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) mx = max(mx, __float_as_uint(v[j][i]) & FP8_MAG);
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
    const uint32_t b = fp4_scale(mx);
    if (h == 0) reinterpret_cast<uint8_t *>(sc)[(8 * c + j) * 4 + wave] = (uint8_t)b;
    st[(8 * c + j) * 16 + ((4 * wave + h) ^ c)] = fp4_pack8(v[j], fp4_inverse(b), b);
  }
  __syncthreads();
  const uint32_t r0 = kt * 128, bytes = fp4_row_bytes(M);
  if (threadIdx.x < 128 && r0 + threadIdx.x < K)
    scale[(size_t)(r0 + threadIdx.x) * mb + mt] = sc[threadIdx.x];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t r = (threadIdx.x >> 2) + 64 * i, p = threadIdx.x & 3, z = r >> 3;
    const u32x4 w = *reinterpret_cast<const u32x4 *>(&st[r * 16 + ((4 * p) ^ (z & ~3u))]);
    u32x4 o = z & 1 ? (u32x4){w.y, w.x, w.w, w.z} : w;
    if (z & 2) o = (u32x4){o.z, o.w, o.x, o.y};
    if (r0 + r < K && mt * 64 + 16 * p < bytes)
      *reinterpret_cast<u32x4 *>(q + (size_t)(r0 + r) * ldq + mt * 64 + 16 * p) = o;
  }
}

// The values of 8 codes a thread.
template <typename YT>
__global__ __launch_bounds__(256) void fp4_values_kernel(const uint8_t *__restrict__ q, size_t ldq,
                                                         const uint8_t *__restrict__ scale, uint32_t M, uint32_t K,
                                                         uint32_t groups, YT *__restrict__ y, size_t ldy) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)M * groups) return;
  const uint32_t m = (uint32_t)(i / groups), k = (uint32_t)(i - (size_t)m * groups) * 8;
  const uint32_t c = *reinterpret_cast<const uint32_t *>(q + (size_t)m * ldq + (k >> 1));
  const float s = fp4_power(scale[(size_t)m * fp4_scale_bytes(K) + (k >> 5)]);
  float v[8];
#define FRX_FP4_PAIR(j)                                                          \
  {                                                                              \
    const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, j);         \
    v[2 * j] = p[0] * s;                                                         \
    v[2 * j + 1] = p[1] * s;                                                     \
  }
  FRX_FP4_PAIR(0) FRX_FP4_PAIR(1) FRX_FP4_PAIR(2) FRX_FP4_PAIR(3)
#undef FRX_FP4_PAIR
  YT *d = y + (size_t)m * ldy + k;
  if constexpr (sizeof(YT) == 4) {
    if (k + 8 <= K) {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; j++) h[j] = __float_as_uint(v[j]);
      reinterpret_cast<u32x4_u *>(d)[0] = (u32x4){h[0], h[1], h[2], h[3]};
      reinterpret_cast<u32x4_u *>(d)[1] = (u32x4){h[4], h[5], h[6], h[7]};
    } else {
      for (uint32_t j = 0; j < 8 && k + j < K; j++) d[j] = v[j];
    }
  } else {
    uint32_t h[8];  // (exact: two bits of significand)
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = __float_as_uint(v[j]) >> 16;
    if (k + 8 <= K) {
      *reinterpret_cast<u32x4_u *>(d) = (u32x4){h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16),
                                               h[6] | (h[7] << 16)};
    } else {
      for (uint32_t j = 0; j < 8 && k + j < K; j++) d[j] = (uint16_t)h[j];
    }
  }
}

template <typename XT>
hipError_t quantize_t(const XT *x, uint32_t M, uint32_t K, size_t ldx, int cols, uint8_t *q, size_t ldq,
                      uint32_t *scale, hipStream_t stream) {
  const uint32_t kb = (K + 127) / 128, mb = (M + 127) / 128;
  const size_t wgs = cols ? (size_t)kb * mb : ((size_t)M * kb + 15) / 16;
  if (wgs > 0xFFFFFFu) return hipErrorInvalidValue;
  if (cols) {
    hipLaunchKernelGGL(fp4_cols_kernel<XT>, dim3((unsigned)wgs), dim3(256), 0, stream, x, M, K, ldx, q, ldq, scale);
  } else {
    hipLaunchKernelGGL(fp4_rows_kernel<XT>, dim3((unsigned)wgs), dim3(256), 0, stream, x, M, K, ldx, kb, q, ldq, scale);
  }
  return hipGetLastError();
}

template <typename YT>
hipError_t values_t(const uint8_t *q, size_t ldq, const uint8_t *scale, uint32_t M, uint32_t K, YT *y, size_t ldy,
                    hipStream_t stream) {
  const uint32_t groups = (K + 7) / 8;
  const size_t wgs = ((size_t)M * groups + 255) / 256;
  if (wgs > 0xFFFFFFu) return hipErrorInvalidValue;
  hipLaunchKernelGGL(fp4_values_kernel<YT>, dim3((unsigned)wgs), dim3(256), 0, stream, q, ldq, scale, M, K, groups, y, ldy);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp4_quantize(const void *x, int xt_bf16, uint32_t M, uint32_t K, size_t ldx, int cols, uint8_t *q,
                               size_t ldq, uint8_t *scale, hipStream_t stream) {
  uint32_t *s = reinterpret_cast<uint32_t *>(scale);
  return xt_bf16 ? quantize_t(static_cast<const uint16_t *>(x), M, K, ldx, cols, q, ldq, s, stream)
                 : quantize_t(static_cast<const float *>(x), M, K, ldx, cols, q, ldq, s, stream);
}

hipError_t launch_fp4_dequantize(const uint8_t *q, size_t ldq, const uint8_t *scale, uint32_t M, uint32_t K, void *y,
                                 int yt_bf16, size_t ldy, hipStream_t stream) {
  return yt_bf16 ? values_t(q, ldq, scale, M, K, static_cast<uint16_t *>(y), ldy, stream)
                 : values_t(q, ldq, scale, M, K, static_cast<float *>(y), ldy, stream);
}

}  // namespace frx
