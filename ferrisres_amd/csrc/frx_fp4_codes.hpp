// frx_fp4_codes.hpp — a block's power of two and its 4-bit codes.
//
// 32 values share a byte b = max(e, 2) - 2, e the biased exponent of the largest
// magnitude, which stands for 2^(b - 127): the largest value lands in [4, 8), where 4 and
// 6 are the format's codes (above 6: 6). x * 2^(127 - b) is exact (a power of two between
// 2^-125 and 2^127), so a code is one rounding, to nearest even, in v_cvt_scalef32_pk_fp4.
// e = 255 (an infinity or a NaN in the block) gives b = 255, the scale that makes a NaN of
// every product, and zeros for codes.
#pragma once
#include "frx_device.hpp"
#include "frx_fp8_codes.hpp"

namespace frx {

// Bytes of a row of K codes, rounded up to whole blocks of 32; of its scales, to whole dwords.
__host__ __device__ constexpr uint32_t fp4_row_bytes(uint32_t K) { return (K + 31) / 32 * 16; }
__host__ __device__ constexpr uint32_t fp4_scale_bytes(uint32_t K) { return (K + 127) / 128 * 4; }

__device__ __forceinline__ uint32_t fp4_scale(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255 ? 255 : max(e, 2u) - 2;
}
__device__ __forceinline__ float fp4_inverse(uint32_t b) { return __uint_as_float((254 - min(b, 252u)) << 23); }
// 2^(b - 127), NaN for 255.
__device__ __forceinline__ float fp4_power(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7FC00000u : b << 23);
}

// Unaligned 16 bytes (a tensor may begin at any element).
typedef u32x4 __attribute__((aligned(2))) u32x4_u;

// Eight values from p on, which may be any element.
__device__ __forceinline__ void ld8u(const float *p, float (&v)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4_u *>(p), b = *reinterpret_cast<const u32x4_u *>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[i] = __uint_as_float(a[i]);
    v[4 + i] = __uint_as_float(b[i]);
  }
}
__device__ __forceinline__ void ld8u(const uint16_t *p, float (&v)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4_u *>(p);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
  }
}

// Eight values times inv as eight codes, the first in the lowest bits; zeros under b = 255.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&v)[8], float inv, uint32_t b) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0] * inv, v[1] * inv, 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2] * inv, v[3] * inv, 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4] * inv, v[5] * inv, 1.0f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6] * inv, v[7] * inv, 1.0f, 3);
  return b == 255 ? 0 : c;
}

// Codes of the 8 values of this lane, in blocks that 4 neighbouring lanes hold; s: the
// bytes of the four blocks of the 16 lanes, in order.
__device__ __forceinline__ uint32_t fp4_block_codes(const float (&v)[8], uint32_t &s) {
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) mx = max(mx, __float_as_uint(v[i]) & FP8_MAG);
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 1));
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 2));
  const uint32_t b = fp4_scale(mx);
  s = b << (8 * ((threadIdx.x >> 2) & 3));
  s |= (uint32_t)__shfl_xor((int)s, 4);
  s |= (uint32_t)__shfl_xor((int)s, 8);
  return fp4_pack8(v, fp4_inverse(b), b);
}

}  // namespace frx
