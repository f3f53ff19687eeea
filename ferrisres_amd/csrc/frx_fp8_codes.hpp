// frx_fp8_codes.hpp — a block's scale and codes, shared by the quantiser and the
// products that quantise their activations on the way.
#pragma once
#include "frx_device.hpp"

namespace frx {

constexpr uint32_t FP8_MAG = 0x7FFFFFFFu;

template <bool E5M2>
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
  const float s = __uint_as_float(amax_bits) * (E5M2 ? 1.0f / 57344.0f : 1.0f / 448.0f);
  return s < 0x1p-126f ? 0x1p-126f : s;  // a NaN stays
}

// Four values as four codes (round to nearest even).
template <bool E5M2>
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  if constexpr (E5M2) {
    const int lo = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, lo, true);
  } else {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
  }
}

// The first n of eight codes, zeros behind them.
__device__ __forceinline__ u32x2 fp8_keep(u32x2 c, uint32_t n) {
  c.x &= n >= 4 ? ~0u : (1u << (8 * n)) - 1;
  c.y &= n >= 8 ? ~0u : n <= 4 ? 0u : (1u << (8 * (n - 4))) - 1;
  return c;
}

__device__ __forceinline__ float ld1(const float *p) { return *p; }
__device__ __forceinline__ float ld1(const uint16_t *p) { return bf16_to_f32(*p); }

// Eight consecutive values (16-byte aligned).
__device__ __forceinline__ void ld8v(const float *p, float (&v)[8]) {
  const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}
__device__ __forceinline__ void ld8v(const uint16_t *p, float (&v)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
  }
}

// Codes and scale of the 1 x 128 block that 16 neighbouring lanes hold, 8
// values each (zeros past its end).
template <bool E5M2>
__device__ __forceinline__ float fp8_block_codes(const float (&v)[8], u32x2 &c) {
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) mx = max(mx, __float_as_uint(v[i]) & FP8_MAG);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o));
  const float s = fp8_scale<E5M2>(mx);
  const float inv = 1.0f / s;
  c.x = fp8_pack4<E5M2>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  c.y = fp8_pack4<E5M2>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
  return s;
}

}  // namespace frx
