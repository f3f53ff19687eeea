// frx_fp4_moe.hip — a whole expert layer for a few tokens, its experts' weights in 4 bits.
//
//   y[t] = sum_j w[t][j] down_e(act(gate_e x_t) * up_e x_t),  e = idx[t][j]
//
// A few tokens read every weight of the experts they reach once: bound by those bytes
// (17/32 a value). So the activations stay as they are: the codes widen to bf16 times
// their block's power of two (exact, one conversion for two codes) and meet x as bf16, or
// an f32 x as three bf16 planes that add up to it exactly; sums in fp32.
//
//   route     the router's logits, top-k and softmax, where the caller has none
//   gate, up  a workgroup per 16 inner columns of an expert: the expert's tokens are
//             gathered 16 at a time; h times the route's weight as bf16 planes, a row for
//             each route
//   down      a workgroup per 16 outputs adds up all experts: tokens are the matrix
//             instruction's columns and an expert's column is its route's row of h, or
//             zeros for a token that it does not serve. So no sum leaves the workgroup and
//             no atomics decide an order.
#include "frx_fp4_codes.hpp"
#include "frx_fp8.hpp"
#include "frx_internal.hpp"

namespace frx {

namespace {

constexpr int WAVES = 8;

// ---- routes ------------------------------------------------------------------------

// Eight values from p on. vec: 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8]) {
  if (vec) {
    ld8v(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = ld1(p + i);
  }
}

// A workgroup of 4 waves per token. The experts of the largest logits, ties to the lowest
// index, a NaN below every number; weights exp(l - l_max) over their sum.
template <typename XT, typename RT>
__global__ __launch_bounds__(256) void fp4_route_kernel(const XT *__restrict__ x, const RT *__restrict__ router,
                                                        uint32_t H, int E, int top_k, uint32_t *__restrict__ idx,
                                                        float *__restrict__ wts, int xvec, int rvec) {
  __shared__ float logit[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const XT *row = x + (size_t)blockIdx.x * H;
  for (int e = wave; e < E; e += 4) {
    float s = 0.f;
    for (uint32_t k = lane * 8; k < H; k += 512) {
      float a[8], b[8];
      load8(row + k, xvec, a);
      load8(router + (size_t)e * H + k, rvec, b);
#pragma unroll
      for (int i = 0; i < 8; i++) s = __builtin_fmaf(a[i], b[i], s);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) logit[e] = s;
  }
  __syncthreads();
  if (wave) return;
  const float mine = lane < E ? logit[lane] + 0.0f : 0.f;  // -0 orders as 0
  const uint32_t bits = __float_as_uint(mine);
  uint64_t key = mine != mine ? 0 : bits >> 31 ? ~bits : bits | 0x80000000u;
  key = lane < E ? ((key + 1) << 6) | (63 - lane) : 0;
  float top = 0.f, sum = 0.f, w = 0.f;
  int place = -1;
  for (int j = 0; j < top_k; j++) {
    uint64_t best = key;
#pragma unroll
    for (int o = 32; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, o));
    const int e = 63 - (int)(best & 63);
    const float l = __shfl(mine, e);
    if (j == 0) top = l;
    const float p = expf(l - top);
    sum += p;
    if (lane == e) {
      key = 0;
      w = p;
      place = j;
    }
  }
  if (place >= 0) {
    idx[(size_t)blockIdx.x * top_k + place] = lane;
    wts[(size_t)blockIdx.x * top_k + place] = w / sum;
  }
}

// The experts that any route goes to, as bits; every thread of the workgroup gets them.
__device__ __forceinline__ uint64_t active_experts(const uint32_t *idx, int slots, int E, uint32_t (&word)[2]) {
  if (threadIdx.x < 2) word[threadIdx.x] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += blockDim.x) {
    const uint32_t e = idx[s];
    if (e < (uint32_t)E) atomicOr(&word[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  return word[0] | ((uint64_t)word[1] << 32);
}

// The a-th set bit's place.
__device__ __forceinline__ int nth_bit(uint64_t m, int a) {
  for (int i = 0; i < a; i++) m &= m - 1;
  return __ffsll((unsigned long long)m) - 1;
}

// ---- operands ----------------------------------------------------------------------

// The 32 codes of a lane times 2^(b - 127) as bf16, 8 to an operand.
__device__ __forceinline__ void widen(const u32x4 &c, uint32_t b, u32x4 (&w)[4]) {
  const float s = fp4_power(b);
#pragma unroll
  for (int q = 0; q < 4; q++) {
    w[q].x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], s, 0));
    w[q].y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], s, 1));
    w[q].z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], s, 2));
    w[q].w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[q], s, 3));
  }
}

// A value as bf16 planes of which each holds the next 8 bits: three add up to it.
__device__ __forceinline__ float cut8(float v, uint32_t &plane) {
  plane = __float_as_uint(v) & 0xFFFF0000u;
  return v - __uint_as_float(plane);
}

// Eight activations as P operands.
template <typename XT, int P>
__device__ __forceinline__ void act8(const XT *p, bool vec, u32x4 (&o)[P]) {
  if constexpr (sizeof(XT) == 2) {
    if (vec) {
      o[0] = *reinterpret_cast<const u32x4 *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) o[0][i] = p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    }
  } else {
    float v[8];
    load8(p, vec, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
      for (int j = 0; j < P; j++) {
        uint32_t u, w;
        a = cut8(a, u);
        b = cut8(b, w);
        o[j][i] = (u >> 16) | w;
      }
    }
  }
}

// ---- gate and up -------------------------------------------------------------------

template <int ACT>
__device__ __forceinline__ float activate(float g) {
  if constexpr (ACT == 0) {
    return g / (1.0f + expf(-g));
  } else {
    return 0.5f * g * (1.0f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g)));
  }
}

struct FewArgs {
  const void *x;
  const uint32_t *idx;
  const float *wts;
  uint16_t *h;
  void *y;
  uint32_t T, H, I;
  int E, top_k, vec;
  const uint8_t *w[2][FP8_MAXE], *s[2][FP8_MAXE];  // gate, up; or down
};

// P: planes of x; HP: planes of h.
template <typename XT, int HP, int ACT>
__global__ __launch_bounds__(WAVES * 64) void fp4_gate_up_kernel(const FewArgs p) {
  constexpr int P = sizeof(XT) == 2 ? 1 : 3;
  __shared__ uint32_t word[2];
  __shared__ uint32_t tok[64], slot[64];
  __shared__ float share[64];
  __shared__ f32x4 red[WAVES][2][64];
  const uint64_t active = active_experts(p.idx, (int)p.T * p.top_k, p.E, word);
  if ((int)blockIdx.y >= __popcll(active)) return;
  const int e = __builtin_amdgcn_readfirstlane(nth_bit(active, blockIdx.y));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  // the expert's tokens, a route taken twice as one of both weights
  int first = -1;
  float w = 0.f;
  if (lane < (int)p.T)
    for (int j = 0; j < p.top_k; j++)
      if (p.idx[lane * p.top_k + j] == (uint32_t)e) {
        if (first < 0) first = j;
        w += p.wts[lane * p.top_k + j];
      }
  const uint64_t mine = __ballot(first >= 0);
  const int n = __popcll(mine);
  if (wave == 0 && first >= 0) {
    const int at = __popcll(mine & ((1ull << lane) - 1));
    tok[at] = lane;
    slot[at] = lane * p.top_k + first;
    share[at] = w;
  }
  __syncthreads();
  const int K = (int)p.H, kbs = (K + 127) >> 7, per = (kbs + WAVES - 1) / WAVES;
  const int kb0 = min(wave * per, kbs), kb1 = min(kb0 + per, kbs);
  const uint32_t n0 = blockIdx.x * 16;
  const size_t row = min(n0 + l16, p.I - 1);
  const uint8_t *wg = p.w[0][e] + row * (K / 2), *wu = p.w[1][e] + row * (K / 2);
  const uint8_t *sg = p.s[0][e] + row * (4 * kbs), *su = p.s[1][e] + row * (4 * kbs);
  for (int c0 = 0; c0 < n; c0 += 16) {
    const XT *x = static_cast<const XT *>(p.x) + (size_t)tok[min(c0 + l16, n - 1)] * K;
    f32x4 ag = {0.f, 0.f, 0.f, 0.f}, au = ag;
    for (int kb = kb0; kb < kb1; kb++) {
      const int blk = min(kb * 4 + g, K / 32 - 1);
      const bool inside = kb * 4 + g < K / 32;
      const u32x4 cg = *reinterpret_cast<const u32x4 *>(wg + 16 * blk), cu = *reinterpret_cast<const u32x4 *>(wu + 16 * blk);
      u32x4 vg[4], vu[4];
      widen(cg, inside ? sg[blk] : 0, vg);
      widen(cu, inside ? su[blk] : 0, vu);
#pragma unroll
      for (int q = 0; q < 4; q++) {
        u32x4 v[P];
        act8<XT, P>(x + 32 * blk + 8 * q, p.vec, v);
#pragma unroll
        for (int j = 0; j < P; j++) {
          if (!inside) v[j] = (u32x4){0, 0, 0, 0};
          ag = mfma16(vg[q], v[j], ag);
          au = mfma16(vu[q], v[j], au);
        }
      }
    }
    red[wave][0][lane] = ag;
    red[wave][1][lane] = au;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 1; i < WAVES; i++) {
        ag += red[i][0][lane];
        au += red[i][1][lane];
      }
      const uint32_t i0 = n0 + 4 * g;
      if (c0 + l16 < n && i0 < p.I) {  // I % 32 == 0: whole quads
        const float sh = share[c0 + l16];
        uint32_t plane[HP][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float v = activate<ACT>(ag[i]) * au[i] * sh;
          if constexpr (HP == 2) {
            plane[0][i] = bf16_rne_nb(v);
            plane[1][i] = bf16_rne_nb(v - __uint_as_float(plane[0][i] << 16));
          } else {
#pragma unroll
            for (int j = 0; j < HP; j++) {
              uint32_t u;
              v = cut8(v, u);
              plane[j][i] = u >> 16;
            }
          }
        }
        uint16_t *d = p.h + (size_t)slot[c0 + l16] * HP * p.I + i0;
#pragma unroll
        for (int j = 0; j < HP; j++)
          *reinterpret_cast<u32x2 *>(d + (size_t)j * p.I) =
              (u32x2){plane[j][0] | (plane[j][1] << 16), plane[j][2] | (plane[j][3] << 16)};
      }
    }
    __syncthreads();
  }
}

// ---- down --------------------------------------------------------------------------

// TT: tiles of 16 tokens.
template <int TT, int HP, typename YT>
__global__ __launch_bounds__(WAVES * 64) void fp4_down_kernel(const FewArgs p) {
  __shared__ uint32_t word[2];
  __shared__ int16_t table[64 * 64];  // [active expert][token]: the route's slot; -1: none
  __shared__ f32x4 red[WAVES][TT][64];
  const int slots = (int)p.T * p.top_k;
  const uint64_t active = active_experts(p.idx, slots, p.E, word);
  const int experts = __popcll(active);
  for (int i = threadIdx.x; i < experts * (int)p.T; i += blockDim.x) table[i] = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += blockDim.x) {
    const uint32_t e = p.idx[s];
    if (e >= (uint32_t)p.E) continue;
    const int t = s / p.top_k;
    bool first = true;
    for (int k = t * p.top_k; k < s; k++) first &= p.idx[k] != e;
    if (first) table[__popcll(active & ((1ull << e) - 1)) * p.T + t] = (int16_t)s;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int K = (int)p.I, kbs = (K + 127) >> 7, units = experts * kbs, per = (units + WAVES - 1) / WAVES;
  const int u0 = min(wave * per, units), u1 = min(u0 + per, units);
  const uint32_t n0 = blockIdx.x * 16;
  const size_t row = min(n0 + l16, p.H - 1);
  f32x4 acc[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int u = u0; u < u1;) {
    const int a = u / kbs, stop = min(u1, (a + 1) * kbs);
    const int e = __builtin_amdgcn_readfirstlane(nth_bit(active, a));
    int slot[TT];
    f32x4 part[TT];  // of this expert: a token that it does not serve drops it, whatever the weights are
#pragma unroll
    for (int t = 0; t < TT; t++) {
      const int tok = 16 * t + l16;
      slot[t] = tok < (int)p.T ? table[a * p.T + tok] : -1;
      part[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    for (; u < stop; u++) {
      const int kb = u - a * kbs;
      const int blk = min(kb * 4 + g, K / 32 - 1);
      const bool inside = kb * 4 + g < K / 32;
      u32x4 w[4];
      widen(*reinterpret_cast<const u32x4 *>(p.w[0][e] + row * (K / 2) + 16 * blk),
            inside ? p.s[0][e][row * (4 * kbs) + blk] : 0, w);
#pragma unroll
      for (int t = 0; t < TT; t++) {
        if (__ballot(slot[t] >= 0) == 0) continue;
        const bool here = slot[t] >= 0 && inside;
        const uint16_t *h = p.h + (size_t)max(slot[t], 0) * HP * p.I + 32 * blk;
#pragma unroll
        for (int j = 0; j < HP; j++)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            u32x4 v = {0, 0, 0, 0};
            if (here) v = *reinterpret_cast<const u32x4 *>(h + (size_t)j * p.I + 8 * q);
            part[t] = mfma16(w[q], v, part[t]);
          }
      }
    }
#pragma unroll
    for (int t = 0; t < TT; t++)
      if (slot[t] >= 0) acc[t] += part[t];
  }
#pragma unroll
  for (int t = 0; t < TT; t++) red[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= TT) return;
  f32x4 v = red[0][wave][lane];
#pragma unroll
  for (int i = 1; i < WAVES; i++) v += red[i][wave][lane];
  const uint32_t n = n0 + 4 * g, m = 16 * wave + l16;
  if (m >= p.T || n >= p.H) return;
  YT *d = static_cast<YT *>(p.y) + (size_t)m * p.H + n;
#pragma unroll
  for (int i = 0; i < 4; i++) {  // H % 32 == 0: whole quads
    if constexpr (sizeof(YT) == 4) d[i] = v[i];
    else d[i] = (uint16_t)bf16_rne_nb(v[i]);
  }
}

template <typename XT>
hipError_t route_go(const Fp4Moe &p, hipStream_t stream) {
  const XT *x = static_cast<const XT *>(p.x);
  const int xvec = ((reinterpret_cast<uintptr_t>(p.x)) & 15) == 0, rvec = ((reinterpret_cast<uintptr_t>(p.router)) & 15) == 0;
  if (p.rt_bf16)
    hipLaunchKernelGGL((fp4_route_kernel<XT, uint16_t>), dim3(p.T), dim3(256), 0, stream, x,
                       static_cast<const uint16_t *>(p.router), p.H, (int)p.E, (int)p.top_k, p.idx, p.wts, xvec, rvec);
  else
    hipLaunchKernelGGL((fp4_route_kernel<XT, float>), dim3(p.T), dim3(256), 0, stream, x,
                       static_cast<const float *>(p.router), p.H, (int)p.E, (int)p.top_k, p.idx, p.wts, xvec, rvec);
  return hipGetLastError();
}

template <typename XT, int HP>
hipError_t gate_up_go(const Fp4Moe &p, const FewArgs &a, hipStream_t stream) {
  const dim3 grid((p.I + 15) / 16, p.E < p.T * p.top_k ? p.E : p.T * p.top_k);
  if (p.act == 0) hipLaunchKernelGGL((fp4_gate_up_kernel<XT, HP, 0>), grid, dim3(WAVES * 64), 0, stream, a);
  else hipLaunchKernelGGL((fp4_gate_up_kernel<XT, HP, 1>), grid, dim3(WAVES * 64), 0, stream, a);
  return hipGetLastError();
}

template <int HP, typename YT>
hipError_t down_go(const Fp4Moe &p, const FewArgs &a, hipStream_t stream) {
  const dim3 grid((p.H + 15) / 16), block(WAVES * 64);
  if (p.T <= 16) hipLaunchKernelGGL((fp4_down_kernel<1, HP, YT>), grid, block, 0, stream, a);
  else if (p.T <= 32) hipLaunchKernelGGL((fp4_down_kernel<2, HP, YT>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((fp4_down_kernel<4, HP, YT>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace

size_t fp4_moe_bytes(uint32_t T, uint32_t I, uint32_t top_k, int yt_bf16) {
  return (size_t)T * top_k * fp4_moe_planes(yt_bf16) * I * 2;
}

hipError_t launch_fp4_moe(const Fp4Moe &p, int cus, hipStream_t stream) {
  (void)cus;
  if (p.router) {
    const hipError_t e = p.xt_bf16 ? route_go<uint16_t>(p, stream) : route_go<float>(p, stream);
    if (e != hipSuccess) return e;
  }
  FewArgs a = {p.x, p.idx, p.wts, p.h, p.y, p.T, p.H, p.I, (int)p.E, (int)p.top_k,
               ((reinterpret_cast<uintptr_t>(p.x)) & 15) == 0, {}, {}};
  for (uint32_t e = 0; e < p.E; e++)
    for (int k = 0; k < 2; k++) {
      a.w[k][e] = p.w[k][e];
      a.s[k][e] = p.s[k][e];
    }
  hipError_t e;
  if (p.yt_bf16) e = p.xt_bf16 ? gate_up_go<uint16_t, 2>(p, a, stream) : gate_up_go<float, 2>(p, a, stream);
  else e = p.xt_bf16 ? gate_up_go<uint16_t, 3>(p, a, stream) : gate_up_go<float, 3>(p, a, stream);
  if (e != hipSuccess) return e;
  for (uint32_t i = 0; i < p.E; i++) {
    a.w[0][i] = p.w[2][i];
    a.s[0][i] = p.s[2][i];
  }
  return p.yt_bf16 ? down_go<2, uint16_t>(p, a, stream) : down_go<3, float>(p, a, stream);
}

}  // namespace frx
