// frx_fp4_moe.hip — a whole expert layer for a few tokens, its experts' weights in 4 bits.
//
//   y[t] = sum_j w[t][j] down_e(act(gate_e x_t) * up_e x_t),  e = idx[t][j]
//
// A few tokens read every weight of the experts they reach once: bound by those bytes
// (17/32 a value). So the activations stay as they are: the codes widen to bf16 times
// their block's power of two (exact, one conversion for two codes) and meet x as bf16, or
// an f32 x as three bf16 planes that hold all of it; sums in fp32.
//
//   route     the router's logits, top-k and softmax, where the caller has none
//   gate, up  h = act(g) * u times the route's weight, as three bf16 planes, a row for each route
//   down      a row of f32 sums for each route (and slice of I)
//   combine   the routes of each token, in order
//
// gate_up and down run one workgroup of 8 waves on each compute unit, which takes an even
// share of the row tiles of an expert in use (of a group of its tokens, where they are many: then
// its weights are read again), one tile of 16 weight rows after the other. The
// waves split K. A wave's slice of the expert's tokens stays in registers as long as the
// expert does not change: columns of the matrix instruction are (token, plane) pairs, the
// expert's tokens gathered. So a tile costs its weights' bytes, the widening, four matrix
// instructions for 128 columns, and one exchange of the waves' sums through LDS. The weights
// of the next tiles are on their way meanwhile, by LDS DMA into a ring that each wave has for
// itself (held in registers they were waited for at every turn of the loop).
//
// h keeps the 24 bits of an f32 number whatever y is: two planes (2^-17 of h) saved a bf16 layer 0.4 us of
// 65 at 8 tokens, 3 of 93 at 64 and 8 of 109 at 64 of 32 experts, and flipped last bits of its outputs.
//
// 16 experts, top 2, H 2048, I 5632, route + gate and up + down + join, us: 1 token bf16 14.5 + 9.6
// + 5.0 (its weights' bytes 7.1 at a copy's rate; a workgroup's way to its first tile is 5 to 6,
// much of it instructions that are fetched for the first time), 8 tokens 6.0 + 31.9 + 20.5 + 4.7
// (37; gate's and up's weights at 4.0 TB/s, down's at 3.0), 61 tokens f32 78.9 + 42.0 + 5.0 (57; of the
// first 46 are the weights' way alone, 10 the products, 17 a tile's sums, activation and stores). Waits that
// leave out a wave's own stores gained nothing, nor did sums by lanes of eight.
#include "frx_fp4.hpp"
#include "frx_internal.hpp"

namespace frx {

namespace {

constexpr int WAVES = 8, NT = WAVES * 64;

// ---- routes ------------------------------------------------------------------------

constexpr int MOST_SLOTS = FP4_MOE_MAX_T * 64;
constexpr int KEPT_SLOTS = 512;

struct FewArgs {
  const void *x, *router;
  uint32_t *idx;
  float *wts;
  uint16_t *h;  // [slot][plane][I]
  float *part;  // [slice][slot][H]
  uint32_t T, K, N;  // columns of a weight row, rows
  int E, top_k, act, rt_bf16, route, slices, per;  // slices of K, steps of 128 in each (down)
  const uint8_t *w[2][FP8_MAXE], *s[2][FP8_MAXE];  // gate, up; or down
};

struct Shared {
  const uint8_t *w[2][FP8_MAXE], *s[2][FP8_MAXE];
  float logit[64];
  uint8_t expert[MOST_SLOTS];  // of each slot; 255: none
  int count[FP8_MAXE];         // the expert's routes
  float wts[KEPT_SLOTS];       // of each slot, where there are few
  float share[64];             // of the expert at hand: its tokens' weights, added where a token names it twice,
  uint16_t slot[64];           // their slots,
  uint8_t token[64];           // and which they are
};

// A token's logits: a wave for each expert.
template <int WAVES, typename XT, typename RT>
__device__ __forceinline__ void router_logits(const XT *x, const RT *router, uint32_t H, int E, float *logit) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int e = wave; e < E; e += WAVES) {
    float s = 0.f;
#pragma unroll 4
    for (uint32_t k = lane * 8; k < H; k += 512) {
      float r[8], v[8];
      ld8u(router + (size_t)e * H + k, r);
      ld8u(x + k, v);
#pragma unroll
      for (int i = 0; i < 8; i++) s = __builtin_fmaf(v[i], r[i], s);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) logit[e] = s;
  }
}

// A wave: the experts of the largest logits, ties to the lowest index, a NaN below every
// number; weights exp(l - l_max) over their sum. Lane e returns its expert's place among
// them (top_k and more: none) and weight.
__device__ __forceinline__ int top_experts(const float *logit, int E, int top_k, float &weight) {
  const int lane = threadIdx.x & 63;
  const float mine = lane < E ? logit[lane] + 0.0f : 0.f;  // -0 orders as 0
  const uint32_t bits = __float_as_uint(mine);
  const uint32_t key = mine != mine ? 0 : bits >> 31 ? ~bits : bits | 0x80000000u;
  int rank = 0;  // experts ahead of this one
  for (int i = 0; i < E; i++) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)key, i);
    rank += other > key || (other == key && i < lane);
  }
  if (lane >= E) rank = 64;
  const int first = __ffsll((unsigned long long)__ballot(rank == 0)) - 1;
  const float top = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)bits, first));
  float w = rank < top_k ? expf(mine - top) : 0.f, sum = w;
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  weight = w / sum;
  return rank;
}

// A workgroup per token: 8 tokens, 16 experts, H 2048 5.9 us (with 8 waves 8.4). Not for a single
// token, whose gate_up routes for itself (fp4_routes_inside).
constexpr int ROUTE_WAVES = 16;
template <typename XT, typename RT>
__global__ __launch_bounds__(ROUTE_WAVES * 64) void fp4_route_kernel(const XT *__restrict__ x,
                                                                     const RT *__restrict__ router,
                                                                     uint32_t H, int E, int top_k, uint32_t *__restrict__ idx,
                                                                     float *__restrict__ wts) {
  __shared__ float logit[64];
  const size_t t = blockIdx.x;
  router_logits<ROUTE_WAVES>(x + t * H, router, H, E, logit);
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float w;
  const int place = top_experts(logit, E, top_k, w);
  if (place < top_k) {
    idx[t * top_k + place] = threadIdx.x;
    wts[t * top_k + place] = w;
  }
}

// Fills the experts' addresses and the routes. ROUTE: by
// the router where the launch says so, workgroup 0 writing the routes for the launches behind.
template <typename XT, bool ROUTE>
__device__ __forceinline__ void read_routes(const FewArgs &p, Shared &sh) {
  const int slots = (int)p.T * p.top_k, lane = threadIdx.x & 63;
  if (threadIdx.x < 2 * FP8_MAXE) {  // (addressed by lane: one wait, beside the routes')
    const int k = threadIdx.x >> 6;
    sh.w[k][lane] = p.w[k][lane];
    sh.s[k][lane] = p.s[k][lane];
  }
  if (threadIdx.x < FP8_MAXE) sh.count[threadIdx.x] = 0;
  __syncthreads();
  if (ROUTE && p.route) {
    const XT *x = static_cast<const XT *>(p.x);
    if (p.rt_bf16) router_logits<WAVES>(x, static_cast<const uint16_t *>(p.router), p.K, p.E, sh.logit);
    else router_logits<WAVES>(x, static_cast<const float *>(p.router), p.K, p.E, sh.logit);
    __syncthreads();
    if (threadIdx.x < 64) {
      float w;
      const int place = top_experts(sh.logit, p.E, p.top_k, w);
      if (place < p.top_k) {
        sh.expert[place] = lane;
        atomicAdd(&sh.count[lane], 1);
        sh.wts[place] = w;
        if (blockIdx.x == 0) {
          p.idx[place] = lane;
          p.wts[place] = w;
        }
      }
    }
  } else {
    for (int s = threadIdx.x; s < slots; s += NT) {
      const uint32_t e = p.idx[s];
      if (s < KEPT_SLOTS) sh.wts[s] = p.wts[s];
      sh.expert[s] = e < (uint32_t)p.E ? e : 255;
      if (e < (uint32_t)p.E) atomicAdd(&sh.count[e], 1);
    }
  }
  __syncthreads();
}

// The experts in use, each as often as `tokens` of its routes at a time take: lane e has
// expert e's.
struct Groups {
  uint64_t active;
  int groups, upto, total;
  __device__ __forceinline__ Groups(const Shared &sh, int E, int tokens) {
    const int lane = threadIdx.x & 63, n = lane < E ? sh.count[lane] : 0;
    active = __ballot(n > 0);
    groups = upto = n > 0;
    if (__ballot(n > tokens) == 0) {
      total = __popcll(active);
    } else {
      groups = 0;
      for (int left = n; left > 0; left -= tokens) groups++;
      upto = groups;
      for (int s = 1; s < 64; s <<= 1) {
        const int v = __shfl_up(upto, s);
        if (lane >= s) upto += v;
      }
      total = __builtin_amdgcn_readlane(upto, 63);
    }
  }
  // Group u's expert, and which of that expert's groups it is.
  __device__ __forceinline__ int find(int u, int &which) const {
    which = 0;
    if (total == __popcll(active)) {  // one of each
      uint64_t m = active;
      for (int i = 0; i < u; i++) m &= m - 1;
      return __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)m) - 1);
    }
    const int e = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(upto > u)) - 1);
    which = u - __builtin_amdgcn_readlane(upto - groups, e);
    return e;
  }
};

// a / b for numbers below 2^22.
__device__ __forceinline__ int div22(int a, int b) {
  const int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));  // one off at most
  const int r = a - q * b;
  return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// Which of `units` (an expert, or a slice of one, with `tiles` row tiles) this workgroup works on, and
// on which tiles: units share the workgroups evenly, so that one belongs to no two of them; where
// there are more units than workgroups, whole units in turn.
struct Share {
  int unit, step, first, last;
  __device__ __forceinline__ Share(int units, int tiles) {
    const int b = blockIdx.x, G = gridDim.x;
    if (units == 0) {  // nothing is routed
      unit = first = last = 0;
      step = 1;
    } else if (units <= G) {
      unit = div22(b * units + units - 1, G);  // of b in [u G / units, (u + 1) G / units)
      const int lo = div22(unit * G, units), n = div22((unit + 1) * G, units) - lo, i = b - lo;
      const int q = div22(tiles, n), r = tiles - q * n;
      first = q * i + min(i, r);
      last = first + q + (i < r);
      step = units;
    } else {
      unit = b;
      step = G;
      first = 0;
      last = tiles;
    }
  }
};

// Expert e's tokens into slot[] (and share[] where WEIGHTS): the first slot of each that
// names it. Every wave finds them; wave 0 writes. Returns their number. The caller puts
// barriers before (nobody reads the lists any more) and behind.
template <bool WEIGHTS>
__device__ __forceinline__ int list_tokens(const FewArgs &p, Shared &sh, int e) {
  const int lane = threadIdx.x & 63;
  const auto weight = [&](int s) { return s < KEPT_SLOTS ? sh.wts[s] : p.wts[s]; };
  int first = -1;
  float w = 0.f;
  if (lane < (int)p.T)
    for (int j = 0; j < p.top_k; j++)
      if (sh.expert[lane * p.top_k + j] == e) {
        if (first < 0) first = lane * p.top_k + j;
        if (WEIGHTS && threadIdx.x < 64) w += weight(lane * p.top_k + j);
      }
  const uint64_t mine = __ballot(first >= 0);
  if (threadIdx.x < 64 && first >= 0) {
    const int at = __popcll(mine & ((1ull << lane) - 1));
    sh.slot[at] = (uint16_t)first;
    sh.token[at] = (uint8_t)lane;
    if (WEIGHTS) sh.share[at] = w;
  }
  return __popcll(mine);
}

// ---- operands ----------------------------------------------------------------------

// Eight codes times 2^(b - 127) as bf16; s = fp4_power(b).
__device__ __forceinline__ u32x4 widen8(uint32_t c, float s) {
  return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

// A value as bf16 planes of which each holds the next 8 bits. What is left of it behind a plane is kept
// times 2^7, then 2^8, which brings it to the plane's own size at most: a bf16 number is a multiple of
// 2^-133, so planes in place would lose the end of values below 2^-110, and all of those below 2^-133.
// So three planes are the value, but for the 2^-149 of an odd multiple of it. (Beside planes in place: 61
// tokens f32, 16 experts, 2048 / 5632, 115.2 us and 114.1; 5 of 8, 8192 / 704, whose x is cut for every
// chunk, 64.0 and 60.6.) The value is an f32 number, not the product that it is the rounding of, as a fused
// multiply-subtract would have it.
__device__ __forceinline__ float cut8(float v, uint32_t &plane, int j) {
#pragma clang fp contract(off)
  plane = __float_as_uint(v) & 0xFFFF0000u;
  return (v - __uint_as_float(plane)) * (j == 0 ? 0x1p7f : 0x1p8f);
}
__device__ __forceinline__ constexpr float plane_unit(int j) { return j == 0 ? 1.0f : j == 1 ? 0x1p-7f : 0x1p-15f; }

// Plane `plane` of eight activations.
__device__ __forceinline__ u32x4 act8(const uint16_t *p, int) { return *reinterpret_cast<const u32x4_u *>(p); }
__device__ __forceinline__ u32x4 act8(const float *p, int plane) {
  float v[8];
  ld8u(p, v);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float left = v[i];
    for (int j = 0; j < 2; j++) {
      uint32_t u;
      const float next = cut8(left, u, j);
      left = j < plane ? next : left;
    }
    h[i] = __float_as_uint(left);
  }
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = (h[2 * i] >> 16) | (h[2 * i + 1] & 0xFFFF0000u);
  return o;
}

// An address that is the same in every lane.
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
  const uint64_t v = reinterpret_cast<uintptr_t>(p);
  return reinterpret_cast<const uint8_t *>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                                           (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// What a wave reads of a tile of 16 rows, STEPS of 128 columns from step kb on: lane (row l16,
// group g) block 4 kb + g of its row, 16 bytes at lane * 16 in LDS, and the scales of 4 blocks
// as a dword, lane (row, step). Blocks from `blocks` on repeat the last one; they count under
// the scale 2^-127 and meet zeros of x.
template <int STEPS>
struct Place {
  static constexpr int DWORDS = STEPS * 256 + (STEPS + 3) / 4 * 64, LOADS = STEPS + (STEPS + 3) / 4;
  uint32_t c[STEPS], s[(STEPS + 3) / 4];
  int inside;  // of the lane's blocks so many are the row's
  __device__ __forceinline__ void set(int K, int kb, int blocks, int l16, int g) {
    const int kbs = (K + 127) >> 7;
#pragma unroll
    for (int i = 0; i < STEPS; i++) c[i] = (uint32_t)(l16 * (K / 2) + 16 * min((kb + i) * 4 + g, blocks - 1));
#pragma unroll
    for (int i = 0; i < (STEPS + 3) / 4; i++) s[i] = (uint32_t)(l16 * kbs + min(kb + 4 * i + g, kbs - 1)) * 4;
    inside = max(0, (blocks - kb * 4 - g + 3) >> 2);
  }
  // codes, scales: of the tile's first row
  __device__ __forceinline__ void load(uint32_t *to, const uint8_t *codes, const uint8_t *scales, int K) const {
    const __amdgpu_buffer_rsrc_t rc = buffer_rsrc(codes, 16u * (uint32_t)(K / 2)), rs = buffer_rsrc(scales, 16u * fp4_scale_bytes(K));
#pragma unroll
    for (int i = 0; i < STEPS; i++) lds_load16(rc, to + i * 256, c[i], 0);
#pragma unroll
    for (int i = 0; i < (STEPS + 3) / 4; i++) lds_load4(rs, to + STEPS * 256 + i * 64, s[i], 0);
  }
};

// from: a wave's piece of a tile, loaded as above; inside: of the lane's blocks so many count.
template <int STEPS, int CT>
__device__ __forceinline__ void multiply(f32x4 (&acc)[CT], const uint32_t *from, const u32x4 (&x)[STEPS][4][CT],
                                         int inside, int cols) {
  const int lane = threadIdx.x & 63;
  const uint8_t *scales = reinterpret_cast<const uint8_t *>(from + STEPS * 256) + (lane & 15) * 4 + (lane >> 4);
#pragma unroll
  for (int i = 0; i < STEPS; i++) {
    const u32x4 c = *reinterpret_cast<const u32x4 *>(from + i * 256 + lane * 4);
    const float s = fp4_power(i < inside ? scales[i * 64] : 0);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const u32x4 v = widen8(c[q], s);
#pragma unroll
      for (int t = 0; t < CT; t++)
        if (CT == 1 || 16 * t < cols) acc[t] = mfma16(v, x[i][q][t], acc[t]);
    }
  }
}

__device__ __forceinline__ float activate(float g, int act) {
  if (act == 0) return g / (1.0f + expf(-g));
  return 0.5f * g * (1.0f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g)));
}

// The waves' sums in LDS, floats: 16 x 16 of a column tile as 4 groups of 4 rows, 80 apart, [column]
// [row of 4] in each: a group's banks are 16 from the next one's.
constexpr int RED = 320;
__device__ __forceinline__ void put_sums(float *red, const f32x4 &v) {
  const int lane = threadIdx.x & 63;
  *reinterpret_cast<f32x4 *>(red + (lane >> 4) * 80 + (lane & 15) * 4) = v;
}
// Sum of a token's planes over the waves, STRIDE apart, for row r of the tile, in order.
template <int P, int STRIDE>
__device__ __forceinline__ float waves_sum(const float *red, int token, int r) {
  float v = 0.f;
#pragma unroll
  for (int j = 0; j < P; j++) {
    const int col = token * P + j;
    const float *at = red + (col >> 4) * RED + (r >> 2) * 80 + (col & 15) * 4 + (r & 3);
#pragma unroll 8
    for (int w = 0; w < WAVES; w++) v = __builtin_fmaf(at[w * STRIDE], plane_unit(j), v);
  }
  return v;
}

// CT column tiles of 16 (token, plane) pairs at a time; D pieces of weights (a tile of gate, the
// same of up, the next tile of gate ...) on their way; RB buffers for the waves' sums, with one
// a second barrier guards it. CHUNKED: K is longer than the waves hold and goes by chunks, x
// loaded anew for each.
template <typename XT, int STEPS, int CT, int D, int RB, bool CHUNKED>
__global__ __launch_bounds__(NT) void fp4_gate_up_kernel(const FewArgs p) {
  constexpr int P = sizeof(XT) == 2 ? 1 : 3, TOKENS = 16 * CT / P, DW = Place<STEPS>::DWORDS;
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ Shared sh;
  read_routes<XT, true>(p, sh);
  const Groups groups(sh, p.E, TOKENS);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int K = (int)p.K, blocks = K / 32, kbs = (K + 127) >> 7, tiles = (int)p.N / 16;
  const int chunks = CHUNKED ? (kbs + WAVES * STEPS - 1) / (WAVES * STEPS) : 1;
  const Share share(groups.total, tiles);
  const int t0 = share.first, count = share.last - t0;
  Place<STEPS> place;
  place.set(K, wave * STEPS, blocks, l16, g);
  uint32_t *ring = lds + wave * (D * DW);
  float *reds = reinterpret_cast<float *>(lds + WAVES * D * DW);
  int phase = 0;
  if (count == 0) return;
  for (int u = share.unit; u < groups.total; u += share.step) {
    int which;
    const int e = groups.find(u, which);
    const uint8_t *wg = uniform(sh.w[0][e]), *wu = uniform(sh.w[1][e]), *sg = uniform(sh.s[0][e]), *su = uniform(sh.s[1][e]);
    const int pieces = 2 * count * chunks;
    // piece j: matrix j % 2, step j / 2 (past the last one it is loaded again: the waits go by the number of loads)
    const auto load_w = [&](int j, int d) {
      j = j < pieces ? j : pieces - 2 + (j & 1);
      const int i = CHUNKED ? (j >> 1) / chunks : j >> 1;
      if (CHUNKED) place.set(K, ((j >> 1) - i * chunks) * WAVES * STEPS + wave * STEPS, blocks, l16, g);
      const size_t c = (size_t)(t0 + i) * 16 * (K / 2), s = (size_t)(t0 + i) * 16 * (4 * kbs);
      place.load(ring + d * DW, (j & 1 ? wu : wg) + c, (j & 1 ? su : sg) + s, K);
    };
    // the first pieces, then x, which arrives behind them, then the others
    constexpr int EARLY = CHUNKED ? D : 2;
#pragma unroll
    for (int d = 0; d < EARLY; d++) load_w(d, d);
    barrier_lds();
    const int n = list_tokens<true>(p, sh, e);
    barrier_lds();
    const int c0 = which * TOKENS, cols = min(n - c0, TOKENS) * P;
    if (cols > 0) {  // (a token may name an expert twice)
      u32x4 x[STEPS][4][CT];
      int inside = 0;
      const auto load_x = [&](int kb0) {
#pragma unroll
        for (int t = 0; t < CT; t++) {
          const int col = 16 * t + l16, tok = sh.token[c0 + min(col, cols - 1) / P];
          const XT *from = static_cast<const XT *>(p.x);
#pragma unroll
          for (int i = 0; i < STEPS; i++) {
            const int b = (kb0 + i) * 4 + g;
            const bool use = b < blocks && col < cols;
            const uint32_t o = (uint32_t)tok * K + 32 * min(b, blocks - 1);
#pragma unroll
            for (int q = 0; q < 4; q++) {
              x[i][q][t] = act8(from + (o + 8 * q), col % P);
              if (!use) x[i][q][t] = (u32x4){0, 0, 0, 0};
            }
            if (sizeof(XT) == 4 && (CT * STEPS > 4) && (i & 1)) __builtin_amdgcn_sched_barrier(0);  // (two values a register: not all at once)
          }
        }
        inside = max(0, (blocks - kb0 * 4 - g + 3) >> 2);
      };
      if (!CHUNKED) {
        __builtin_amdgcn_sched_barrier(0);
        load_x(wave * STEPS);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = EARLY; d < D; d++) load_w(d, d);
      }
      f32x4 acc[2][CT];
      int chunk = 0, tile = t0, d = 0;
      for (int j = 0; j < pieces; j += 2) {
        if (CHUNKED) load_x(chunk * WAVES * STEPS + wave * STEPS);
        if (!CHUNKED || chunk == 0)
#pragma unroll
          for (int t = 0; t < CT; t++) acc[0][t] = acc[1][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < 2; m++) {
          wait_vmcnt<(D - 1) * Place<STEPS>::LOADS>();
          __builtin_amdgcn_sched_barrier(0);
          multiply<STEPS, CT>(acc[m], ring + d * DW, x, inside, cols);
          __builtin_amdgcn_sched_barrier(0);
          load_w(j + m + D, d);
          d = d + 1 == D ? 0 : d + 1;
        }
        if (CHUNKED && ++chunk < chunks) continue;
        chunk = 0;
        constexpr int MAT = CT * RED + 32, WAVE = 2 * MAT;  // [wave][matrix][column tile]
        float *red = reds + phase * (WAVES * WAVE);
        if (RB == 2) phase ^= 1;
        else barrier_lds();
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int t = 0; t < CT; t++)
            if (16 * t < cols) put_sums(red + wave * WAVE + m * MAT + t * RED, acc[m][t]);
        barrier_lds();
        // a thread an inner column (of 16), matrix and token
        const int r = threadIdx.x & 15, m = (threadIdx.x >> 4) & 1;
        for (int token = threadIdx.x >> 5; token * P < cols; token += NT / 32) {
          const float sum = waves_sum<P, WAVE>(red + m * MAT, token, r);
          const float other = __shfl_xor(sum, 16);
          if (m) continue;
          const float v = activate(sum, p.act) * other * sh.share[c0 + token];
          uint16_t *to = p.h + (size_t)sh.slot[c0 + token] * FP4_MOE_PLANES * p.N + (uint32_t)tile * 16 + r;
          uint32_t u;
          float left = v;
#pragma unroll
          for (int j = 0; j < FP4_MOE_PLANES; j++) {
            left = cut8(left, u, j);
            to[j * (size_t)p.N] = (uint16_t)(u >> 16);
          }
        }
        tile++;
      }
    }
    wait_vmcnt<0>();  // nothing is in flight into the ring any more
  }
}

// ---- down --------------------------------------------------------------------------

// A unit is a group of an expert's tokens and a slice of K; D tiles' weights on their way.
template <int STEPS, int CT, int D>
__global__ __launch_bounds__(NT) void fp4_down_kernel(const FewArgs p) {
  constexpr int P = FP4_MOE_PLANES, TOKENS = 16 * CT / P;
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ Shared sh;
  read_routes<uint16_t, false>(p, sh);
  const Groups groups(sh, p.E, TOKENS);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int K = (int)p.K, blocks = K / 32, kbs = (K + 127) >> 7, tiles = (int)p.N / 16;
  const int units = groups.total * p.slices, slots = (int)p.T * p.top_k;
  const Share share(units, tiles);
  const int t0 = share.first, count = share.last - t0;
  constexpr int DW = Place<STEPS>::DWORDS;
  uint32_t *ring = lds + wave * (D * DW);
  float *reds = reinterpret_cast<float *>(lds + WAVES * D * DW);
  int phase = 0;
  if (count == 0) return;
  for (int u = share.unit; u < units; u += share.step) {
    const int group = div22(u, p.slices), slice = u - group * p.slices;
    int which;
    const int e = groups.find(group, which);
    const uint8_t *wd = uniform(sh.w[0][e]), *sd = uniform(sh.s[0][e]);
    const int kb = slice * p.per + wave * STEPS;
    const int stop = min((slice + 1) * p.per * 4, blocks);  // the slice's blocks
    Place<STEPS> place;
    place.set(K, kb, stop, l16, g);
    const auto load_w = [&](int j, int d) {
      const size_t row = (size_t)(t0 + min(j, count - 1)) * 16;
      place.load(ring + d * DW, wd + row * (K / 2), sd + row * (4 * kbs), K);
    };
    load_w(0, 0);
    barrier_lds();
    const int n = list_tokens<false>(p, sh, e);
    barrier_lds();
    const int c0 = which * TOKENS, cols = min(n - c0, TOKENS) * P;
    if (cols > 0) {
      __builtin_amdgcn_sched_barrier(0);
      u32x4 x[STEPS][4][CT];
#pragma unroll
      for (int t = 0; t < CT; t++) {
        const int col = 16 * t + l16, cc = min(col, cols - 1);
        const uint16_t *row = p.h + ((size_t)sh.slot[c0 + cc / P] * P + cc % P) * K;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
          const int b = (kb + i) * 4 + g;
#pragma unroll
          for (int q = 0; q < 4; q++)
            x[i][q][t] = *reinterpret_cast<const u32x4 *>(row + 32 * min(b, stop - 1) + 8 * q);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 1; d < D; d++) load_w(d, d);
      wait_vmcnt<(D - 1) * Place<STEPS>::LOADS>();
#pragma unroll
      for (int t = 0; t < CT; t++)
#pragma unroll
        for (int i = 0; i < STEPS; i++)
          if ((kb + i) * 4 + g >= stop || 16 * t + l16 >= cols)
#pragma unroll
            for (int q = 0; q < 4; q++) x[i][q][t] = (u32x4){0, 0, 0, 0};
      int d = 0;
      for (int j = 0; j < count; j++) {
        f32x4 acc[CT];
#pragma unroll
        for (int t = 0; t < CT; t++) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        wait_vmcnt<(D - 1) * Place<STEPS>::LOADS>();
        __builtin_amdgcn_sched_barrier(0);
        multiply<STEPS, CT>(acc, ring + d * DW, x, place.inside, cols);
        __builtin_amdgcn_sched_barrier(0);
        load_w(j + D, d);
        d = d + 1 == D ? 0 : d + 1;
        float *red = reds + phase * (WAVES * CT * RED);
        phase ^= 1;
#pragma unroll
        for (int t = 0; t < CT; t++)
          if (16 * t < cols) put_sums(red + (wave * CT + t) * RED, acc[t]);
        barrier_lds();
        for (int token = threadIdx.x >> 4; token * P < cols; token += NT / 16) {
          const int r = threadIdx.x & 15;
          p.part[((size_t)slice * slots + sh.slot[c0 + token]) * p.N + (uint32_t)(t0 + j) * 16 + r] =
              waves_sum<P, CT * RED>(red, token, r);
        }
      }
    }
    wait_vmcnt<0>();  // nothing is in flight into the ring any more
  }
}

// y[t] = its routes' sums over the slices, in the order of the routes. A route that goes
// nowhere, and a later one to an expert that the token has named, has none. 5 us, most of it a
// launch's own; joined in down by the last workgroup at each tile 61 tokens took 20 us more, 8
// two more, 1 as long.
template <typename YT>
__global__ __launch_bounds__(256) void fp4_join_kernel(const FewArgs p, YT *__restrict__ y) {
  const uint32_t t = blockIdx.y, n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= p.N) return;
  const uint32_t *idx = p.idx + t * p.top_k;
  const size_t slots = (size_t)p.T * p.top_k;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < p.top_k; j++) {
    bool use = idx[j] < (uint32_t)p.E;
    for (int k = 0; k < j; k++) use &= idx[k] != idx[j];
    if (!use) continue;
    for (int c = 0; c < p.slices; c++)
      v += *reinterpret_cast<const f32x4 *>(p.part + (c * slots + t * p.top_k + j) * p.N + n);
  }
  YT *d = y + (size_t)t * p.N + n;
#pragma unroll
  for (int i = 0; i < 4; i++) {  // N % 32 == 0: whole quads
    if constexpr (sizeof(YT) == 4) d[i] = v[i];
    else d[i] = (uint16_t)bf16_rne_nb(v[i]);
  }
}

template <typename XT>
hipError_t route_go(const Fp4Moe &p, hipStream_t stream) {
  const XT *x = static_cast<const XT *>(p.x);
  if (p.rt_bf16)
    hipLaunchKernelGGL((fp4_route_kernel<XT, uint16_t>), dim3(p.T), dim3(ROUTE_WAVES * 64), 0, stream, x,
                       static_cast<const uint16_t *>(p.router), p.H, (int)p.E, (int)p.top_k, p.idx, p.wts);
  else
    hipLaunchKernelGGL((fp4_route_kernel<XT, float>), dim3(p.T), dim3(ROUTE_WAVES * 64), 0, stream, x,
                       static_cast<const float *>(p.router), p.H, (int)p.E, (int)p.top_k, p.idx, p.wts);
  return hipGetLastError();
}

template <typename Kernel>
hipError_t few_go(Kernel kernel, std::atomic<uint64_t> &done, int lds, int cus, const FewArgs &a, hipStream_t stream) {
  const hipError_t e = opt_in_lds(reinterpret_cast<const void *>(kernel), lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3(cus), dim3(NT), lds, stream, a);
  return hipGetLastError();
}

template <typename XT, int STEPS, int CT, int D, int RB, bool CHUNKED>
hipError_t gate_up_go(const FewArgs &a, int cus, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = WAVES * D * Place<STEPS>::DWORDS * 4 + RB * WAVES * 2 * (CT * RED + 32) * 4;
  static_assert(lds + sizeof(Shared) <= 160 << 10, "LDS");
  return few_go(fp4_gate_up_kernel<XT, STEPS, CT, D, RB, CHUNKED>, done, lds, cus, a, stream);
}

template <typename XT>
hipError_t gate_up(const FewArgs &a, const Fp4FewPlan &plan, int cus, hipStream_t stream) {
  if (plan.slices > 1) return gate_up_go<XT, 4, 1, 3, 1, true>(a, cus, stream);
  if (plan.steps == 4) {
    if constexpr (sizeof(XT) == 2)
      if (plan.tiles == 2) return gate_up_go<XT, 4, 2, 2, 1, false>(a, cus, stream);
    return gate_up_go<XT, 4, 1, 3, 1, false>(a, cus, stream);
  }
  if (plan.tiles == 1) return gate_up_go<XT, 2, 1, 5, 2, false>(a, cus, stream);
  return plan.tiles == 2 ? gate_up_go<XT, 2, 2, 3, 2, false>(a, cus, stream) : gate_up_go<XT, 2, 3, 4, 1, false>(a, cus, stream);
}

template <int STEPS, int CT, int D>
hipError_t down_go(const FewArgs &a, int cus, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = WAVES * D * Place<STEPS>::DWORDS * 4 + 2 * WAVES * CT * RED * 4;
  static_assert(lds + sizeof(Shared) <= 160 << 10, "LDS");
  return few_go(fp4_down_kernel<STEPS, CT, D>, done, lds, cus, a, stream);
}

hipError_t down(const FewArgs &a, const Fp4FewPlan &plan, int cus, hipStream_t stream) {
  if (plan.tiles == 3) return plan.steps == 2 ? down_go<2, 3, 4>(a, cus, stream) : down_go<3, 3, 3>(a, cus, stream);
  if (plan.tiles == 2) return plan.steps == 2 ? down_go<2, 2, 5>(a, cus, stream) : down_go<3, 2, 3>(a, cus, stream);
  if (plan.steps == 2) return down_go<2, 1, 5>(a, cus, stream);
  return plan.steps == 3 ? down_go<3, 1, 4>(a, cus, stream) : down_go<4, 1, 3>(a, cus, stream);
}

}  // namespace

size_t fp4_moe_h_bytes(uint32_t T, uint32_t I, uint32_t top_k) {
  return (size_t)T * top_k * FP4_MOE_PLANES * I * 2;
}
size_t fp4_moe_part_bytes(uint32_t T, uint32_t H, uint32_t I, uint32_t E, uint32_t top_k) {
  return (size_t)fp4_down_plan(T, I, E, top_k, FP4_MOE_PLANES).slices * T * top_k * H * 4;
}

hipError_t launch_fp4_moe(const Fp4Moe &p, int cus, hipStream_t stream) {
  const bool fused = p.router && fp4_routes_inside(p.T);
  if (p.router && !fused) {
    const hipError_t e = p.xt_bf16 ? route_go<uint16_t>(p, stream) : route_go<float>(p, stream);
    if (e != hipSuccess) return e;
  }
  FewArgs a = {p.x,      p.router, p.idx,    p.wts, p.h, p.part, p.T, p.H, p.I, (int)p.E, (int)p.top_k, p.act,
               p.rt_bf16, fused,    1,        0,     {},  {}};
  for (uint32_t e = 0; e < p.E; e++)
    for (int k = 0; k < 2; k++) {
      a.w[k][e] = p.w[k][e];
      a.s[k][e] = p.s[k][e];
    }
  const Fp4FewPlan up = fp4_gate_up_plan(p.T, p.H, p.E, p.top_k, p.xt_bf16 ? 1 : 3);
  hipError_t e = p.xt_bf16 ? gate_up<uint16_t>(a, up, cus, stream) : gate_up<float>(a, up, cus, stream);
  if (e != hipSuccess) return e;
  for (uint32_t i = 0; i < p.E; i++) {
    a.w[0][i] = p.w[2][i];
    a.s[0][i] = p.s[2][i];
  }
  const Fp4FewPlan dn = fp4_down_plan(p.T, p.I, p.E, p.top_k, FP4_MOE_PLANES);
  a.route = 0;
  a.K = p.I;
  a.N = p.H;
  a.slices = dn.slices;
  a.per = dn.per;
  e = down(a, dn, cus, stream);
  if (e != hipSuccess) return e;
  const dim3 grid((p.H + 1023) / 1024, p.T);
  if (p.yt_bf16) hipLaunchKernelGGL(fp4_join_kernel<uint16_t>, grid, dim3(256), 0, stream, a, static_cast<uint16_t *>(p.y));
  else hipLaunchKernelGGL(fp4_join_kernel<float>, grid, dim3(256), 0, stream, a, static_cast<float *>(p.y));
  return hipGetLastError();
}

}  // namespace frx
