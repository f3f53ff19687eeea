// frx_route.hip — tokens into rows sorted by expert, and back, with gradients.
//
// sort: a stable counting sort of the slots t * top_k + j by expert; segments
// start at multiples of `align`.
// dispatch: xs[row] = x[token of row].   combine: y[t] = sum_j w[t][j] ys[row_of[t][j]].
// combine_backward: dys[row] = w[slot] dy[token], dw[t][j] = <dy[t], ys[row_of[t][j]]>.
// All but the sort are bound by memory. us, 8192 tokens of 4096 bf16 columns, two
// routes each: dispatch 38.6 (201 MB, 5.2 TB/s with tokens read once from HBM),
// combine 49 (4.1 TB/s), combine_backward 57 (336 MB, 5.9 TB/s), sort 10 (two
// launches); 33 tokens of four routes 2.4 to 4.3 each.
#include "frx_device.hpp"
#include "frx_internal.hpp"

namespace frx {

namespace {

constexpr int ROUTE_MAXE = 64;
constexpr uint32_t kNone = 0xFFFFFFFFu;

constexpr int SORT_NT = 1024;     // slots of a chunk, one a thread
constexpr int ROUTE_RUNS = 1024;  // runs of chunks: each reads the counts of all

// Counts of one chunk by expert, wave by wave, and each thread's rank among
// the slots of its expert in its wave. e >= E: no expert. A wave finds the
// lanes of equal expert with a ballot for each bit of the index.
__device__ __forceinline__ int chunk_ranks(uint32_t e, int E, int (*wave_cnt)[ROUTE_MAXE]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  wave_cnt[wave][lane] = 0;
  __builtin_amdgcn_wave_barrier();  // lanes of one wave: its LDS stores keep their order
  const bool in = e < (uint32_t)E;
  unsigned long long same = __ballot(in);
#pragma unroll
  for (int b = 0; b < 6; b++) {
    const unsigned long long m = __ballot((e >> b) & 1);
    same &= (e >> b) & 1 ? m : ~m;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1ull));
  if (in && rank == 0) wave_cnt[wave][e] = __popcll(same);
  return rank;
}

// Exclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_before(int v) {
  int x = v;
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if ((threadIdx.x & 63) >= o) x += y;
  }
  return x - v;
}

// One workgroup, chunk after chunk: counts first, then rows.
__global__ __launch_bounds__(SORT_NT) void route_sort_kernel(const uint32_t *__restrict__ idx, RouteRows r) {
  __shared__ int wave_cnt[16][ROUTE_MAXE];
  __shared__ int base[ROUTE_MAXE];  // next row of each expert
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int A = r.T * r.top_k, E = r.E;
  if (tid < ROUTE_MAXE) base[tid] = 0;
  for (int i = tid; i < r.R; i += SORT_NT) r.slot_of[i] = kNone;
  uint32_t e = kNone;
  int rank = 0;
  for (int c0 = 0; c0 < A; c0 += SORT_NT) {
    __syncthreads();
    e = c0 + tid < A ? idx[c0 + tid] : kNone;
    rank = chunk_ranks(e, E, wave_cnt);
    __syncthreads();
    if (tid < E) {
      int s = 0;
      for (int w = 0; w < 16; w++) s += wave_cnt[w][tid];
      base[tid] += s;
    }
  }
  __syncthreads();
  if (wave == 0) {
    const int c = lane < E ? (base[lane] + r.align - 1) & -r.align : 0;
    const int at = wave_before(c);
    base[lane] = at;
    if (lane < E) r.offsets[lane] = (uint32_t)at;
    if (lane == E - 1) r.offsets[E] = (uint32_t)(at + c);
  }
  for (int c0 = 0; c0 < A; c0 += SORT_NT) {
    __syncthreads();  // (the first also orders the cleared slot_of before the rows below)
    if (A > SORT_NT) {  // one chunk: its ranks are still there
      e = c0 + tid < A ? idx[c0 + tid] : kNone;
      rank = chunk_ranks(e, E, wave_cnt);
      __syncthreads();
    }
    if (c0 + tid < A) {
      uint32_t row = kNone;
      if (e < (uint32_t)E) {
        int before = base[e];
        for (int w = 0; w < wave; w++) before += wave_cnt[w][e];
        row = (uint32_t)(before + rank);
        r.slot_of[row] = (uint32_t)(c0 + tid);
      }
      r.row_of[c0 + tid] = row;
    }
    __syncthreads();
    if (tid < E) {
      int s = 0;
      for (int w = 0; w < 16; w++) s += wave_cnt[w][tid];
      base[tid] += s;
    }
  }
}

// Many chunks: runs of `per` of them (1 up to ROUTE_RUNS chunks), a workgroup a
// run. hist[run][expert], then (a launch later) every workgroup adds up the runs
// before its own.
__global__ __launch_bounds__(SORT_NT) void route_count_kernel(const uint32_t *__restrict__ idx, int A, int E, int per,
                                                              int *__restrict__ hist) {
  __shared__ int wave_cnt[16][ROUTE_MAXE];
  const int tid = threadIdx.x, first = blockIdx.x * per * SORT_NT;
  int s = 0;
  for (int a = first; a < A && a < first + per * SORT_NT; a += SORT_NT) {
    if (a > first) __syncthreads();  // the counts before are added up
    chunk_ranks(a + tid < A ? idx[a + tid] : kNone, E, wave_cnt);
    __syncthreads();
    if (tid < ROUTE_MAXE)
      for (int w = 0; w < 16; w++) s += wave_cnt[w][tid];
  }
  if (tid < ROUTE_MAXE) hist[blockIdx.x * ROUTE_MAXE + tid] = s;
}

__global__ __launch_bounds__(SORT_NT) void route_place_kernel(const uint32_t *__restrict__ idx, RouteRows r, int per,
                                                              const int *__restrict__ hist) {
  __shared__ int wave_cnt[16][ROUTE_MAXE];
  __shared__ int part[2][16][ROUTE_MAXE];  // counts of the runs before this one; of all
  __shared__ int first[ROUTE_MAXE], count[ROUTE_MAXE], base[ROUTE_MAXE], end;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int A = r.T * r.top_k, E = r.E, G = gridDim.x, g = blockIdx.x;
  const int a0 = g * per * SORT_NT;
  uint32_t e = a0 + tid < A ? idx[a0 + tid] : kNone;
  int rank = chunk_ranks(e, E, wave_cnt);
  int before = 0, all = 0;
  for (int c = wave; c < G; c += 16) {
    const int h = hist[c * ROUTE_MAXE + lane];
    all += h;
    before += c < g ? h : 0;
  }
  part[0][wave][lane] = before;
  part[1][wave][lane] = all;
  __syncthreads();
  if (wave == 0) {
    before = all = 0;
    for (int w = 0; w < 16; w++) {
      before += part[0][w][lane];
      all += part[1][w][lane];
    }
    const int c = (all + r.align - 1) & -r.align;  // experts past E have none
    const int at = wave_before(c);
    first[lane] = at;
    count[lane] = all;
    base[lane] = at + before;
    if (lane == 63) end = at + c;
    if (g == 0) {
      if (lane < E) r.offsets[lane] = (uint32_t)at;
      if (lane == 63) r.offsets[E] = (uint32_t)(at + c);
    }
  }
  __syncthreads();
  for (int a = a0;;) {
    if (a + tid < A) {
      uint32_t row = kNone;
      if (e < (uint32_t)E) {
        int at = base[e];
        for (int w = 0; w < wave; w++) at += wave_cnt[w][e];
        row = (uint32_t)(at + rank);
        r.slot_of[row] = (uint32_t)(a + tid);
      }
      r.row_of[a + tid] = row;
    }
    a += SORT_NT;
    if (a >= A || a >= a0 + per * SORT_NT) break;
    __syncthreads();
    if (tid < ROUTE_MAXE)
      for (int w = 0; w < 16; w++) base[tid] += wave_cnt[w][tid];
    __syncthreads();
    e = a + tid < A ? idx[a + tid] : kNone;
    rank = chunk_ranks(e, E, wave_cnt);
    __syncthreads();
  }
  // rows of no route: between the segments (a wave an expert), and from the end on
  for (int x = g * 16 + wave; x < E; x += G * 16) {
    const int z = x + 1 < E ? first[x + 1] : end;
    for (int i = first[x] + count[x] + lane; i < z; i += 64) r.slot_of[i] = kNone;
  }
  for (int i = end + g * SORT_NT + tid; i < r.R; i += G * SORT_NT) r.slot_of[i] = kNone;
}

// One row per wave, W bytes per lane and load.
template <typename V>
__global__ __launch_bounds__(256) void route_dispatch_kernel(const char *__restrict__ x, size_t row_bytes,
                                                             RouteRows r, char *__restrict__ xs) {
  const int lane = threadIdx.x & 63;
  const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (size_t)r.R) return;
  const uint32_t slot = r.slot_of[row];
  const uint32_t A = (uint32_t)r.T * (uint32_t)r.top_k;
  if (slot >= A && row >= r.offsets[r.E]) return;
  const V *src = reinterpret_cast<const V *>(x + (size_t)(slot >= A ? 0 : slot / r.top_k) * row_bytes);
  V *dst = reinterpret_cast<V *>(xs + row * row_bytes);
  for (size_t i = lane; i < row_bytes / sizeof(V); i += 64) dst[i] = slot >= A ? V{} : src[i];
}

// Q consecutive values; the vector forms need 16-byte aligned rows (and Q
// dividing them).
__device__ __forceinline__ void ldq(const float *p, float (&v)[4]) {
  const f32x4 a = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = a[i];
}
__device__ __forceinline__ void ldq(const float *p, float (&v)[8]) {
  float a[4], b[4];
  ldq(p, a);
  ldq(p + 4, b);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}
__device__ __forceinline__ void ldq(const uint16_t *p, float (&v)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void ldq(const float *p, float (&v)[1]) { v[0] = *p; }
__device__ __forceinline__ void ldq(const uint16_t *p, float (&v)[1]) { v[0] = bf16_to_f32(*p); }
template <int Q>
__device__ __forceinline__ void stq(float *p, const float (&v)[Q]) {
  if constexpr (Q == 1) *p = v[0];
  else
#pragma unroll
    for (int i = 0; i < Q; i += 4) *reinterpret_cast<f32x4 *>(p + i) = (f32x4){v[i], v[i + 1], v[i + 2], v[i + 3]};
}
template <int Q>
__device__ __forceinline__ void stq(uint16_t *p, const float (&v)[Q]) {
  uint32_t h[Q];
#pragma unroll
  for (int i = 0; i < Q; i++) h[i] = bf16_rne_nb(v[i]);
  if constexpr (Q == 1) *p = (uint16_t)h[0];
  else
    *reinterpret_cast<u32x4 *>(p) = (u32x4){h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
}

#pragma clang fp contract(off)
// Q columns of one token a thread; 1 << tb threads a token (256 and several
// workgroups for long rows, several tokens a workgroup for short ones). The
// rows of four routes are loaded before the first is added.
template <typename ST, typename YT, int Q>
__global__ __launch_bounds__(256) void route_combine_kernel(const ST *__restrict__ ys, RouteRows r,
                                                            const float *__restrict__ w, YT *__restrict__ y,
                                                            uint32_t H, int tb) {
  constexpr int C = 4;
  const size_t t = (size_t)blockIdx.x * (256 >> tb) + (threadIdx.x >> tb);
  const uint32_t h = (blockIdx.y * 256 + (threadIdx.x & ((1 << tb) - 1))) * Q;
  if (t >= (size_t)r.T || h >= H) return;
  const uint32_t *row_of = r.row_of + t * r.top_k;
  float acc[Q];
#pragma unroll
  for (int q = 0; q < Q; q++) acc[q] = 0.0f;
  for (int j0 = 0; j0 < r.top_k; j0 += C) {
    uint32_t row[C];
    float g[C], v[C][Q];
#pragma unroll
    for (int c = 0; c < C; c++) {
      row[c] = j0 + c < r.top_k ? row_of[j0 + c] : kNone;
      g[c] = w && j0 + c < r.top_k ? w[t * r.top_k + j0 + c] : 1.0f;
    }
#pragma unroll
    for (int c = 0; c < C; c++)
      if (row[c] < (uint32_t)r.R) ldq(ys + (size_t)row[c] * H + h, v[c]);
#pragma unroll
    for (int c = 0; c < C; c++)
      if (row[c] < (uint32_t)r.R)
#pragma unroll
        for (int q = 0; q < Q; q++) acc[q] = acc[q] + g[c] * v[c][q];
  }
  stq<Q>(y + t * H + h, acc);
}

// A wave a route: dy's row is read once for each of its token's routes, from
// cache after the first (neighbouring waves). Then (align > 1) a wave a row,
// for those of no route.
template <typename DT, typename ST, int Q>
__global__ __launch_bounds__(256) void route_combine_backward_kernel(const DT *__restrict__ dy,
                                                                     const ST *__restrict__ ys, RouteRows r,
                                                                     const float *__restrict__ w,
                                                                     ST *__restrict__ dys, float *__restrict__ dw,
                                                                     uint32_t H) {
  const int lane = threadIdx.x & 63;
  const uint32_t A = (uint32_t)r.T * (uint32_t)r.top_k;
  const uint32_t slot = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (slot >= A) {
    const uint32_t row = slot - A;
    if (row >= (uint32_t)r.R || row >= r.offsets[r.E] || r.slot_of[row] != kNone) return;
    const float z[Q] = {};
    for (uint32_t h = lane * Q; h < H; h += 64 * Q) stq<Q>(dys + (size_t)row * H + h, z);
    return;
  }
  const uint32_t row = r.row_of[slot];
  // a lane's sum goes by 8 products at a time, fused: 8 + H / 512 roundings instead of H / 32
  constexpr uint32_t EVERY = Q < 8 ? 8 / Q : 1;
  float dot = 0.0f, part = 0.0f;
  uint32_t n = 0;
  if (row < (uint32_t)r.R) {
    const float g = w ? w[slot] : 1.0f;
    const DT *src = dy + (size_t)(slot / r.top_k) * H;
    const ST *other = ys + (size_t)row * H;
    ST *d = dys + (size_t)row * H;
#pragma unroll 4
    for (uint32_t h = lane * Q; h < H; h += 64 * Q) {
      float a[Q], p[Q];
      ldq(src + h, a);
#pragma unroll
      for (int q = 0; q < Q; q++) p[q] = g * a[q];
      if (ys) {
        float b[Q];
        ldq(other + h, b);
#pragma unroll
        for (int q = 0; q < Q; q++) part = __builtin_fmaf(a[q], b[q], part);
        if (++n % EVERY == 0) {
          dot = dot + part;
          part = 0.0f;
        }
      }
      stq<Q>(d + h, p);
    }
  }
  if (!dw) return;
  dot = dot + part;
  for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
  if (lane == 0) dw[slot] = dot;
}
#pragma clang fp contract(on)

}  // namespace

// Chunks of a run, and the runs there are.
static int sort_runs(const RouteRows &r, int &per) {
  const int chunks = (r.T * r.top_k + SORT_NT - 1) / SORT_NT;
  per = (chunks + ROUTE_RUNS - 1) / ROUTE_RUNS;
  return (chunks + per - 1) / per;
}

size_t route_sort_bytes(const RouteRows &r) {
  int per;
  return r.T * r.top_k <= ROUTE_ONE_WG ? 0 : sort_runs(r, per) * ROUTE_MAXE * sizeof(int);
}

hipError_t launch_route_sort(const uint32_t *idx, const RouteRows &r, int *hist, hipStream_t stream) {
  if (!hist) {
    hipLaunchKernelGGL(route_sort_kernel, dim3(1), dim3(SORT_NT), 0, stream, idx, r);
    return hipGetLastError();
  }
  int per;
  const dim3 grid(sort_runs(r, per));
  hipLaunchKernelGGL(route_count_kernel, grid, dim3(SORT_NT), 0, stream, idx, r.T * r.top_k, r.E, per, hist);
  hipLaunchKernelGGL(route_place_kernel, grid, dim3(SORT_NT), 0, stream, idx, r, per, hist);
  return hipGetLastError();
}

hipError_t launch_route_dispatch(const void *x, size_t row_bytes, const RouteRows &r, void *xs, hipStream_t stream) {
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xs) | row_bytes) & 15) == 0;
  const dim3 grid((unsigned)((r.R + 3) / 4));
  const char *src = static_cast<const char *>(x);
  char *dst = static_cast<char *>(xs);
  if (vec) hipLaunchKernelGGL(route_dispatch_kernel<u32x4>, grid, dim3(256), 0, stream, src, row_bytes, r, dst);
  else hipLaunchKernelGGL(route_dispatch_kernel<uint32_t>, grid, dim3(256), 0, stream, src, row_bytes, r, dst);
  return hipGetLastError();
}

// Whether rows of `bytes` from each of the pointers on are 16-byte aligned.
static bool rows16(const void *a, const void *b, const void *c, size_t bytes) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | bytes) &
          15) == 0;
}

template <typename ST, typename YT, int Q>
static hipError_t combine_go(const ST *ys, const RouteRows &r, const float *w, YT *y, uint32_t H, hipStream_t stream) {
  const uint32_t need = (H + Q - 1) / Q;
  int tb = 0;
  while (tb < 8 && (1u << tb) < need) tb++;
  const dim3 grid((unsigned)((r.T + (256 >> tb) - 1) / (256 >> tb)), (need + 255) / 256);
  hipLaunchKernelGGL((route_combine_kernel<ST, YT, Q>), grid, dim3(256), 0, stream, ys, r, w, y, H, tb);
  return hipGetLastError();
}

template <typename ST, typename YT>
static hipError_t combine_q(const ST *ys, const RouteRows &r, const float *w, YT *y, uint32_t H, hipStream_t stream) {
  // 16 bytes of the narrower type a thread
  constexpr int Q = sizeof(ST) == 4 && sizeof(YT) == 4 ? 4 : 8;
  if (rows16(ys, y, nullptr, (size_t)H * 2) && H % Q == 0) return combine_go<ST, YT, Q>(ys, r, w, y, H, stream);
  return combine_go<ST, YT, 1>(ys, r, w, y, H, stream);
}

template <typename ST>
static hipError_t combine_t(const ST *ys, const RouteRows &r, const float *w, void *y, int yt_bf16, uint32_t H,
                            hipStream_t stream) {
  return yt_bf16 ? combine_q(ys, r, w, static_cast<uint16_t *>(y), H, stream)
                 : combine_q(ys, r, w, static_cast<float *>(y), H, stream);
}

hipError_t launch_route_combine(const void *ys, int st_bf16, const RouteRows &r, const float *w, void *y, int yt_bf16,
                                uint32_t H, hipStream_t stream) {
  return st_bf16 ? combine_t(static_cast<const uint16_t *>(ys), r, w, y, yt_bf16, H, stream)
                 : combine_t(static_cast<const float *>(ys), r, w, y, yt_bf16, H, stream);
}

template <typename DT, typename ST>
static hipError_t combine_backward_t(const void *dy, const void *ys, const RouteRows &r, const float *w, void *dys,
                                     float *dw, uint32_t H, hipStream_t stream) {
  constexpr int Q = sizeof(DT) == 4 && sizeof(ST) == 4 ? 4 : 8;
  const size_t waves = (size_t)r.T * r.top_k + (r.align > 1 ? r.R : 0);
  const dim3 grid((unsigned)((waves + 3) / 4));
  if (rows16(dy, ys, dys, (size_t)H * 2) && H % Q == 0)
    hipLaunchKernelGGL((route_combine_backward_kernel<DT, ST, Q>), grid, dim3(256), 0, stream,
                       static_cast<const DT *>(dy), static_cast<const ST *>(ys), r, w, static_cast<ST *>(dys), dw, H);
  else
    hipLaunchKernelGGL((route_combine_backward_kernel<DT, ST, 1>), grid, dim3(256), 0, stream,
                       static_cast<const DT *>(dy), static_cast<const ST *>(ys), r, w, static_cast<ST *>(dys), dw, H);
  return hipGetLastError();
}

hipError_t launch_route_combine_backward(const void *dy, int dt_bf16, const void *ys, int st_bf16, const RouteRows &r,
                                         const float *w, void *dys, float *dw, uint32_t H, hipStream_t stream) {
  if (dt_bf16)
    return st_bf16 ? combine_backward_t<uint16_t, uint16_t>(dy, ys, r, w, dys, dw, H, stream)
                   : combine_backward_t<uint16_t, float>(dy, ys, r, w, dys, dw, H, stream);
  return st_bf16 ? combine_backward_t<float, uint16_t>(dy, ys, r, w, dys, dw, H, stream)
                 : combine_backward_t<float, float>(dy, ys, r, w, dys, dw, H, stream);
}

}  // namespace frx
