// frx_route.hip — tokens into rows sorted by expert, and back, with gradients.
//
// sort: a stable counting sort of the slots t * top_k + j by expert; segments
// start at multiples of `align`.
// dispatch: xs[row] = x[token of row].   combine: y[t] = sum_j w[t][j] ys[row_of[t][j]].
// combine_backward: dys[row] = w[slot] dy[token], dw[t][j] = <dy[t], ys[row_of[t][j]]>.
// All but the sort are bound by memory.
#include "frx_device.hpp"
#include "frx_internal.hpp"

namespace frx {

namespace {

constexpr int ROUTE_MAXE = 64;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// One workgroup: counts, then ranks chunk by chunk in slot order.
__global__ __launch_bounds__(1024) void route_sort_kernel(const uint32_t *__restrict__ idx, RouteRows r) {
  __shared__ int wave_cnt[16][ROUTE_MAXE];
  __shared__ int base[ROUTE_MAXE];  // next row of each expert
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int A = r.T * r.top_k, E = r.E;
  for (int i = tid; i < 16 * ROUTE_MAXE; i += 1024) wave_cnt[i / ROUTE_MAXE][i % ROUTE_MAXE] = 0;
  for (int i = tid; i < r.R; i += 1024) r.slot_of[i] = kNone;
  __syncthreads();
  for (int a = tid; a < A; a += 1024) {
    const uint32_t e = idx[a];
    if (e < (uint32_t)E) atomicAdd(&wave_cnt[wave][e], 1);
  }
  __syncthreads();
  if (wave == 0) {
    int c = 0;
    if (lane < E)
      for (int w = 0; w < 16; w++) c += wave_cnt[w][lane];
    c = (c + r.align - 1) / r.align * r.align;
    int x = c;
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    base[lane] = x - c;
    if (lane < E) r.offsets[lane] = (uint32_t)(x - c);
    if (lane == E - 1) r.offsets[E] = (uint32_t)x;
  }
  __syncthreads();  // also orders the cleared slot_of before the rows below
  for (int c0 = 0; c0 < A; c0 += 1024) {
    const int a = c0 + tid;
    const uint32_t e = a < A ? idx[a] : kNone;
    int rank = 0;
    for (int ee = 0; ee < E; ee++) {
      const unsigned long long m = __ballot(e == (uint32_t)ee);
      if (lane == 0) wave_cnt[wave][ee] = __popcll(m);
      if (e == (uint32_t)ee) rank = __popcll(m & ((1ull << lane) - 1ull));
    }
    __syncthreads();
    if (a < A) {
      uint32_t row = kNone;
      if (e < (uint32_t)E) {
        int before = base[e];
        for (int w = 0; w < wave; w++) before += wave_cnt[w][e];
        row = (uint32_t)(before + rank);
        r.slot_of[row] = (uint32_t)a;
      }
      r.row_of[a] = row;
    }
    __syncthreads();
    if (tid < E) {
      int s = 0;
      for (int w = 0; w < 16; w++) s += wave_cnt[w][tid];
      base[tid] += s;
    }
    __syncthreads();
  }
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

__device__ __forceinline__ float ldf(const float *p, size_t i) { return p[i]; }
__device__ __forceinline__ float ldf(const uint16_t *p, size_t i) { return bf16_to_f32(p[i]); }
__device__ __forceinline__ void stf(float *p, size_t i, float v) { p[i] = v; }
__device__ __forceinline__ void stf(uint16_t *p, size_t i, float v) { p[i] = (uint16_t)bf16_rne_nb(v); }

#pragma clang fp contract(off)
template <typename ST, typename YT>
__global__ __launch_bounds__(256) void route_combine_kernel(const ST *__restrict__ ys, RouteRows r,
                                                            const float *__restrict__ w, YT *__restrict__ y,
                                                            uint32_t H) {
  const size_t t = blockIdx.x;
  for (uint32_t h = threadIdx.x; h < H; h += 256) {
    float acc = 0.0f;
    for (int j = 0; j < r.top_k; j++) {
      const uint32_t row = r.row_of[t * r.top_k + j];
      if (row >= (uint32_t)r.R) continue;
      const float p = (w ? w[t * r.top_k + j] : 1.0f) * ldf(ys, (size_t)row * H + h);
      acc = acc + p;
    }
    stf(y, t * H + h, acc);
  }
}
#pragma clang fp contract(on)

// A workgroup per token; then one per 4 rows for the rows of no route.
template <typename DT, typename ST>
__global__ __launch_bounds__(256) void route_combine_backward_kernel(const DT *__restrict__ dy,
                                                                     const ST *__restrict__ ys, RouteRows r,
                                                                     const float *__restrict__ w,
                                                                     ST *__restrict__ dys, float *__restrict__ dw,
                                                                     uint32_t H) {
  __shared__ float part[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x >= (unsigned)r.T) {
    const size_t row = (size_t)(blockIdx.x - r.T) * 4 + wave;
    if (row >= r.R || row >= r.offsets[r.E] || r.slot_of[row] != kNone) return;
    for (uint32_t h = lane; h < H; h += 64) stf(dys, row * H + h, 0.0f);
    return;
  }
  const size_t t = blockIdx.x;
  for (int j = 0; j < r.top_k; j++) {
    const uint32_t row = r.row_of[t * r.top_k + j];
    float dot = 0.0f;
    if (row < (uint32_t)r.R) {
      const float g = w ? w[t * r.top_k + j] : 1.0f;
      for (uint32_t h = threadIdx.x; h < H; h += 256) {
        const float d = ldf(dy, t * H + h);
        stf(dys, (size_t)row * H + h, g * d);
        if (ys) dot += d * ldf(ys, (size_t)row * H + h);
      }
    }
    if (!dw) continue;
    for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
    if (lane == 0) part[wave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) dw[t * r.top_k + j] = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_route_sort(const uint32_t *idx, const RouteRows &r, hipStream_t stream) {
  hipLaunchKernelGGL(route_sort_kernel, dim3(1), dim3(1024), 0, stream, idx, r);
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

template <typename ST>
static hipError_t combine_t(const ST *ys, const RouteRows &r, const float *w, void *y, int yt_bf16, uint32_t H,
                            hipStream_t stream) {
  if (yt_bf16)
    hipLaunchKernelGGL((route_combine_kernel<ST, uint16_t>), dim3(r.T), dim3(256), 0, stream, ys, r, w,
                       static_cast<uint16_t *>(y), H);
  else
    hipLaunchKernelGGL((route_combine_kernel<ST, float>), dim3(r.T), dim3(256), 0, stream, ys, r, w,
                       static_cast<float *>(y), H);
  return hipGetLastError();
}

hipError_t launch_route_combine(const void *ys, int st_bf16, const RouteRows &r, const float *w, void *y, int yt_bf16,
                                uint32_t H, hipStream_t stream) {
  return st_bf16 ? combine_t(static_cast<const uint16_t *>(ys), r, w, y, yt_bf16, H, stream)
                 : combine_t(static_cast<const float *>(ys), r, w, y, yt_bf16, H, stream);
}

template <typename DT, typename ST>
static hipError_t combine_backward_t(const void *dy, const void *ys, const RouteRows &r, const float *w, void *dys,
                                     float *dw, uint32_t H, hipStream_t stream) {
  hipLaunchKernelGGL((route_combine_backward_kernel<DT, ST>), dim3((unsigned)(r.T + (r.R + 3) / 4)), dim3(256), 0,
                     stream, static_cast<const DT *>(dy), static_cast<const ST *>(ys), r, w,
                     static_cast<ST *>(dys), dw, H);
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
