// adapters.h — low-rank adapters of many rows beside a shared projection (part of ops.hip).
//
// Row t with the adapter w = which[t]: y[t] += scales[w] B_w h[t], h[t] = A_w x[t]. Two launches: h, then the sum into y.
// Rows are taken 64 at a time, one per lane, and the adapters that occur among them one after another, so that an
// adapter's weights are read once for all of its rows there, whatever their order.
#pragma once

namespace wgd {

constexpr uint32_t AD_ROWS = 64;

// The rows of the j-th adapter among the 64 (in order of first rows), as bits; 0 where there are fewer.
struct AdapterRows { uint64_t rows; int32_t w; };
__device__ __forceinline__ AdapterRows adapter_rows(int32_t mine, uint64_t &left) {
  if (!left) return {0, -1};
  const int32_t w = __builtin_amdgcn_readlane(mine, (int)__ffsll((unsigned long long)left) - 1);
  const uint64_t rows = __ballot(mine == w) & left;
  left &= ~rows;
  return {rows, w};
}
__device__ __forceinline__ int32_t adapter_of(const AdaptersArgs &a, uint32_t t) {
  const int32_t w = t < a.batch ? a.which[t] : -1;
  return w >= 0 && (uint32_t)w < a.adapters ? w : -1;
}
template <class E> __device__ __forceinline__ float adapter_get(const void *p, uint64_t i) { return (float)((const E *)p)[i]; }

// A wavefront per (row, rank).
template <class E>
__global__ __launch_bounds__(256) void k_adapters_down(AdaptersArgs a) {
  const uint32_t lane = threadIdx.x & 63, t = blockIdx.x, k = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int32_t w = adapter_of(a, t);
  if (w < 0 || k >= a.rank) return;
  const uint64_t at = ((uint64_t)w * a.rank + k) * a.cols;
  const float *x = a.x + (uint64_t)t * a.cols;
  float s = 0.f;
  for (uint32_t c = lane; c < a.cols; c += 64) s += adapter_get<E>(a.a, at + c) * x[c];
  s = wave_sum(s);
  if (lane == 0) a.partial[(uint64_t)t * a.rank + k] = s;
}

// A thread per element of y.
template <class E>
__global__ __launch_bounds__(256) void k_adapters_up(AdaptersArgs a) {
  const uint32_t t = blockIdx.x, r = blockIdx.y * 256 + threadIdx.x;
  const int32_t w = adapter_of(a, t);
  if (w < 0 || r >= a.rows) return;
  const float *h = a.partial + (uint64_t)t * a.rank;
  const uint64_t at = ((uint64_t)w * a.rows + r) * a.rank;
  float s = 0.f;
  for (uint32_t k = 0; k < a.rank; k++) s += adapter_get<E>(a.b, at + k) * h[k];
  a.y[(uint64_t)t * a.stride + r] += a.scales[w] * s;
}

uint64_t adapters_scratch_floats(const AdaptersArgs &a) { return (uint64_t)a.batch * a.rank; }

hipError_t adapters(hipStream_t s, const AdaptersArgs &a) {
  if (!a.batch || !a.rank || !a.rows || !a.cols || !a.adapters) return hipSuccess;
  const dim3 down(a.batch, (a.rank + 3) / 4), up(a.batch, (a.rows + 255) / 256);
  if (a.half) hipLaunchKernelGGL(k_adapters_down<_Float16>, down, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_adapters_down<float>, down, dim3(256), 0, s, a);
  WGD_HIP(hipGetLastError());
  if (a.half) hipLaunchKernelGGL(k_adapters_up<_Float16>, up, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_adapters_up<float>, up, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace wgd
