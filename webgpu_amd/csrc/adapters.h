// adapters.h — low-rank adapters of many rows beside a shared projection (part of ops.hip).
//
// Row t with the adapter w = which[t]: y[t] += scales[w] B_w h[t], h[t] = A_w x[t]. Two launches: h, then the sum into y.
// Rows are taken 64 at a time, one per lane, and the adapters that occur among them one after another, so that an
// adapter's weights are read once for all of its rows there, whatever their order, and no list of rows has to be made first. Products are those of
// v_mfma_f32_16x16x4_f32: halves are widened exactly, products and sums are f32. The order of the sums depends on the sizes alone.
#pragma once

namespace wgd {

constexpr uint32_t AD_ROWS = 64, AD_RANKS = 64, AD_OUT = 512, AD_SPLITS = 16;

// The rows of the next adapter among the 64 (in order of their first rows), as bits; 0 where there are no more.
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
// Lane i: the lane of the i-th of `rows`.
__device__ __forceinline__ uint32_t adapter_order(uint64_t rows) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1;
  const uint32_t to = rows >> lane & 1 ? (uint32_t)__popcll(rows & below) : (uint32_t)(__popcll(rows) + __popcll(~rows & below));
  return (uint32_t)__builtin_amdgcn_ds_permute((int)(4 * to), (int)lane);
}
// N elements p[i] .., 0 from n on. VEC: they lie on 16 bytes (8 for four halves), and n is a multiple of N, or 0 with N of them to read.
template <class E, uint32_t N, bool VEC> __device__ __forceinline__ void adapter_get(const E *p, uint32_t i, uint32_t n, E (&v)[N]) {
  typedef E en __attribute__((ext_vector_type(N)));
  if constexpr (VEC) {
    const en e = *(const en *)(p + (i < n ? i : 0));
#pragma unroll
    for (uint32_t u = 0; u < N; u++) v[u] = i < n ? e[u] : (E)0.f;
  } else {
#pragma unroll
    for (uint32_t u = 0; u < N; u++) v[u] = i + u < n ? p[i + u] : (E)0.f;
  }
}
typedef float ad4 __attribute__((ext_vector_type(4)));

// Sums of a wavefront's steps from, from + by, .. below `to` for NK tiles of 16 ranks, the loads of U steps ahead of their products.
template <class E, uint32_t NK, uint32_t U, bool VEC>
__device__ __forceinline__ void adapter_steps(const E *(&w)[AD_RANKS / 16], const float *x, bool row, uint32_t from, uint32_t by, uint32_t to,
                                              ad4 (&acc)[AD_RANKS / 16]) {
  constexpr uint32_t W = 16 / sizeof(E);
  const uint32_t mine = W * ((threadIdx.x & 63) >> 4);
  for (uint32_t s = from; s < to; s += U * by) {
    float xv[U][W];
    E wv[U][NK][W];
#pragma unroll
    for (uint32_t e = 0; e < U; e++) {
      const uint32_t k = s + e * by + mine;
#pragma unroll
      for (uint32_t i = 0; i < NK; i++) adapter_get<E, W, VEC>(w[i], k, to, wv[e][i]);
      adapter_get<float, W, VEC>(x, k, row ? to : 0, xv[e]);
    }
#pragma unroll
    for (uint32_t e = 0; e < U; e++)
#pragma unroll
      for (uint32_t u = 0; u < W; u++)
#pragma unroll
        for (uint32_t i = 0; i < NK; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)wv[e][i][u], xv[e][u], acc[i], 0, 0, 0);
  }
}

// h of 16 rows of one adapter: a wavefront takes every fourth step of 4 W columns of its workgroup's, for up to four tiles of 16
// ranks; lane (g, c) = (lane / 16, lane % 16) has W columns at W g of rank c and of row c. The wavefronts' sums meet in LDS, those of
// several column ranges (blockIdx.z) in the next launch.
template <class E, bool VEC>
__global__ __launch_bounds__(256) void k_adapters_down(AdaptersArgs a, uint32_t tiles, uint32_t splits, uint32_t span) {
  constexpr uint32_t W = 16 / sizeof(E), STEP = 4 * W;
  __shared__ ad4 red[4][AD_RANKS / 16][64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t t0 = blockIdx.x / tiles * AD_ROWS, tile = blockIdx.x % tiles, z = blockIdx.z % splits, k0 = blockIdx.z / splits * AD_RANKS;
  const uint32_t from = z * span, to = min(a.cols, from + span);
  const int32_t mine = adapter_of(a, t0 + lane);
  uint64_t left = __ballot(mine >= 0);
  for (uint32_t j = 0;; j++) {
    const AdapterRows r = adapter_rows(mine, left);
    if (!r.rows) return;
    const uint32_t n = (uint32_t)__popcll(r.rows);
    if (j % gridDim.y != blockIdx.y || 16 * tile >= n) continue;
    const uint32_t order = adapter_order(r.rows), at = 16 * tile + c;
    const bool row = at < n;
    const uint32_t t = t0 + (uint32_t)__shfl((int)order, (int)at, 64);
    const float *x = a.x + (uint64_t)(row ? t : t0) * a.cols;
    const E *w[AD_RANKS / 16];
#pragma unroll
    for (uint32_t i = 0; i < AD_RANKS / 16; i++) w[i] = (const E *)a.a + ((uint64_t)r.w * a.rank + min(k0 + 16 * i + c, a.rank - 1)) * a.cols;
    ad4 acc[AD_RANKS / 16] = {};
    if (a.rank - k0 <= 16) adapter_steps<E, 1, 4, VEC>(w, x, row, from + wave * STEP, 4 * STEP, to, acc);
    else adapter_steps<E, AD_RANKS / 16, 2, VEC>(w, x, row, from + wave * STEP, 4 * STEP, to, acc);
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < AD_RANKS / 16; i++) red[wave][i][lane] = acc[i];
    __syncthreads();
    // wavefront i: ranks 4 g .. + 4 of tile i, row c
    const ad4 h = red[0][wave][lane] + red[1][wave][lane] + red[2][wave][lane] + red[3][wave][lane];
    if (!row) continue;
    const uint32_t k = k0 + 16 * wave + 4 * g;
    float *out = a.partial + ((uint64_t)z * a.batch + t) * a.rank + k;
    if (a.rank % 4 == 0) {
      if (k < a.rank) *(ad4 *)out = h;
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; e++)
        if (k + e < a.rank) out[e] = h[e];
    }
  }
}

// The sums of h's column ranges, in order, of the rows `order` of an adapter (n of them, filled up to `tiles` of 16) and the ranks k0 .. + 64, into LDS.
constexpr uint32_t AD_HS = AD_RANKS + 4;
__device__ __forceinline__ void adapter_h(const AdaptersArgs &a, float *h, uint32_t t0, uint32_t order, uint32_t n, uint32_t tiles, uint32_t k0,
                                          uint32_t splits) {
  const uint64_t next = (uint64_t)a.batch * a.rank;
  if (a.rank % 4 == 0) {
    const uint32_t k = threadIdx.x % 16 * 4;
#pragma unroll
    for (uint32_t b = 0; b < 4; b++) {
      if (b >= tiles) break;
      const uint32_t at = 16 * b + threadIdx.x / 16;
      const uint32_t t = t0 + (uint32_t)__shfl((int)order, (int)at, 64);
      ad4 s = {0, 0, 0, 0};
      if (at < n && k0 + k < a.rank) {
        const float *p = a.partial + (uint64_t)t * a.rank + k0 + k;
#pragma unroll 4
        for (uint32_t z = 0; z < splits; z++) s += *(const ad4 *)(p + z * next);
      }
      *(ad4 *)(h + at * AD_HS + k) = s;
    }
  } else {
    for (uint32_t i = threadIdx.x; i < 16 * tiles * AD_RANKS; i += 256) {
      const uint32_t at = i / AD_RANKS, k = k0 + i % AD_RANKS;
      const uint32_t t = t0 + (uint32_t)__shfl((int)order, (int)at, 64);
      float s = 0.f;
      if (at < n && k < a.rank)
        for (uint32_t z = 0; z < splits; z++) s += a.partial[z * next + (uint64_t)t * a.rank + k];
      h[at * AD_HS + i % AD_RANKS] = s;
    }
  }
}

// y of `last - first` elements and TILES tiles of 16 rows, M tiles of 16 elements a wavefront at a time. Lane (g, c) has
// W ranks at W g of element c and of row c; the result's 4 elements at 4 g of row c lie side by side in y.
template <class E, uint32_t M, uint32_t TILES, bool VEC, bool YVEC>
__device__ __forceinline__ void adapter_sum(const AdaptersArgs &a, float *h, uint32_t t0, uint32_t order, uint32_t n, int32_t kind, uint32_t first,
                                            uint32_t last, uint32_t splits) {
  constexpr uint32_t W = 16 / sizeof(E), STEP = 4 * W;
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float scale = a.scales[kind];
  const E *w0 = (const E *)a.b + (uint64_t)kind * a.rows * a.rank;
  float *y[TILES];
  bool row[TILES];
#pragma unroll
  for (uint32_t b = 0; b < TILES; b++) {
    row[b] = 16 * b + c < n;
    y[b] = a.y + (uint64_t)(t0 + (uint32_t)__shfl((int)order, (int)(16 * b + c), 64)) * a.stride;
  }
  for (uint32_t o0 = first; o0 < last; o0 += 64 * M) {
    const uint32_t o = o0 + 16 * M * wave;
    ad4 old[M][TILES] = {}, acc[M][TILES] = {};
    E wv[M][W];
#pragma unroll
    for (uint32_t m = 0; m < M; m++) {
      adapter_get<E, W, VEC>(w0 + (uint64_t)min(o + 16 * m + c, a.rows - 1) * a.rank, W * g, a.rank, wv[m]);
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) {
        const uint32_t e = o + 16 * m + 4 * g;
        if constexpr (YVEC) {
          if (row[b] && e < last) old[m][b] = *(const ad4 *)(y[b] + e);
        } else {
#pragma unroll
          for (uint32_t u = 0; u < 4; u++)
            if (row[b] && e + u < last) old[m][b][u] = y[b][e + u];
        }
      }
    }
    for (uint32_t k0 = 0; k0 < a.rank; k0 += AD_RANKS) {
      if (o0 == first || a.rank > AD_RANKS) {
        __syncthreads();
        adapter_h(a, h, t0, order, n, TILES, k0, splits);
        __syncthreads();
      }
      for (uint32_t s = 0; s < AD_RANKS && k0 + s < a.rank; s += STEP) {
        float hv[TILES][W];
#pragma unroll
        for (uint32_t b = 0; b < TILES; b++)
#pragma unroll
          for (uint32_t u = 0; u < W; u += 4) {
            const ad4 q = *(const ad4 *)(h + (16 * b + c) * AD_HS + s + W * g + u);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) hv[b][u + e] = q[e];
          }
#pragma unroll
        for (uint32_t m = 0; m < M; m++)
#pragma unroll
          for (uint32_t u = 0; u < W; u++)
#pragma unroll
            for (uint32_t b = 0; b < TILES; b++) acc[m][b] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)wv[m][u], hv[b][u], acc[m][b], 0, 0, 0);
        const uint32_t next = k0 + s + STEP;
        if (next < a.rank)
#pragma unroll
          for (uint32_t m = 0; m < M; m++) adapter_get<E, W, VEC>(w0 + (uint64_t)min(o + 16 * m + c, a.rows - 1) * a.rank, next + W * g, a.rank, wv[m]);
      }
    }
#pragma unroll
    for (uint32_t m = 0; m < M; m++)
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) {
        const uint32_t e = o + 16 * m + 4 * g;
        const ad4 v = old[m][b] + acc[m][b] * scale;
        if constexpr (YVEC) {
          if (row[b] && e < last) *(ad4 *)(y[b] + e) = v;
        } else {
#pragma unroll
          for (uint32_t u = 0; u < 4; u++)
            if (row[b] && e + u < last) y[b][e + u] = v[u];
        }
      }
  }
}

// The sum into y: `span` elements of the 64 rows' y by one workgroup; with 16 rows of an adapter or fewer, 512 of them at a time.
template <class E, bool VEC, bool YVEC>
__global__ __launch_bounds__(256) void k_adapters_up(AdaptersArgs a, uint32_t chunks, uint32_t splits, uint32_t span) {
  __shared__ __attribute__((aligned(16))) float h[AD_ROWS * AD_HS];
  const uint32_t t0 = blockIdx.x / chunks * AD_ROWS, first = blockIdx.x % chunks * span, last = min(a.rows, first + span);
  const int32_t mine = adapter_of(a, t0 + (threadIdx.x & 63));
  uint64_t left = __ballot(mine >= 0);
  for (uint32_t j = 0;; j++) {
    const AdapterRows r = adapter_rows(mine, left);
    if (!r.rows) return;
    if (j % gridDim.y != blockIdx.y) continue;
    const uint32_t n = (uint32_t)__popcll(r.rows), order = adapter_order(r.rows);
    if (n <= 16) adapter_sum<E, 8, 1, VEC, YVEC>(a, h, t0, order, n, r.w, first, last, splits);
    else adapter_sum<E, 2, 4, VEC, YVEC>(a, h, t0, order, n, r.w, first, last, splits);
  }
}

// The column ranges of h: as many as give about 512 workgroups, of two steps for each wavefront at least.
struct AdaptersPlan { uint32_t blocks, tiles, kinds, splits, span, chunks, out; };
static AdaptersPlan adapters_plan(const AdaptersArgs &a) {
  AdaptersPlan p;
  p.blocks = (a.batch + AD_ROWS - 1) / AD_ROWS;
  p.tiles = (std::min(a.batch, AD_ROWS) + 15) / 16;
  const uint32_t most = std::min({AD_ROWS, a.batch, a.adapters});  // adapters among 64 rows
  p.kinds = std::min(most, std::max(1u, 64 / p.blocks));
  const uint32_t step = a.half ? 256 : 128;
  p.splits = std::min({AD_SPLITS, std::max(1u, 512 / (p.blocks * p.tiles)), (a.cols + step - 1) / step});
  p.span = ((a.cols + p.splits - 1) / p.splits + step - 1) / step * step;
  p.splits = (a.cols + p.span - 1) / p.span;
  const uint32_t outs = (a.rows + AD_OUT - 1) / AD_OUT;
  p.chunks = std::min(outs, std::max(1u, 1024 / p.blocks));
  p.out = (outs + p.chunks - 1) / p.chunks * AD_OUT;
  p.chunks = (a.rows + p.out - 1) / p.out;
  return p;
}
uint64_t adapters_scratch_floats(const AdaptersArgs &a) { return (uint64_t)adapters_plan(a).splits * a.batch * a.rank; }

template <class E, bool VEC> static hipError_t launch_adapters(hipStream_t s, const AdaptersArgs &a) {
  const AdaptersPlan p = adapters_plan(a);
  const uint32_t ranks = (a.rank + AD_RANKS - 1) / AD_RANKS;
  hipLaunchKernelGGL((k_adapters_down<E, VEC>), dim3(p.blocks * p.tiles, p.kinds, p.splits * ranks), dim3(256), 0, s, a, p.tiles, p.splits, p.span);
  WGD_HIP(hipGetLastError());
  return hipSuccess;
}
template <class E, bool VEC, bool YVEC> static hipError_t launch_adapters_up(hipStream_t s, const AdaptersArgs &a) {
  const AdaptersPlan p = adapters_plan(a);
  hipLaunchKernelGGL((k_adapters_up<E, VEC, YVEC>), dim3(p.blocks * p.chunks, p.kinds), dim3(256), 0, s, a, p.chunks, p.splits, p.out);
  return hipGetLastError();
}
template <class E> static hipError_t launch_adapters_of(hipStream_t s, const AdaptersArgs &a) {
  constexpr uint32_t W = 16 / sizeof(E);
  if (a.cols % W == 0) WGD_HIP((launch_adapters<E, true>(s, a)));
  else WGD_HIP((launch_adapters<E, false>(s, a)));
  const bool yvec = (uintptr_t)a.y % 16 == 0 && a.rows % 4 == 0 && a.stride % 4 == 0, vec = a.rank % W == 0;
  if (vec) return yvec ? launch_adapters_up<E, true, true>(s, a) : launch_adapters_up<E, true, false>(s, a);
  return yvec ? launch_adapters_up<E, false, true>(s, a) : launch_adapters_up<E, false, false>(s, a);
}

hipError_t adapters(hipStream_t s, const AdaptersArgs &a) {
  if (!a.batch || !a.rank || !a.rows || !a.cols || !a.adapters) return hipSuccess;
  return a.half ? launch_adapters_of<_Float16>(s, a) : launch_adapters_of<float>(s, a);
}

}  // namespace wgd
