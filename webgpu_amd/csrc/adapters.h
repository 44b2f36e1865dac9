// adapters.h — low-rank adapters of many rows beside a shared projection (part of ops.hip).
//
// Row t with the adapter w = which[t]: y[t] += scales[w] B_w h[t], h[t] = A_w x[t]. Two launches: h, then the sum into y.
// Rows are taken 64 at a time, one per lane, and the adapters that occur among them one after another, so that an
// adapter's weights are read once for all of its rows there, whatever their order, and no list of rows has to be made first.
//   f32 weights (v_mfma_f32_16x16x4_f32): f32 products and sums.
//   f16 weights (v_mfma_f32_16x16x32_f16): the weights are operands as they are, x and h are split into f16 hi + lo over a power of two per
//     row that puts its largest magnitude into [2^14, 2^15): each entry is off by 2^-22 of itself and 2^-39 of that largest one. Two products of f16
//     in place of one of f32, whose rate is an eighth: down and up at 1536 rows, rank 64, 4096 x 4096 took 17.4 and 21.8 us with f32 products.
// The order of the sums depends on the sizes alone.
// What bounds it: few rows, the latency of two launches, each of loads that depend on which[] (4 rows of rank 8, 1024 x 2048: 3.7 and 5.0 us;
// 64 rows of 24 adapters of rank 16, 4096 x 14336, 12 MB of weights: 5.9 and 8.6). Many rows, the bytes of x and y: 1536 rows of rank 64, 4096 x
// 4096: down 14.2 (25 MB), up 17.7 (50 MB), where two thirds of a wavefront's life wait for loads.
#pragma once

namespace wgd {

constexpr uint32_t AD_ROWS = 64, AD_RANKS = 64, AD_OUT = 128, AD_SPLITS = 16;

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
// N elements p[i] .., 0 from n on, side by side in registers. VEC: they lie on 16 bytes, and n is a multiple of N. WHOLE: all are
// there, so nothing waits for the load but its use.
template <class E, uint32_t N> using ad_vec = E __attribute__((ext_vector_type(N)));
template <class E, uint32_t N, bool VEC, bool WHOLE> __device__ __forceinline__ ad_vec<E, N> adapter_get(const E *p, uint32_t i, uint32_t n) {
  if constexpr (VEC) {
    typedef uint32_t words __attribute__((ext_vector_type(N * sizeof(E) / 4)));
    if constexpr (WHOLE) return __builtin_bit_cast(ad_vec<E, N>, *(const words *)(p + i));
    const words v = *(const words *)(p + (i < n ? i : 0)), none = {};
    return __builtin_bit_cast(ad_vec<E, N>, i < n ? v : none);
  } else {
    ad_vec<E, N> v;
#pragma unroll
    for (uint32_t u = 0; u < N; u++) v[u] = WHOLE || i + u < n ? p[i + u] : (E)0.f;
    return v;
  }
}
typedef float ad4 __attribute__((ext_vector_type(4)));
typedef uint32_t adw __attribute__((ext_vector_type(4)));
typedef _Float16 ad8 __attribute__((ext_vector_type(8)));

// A power of two by its exponent field, and the largest exponent field of magnitudes given as bits; both it and its inverse are normal.
__device__ __forceinline__ uint32_t adapter_exponent(uint32_t bits) { return min(max(bits >> 23, 16u), 254u) - 14u; }
__device__ __forceinline__ float adapter_power(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ float adapter_inverse(uint32_t e) { return __uint_as_float((254u - e) << 23); }

// Sums of a wavefront's steps from, from + by, .. below `to` for NK tiles of 16 ranks, the loads of AD_AHEAD steps under way ahead of
// their products.
constexpr uint32_t AD_AHEAD = 4;
template <class E, uint32_t NK, bool VEC>
__device__ __forceinline__ void adapter_steps(const E *(&w)[AD_RANKS / 16], const float *x, uint32_t from, uint32_t by, uint32_t to,
                                              ad4 (&acc)[AD_RANKS / 16]) {
  constexpr uint32_t W = 16 / sizeof(E), STEP = 4 * W;
  const uint32_t mine = W * ((threadIdx.x & 63) >> 4);
  typedef ad_vec<E, W> wvec;
  typedef ad_vec<float, W> xvec;
  uint32_t exponent = 2;  // of the row's power of two
  xvec xv[AD_AHEAD];
  wvec wv[AD_AHEAD][NK];
  auto load = [&](auto whole, uint32_t k, xvec &xb, wvec (&wb)[NK]) {
#pragma unroll
    for (uint32_t i = 0; i < NK; i++) wb[i] = adapter_get<E, W, VEC, decltype(whole)::value>(w[i], k + mine, to);
    xb = adapter_get<float, W, VEC, decltype(whole)::value>(x, k + mine, to);
  };
  const std::true_type all;
  const std::false_type some;
  auto add = [&](const xvec &xb, const wvec (&wb)[NK]) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (uint32_t u = 0; u < W; u++)
#pragma unroll
        for (uint32_t i = 0; i < NK; i++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(wb[i][u], xb[u], acc[i], 0, 0, 0);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (uint32_t u = 0; u < W; u++) m = max(m, __float_as_uint(xb[u]) & 0x7FFFFFFFu);
      if (__any(m >> 23 > exponent + 14u && exponent < 240u)) {  // larger than what the row had so far: its sums move along
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        const uint32_t to = max(exponent, adapter_exponent(m));
        const float f = adapter_power(exponent) * adapter_inverse(to);
        exponent = to;
#pragma unroll
        for (uint32_t i = 0; i < NK; i++) acc[i] *= f;
      }
      const float inv = adapter_inverse(exponent);
      adw hi, lo;
#pragma unroll
      for (uint32_t u = 0; u < 4; u++) {
        uint32_t h, l;
        split2(xb[2 * u] * inv, xb[2 * u + 1] * inv, h, l);
        hi[u] = h;
        lo[u] = l;
      }
#pragma unroll
      for (uint32_t i = 0; i < NK; i++) {
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb[i], __builtin_bit_cast(ad8, hi), acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb[i], __builtin_bit_cast(ad8, lo), acc[i], 0, 0, 0);
      }
    }
  };
  const uint32_t whole = from + STEP <= to ? (to - from - STEP) / by + 1 : 0;  // steps of which all columns are there
  if (whole) {
    // no load depends on a branch, so that each is waited for by itself: past the end they repeat the last step
    auto step = [&](uint32_t e) { return from + min(e, whole - 1) * by; };
#pragma unroll
    for (uint32_t e = 0; e < AD_AHEAD; e++) load(all, step(e), xv[e], wv[e]);
    uint32_t s = 0;
    for (; s + AD_AHEAD < whole; s += AD_AHEAD)
#pragma unroll
      for (uint32_t e = 0; e < AD_AHEAD; e++) {
        add(xv[e], wv[e]);
        load(all, step(s + e + AD_AHEAD), xv[e], wv[e]);
      }
#pragma unroll
    for (uint32_t e = 0; e < AD_AHEAD; e++)
      if (s + e < whole) add(xv[e], wv[e]);
  }
  if (from + whole * by < to) {  // the last columns
    load(some, from + whole * by, xv[0], wv[0]);
    add(xv[0], wv[0]);
  }
  if constexpr (sizeof(E) == 2) {
    const float f = adapter_power(exponent);
#pragma unroll
    for (uint32_t i = 0; i < NK; i++) acc[i] *= f;
  }
}

// h of 16 rows of one adapter: a wavefront takes every fourth step of 4 W columns of its workgroup's, for up to four tiles of 16
// ranks; lane (g, c) = (lane / 16, lane % 16) has W columns at W g of rank c and of row c. The wavefronts' sums meet in LDS, those of
// several column ranges (blockIdx.z) in the next launch.
template <class E, bool VEC>
__global__ __launch_bounds__(256) void k_adapters_down(AdaptersArgs a, uint32_t splits, uint32_t span) {
  constexpr uint32_t W = 16 / sizeof(E), STEP = 4 * W;
  __shared__ ad4 red[4][AD_RANKS / 16][64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t t0 = blockIdx.x * AD_ROWS, z = blockIdx.z % splits, k0 = blockIdx.z / splits * AD_RANKS;
  const uint32_t from = z * span, to = min(a.cols, from + span);
  const int32_t mine = adapter_of(a, t0 + lane);
  uint64_t left = __ballot(mine >= 0);
  AdapterRows r = {0, -1};
  uint32_t n = 0;
  for (uint32_t i = 0, tile = 0, next = blockIdx.y;; i++, tile++) {  // the tiles of 16 rows of all adapters, one after another
    if (16 * tile >= n) {
      r = adapter_rows(mine, left);
      if (!r.rows) return;
      n = (uint32_t)__popcll(r.rows);
      tile = 0;
    }
    if (i != next) continue;
    next += gridDim.y;
    const uint32_t order = adapter_order(r.rows), at = 16 * tile + c;
    const bool row = at < n;
    const uint32_t t = t0 + (uint32_t)__shfl((int)order, (int)at, 64);
    const float *x = a.x + (uint64_t)(row ? t : t0) * a.cols;  // (what a column without a row holds is not written)
    const E *w[AD_RANKS / 16];
#pragma unroll
    for (uint32_t i = 0; i < AD_RANKS / 16; i++) w[i] = (const E *)a.a + ((uint64_t)r.w * a.rank + min(k0 + 16 * i + c, a.rank - 1)) * a.cols;
    ad4 acc[AD_RANKS / 16] = {};
    if (a.rank - k0 <= 16) adapter_steps<E, 1, VEC>(w, x, from + wave * STEP, 4 * STEP, to, acc);
    else adapter_steps<E, AD_RANKS / 16, VEC>(w, x, from + wave * STEP, 4 * STEP, to, acc);
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

// The sums of h's column ranges, in order, of the rows `order` of an adapter (n of them, filled up to TILES tiles of 16 with zeros) and the
// ranks k0 .. + 64, into LDS: f32, or split into hi and lo with the power of two taken out of the row. All loads are of places that
// are there, so that none waits for a branch.
constexpr uint32_t AD_HS = AD_RANKS + 4, AD_HH = AD_RANKS + 8;
template <class E> struct AdapterH { __attribute__((aligned(16))) float h[AD_ROWS * AD_HS]; };
template <> struct AdapterH<_Float16> { __attribute__((aligned(16))) _Float16 hi[AD_ROWS * AD_HH], lo[AD_ROWS * AD_HH]; float power[AD_ROWS]; };
template <class E, uint32_t TILES>
__device__ __forceinline__ void adapter_h(const AdaptersArgs &a, AdapterH<E> &H, uint32_t t0, uint32_t order, uint32_t n, uint32_t k0, uint32_t splits) {
  const uint64_t next = (uint64_t)a.batch * a.rank;
  const uint32_t k = threadIdx.x % 16 * 4, at = threadIdx.x / 16;
  const float *p[TILES];
  ad4 s[TILES] = {};
#pragma unroll
  for (uint32_t b = 0; b < TILES; b++)
    p[b] = a.partial + (uint64_t)(t0 + (uint32_t)__shfl((int)order, (int)min(16 * b + at, n - 1), 64)) * a.rank;
  if (a.rank % 4 == 0) {
    const uint32_t from = min(k0 + k, a.rank - 4);
#pragma unroll 4
    for (uint32_t z = 0; z < splits; z++)
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) s[b] += *(const ad4 *)(p[b] + z * next + from);
  } else {
    for (uint32_t z = 0; z < splits; z++)
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) s[b][e] += p[b][z * next + min(k0 + k + e, a.rank - 1)];
  }
#pragma unroll
  for (uint32_t b = 0; b < TILES; b++) {
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) s[b][e] = 16 * b + at < n && k0 + k + e < a.rank ? s[b][e] : 0.f;
    if constexpr (sizeof(E) == 4) {
      *(ad4 *)(H.h + (16 * b + at) * AD_HS + k) = s[b];
    } else {
      uint32_t m = 0;
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) m = max(m, __float_as_uint(s[b][e]) & 0x7FFFFFFFu);
      m = max(m, row_other<0xB1>(m));   // over the 16 lanes of the row
      m = max(m, row_other<0x4E>(m));
      m = max(m, row_other<0x141>(m));
      m = max(m, row_other<0x140>(m));
      const uint32_t ex = adapter_exponent(m);
      const float inv = adapter_inverse(ex);
      uint2 hi, lo;
      split2(s[b][0] * inv, s[b][1] * inv, hi.x, lo.x);
      split2(s[b][2] * inv, s[b][3] * inv, hi.y, lo.y);
      *(uint2 *)(H.hi + (16 * b + at) * AD_HH + k) = hi;
      *(uint2 *)(H.lo + (16 * b + at) * AD_HH + k) = lo;
      if (k == 0) H.power[16 * b + at] = adapter_power(ex);
    }
  }
}

// y of `last - first` elements and TILES tiles of 16 rows, M tiles of 16 elements a wavefront at a time. Lane (g, c) has
// W ranks at W g of element c and of row c; the result's 4 elements at 4 g of row c lie side by side in y. y and the first ranks of B are
// asked for a step ahead; places that are not there read one that is, and are masked where they are used. MANY: more than AD_RANKS ranks, whose
// sums meet before y is added to them, once: f32 ones in the accumulators, others (over a power of two for each AD_RANKS of a row) in `sum`, with the next ranks' B asked for
// ahead of their h. (With that for all ranks, 4 rows of rank 8 took 9.3 us in place of 7.8. 4 and 64 rows of rank 128, 1024 x 2048: 15.5 and 21.3 f32, 12.6 and 17.5
// f16; with f32's four steps unrolled 17.4 and 20.9, f16 without B ahead 13.3 and 17.6.)
template <class E, uint32_t M, uint32_t TILES, bool VEC, bool YVEC, bool MANY>
__device__ __forceinline__ void adapter_sum(const AdaptersArgs &a, AdapterH<E> &H, uint32_t t0, uint32_t order, uint32_t n, int32_t kind, uint32_t first,
                                            uint32_t last, uint32_t splits) {
  constexpr bool AHEAD = MANY && sizeof(E) == 2, CARRY = MANY && sizeof(E) == 4;
  constexpr uint32_t W = 16 / sizeof(E), STEP = 4 * W, UNROLL = CARRY ? 1 : AD_RANKS / STEP;
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float scale = a.scales[kind];
  typedef ad_vec<E, W> wvec;
  const E *w0 = (const E *)a.b + (uint64_t)kind * a.rows * a.rank;
  float *y[TILES];
#pragma unroll
  for (uint32_t b = 0; b < TILES; b++) y[b] = a.y + (uint64_t)(t0 + (uint32_t)__shfl((int)order, (int)min(16 * b + c, n - 1), 64)) * a.stride;
  auto get = [&](uint32_t o, uint32_t k) {
    const E *p = w0 + (uint64_t)min(o + c, a.rows - 1) * a.rank;
    if constexpr (VEC) return adapter_get<E, W, true, true>(p, min(k + W * g, a.rank - W), 0);
    else return adapter_get<E, W, false, false>(p, k + W * g, a.rank);
  };
  auto load = [&](uint32_t o, ad4 (&old)[M][TILES], wvec (&wv)[M]) {
#pragma unroll
    for (uint32_t m = 0; m < M; m++) {
      wv[m] = get(o + 16 * m, 0);
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) {
        const uint32_t e = o + 16 * m + 4 * g;
        if constexpr (YVEC) {
          old[m][b] = *(const ad4 *)(y[b] + min(e, last - 4));
        } else {
#pragma unroll
          for (uint32_t u = 0; u < 4; u++) old[m][b][u] = y[b][min(e + u, last - 1)];
        }
      }
    }
  };
  ad4 old[M][TILES], ahead[M][TILES];
  wvec wv[M], wahead[M];
  load(first + 16 * M * wave, ahead, wahead);
  for (uint32_t o0 = first; o0 < last; o0 += 64 * M) {
    const uint32_t o = o0 + 16 * M * wave;
    ad4 acc[M][TILES] = {}, sum[M][TILES] = {};
#pragma unroll
    for (uint32_t m = 0; m < M; m++) {
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) old[m][b] = ahead[m][b];
      wv[m] = wahead[m];
    }
    load(min(o + 64 * M, last - 1), ahead, wahead);
    for (uint32_t k0 = 0; k0 < a.rank; k0 += AD_RANKS) {
      if constexpr (AHEAD)
        if (k0)
#pragma unroll
          for (uint32_t m = 0; m < M; m++) wv[m] = get(o + 16 * m, k0);
      if (o0 == first || MANY) {
        __syncthreads();
        adapter_h<E, TILES>(a, H, t0, order, n, k0, splits);
        __syncthreads();
      }
#pragma unroll UNROLL
      for (uint32_t s = 0; s < AD_RANKS && k0 + s < a.rank; s += STEP) {
        wvec wn[M] = {};
        if (!AHEAD || s + STEP < AD_RANKS)
#pragma unroll
          for (uint32_t m = 0; m < M; m++) wn[m] = get(o + 16 * m, k0 + s + STEP);
        const bool there = !VEC || k0 + s + W * g < a.rank;
        wvec w[M];
#pragma unroll
        for (uint32_t m = 0; m < M; m++) {
          w[m] = __builtin_bit_cast(wvec, there ? __builtin_bit_cast(adw, wv[m]) : adw{0, 0, 0, 0});
          wv[m] = wn[m];
        }
#pragma unroll
        for (uint32_t b = 0; b < TILES; b++) {
          if constexpr (sizeof(E) == 4) {
            const ad4 hv = *(const ad4 *)(H.h + (16 * b + c) * AD_HS + s + W * g);
#pragma unroll
            for (uint32_t u = 0; u < W; u++)
#pragma unroll
              for (uint32_t m = 0; m < M; m++) acc[m][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[m][u], hv[u], acc[m][b], 0, 0, 0);
          } else {
            const ad8 hi = *(const ad8 *)(H.hi + (16 * b + c) * AD_HH + s + W * g), lo = *(const ad8 *)(H.lo + (16 * b + c) * AD_HH + s + W * g);
#pragma unroll
            for (uint32_t m = 0; m < M; m++) {
              acc[m][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[m], hi, acc[m][b], 0, 0, 0);
              acc[m][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[m], lo, acc[m][b], 0, 0, 0);
            }
          }
        }
      }
      // these ranks' sums, over the row's power of two (before the scale: the product of both may leave f32's range)
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) {
        float power = 1.f;
        if constexpr (sizeof(E) == 2) power = H.power[16 * b + c];
#pragma unroll
        for (uint32_t m = 0; m < M; m++) {
          if constexpr (CARRY) continue;
          if constexpr (MANY) sum[m][b] += acc[m][b] * power;
          else old[m][b] += acc[m][b] * power * scale;
          acc[m][b] = ad4{0, 0, 0, 0};
        }
      }
    }
#pragma unroll
    for (uint32_t m = 0; m < M; m++)
#pragma unroll
      for (uint32_t b = 0; b < TILES; b++) {
        const uint32_t e = o + 16 * m + 4 * g;
        ad4 v = old[m][b];
        if constexpr (MANY) v += (CARRY ? acc[m][b] : sum[m][b]) * scale;
        if constexpr (YVEC) {
          if (16 * b + c < n && e < last) *(ad4 *)(y[b] + e) = v;
        } else {
#pragma unroll
          for (uint32_t u = 0; u < 4; u++)
            if (16 * b + c < n && e + u < last) y[b][e + u] = v[u];
        }
      }
  }
}

// The sum into y: `span` elements of the 64 rows' y by one workgroup; 64 or, with 16 rows of an adapter or fewer, 256 of them at a time.
template <class E, bool VEC, bool YVEC, bool MANY>
__global__ __launch_bounds__(256) void k_adapters_up(AdaptersArgs a, uint32_t chunks, uint32_t splits, uint32_t span) {
  __shared__ AdapterH<E> h;
  const uint32_t t0 = blockIdx.x / chunks * AD_ROWS, first = blockIdx.x % chunks * span, last = min(a.rows, first + span);
  const int32_t mine = adapter_of(a, t0 + (threadIdx.x & 63));
  uint64_t left = __ballot(mine >= 0);
  for (uint32_t j = 0, next = blockIdx.y;; j++) {
    const AdapterRows r = adapter_rows(mine, left);
    if (!r.rows) return;
    if (j != next) continue;
    next += gridDim.y;
    const uint32_t n = (uint32_t)__popcll(r.rows), order = adapter_order(r.rows);
    if (n <= 16) adapter_sum<E, 4, 1, VEC, YVEC, MANY>(a, h, t0, order, n, r.w, first, last, splits);
    else adapter_sum<E, 1, 4, VEC, YVEC, MANY>(a, h, t0, order, n, r.w, first, last, splits);
  }
}

// The column ranges of h: as many as give about 256 workgroups (four tiles of rows to a block), of two steps for each wavefront at least, since
// the next launch reads the sums of each. Elements of y: about 1024 workgroups, of AD_OUT at least. 1536 rows of rank 64, 4096 x 4096: two
// ranges 14.2 and 17.8 us, four 14.4 and 20.8, eight 16.5 and 33.
struct AdaptersPlan { uint32_t blocks, tiles, kinds, splits, span, chunks, out; };  // tiles, kinds: workgroups for those of 64 rows
static AdaptersPlan adapters_plan(const AdaptersArgs &a) {
  AdaptersPlan p;
  p.blocks = (a.batch + AD_ROWS - 1) / AD_ROWS;
  const uint32_t most = std::min({AD_ROWS, a.batch, a.adapters});  // adapters among 64 rows
  p.kinds = std::min(most, std::max(1u, 64 / p.blocks));
  p.tiles = std::min(most + (std::min(a.batch, AD_ROWS) - most) / 16, std::max(4u, 64 / p.blocks));
  const uint32_t step = a.half ? 256 : 128;
  p.splits = std::min({AD_SPLITS, std::max(1u, 256 / (p.blocks * std::min(p.tiles, 4u))), (a.cols + step - 1) / step});
  p.span = ((a.cols + p.splits - 1) / p.splits + step - 1) / step * step;
  p.splits = (a.cols + p.span - 1) / p.span;
  const uint32_t outs = (a.rows + AD_OUT - 1) / AD_OUT;
  p.chunks = std::min(outs, std::max(1u, 1024 / (p.blocks * p.kinds)));
  p.out = (outs + p.chunks - 1) / p.chunks * AD_OUT;
  p.chunks = (a.rows + p.out - 1) / p.out;
  return p;
}
uint64_t adapters_scratch_floats(const AdaptersArgs &a) { return (uint64_t)adapters_plan(a).splits * a.batch * a.rank; }

template <class E, bool VEC> static hipError_t launch_adapters(hipStream_t s, const AdaptersArgs &a) {
  const AdaptersPlan p = adapters_plan(a);
  const uint32_t ranks = (a.rank + AD_RANKS - 1) / AD_RANKS;
  hipLaunchKernelGGL((k_adapters_down<E, VEC>), dim3(p.blocks, p.tiles, p.splits * ranks), dim3(256), 0, s, a, p.splits, p.span);
  WGD_HIP(hipGetLastError());
  return hipSuccess;
}
template <class E, bool VEC, bool YVEC> static hipError_t launch_adapters_up(hipStream_t s, const AdaptersArgs &a) {
  const AdaptersPlan p = adapters_plan(a);
  const dim3 grid(p.blocks * p.chunks, p.kinds);
  if (a.rank > AD_RANKS) hipLaunchKernelGGL((k_adapters_up<E, VEC, YVEC, true>), grid, dim3(256), 0, s, a, p.chunks, p.splits, p.out);
  else hipLaunchKernelGGL((k_adapters_up<E, VEC, YVEC, false>), grid, dim3(256), 0, s, a, p.chunks, p.splits, p.out);
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
