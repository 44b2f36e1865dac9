// sample.hip — temperature / top-k / top-p sampling of one logits row on the device.
//
// Replaces sample() (src/core/engine.ts:305-324), whose steps it keeps:
//   * the best finite logit (first index of the maximum; none finite is an error);
//   * temperature 0: that index;
//   * the top-k finite logits in descending order, ties to the lower index (the order the
//     reference's stable insertion sort leaves);
//   * probabilities exp((l - best) / T) in f64, their sum, the shortest prefix whose share
//     reaches top-p, and a draw u * retained walked down that prefix.
// Math.random() becomes the index-th output of splitmix64(seed) (Steele, Lea and Flood,
// "Fast splittable pseudorandom number generators", OOPSLA 2014), scaled to [0, 1) with 53
// bits: the index is the position the sampled token will take, so a sequence is the same
// whether it is decoded one token per call, in device chunks or by graph replays.
//
// Every finite logit has a unique 64-bit composite: an order-preserving 32-bit key of its
// value above the complement of its index, so larger composites are larger logits and,
// among equal logits, lower indices. Two launches:
//   * k_sample_local, one workgroup per slice of about 2K logits (one workgroup's loads
//     cannot stream a 500 KB row quickly): the slice's finite count and best composite, a
//     histogram of the top 12 key bits, and every composite at or above the bin holding the
//     slice's k-th largest. That is a superset of the slice's top k, so together the slices
//     hold the row's top k.
//   * k_sample, one workgroup of 1024 threads over those candidates. With at least k slices, the
//     k-th largest of the slices' best composites is a lower bound of the row's k-th
//     largest (k composites reach it), and few candidates lie above it: they are gathered
//     into LDS at once (each wavefront reads its slices' lists, the first 64 entries loaded
//     before the bound is known). Otherwise, or if more than 1024 lie above it, a 4096-bin
//     histogram of the top 12 composite bits and a block scan find the bin holding the k-th
//     largest; if it and the bins above hold at most 1024 candidates they are gathered into
//     LDS, else the next 12 bits of that bin are histogrammed (values that tie over many
//     indices) until they fit. Each gathered composite's rank orders them; then the
//     probabilities, their running sum (one thread, in order) and the draw.
//     It is a chain of latencies in one workgroup, not of bytes: 128256 logits, k = 40, took
//     19.9 us by the histogram and serial sums with a division per step, 12.1 us so.
#include <algorithm>
#include <cmath>

#include "internal.h"
#include "decode.h"

namespace wgd {

constexpr uint32_t SMP_T = 1024, SMP_BINS = 4096, SMP_CAND = 1024;
constexpr uint32_t SL_T = 256, SL_MAX = 256, SL_SLICE = 1024;  // local kernel: threads, slices, slice floor
constexpr uint32_t SL_E = 4;  // logits per thread per step of the local kernel, loaded before use
constexpr uint32_t SMP_R = 16;  // candidates per thread held in registers by the selection

__host__ __device__ inline uint64_t splitmix64_at(uint64_t seed, uint64_t index) {
  uint64_t z = seed + (index + 1) * 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

// Order-preserving key of a finite float (-0 and +0 equal, as the reference compares them).
__device__ __forceinline__ uint32_t order_key(float v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) == 0) u = 0;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ bool finite_f(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ uint32_t comp_index(uint64_t c) { return 0xFFFFFFFFu - (uint32_t)c; }
// The logit of a composite (order_key undone; -0 comes back as +0).
__device__ __forceinline__ float comp_value(uint64_t c) {
  const uint32_t k = (uint32_t)(c >> 32);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  return v;
}

// The bin of hist[0..NB) holding the K-th largest entry when `above` entries are larger
// than every bin, and the count above that bin, to *out_bin / *out_above. Each of the T
// threads owns NB / T consecutive bins. Every thread calls it; K <= above + the total.
template <uint32_t T, uint32_t NB>
__device__ __forceinline__ void find_bin(const uint32_t *hist, uint32_t above, uint32_t K, uint32_t *wsum,
                                         uint32_t *out_bin, uint32_t *out_above) {
  constexpr uint32_t PER = NB / T;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const uint32_t b0 = PER * tid;
  uint32_t s = 0;
#pragma unroll
  for (uint32_t j = 0; j < PER; j++) s += hist[b0 + j];
  uint32_t incl = s;  // the sum of s over this and the higher lanes
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t w = __shfl_down(incl, o);
    if (lane + o < 64) incl += w;
  }
  __syncthreads();
  if (lane == 0) wsum[wv] = incl;
  __syncthreads();
  uint32_t higher = above + incl - s;  // entries in the bins above this thread's
  for (uint32_t w = wv + 1; w < T / 64; w++) higher += wsum[w];
  if (higher < K && higher + s >= K) {
    uint32_t h = higher;
    for (int j = (int)PER - 1; j >= 0; j--) {
      const uint32_t c = hist[b0 + j];
      if (h + c >= K) { *out_bin = b0 + j; *out_above = h; break; }
      h += c;
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------ per-slice candidates

struct SliceOut { uint64_t best; uint32_t finite, count; };

__global__ __launch_bounds__(SL_T) void k_sample_local(const float *logits, uint32_t n, uint32_t slice,
                                                       const SampleParams *prm, SampleParams value, uint64_t *cand,
                                                       SliceOut *so) {
  __shared__ uint32_t hist[SMP_BINS];
  __shared__ uint32_t wsum[SL_T / 64];
  __shared__ uint64_t wmax[SL_T / 64];
  __shared__ uint32_t sh_bin, sh_above, sh_count;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, w = blockIdx.x;
  const uint32_t lo = w * slice, hi = lo + slice < n ? lo + slice : n;
  for (uint32_t b = tid; b < SMP_BINS; b += SL_T) hist[b] = 0;
  if (tid == 0) { sh_count = 0; sh_bin = 0; sh_above = 0; }
  __syncthreads();
  // the slice is read twice; the second time from this CU's caches
  uint32_t cnt = 0;
  uint64_t best = 0;
  for (uint32_t i0 = lo; i0 < hi; i0 += SL_T * SL_E) {
    float v[SL_E];
#pragma unroll
    for (uint32_t e = 0; e < SL_E; e++) {
      const uint32_t i = i0 + e * SL_T + tid;
      v[e] = i < hi ? logits[i] : __uint_as_float(0x7FC00000u);
    }
#pragma unroll
    for (uint32_t e = 0; e < SL_E; e++) {
      if (!finite_f(v[e])) continue;
      const uint32_t i = i0 + e * SL_T + tid;
      const uint32_t k = order_key(v[e]);
      const uint64_t c = ((uint64_t)k << 32) | (0xFFFFFFFFu - i);
      best = c > best ? c : best;
      cnt++;
      atomicAdd(&hist[k >> 20], 1u);
    }
  }
  cnt = wave_sum_u32(cnt);
  best = wave_max_u64(best);
  if (lane == 0) { wsum[wv] = cnt; wmax[wv] = best; }
  __syncthreads();
  cnt = 0; best = 0;
  for (uint32_t u = 0; u < SL_T / 64; u++) {
    cnt += wsum[u];
    best = wmax[u] > best ? wmax[u] : best;
  }
  const SampleParams p = prm ? *prm : value;
  const uint32_t K = p.top_k < cnt ? p.top_k : cnt;
  const bool gather = p.temperature != 0.0 && K > 0;
  if (gather) {
    find_bin<SL_T, SMP_BINS>(hist, 0, K, wsum, &sh_bin, &sh_above);
    const uint32_t lo_key = sh_bin << 20;
    uint64_t *out = cand + (uint64_t)w * slice;
    for (uint32_t i0 = lo; i0 < hi; i0 += SL_T) {
      const uint32_t i = i0 + tid;
      const float v = i < hi ? logits[i] : __uint_as_float(0x7FC00000u);
      const bool fin = finite_f(v);
      const uint32_t k = fin ? order_key(v) : 0;
      const bool take = fin && k >= lo_key;
      const uint64_t m = __ballot(take);
      if (m) {
        uint32_t base = 0;
        if (lane == 0) base = atomicAdd(&sh_count, (uint32_t)__popcll(m));
        base = __shfl(base, 0);
        if (take) out[base + (uint32_t)__popcll(m & ((1ull << lane) - 1))] = ((uint64_t)k << 32) | (0xFFFFFFFFu - i);
      }
    }
    __syncthreads();
  }
  if (tid == 0) so[w] = SliceOut{best, cnt, gather ? sh_count : 0u};
}

// ------------------------------------------------------------------ selection and draw

struct SampleLds {
  uint32_t hist[SMP_BINS];
  uint64_t cand[SMP_CAND];
  double prob[256], cum[256];
  uint64_t top[SL_MAX];
  uint32_t counts[SL_MAX];
  uint32_t offs[SL_MAX + 1];
  uint32_t wsum[16];
  uint64_t wmax[16];
  uint64_t bound;
  uint32_t bin, above, ncand, cutoff;
};

// What select() starts from: the offsets of the slices' candidate lists in one flat range, and an
// empty histogram.
__device__ __forceinline__ void select_begin(SampleLds &L, uint32_t nslices) {
  if (threadIdx.x == 0) {
    L.offs[0] = 0;
    for (uint32_t w = 0; w < nslices; w++) L.offs[w + 1] = L.offs[w] + L.counts[w];
  }
  for (uint32_t b = threadIdx.x; b < SMP_BINS; b += SMP_T) L.hist[b] = 0;
}

// The histogram selection of k_sample: the candidates at or above a bin's start that hold the
// K largest, through put().
template <class Put>
__device__ __forceinline__ void select(SampleLds &L, const uint64_t *cand, uint32_t slice, uint32_t nslices, uint32_t K,
                                       Put put) {
  const uint32_t tid = threadIdx.x;
  __syncthreads();
  const uint32_t C = L.offs[nslices];
  auto at = [&](uint32_t i) -> uint64_t {  // flat candidate i: binary search over the offsets
    uint32_t a = 0, b = nslices;
    while (b - a > 1) {
      const uint32_t mid = (a + b) >> 1;
      if (L.offs[mid] <= i) a = mid; else b = mid;
    }
    return cand[(uint64_t)a * slice + (i - L.offs[a])];
  };
  // The candidates, loaded once: all loads issued together, then kept in registers for every
  // pass (up to SMP_T * SMP_R of them; more are read again per pass).
  const bool resident = C <= SMP_T * SMP_R;
  uint64_t cr[SMP_R];
#pragma unroll
  for (uint32_t r = 0; r < SMP_R; r++) {
    const uint32_t i = r * SMP_T + tid;
    cr[r] = resident && i < C ? at(i) : 0;
  }
  // f(c) over every candidate c this thread owns (uniform control flow: f may use ballots)
  auto each = [&](auto f) {
    if (resident) {
#pragma unroll
      for (uint32_t r = 0; r < SMP_R; r++) {
        const uint32_t i = r * SMP_T + tid;
        f(i < C, cr[r]);
      }
    } else {
      for (uint32_t i0 = 0; i0 < C; i0 += SMP_T) {
        const uint32_t i = i0 + tid;
        f(i < C, i < C ? at(i) : 0);
      }
    }
  };
  each([&](bool ok, uint64_t c) { if (ok) atomicAdd(&L.hist[c >> 52], 1u); });
  __syncthreads();
  // refine until the bin holding the K-th largest, and everything above it, fits in LDS
  uint64_t prefix = 0;   // composite bits fixed so far
  uint32_t shift = 52;   // the current field starts here: 12 bits, the last one 4 (bits 3..0)
  uint32_t above = 0;    // candidates above the current prefix range: all in the top K
  for (;;) {
    find_bin<SMP_T, SMP_BINS>(L.hist, above, K, L.wsum, &L.bin, &L.above);
    const uint32_t bin = L.bin;
    above = L.above;
    const uint32_t inbin = L.hist[bin];
    prefix |= (uint64_t)bin << shift;
    __syncthreads();
    if (above + inbin <= SMP_CAND || shift == 0) break;
    const uint32_t nshift = shift >= 12 ? shift - 12 : 0;
    const uint64_t hi_mask = ~((1ull << shift) - 1);                   // bits fixed so far
    const uint32_t fmask = shift >= 12 ? 0xFFFu : (1u << shift) - 1;  // the next field's width
    for (uint32_t b = tid; b < SMP_BINS; b += SMP_T) L.hist[b] = 0;
    __syncthreads();
    each([&](bool ok, uint64_t c) {
      if (ok && (c & hi_mask) == prefix) atomicAdd(&L.hist[(uint32_t)((c >> nshift) & fmask)], 1u);
    });
    __syncthreads();
    shift = nshift;
  }
  // every candidate at or above the selected bin's range start (prefix: zeros below it)
  if (tid == 0) L.ncand = 0;
  __syncthreads();
  each([&](bool ok, uint64_t c) { put(ok && c >= prefix, c); });
  __syncthreads();
}

// The token from the slices' candidates; st (optional) receives it as k_argmax_advance would.
__global__ __launch_bounds__(SMP_T) void k_sample(const uint64_t *cand, const SliceOut *so, uint32_t nslices,
                                                  uint32_t slice, const SampleParams *prm, SampleParams value,
                                                  int32_t index, StepState *st, int32_t *out, int32_t *tokens,
                                                  uint32_t cap, int advance) {
  __shared__ SampleLds L;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const SampleParams p = prm ? *prm : value;
  // the slices' totals and best composites, and this wavefront's slices' first 64 candidates
  // (slices wv, wv + 16, ...; a list has room for more than 64, entries past its count are not used)
  const uint32_t wv = tid >> 6;
  const SliceOut mine_so = tid < nslices ? so[tid] : SliceOut{0, 0, 0};
  constexpr uint32_t WV = SMP_T / 64, SR = SL_MAX / WV;
  uint64_t first[SR];
#pragma unroll
  for (uint32_t r = 0; r < SR; r++) {
    const uint32_t w = r * WV + wv;
    first[r] = w < nslices ? cand[(uint64_t)w * slice + lane] : 0;
  }
  if (tid < SL_MAX) { L.top[tid] = mine_so.best; L.counts[tid] = mine_so.count; }
  uint32_t cnt = wave_sum_u32(mine_so.finite);
  uint64_t best = wave_max_u64(mine_so.best);
  if (lane == 0) { L.wsum[wv] = cnt; L.wmax[wv] = best; }
  if (tid == 0) { L.ncand = 0; L.bound = 0; L.cutoff = 0xFFFFFFFFu; }
  __syncthreads();
  if (p.top_k > nslices) select_begin(L, nslices);  // beside the sums below
  cnt = 0; best = 0;
  for (uint32_t u = 0; u < SMP_T / 64; u++) {
    cnt += L.wsum[u];
    best = L.wmax[u] > best ? L.wmax[u] : best;
  }
  // the candidates that this wavefront takes, into L.cand (uniform control flow)
  auto put = [&](bool take, uint64_t c) {
    const uint64_t m = __ballot(take);
    if (m) {
      uint32_t slot0 = 0;
      if (lane == 0) slot0 = atomicAdd(&L.ncand, (uint32_t)__popcll(m));
      slot0 = __shfl(slot0, 0);
      const uint32_t slot = slot0 + (uint32_t)__popcll(m & ((1ull << lane) - 1));
      if (take && slot < SMP_CAND) L.cand[slot] = c;
    }
  };
  int32_t token = -1;
  const uint32_t K = p.top_k < cnt ? p.top_k : cnt;
  if (cnt > 0 && (p.temperature == 0.0 || K == 1)) {
    token = (int32_t)comp_index(best);  // one candidate is drawn whatever its probability
  } else if (cnt > 0) {
    bool gathered = false;
    if (p.top_k <= nslices) {
      // the K-th largest best: the one with K - 1 larger (zeros, slices without a finite
      // logit, are below every composite; with fewer than K bests the bound stays 0)
      if (tid < nslices && mine_so.best) {
        uint32_t larger = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < nslices; j++) larger += L.top[j] > mine_so.best ? 1u : 0u;
        if (larger == K - 1) L.bound = mine_so.best;
      }
      __syncthreads();
      const uint64_t bound = L.bound;
#pragma unroll
      for (uint32_t r = 0; r < SR; r++) {
        const uint32_t w = r * WV + wv, n = w < nslices ? L.counts[w] : 0;
        put(lane < n && first[r] >= bound, first[r]);
        for (uint32_t i0 = 64; i0 < n; i0 += 64) {
          const uint64_t c = i0 + lane < n ? cand[(uint64_t)w * slice + i0 + lane] : 0;
          put(i0 + lane < n && c >= bound, c);
        }
      }
      __syncthreads();
      gathered = L.ncand <= SMP_CAND;
    }
    if (!gathered) {
      if (p.top_k <= nslices) select_begin(L, nslices);
      select(L, cand, slice, nslices, K, put);
    }
    // rank sort, descending: the composites are unique, so each one's place is the count of
    // larger ones
    const uint32_t nc = L.ncand < SMP_CAND ? L.ncand : SMP_CAND;
    uint64_t mine = 0;
    uint32_t rank = 0;
    if (tid < nc) {
      mine = L.cand[tid];
      for (uint32_t j = 0; j < nc; j++) rank += L.cand[j] > mine ? 1u : 0u;
    }
    __syncthreads();
    if (tid < nc) L.cand[rank] = mine;
    __syncthreads();
    // probabilities of the top K (f64, as the reference's numbers)
    if (tid < K) L.prob[tid] = exp(((double)comp_value(L.cand[tid]) - (double)comp_value(best)) / p.temperature);
    __syncthreads();
    if (tid == 0) {
      double sum = 0.0, q[8];
#pragma unroll
      for (uint32_t e = 0; e < 8; e++) q[e] = L.prob[e];
      for (uint32_t j0 = 0; j0 < K; j0 += 8) {  // K <= 200, prob and cum hold 256
        double next[8];  // loaded beside the sums of this chunk
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) next[e] = L.prob[j0 + 8 + e];
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) {
          sum += q[e];
          L.cum[j0 + e] = sum;
          q[e] = next[e];
        }
      }
    }
    __syncthreads();
    // the shortest prefix whose share reaches top-p (all K where none does): a share never
    // falls along the prefix, so the first is the least index of those that reach it
    if (tid < K && L.cum[tid] / L.cum[K - 1] >= p.top_p) atomicMin(&L.cutoff, tid + 1);
    __syncthreads();
    if (tid == 0) {
      const uint32_t cutoff = L.cutoff < K ? L.cutoff : K;
      const int64_t at_pos = index >= 0 ? (int64_t)index : (int64_t)st->pos + 1;
      const double u = (double)(splitmix64_at(p.seed, (uint64_t)at_pos) >> 11) * 0x1.0p-53;
      double draw = u * L.cum[cutoff - 1];
      token = (int32_t)comp_index(best);
      uint32_t at = cutoff;  // no early exit: the loads of a chunk go out together
      for (uint32_t j0 = 0; j0 < cutoff && at == cutoff; j0 += 8) {
        double q[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) q[e] = L.prob[j0 + e];  // within prob; entries past the cutoff are not used
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) {
          draw -= q[e];
          if (draw <= 0.0 && at == cutoff && j0 + e < cutoff) at = j0 + e;
        }
      }
      if (at < cutoff) token = (int32_t)comp_index(L.cand[at]);
    }
  }
  if (tid != 0) return;
  *out = token;
  if (!advance) return;
  int32_t t = token;
  if (t < 0) { st->error = 1; t = 0; }
  if ((uint32_t)st->step < cap) tokens[st->step] = t;
  st->token = t;
  st->pos += 1;
  st->step += 1;
}

// Slices of at least SL_SLICE logits (a multiple of 4), at most SL_MAX of them.
static void slicing(uint32_t n, uint32_t *nslices, uint32_t *slice) {
  uint32_t s = (n + SL_MAX - 1) / SL_MAX;
  if (s < SL_SLICE) s = SL_SLICE;
  s = (s + 3) & ~3u;
  *slice = s;
  *nslices = (n + s - 1) / s;
}

static uint64_t cand_bytes(uint32_t nslices, uint32_t slice) { return ((uint64_t)nslices * slice * 8 + 255) / 256 * 256; }

uint64_t sample_scratch_bytes(uint32_t n) {
  uint32_t ns, sl;
  slicing(n, &ns, &sl);
  return cand_bytes(ns, sl) + SL_MAX * sizeof(SliceOut);
}

hipError_t sample(hipStream_t s, const float *logits, uint32_t n, const SampleParams *params, int32_t index,
                  StepState *st, int32_t *out, int32_t *tokens, uint32_t cap, bool advance, void *scratch,
                  const SampleParams *host_params) {
  if (!n || !scratch || (!params && !host_params) || (index < 0 && !st) || (advance && (!st || !tokens))) return hipErrorInvalidValue;
  const SampleParams value = host_params ? *host_params : SampleParams{};
  uint32_t ns, sl;
  slicing(n, &ns, &sl);
  uint64_t *cand = (uint64_t *)scratch;
  SliceOut *so = (SliceOut *)((uint8_t *)scratch + cand_bytes(ns, sl));
  hipLaunchKernelGGL(k_sample_local, dim3(ns), dim3(SL_T), 0, s, logits, n, sl, params, value, cand, so);
  WGD_HIP(hipGetLastError());
  hipLaunchKernelGGL(k_sample, dim3(1), dim3(SMP_T), 0, s, (const uint64_t *)cand, (const SliceOut *)so, ns, sl, params,
                     value, index, st, out, tokens, cap, advance ? 1 : 0);
  return hipGetLastError();
}

// ------------------------------------------------------------------ rows with given uniforms
//
// wgd_sample_rows: for every row the finite logits in descending order (composites, as above) have the
// weights w = exp((l - best) / T) in f64, rounded to integers of 2^-shift with shift = 62 - ceil(log2 n), at most 51: their sums fit
// 64 bits, are exact, and do not depend on the order of the adds, so atomics give the same token every time.
// A top-k, top-p or min-p cut and the draw itself are all "the first token whose running count reaches A or whose
// running weight reaches X". Two ways, by top_k alone:
//
// Few (2 <= top_k <= RS_FEW and half the row's groups, or a row that fits a list), two launches or one:
//   * k_rows_groups reads the row once and leaves the largest key of every group of 16 to 128 logits;
//   * k_rows_few, a workgroup a row: the bin (below) that holds the top_k-th largest of those keys bounds the bin of the
//     top_k-th largest logit (top_k logits reach it). Only groups that reach it are read again; of their
//     logits little more than top_k do, which are sorted and summed in LDS. A row of at most RS_CAP logits is one list.
// Many (top_k 0 or above), four or five launches, each a pass over the rows by all CUs:
//   * k_rows_best: the best composite and the count of finite logits, by slices;
//   * k_rows_hist: counts (for a top-k cut) and weights over RS_BINS bins of (best - l) / T, which is monotonic in l;
//   * k_rows_topk where top_k cuts: the bin of its token, from the running histogram, and that bin's tokens into a list;
//   * k_rows_cuts: the same for top-p, and for the draw: what top-p keeps is known to within its bin, so the bins
//     that the draw can fall into are known too, one or two;
//   * k_rows_last: what top-p keeps and the token, from their lists.
// Few is bound by the row's one read where there are many rows and by latency else: 64 rows of 128256, top-k 40: groups 7.0 us
// (4.7 TB/s), few 6.0; one row of 151936: 3.2 and 5.6. Up to 64 candidates are cut in one wavefront, without barriers (all
// 512 threads: 11.5). Many is bound by latency and by atomics: 16 rows of 262144, top-p 0.95: best 4.0, hist 12.1, cuts 11.7,
// last 7.6.
// A cut's token is found in its list by a histogram of RS_SUB parts of the bin and a sort of the one part
// that holds it (a sort of the whole list took four times as long).
// A bin with more tokens than its list holds (RS_LIST in all, RS_CAP from one workgroup and in one part of the bin: ties, or
// logits that lie within a few tens of bins, so less than the temperature apart), or more than RS_CAP candidates of a
// small top-k, send a row through pick_row, which refines by 11 bits of the composite at a time, in one workgroup. 16 rows
// of 262144, top-p: 40 us where that bin holds 700 tokens, 49 where it holds 2300 (650 by pick_row, with lists of
// RS_CAP), 5.0 ms where all are equal; top-k 40 of equal logits 7.4 ms.
constexpr uint32_t RS_T = 512, RS_BINS = 2048, RS_CAP = 2048, RS_LIST = 8192, RS_SUB = 1024;
constexpr uint32_t RS_ROWS = 256;  // rows per launch: the histograms of more would only fill memory
constexpr float RS_SPAN = 48.f;    // bins cover exp(0) to exp(-48) < 2^-62; the last one all below
constexpr uint32_t RS_SLICES = 64, RS_SLICE = 4096;  // most slices of a row, least logits of one
constexpr uint32_t RS_FEW = 512, RS_GROUPS = 2048;   // top_k by groups; most groups of a row
constexpr uint32_t RG_T = 256, RG_STEP = 256;        // k_rows_groups: threads; logits of a wavefront's step
enum RowCut : uint32_t { CUT_K = 0, CUT_P = 1, CUT_DRAW = 2 };

struct RowSlice { uint64_t best; uint32_t finite, pad; };
struct RowHist {
  uint64_t mass[RS_BINS];
  uint32_t count[RS_BINS];
  uint64_t list[3][RS_LIST];                 // of top-k, top-p and the draw
  uint32_t nlist[3], slow[2];                // slow: k_rows_topk or k_rows_cuts has a list that is full
  uint64_t minp, s;                          // the weights that min-p and top-k keep
  uint64_t pmass, dmass;                     // the weights before top-p's bin and before the draw's bins b0 .. b1
  uint32_t pbin, b0, b1;
  RowSlice slice[RS_SLICES];
};
struct RowGroups { uint32_t key[RS_GROUPS]; };

struct RowsK {
  const float *logits; uint32_t n, slice; uint64_t stride;
  const double *uniforms; int32_t *tokens; RowHist *hist; RowGroups *groups;
  double inv_t, top_p, min_p, unit;  // 1 / temperature; unit: 2^shift
  float bins;                        // bins per unit of logit
  uint32_t top_k, steps, ngroups, aligned, bslice, bslices;  // b..: slices of k_rows_best
};

__device__ __forceinline__ uint32_t row_bin(const RowsK &a, float best, float l) {
  return (uint32_t)fminf((best - l) * a.bins, (float)(RS_BINS - 1));
}
// exp((l - best) / T) to 2^-45 of it, which is finer than the grid of all but the largest weights: 2^k times the Taylor sum of the
// rest r, |r| <= ln 2 / 2. The next term is below 9e-15 of it, the roundings of 1 / T, of the quotient and of r add up to 1.1e-14
// at 48; measured 1.33e-14. More terms would lengthen a chain that bounds k_rows_hist as it is.
// Below 2^-70 it is 0: less than half of the least integer below, whatever n.
__device__ __forceinline__ double row_weight(const RowsK &a, float best, float l) {
  const double x = fmax(((double)l - (double)best) * a.inv_t, -64.0);
  const double k = rint(x * 1.44269504088896340736);
  const double r = fma(-k, 0.69314718055994530942, x);
  double p = 1.0 / 39916800;
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return x <= -48.6 ? 0.0 : ldexp(p, (int)k);
}
// w times 2^shift (at most 2^51) as an integer: the low bits of its sum with 2^52, which rounds it.
__device__ __forceinline__ uint64_t row_mass(const RowsK &a, double w) {
  return (uint64_t)__double_as_longlong(w * a.unit + 0x1p52) & ((1ull << 52) - 1);
}
__device__ __forceinline__ uint64_t composite(float l, uint32_t i) { return ((uint64_t)order_key(l) << 32) | (0xFFFFFFFFu - i); }
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max_f(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
// The values of the lanes up to and with this one, combined: row_shr 1, 2, 4, 8, then row_bcast15 into rows 1 and 3 and
// row_bcast31 into rows 2 and 3. Lanes without a source take 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  return (uint64_t)dpp_u32<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp_u32<CTRL, ROWS>((uint32_t)v);
}
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
  v += dpp_u64<0x111, 0xf>(v);
  v += dpp_u64<0x112, 0xf>(v);
  v += dpp_u64<0x114, 0xf>(v);
  v += dpp_u64<0x118, 0xf>(v);
  v += dpp_u64<0x142, 0xa>(v);
  v += dpp_u64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
  v += dpp_u32<0x111, 0xf>(v);
  v += dpp_u32<0x112, 0xf>(v);
  v += dpp_u32<0x114, 0xf>(v);
  v += dpp_u32<0x118, 0xf>(v);
  v += dpp_u32<0x142, 0xa>(v);
  v += dpp_u32<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t wave_top_u32(uint32_t v) {  // the largest, in every lane
  v = max(v, dpp_u32<0x111, 0xf>(v));
  v = max(v, dpp_u32<0x112, 0xf>(v));
  v = max(v, dpp_u32<0x114, 0xf>(v));
  v = max(v, dpp_u32<0x118, 0xf>(v));
  v = max(v, dpp_u32<0x142, 0xa>(v));
  v = max(v, dpp_u32<0x143, 0xc>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, uint32_t lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), (int)lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, (int)lane);
}
// At least x and 1, at most `most`.
__device__ __forceinline__ uint64_t at_least(double x, uint64_t most) { return min(max((uint64_t)ceil(x), (uint64_t)1), most); }

// Logits i .. i + 4 of a row of n, NaN past its end; 16 bytes at once where every row starts on 16.
__device__ __forceinline__ float4 row_load4(const RowsK &a, const float *row, uint32_t i) {
  const float none = __uint_as_float(0x7FC00000u);
  if (a.aligned && i + 4 <= a.n) return *(const float4 *)(row + i);
  return make_float4(i < a.n ? row[i] : none, i + 1 < a.n ? row[i + 1] : none, i + 2 < a.n ? row[i + 2] : none,
                     i + 3 < a.n ? row[i + 3] : none);
}
// Logits of T threads on their way: 16 a thread, four in a row.
struct RowQuads { float4 v[4]; };
template <uint32_t T>
__device__ __forceinline__ RowQuads load_quads(const RowsK &a, const float *row, uint32_t i0, uint32_t hi) {
  const float none = __uint_as_float(0x7FC00000u);
  RowQuads q;
#pragma unroll
  for (uint32_t e = 0; e < 4; e++) {
    const uint32_t i = i0 + 4 * (e * T + threadIdx.x);
    q.v[e] = i < hi ? row_load4(a, row, i) : make_float4(none, none, none, none);
  }
  return q;
}
// f(finite, logit, index) over the logits [lo, hi) (lo a multiple of 4), for every thread of T alike. `now` are the first
// of them, which a caller loads ahead of what it waits for.
template <uint32_t T, class F>
__device__ __forceinline__ void each_logit(const RowsK &a, const float *row, uint32_t lo, uint32_t hi, RowQuads now, F f) {
  for (uint32_t i0 = lo; i0 < hi; i0 += 16 * T) {
    RowQuads next = {};
    if (i0 + 16 * T < hi) next = load_quads<T>(a, row, i0 + 16 * T, hi);
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
      const uint32_t i = i0 + 4 * (e * T + threadIdx.x);
      const float4 v = now.v[e];
      f(finite_f(v.x) && i < hi, v.x, i);
      f(finite_f(v.y) && i + 1 < hi, v.y, i + 1);
      f(finite_f(v.z) && i + 2 < hi, v.z, i + 2);
      f(finite_f(v.w) && i + 3 < hi, v.w, i + 3);
    }
    now = next;
  }
}
template <uint32_t T, class F>
__device__ __forceinline__ void each_logit(const RowsK &a, const float *row, uint32_t lo, uint32_t hi, F f) {
  each_logit<T>(a, row, lo, hi, load_quads<T>(a, row, lo, hi), f);
}

__global__ __launch_bounds__(256) void k_rows_best(RowsK a) {
  __shared__ uint64_t wmax[4];
  __shared__ uint32_t wsum[4];
  const uint32_t tid = threadIdx.x, lo = blockIdx.x * a.bslice, hi = min(lo + a.bslice, a.n);
  RowHist &h = a.hist[blockIdx.y];
  float top = -INFINITY;
  uint32_t at = 0, cnt = 0;
  // a thread meets its logits in order: the first of equal ones stays
  each_logit<256>(a, a.logits + blockIdx.y * a.stride, lo, hi, [&](bool ok, float v, uint32_t i) {
    cnt += ok;
    if (ok && (v > top || cnt == 1)) { top = v; at = i; }
  });
  uint64_t best = wave_max_u64(cnt ? composite(top, at) : 0);
  cnt = wave_sum_u32(cnt);
  if ((tid & 63) == 0) { wmax[tid >> 6] = best; wsum[tid >> 6] = cnt; }
  // this slice's share of what the launches behind it add to
  for (uint32_t b = blockIdx.x * 256 + tid; b < RS_BINS; b += a.bslices * 256) { h.mass[b] = 0; h.count[b] = 0; }
  if (blockIdx.x == 0 && tid == 0) {
    h.minp = 0;
    h.nlist[0] = h.nlist[1] = h.nlist[2] = h.slow[0] = h.slow[1] = 0;
  }
  __syncthreads();
  if (tid != 0) return;
  for (uint32_t w = 1; w < 4; w++) { best = wmax[w] > best ? wmax[w] : best; cnt += wsum[w]; }
  h.slice[blockIdx.x] = RowSlice{best, cnt, 0};
}

// The row's best composite and finite count, in every thread of a wavefront.
__device__ __forceinline__ void row_best(const RowsK &a, const RowHist &h, uint64_t *best, uint32_t *finite) {
  const uint32_t lane = threadIdx.x & 63;
  const RowSlice s = lane < a.bslices ? h.slice[lane] : RowSlice{0, 0, 0};
  const uint32_t key = wave_top_u32((uint32_t)(s.best >> 32));
  *best = (uint64_t)key << 32 | wave_top_u32((uint32_t)(s.best >> 32) == key ? (uint32_t)s.best : 0);
  *finite = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(s.finite), 63);
}

// One token's weight, and with COUNT the token, into a histogram in LDS.
template <bool COUNT>
__device__ __forceinline__ void hist_add(uint64_t *mass, uint32_t *count, bool ok, uint32_t bin, uint64_t m) {
  if (!ok) return;
  if (COUNT) atomicAdd(&count[bin], 1u);
  if (m) atomicAdd((unsigned long long *)&mass[bin], (unsigned long long)m);
}

template <bool COUNT>
__global__ __launch_bounds__(RS_T) void k_rows_hist(RowsK a) {
  __shared__ uint64_t mass[RS_BINS];
  __shared__ uint32_t count[COUNT ? RS_BINS : 1];
  const uint32_t tid = threadIdx.x;
  RowHist &h = a.hist[blockIdx.y];
  const uint32_t lo = blockIdx.x * a.slice, hi = min(lo + a.slice, a.n);
  const float *row = a.logits + blockIdx.y * a.stride;
  const RowQuads first = load_quads<RS_T>(a, row, lo, hi);
  uint64_t best;
  uint32_t finite;
  row_best(a, h, &best, &finite);
  if (!finite) return;
  const float bv = comp_value(best);
  for (uint32_t b = tid; b < RS_BINS; b += RS_T) {
    mass[b] = 0;
    if (COUNT) count[b] = 0;
  }
  __syncthreads();
  uint64_t minp = 0;
  each_logit<RS_T>(a, row, lo, hi, first, [&](bool ok, float v, uint32_t) {
    const double w = ok ? row_weight(a, bv, v) : 0.0;
    const uint64_t m = row_mass(a, w);
    if (ok && w >= a.min_p) minp += m;
    hist_add<COUNT>(mass, count, ok, ok ? row_bin(a, bv, v) : 0, m);
  });
  __syncthreads();
  for (uint32_t b = tid; b < RS_BINS; b += RS_T) {
    if (COUNT && count[b]) atomicAdd(&h.count[b], count[b]);
    if (mass[b]) atomicAdd((unsigned long long *)&h.mass[b], (unsigned long long)mass[b]);
  }
  minp = wave_sum_u64(minp);
  if ((tid & 63) == 0 && minp) atomicAdd((unsigned long long *)&h.minp, (unsigned long long)minp);
}

struct PickLds {
  uint64_t mass[RS_BINS];
  uint32_t count[RS_BINS];         // both with what lies in the bins before, once scanned
  uint64_t smass[RS_SUB];
  uint32_t scount[RS_SUB];         // the same of the parts of one bin
  uint64_t list[RS_CAP], cum[RS_CAP];
  uint64_t part[RS_CAP];           // one bin's tokens; tokens on their way to a list
  uint64_t wmass[RS_T / 64];
  uint32_t wcount[RS_T / 64];
  uint64_t x_mass;                 // of find_cross: the weight and count before the bin
  uint32_t x_bin, x_count, nlist, npart, at;
};

// Running sums of the bins, in place.
template <uint32_t BINS>
__device__ __forceinline__ void scan_bins(PickLds &L, uint64_t *mass, uint32_t *count) {
  constexpr uint32_t PER = BINS / RS_T;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  uint64_t m[PER], ms = 0;
  uint32_t c[PER], cs = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t e = 0; e < PER; e++) {
    m[e] = ms += mass[PER * tid + e];
    c[e] = cs += count[PER * tid + e];
  }
  const uint64_t mi = wave_scan_u64(ms);
  const uint32_t ci = wave_scan_u32(cs);
  if (lane == 63) { L.wmass[wv] = mi; L.wcount[wv] = ci; }
  __syncthreads();
  uint64_t mb = mi - ms;
  uint32_t cb = ci - cs;
  for (uint32_t w = 0; w < wv; w++) { mb += L.wmass[w]; cb += L.wcount[w]; }
#pragma unroll
  for (uint32_t e = 0; e < PER; e++) {
    mass[PER * tid + e] = mb + m[e];
    count[PER * tid + e] = cb + c[e];
  }
  __syncthreads();
}

// The first bin of scanned ones at which the running count reaches A or the running weight X, from count0 and mass0
// on, and both before that bin. Callers ask only for what the bins hold; without such a bin x_bin is BINS.
template <uint32_t BINS>
__device__ __forceinline__ void find_cross(PickLds &L, const uint64_t *mass, const uint32_t *count, uint32_t count0, uint64_t mass0, uint64_t A,
                                           uint64_t X) {
  __syncthreads();
  if (threadIdx.x == 0) L.x_bin = BINS;
  __syncthreads();
#pragma unroll
  for (uint32_t b = threadIdx.x; b < BINS; b += RS_T) {
    const uint64_t c1 = (uint64_t)count0 + count[b], m1 = mass0 + mass[b];
    const uint64_t cb = b ? (uint64_t)count0 + count[b - 1] : count0, mb = b ? mass0 + mass[b - 1] : mass0;
    if (cb < A && mb < X && (c1 >= A || m1 >= X)) { L.x_bin = b; L.x_count = (uint32_t)cb; L.x_mass = mb; }
  }
  __syncthreads();
}
__device__ __forceinline__ void find_cross(PickLds &L, uint64_t A, uint64_t X) { find_cross<RS_BINS>(L, L.mass, L.count, 0, 0, A, X); }

// L.list[0 .. L.nlist) (at most RS_CAP) in descending order, and its running weights in L.cum. Up to RS_RANK tokens are
// placed by the count of larger ones, without a barrier per step.
constexpr uint32_t RS_RANK = 256;
__device__ __forceinline__ void sort_list(const RowsK &a, PickLds &L, float bv) {
  constexpr uint32_t PER = RS_CAP / RS_T;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, nl = min(L.nlist, RS_CAP);
  if (nl <= RS_RANK) {
    uint64_t mine = 0;
    uint32_t rank = 0;
    if (tid < nl) {
      mine = L.list[tid];
#pragma unroll 8
      for (uint32_t j = 0; j < nl; j++) rank += L.list[j] > mine ? 1u : 0u;
    }
    __syncthreads();
    if (tid < nl) L.list[rank] = mine;
  } else {
    uint32_t size = 2;
    while (size < nl) size <<= 1;
    for (uint32_t j = nl + tid; j < size; j += RS_T) L.list[j] = 0;
    for (uint32_t k = 2; k <= size; k <<= 1)  // bitonic
      for (uint32_t j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (uint32_t t = tid; t < size / 2; t += RS_T) {
          const uint32_t i = 2 * t - (t & (j - 1)), p = i + j;
          const uint64_t x = L.list[i], y = L.list[p];
          if ((x < y) == ((i & k) == 0)) { L.list[i] = y; L.list[p] = x; }
        }
      }
  }
  __syncthreads();
  uint64_t m[PER], incl = 0;
#pragma unroll
  for (uint32_t e = 0; e < PER; e++) {
    const uint32_t j = PER * tid + e;
    m[e] = j < nl ? row_mass(a, row_weight(a, bv, comp_value(L.list[j]))) : 0;
    incl += m[e];
  }
  incl = wave_scan_u64(incl);
  if (lane == 63) L.wmass[wv] = incl;
  __syncthreads();
  for (uint32_t w = 0; w < wv; w++) incl += L.wmass[w];
#pragma unroll
  for (int e = (int)PER - 1; e >= 0; e--) {
    L.cum[PER * tid + e] = incl;
    incl -= m[e];
  }
  __syncthreads();
}

// L.list[0 .. nl) with nl <= 64 in descending order, one token a lane of this wavefront, each with its weight and the
// running weights.
struct WaveList { uint64_t c, cum; double w; };
__device__ __forceinline__ WaveList wave_list(const RowsK &a, const PickLds &L, float bv, uint32_t nl) {
  const uint32_t lane = threadIdx.x & 63;
  WaveList t;
  t.c = lane < nl ? L.list[lane] : 0;
  uint32_t rank = 0;
#pragma unroll 8
  for (uint32_t j = 0; j < nl; j++) rank += L.list[j] > t.c ? 1u : 0u;
  if (lane >= nl) rank = lane;
  t.c = (uint64_t)(uint32_t)__builtin_amdgcn_ds_permute((int)(4 * rank), (int)(uint32_t)(t.c >> 32)) << 32 |
        (uint32_t)__builtin_amdgcn_ds_permute((int)(4 * rank), (int)(uint32_t)t.c);
  t.w = lane < nl ? row_weight(a, bv, comp_value(t.c)) : 0.0;
  t.cum = wave_scan_u64(row_mass(a, t.w));
  return t;
}

// The place in L.list at which the running count (1 for the first) reaches A or mass0 and the running
// weight reach X; the last place if none does.
__device__ __forceinline__ uint32_t find_place(PickLds &L, uint64_t mass0, uint64_t A, uint64_t X) {
  const uint32_t nl = min(L.nlist, RS_CAP);
  __syncthreads();
  if (threadIdx.x == 0) L.at = max(nl, 1u) - 1;
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < nl; j += RS_T)
    if (j + 1 >= A || mass0 + L.cum[j] >= X) { atomicMin(&L.at, j); break; }
  __syncthreads();
  return L.at;
}

// The row's histogram, scanned: the last bin has the sum of all weights.
__device__ __forceinline__ void load_hist(PickLds &L, const RowHist &h) {
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < RS_BINS; b += RS_T) { L.mass[b] = h.mass[b]; L.count[b] = h.count[b]; }
  scan_bins<RS_BINS>(L, L.mass, L.count);
}

// Appends the wavefront's tokens for which `take` holds to a list with room for RS_CAP; the count goes on past it.
__device__ __forceinline__ void append(uint64_t *list, uint32_t *nlist, bool take, uint64_t c) {
  const uint64_t m = __ballot(take);
  if (!m) return;
  const uint32_t lane = threadIdx.x & 63;
  uint32_t base = 0;
  if (lane == 0) base = atomicAdd(nlist, (uint32_t)__popcll(m));
  base = (uint32_t)__builtin_amdgcn_readfirstlane((int)base) + (uint32_t)__popcll(m & ((1ull << lane) - 1));
  if (take && base < RS_CAP) list[base] = c;
}

// The first token of L.list whose running count (1 for the first) reaches A or mass0 and the running weight reach X (the
// last if none does): its composite, and the weight up to and with it.
__device__ __forceinline__ uint64_t cut_sorted(const RowsK &a, PickLds &L, float bv, uint64_t mass0, uint64_t A, uint64_t X, uint64_t *mass) {
  const uint32_t nl = min(L.nlist, RS_CAP), lane = threadIdx.x & 63;
  if (nl > 64) {
    sort_list(a, L, bv);
    const uint32_t at = find_place(L, mass0, A, X);
    *mass = mass0 + L.cum[at];
    return L.list[at];
  }
  if (threadIdx.x < 64) {
    const WaveList t = wave_list(a, L, bv, nl);
    const uint64_t m = __ballot(lane < nl && (lane + 1 >= A || mass0 + t.cum >= X));
    if (lane == (m ? (uint32_t)__builtin_ctzll(m) : max(nl, 1u) - 1)) { L.cum[0] = t.cum; L.part[0] = t.c; }
  }
  __syncthreads();
  *mass = mass0 + L.cum[0];
  return L.part[0];
}

// The same of n tokens in memory, in any order and with the bins b0 .. b1, before which lie the count `before` and the
// weight mbefore. *ok is off if too many tokens lie in one part of the bins.
__device__ __forceinline__ uint64_t cut_list(const RowsK &a, PickLds &L, float bv, const uint64_t *from, uint32_t n, uint32_t b0, uint32_t b1,
                                             uint32_t before, uint64_t mbefore, uint64_t A, uint64_t X, uint64_t *mass, bool *ok) {
  const float parts = (float)RS_SUB / (float)(b1 - b0 + 1);
  auto part = [&](uint64_t c) {  // monotonic, as row_bin is
    const float x = (bv - comp_value(c)) * a.bins - (float)b0;
    return (uint32_t)fminf(fmaxf(x, 0.f) * parts, (float)(RS_SUB - 1));
  };
  __syncthreads();
  if (threadIdx.x == 0) L.nlist = 0;
  if (n <= 64) {
    if (threadIdx.x < n) L.list[threadIdx.x] = from[threadIdx.x];
    if (threadIdx.x == 0) L.nlist = n;
  } else {
    for (uint32_t b = threadIdx.x; b < RS_SUB; b += RS_T) { L.smass[b] = 0; L.scount[b] = 0; }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < n; j += RS_T)
      hist_add<true>(L.smass, L.scount, true, part(from[j]), row_mass(a, row_weight(a, bv, comp_value(from[j]))));
    scan_bins<RS_SUB>(L, L.smass, L.scount);
    find_cross<RS_SUB>(L, L.smass, L.scount, before, mbefore, A, X);
    const uint32_t sub = L.x_bin;
    for (uint32_t j0 = 0; j0 < n; j0 += RS_T) {
      const uint32_t j = j0 + threadIdx.x;
      const uint64_t c = j < n ? from[j] : 0;
      append(L.list, &L.nlist, j < n && (sub >= RS_SUB || part(c) == sub), c);
    }
    if (sub < RS_SUB) { before = L.x_count; mbefore = L.x_mass; }
  }
  __syncthreads();
  *ok = L.nlist <= RS_CAP;
  return cut_sorted(a, L, bv, mbefore, A > before ? A - before : 1, X, mass);
}

// ------------------------------------------------------------------ rows: one workgroup, any bins

// The first token of the row whose running count reaches A or whose running weight reaches X: its
// composite, and the weight up to and with it.
__device__ __forceinline__ uint64_t first_token(const RowsK &a, PickLds &L, const RowHist &h, const float *row, float bv,
                                                uint64_t A, uint64_t X, uint64_t *mass) {
  load_hist(L, h);
  find_cross(L, A, X);
  auto in_bin = [&](uint32_t b) { return b < RS_BINS ? L.count[b] - (b ? L.count[b - 1] : 0) : 0; };
  const uint32_t bin = L.x_bin;
  uint32_t before = L.x_count, inside = in_bin(bin);
  uint64_t mbefore = L.x_mass, prefix = 0, hi_mask = 0;
  uint32_t shift = 64;
  while (inside > RS_CAP && shift > 0) {
    const uint32_t next = shift >= 11 ? shift - 11 : 0, fmask = (1u << (shift - next)) - 1;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < RS_BINS; b += RS_T) { L.mass[b] = 0; L.count[b] = 0; }
    __syncthreads();
    each_logit<RS_T>(a, row, 0, a.n, [&](bool ok, float v, uint32_t i) {
      const uint64_t c = composite(v, i);
      ok = ok && row_bin(a, bv, v) == bin && (c & hi_mask) == prefix;
      // larger composites first
      hist_add<true>(L.mass, L.count, ok, RS_BINS - 1 - ((uint32_t)(c >> next) & fmask), ok ? row_mass(a, row_weight(a, bv, v)) : 0);
    });
    scan_bins<RS_BINS>(L, L.mass, L.count);
    find_cross<RS_BINS>(L, L.mass, L.count, before, mbefore, A, X);
    before = L.x_count;
    mbefore = L.x_mass;
    inside = in_bin(L.x_bin);
    prefix |= (uint64_t)(RS_BINS - 1 - L.x_bin) << next;
    hi_mask = ~((1ull << next) - 1);
    shift = next;
    __syncthreads();
  }
  if (threadIdx.x == 0) L.nlist = 0;
  __syncthreads();
  each_logit<RS_T>(a, row, 0, a.n, [&](bool ok, float v, uint32_t i) {
    const uint64_t c = composite(v, i);
    append(L.list, &L.nlist, ok && row_bin(a, bv, v) == bin && (c & hi_mask) == prefix, c);
  });
  __syncthreads();
  return cut_sorted(a, L, bv, mbefore, A > before ? A - before : 1, X, mass);
}

// The row's histogram, and the weight that min-p keeps, by this workgroup alone, into h.
__device__ __forceinline__ void row_hist(const RowsK &a, PickLds &L, RowHist &h, const float *row, float bv) {
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < RS_BINS; b += RS_T) { L.mass[b] = 0; L.count[b] = 0; }
  if (threadIdx.x == 0) L.x_mass = 0;
  __syncthreads();
  uint64_t minp = 0;
  each_logit<RS_T>(a, row, 0, a.n, [&](bool ok, float v, uint32_t) {
    const double w = ok ? row_weight(a, bv, v) : 0.0;
    if (ok && w >= a.min_p) minp += row_mass(a, w);
    hist_add<true>(L.mass, L.count, ok, ok ? row_bin(a, bv, v) : 0, row_mass(a, w));
  });
  minp = wave_sum_u64(minp);
  if ((threadIdx.x & 63) == 0) atomicAdd((unsigned long long *)&L.x_mass, (unsigned long long)minp);
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < RS_BINS; b += RS_T) { h.mass[b] = L.mass[b]; h.count[b] = L.count[b]; }
  if (threadIdx.x == 0) h.minp = L.x_mass;
  __syncthreads();
}

// The row's token from its histogram (row_hist's), cut after cut.
__device__ __forceinline__ int32_t pick_row(const RowsK &a, PickLds &L, const RowHist &h, const float *row, float bv, uint32_t finite,
                                            double u) {
  constexpr uint64_t ALL = ~0ull;
  uint64_t S, R, unused;
  if (a.top_k && a.top_k < finite) {
    first_token(a, L, h, row, bv, a.top_k, ALL, &S);
  } else {
    load_hist(L, h);
    S = L.mass[RS_BINS - 1];
  }
  R = S;
  if (a.top_p < 1.0) first_token(a, L, h, row, bv, ALL, at_least(a.top_p * (double)S, S), &R);
  R = min(R, h.minp);
  return (int32_t)comp_index(first_token(a, L, h, row, bv, ALL, at_least(u * (double)R, R), &unused));
}

// ------------------------------------------------------------------ rows: many

// This workgroup's n tokens from LDS into a list of the row, with one atomic on the list's count. Whichever workgroup
// finds the list full says so.
__device__ __forceinline__ void put_list(PickLds &L, const uint64_t *from, uint32_t n, uint64_t *list, uint32_t cap, uint32_t *nlist,
                                         uint32_t *slow) {
  if (threadIdx.x == 0) L.at = n ? atomicAdd(nlist, n) : 0;
  __syncthreads();
  const uint32_t at = L.at;
  __syncthreads();
  if (n > RS_CAP || at + n > cap) {
    if (threadIdx.x == 0) *slow = 1;
    return;
  }
  for (uint32_t j = threadIdx.x; j < n; j += RS_T) list[at + j] = from[j];
}

__global__ __launch_bounds__(RS_T) void k_rows_topk(RowsK a) {
  extern __shared__ uint64_t pick_lds[];
  PickLds &L = *(PickLds *)pick_lds;
  RowHist &h = a.hist[blockIdx.y];
  const uint32_t lo = blockIdx.x * a.slice, hi = min(lo + a.slice, a.n);
  const float *row = a.logits + blockIdx.y * a.stride;
  const RowQuads first = load_quads<RS_T>(a, row, lo, hi);
  uint64_t best;
  uint32_t finite;
  row_best(a, h, &best, &finite);
  if (a.top_k >= finite) return;
  load_hist(L, h);
  find_cross(L, a.top_k, ~0ull);
  const uint32_t bin = L.x_bin;
  const float bv = comp_value(best);
  if (threadIdx.x == 0) L.nlist = 0;
  __syncthreads();
  each_logit<RS_T>(a, row, lo, hi, first, [&](bool ok, float v, uint32_t i) {
    append(L.list, &L.nlist, ok && row_bin(a, bv, v) == bin, composite(v, i));
  });
  __syncthreads();
  put_list(L, L.list, L.nlist, h.list[CUT_K], RS_LIST, &h.nlist[CUT_K], &h.slow[0]);
}

// The weight that the top-k cut leaves, from its list (*ok as cut_list's).
__device__ __forceinline__ uint64_t topk_mass(const RowsK &a, PickLds &L, const RowHist &h, float bv, bool *ok) {
  uint64_t m;
  find_cross(L, a.top_k, ~0ull);
  const uint32_t bin = L.x_bin, before = L.x_count, n = min(h.nlist[CUT_K], RS_LIST);
  const uint64_t mbefore = L.x_mass;
  cut_list(a, L, bv, h.list[CUT_K], n, bin, bin, before, mbefore, a.top_k, ~0ull, &m, ok);
  return m;
}

__global__ __launch_bounds__(RS_T) void k_rows_cuts(RowsK a) {
  extern __shared__ uint64_t pick_lds[];
  PickLds &L = *(PickLds *)pick_lds;
  RowHist &h = a.hist[blockIdx.y];
  const uint32_t lo = blockIdx.x * a.slice, hi = min(lo + a.slice, a.n);
  const float *row = a.logits + blockIdx.y * a.stride;
  const RowQuads first = load_quads<RS_T>(a, row, lo, hi);
  uint64_t best;
  uint32_t finite;
  row_best(a, h, &best, &finite);
  const double u = a.uniforms[blockIdx.y];
  if (!finite || h.slow[0] || !(u > 0.0 && u < 1.0)) return;  // slow[0]: of the launch before
  const float bv = comp_value(best);
  load_hist(L, h);
  bool ok = true;
  const uint64_t S = a.top_k && a.top_k < finite ? topk_mass(a, L, h, bv, &ok) : L.mass[RS_BINS - 1];
  if (!ok) {  // as every workgroup of the row finds
    if (threadIdx.x == 0) h.slow[1] = 1;
    return;
  }
  uint64_t least = S, most = S, pmass = 0;  // of the weight that top-p keeps; before its bin
  uint32_t pbin = RS_BINS;                  // none
  if (a.top_p < 1.0) {
    least = at_least(a.top_p * (double)S, S);
    find_cross(L, ~0ull, least);
    pbin = min(L.x_bin, RS_BINS - 1);
    pmass = L.x_mass;
    most = min(L.mass[pbin], S);
  }
  least = min(least, h.minp);
  most = min(most, h.minp);
  least = at_least(u * (double)least, least);
  most = at_least(u * (double)most, most);
  __syncthreads();
#pragma unroll
  for (uint32_t b = threadIdx.x; b < RS_BINS; b += RS_T) {
    const uint64_t m1 = L.mass[b], mb = b ? L.mass[b - 1] : 0;
    if (mb < least && m1 >= least) { L.x_bin = b; L.x_mass = mb; }
    if (mb < most && m1 >= most) L.at = b;
  }
  __syncthreads();
  const uint32_t b0 = L.x_bin, b1 = L.at;
  if (blockIdx.x == 0 && threadIdx.x == 0) { h.s = S; h.pbin = pbin; h.pmass = pmass; h.b0 = b0; h.b1 = b1; h.dmass = L.x_mass; }
  if (threadIdx.x == 0) L.nlist = L.npart = 0;
  __syncthreads();
  each_logit<RS_T>(a, row, lo, hi, first, [&](bool ok, float v, uint32_t i) {
    const uint32_t b = ok ? row_bin(a, bv, v) : RS_BINS + 1;
    append(L.list, &L.nlist, b == pbin, composite(v, i));
    append(L.part, &L.npart, b >= b0 && b <= b1, composite(v, i));
  });
  __syncthreads();
  put_list(L, L.list, L.nlist, h.list[CUT_P], RS_LIST, &h.nlist[CUT_P], &h.slow[1]);
  put_list(L, L.part, L.npart, h.list[CUT_DRAW], RS_LIST, &h.nlist[CUT_DRAW], &h.slow[1]);
}

// The token: the best where nothing is drawn, else from the lists.
__global__ __launch_bounds__(RS_T) void k_rows_last(RowsK a, uint32_t drawn) {
  extern __shared__ uint64_t pick_lds[];
  PickLds &L = *(PickLds *)pick_lds;
  RowHist &h = a.hist[blockIdx.x];
  const uint32_t tid = threadIdx.x;
  uint64_t best;
  uint32_t finite;
  row_best(a, h, &best, &finite);
  const double u = a.uniforms[blockIdx.x];
  int32_t token = finite ? (int32_t)comp_index(best) : -1;
  if (finite && drawn && u > 0.0 && u < 1.0) {
    const float bv = comp_value(best);
    bool slow = h.slow[0] || h.slow[1];
    if (!slow) {
      uint64_t R = h.s, unused;
      bool ok = true;
      if (a.top_p < 1.0)
        cut_list(a, L, bv, h.list[CUT_P], min(h.nlist[CUT_P], RS_LIST), h.pbin, h.pbin, 0, h.pmass, ~0ull, at_least(a.top_p * (double)R, R), &R, &ok);
      slow = !ok;
      if (!slow) {
        R = min(R, h.minp);
        const uint64_t c = cut_list(a, L, bv, h.list[CUT_DRAW], min(h.nlist[CUT_DRAW], RS_LIST), h.b0, h.b1, 0, h.dmass, ~0ull,
                                    at_least(u * (double)R, R), &unused, &ok);
        slow = !ok;
        token = (int32_t)comp_index(c);
      }
    }
    if (slow) {
      row_hist(a, L, h, a.logits + blockIdx.x * a.stride, bv);
      token = pick_row(a, L, h, a.logits + blockIdx.x * a.stride, bv, finite, u);
    }
  }
  if (tid == 0) a.tokens[blockIdx.x] = token;
}

// ------------------------------------------------------------------ rows: few

// Group j of 4 lanes of a wavefront's part of the row (a.steps steps of 256 logits): its largest key, 0 without a
// finite logit. Lane l of step s reads logits 256 s + 4 l .. + 4 of the part.
__global__ __launch_bounds__(RG_T) void k_rows_groups(RowsK a) {
  const uint32_t lane = threadIdx.x & 63, part = blockIdx.x * (RG_T / 64) + (threadIdx.x >> 6);
  const uint32_t lo = part * a.steps * RG_STEP;
  if (lo >= a.n) return;
  const float *row = a.logits + blockIdx.y * a.stride;
  uint32_t key = 0;
  auto take = [&](float v) { key = max(key, finite_f(v) ? order_key(v) : 0u); };
  for (uint32_t s0 = 0; s0 < a.steps; s0 += 8) {
    float4 v[8];
#pragma unroll
    for (uint32_t e = 0; e < 8; e++) v[e] = s0 + e < a.steps ? row_load4(a, row, lo + (s0 + e) * RG_STEP + 4 * lane) : make_float4(NAN, NAN, NAN, NAN);
#pragma unroll
    for (uint32_t e = 0; e < 8; e++) { take(v[e].x); take(v[e].y); take(v[e].z); take(v[e].w); }
  }
  key = max(key, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)key, 0xB1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  key = max(key, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)key, 0x4E, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  if ((lane & 3) == 0) a.groups[blockIdx.y].key[16 * part + lane / 4] = key;
}

// The token of a row whose candidates, L.list[0 .. nl) with 0 < nl <= 64, fit a wavefront: all cuts, in this one.
__device__ __forceinline__ int32_t pick_wave(const RowsK &a, const PickLds &L, float bv, double u, uint32_t nl) {
  const uint32_t lane = threadIdx.x & 63;
  const WaveList t = wave_list(a, L, bv, nl);
  uint32_t at = 0;
  if (u > 0.0 && u < 1.0) {
    // the first lane at which the running weight reaches x, the last candidate if none does
    auto place = [&](uint64_t x) {
      const uint64_t m = __ballot(lane < nl && t.cum >= x);
      return m ? (uint32_t)__builtin_ctzll(m) : nl - 1;
    };
    uint32_t last = (a.top_k ? min(a.top_k, nl) : nl) - 1;
    const uint64_t S = lane_u64(t.cum, last);
    if (a.top_p < 1.0) last = min(last, place(at_least(a.top_p * (double)S, S)));
    if (a.min_p > 0.0) {  // weights fall along the lanes
      const uint32_t kept = (uint32_t)__popcll(__ballot(lane <= last && t.w >= a.min_p));
      last = min(last, max(kept, 1u) - 1);
    }
    const uint64_t R = lane_u64(t.cum, last);
    at = place(at_least(u * (double)R, R));
  }
  return (int32_t)comp_index(lane_u64(t.c, at));
}

__global__ __launch_bounds__(RS_T) void k_rows_few(RowsK a) {
  extern __shared__ uint64_t pick_lds[];
  PickLds &L = *(PickLds *)pick_lds;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const float *row = a.logits + blockIdx.x * a.stride;
  const double u = a.uniforms[blockIdx.x];
  float bv = 0.f;
  if (a.n <= RS_CAP) {
    if (tid == 0) L.nlist = 0;
    __syncthreads();
    float top = -INFINITY;
    for (uint32_t i0 = 0; i0 < a.n; i0 += RS_T) {
      const float v = i0 + tid < a.n ? row[i0 + tid] : NAN;
      append(L.list, &L.nlist, finite_f(v), composite(v, i0 + tid));
      top = finite_f(v) ? fmaxf(top, v) : top;
    }
    top = wave_max_f(top);
    if (lane == 0) L.wcount[tid >> 6] = __float_as_uint(top);
    __syncthreads();
    for (uint32_t w = 0; w < RS_T / 64; w++) top = fmaxf(top, __uint_as_float(L.wcount[w]));
    if (L.nlist == 0) {
      if (tid == 0) a.tokens[blockIdx.x] = -1;
      return;
    }
    bv = top;
    __syncthreads();
  } else {
    uint32_t *chosen = (uint32_t *)L.cum;  // groups that reach the bound
    const uint32_t *keys = a.groups[blockIdx.x].key;
    constexpr uint32_t PER = RS_GROUPS / RS_T;
    uint32_t key[PER], top_key = 0;
    for (uint32_t b = tid; b < RS_BINS; b += RS_T) L.count[b] = 0;
    if (tid == 0) { L.nlist = 0; L.at = 0; L.x_bin = RS_BINS; }
#pragma unroll
    for (uint32_t e = 0; e < PER; e++) {
      key[e] = e * RS_T + tid < a.ngroups ? keys[e * RS_T + tid] : 0;
      top_key = max(top_key, key[e]);
    }
    top_key = wave_top_u32(top_key);
    if (lane == 0) L.wcount[tid >> 6] = top_key;
    __syncthreads();
    for (uint32_t w = 0; w < RS_T / 64; w++) top_key = max(top_key, L.wcount[w]);
    if (!top_key) {  // nothing finite
      if (tid == 0) a.tokens[blockIdx.x] = -1;
      return;
    }
    bv = comp_value((uint64_t)top_key << 32);
#pragma unroll
    for (uint32_t e = 0; e < PER; e++)
      if (key[e]) atomicAdd(&L.count[row_bin(a, bv, comp_value((uint64_t)key[e] << 32))], 1u);
    __syncthreads();
    // the bin at which their running count reaches top_k
    constexpr uint32_t B = RS_BINS / RS_T;
    uint32_t c[B], upto = 0;
#pragma unroll
    for (uint32_t e = 0; e < B; e++) c[e] = upto += L.count[B * tid + e];
    const uint32_t incl = wave_scan_u32(upto);
    if (lane == 63) L.scount[tid >> 6] = incl;
    __syncthreads();
    uint32_t before = incl - upto;
    for (uint32_t w = 0; w < tid >> 6; w++) before += L.scount[w];
#pragma unroll
    for (uint32_t e = 0; e < B; e++)
      if (before + c[e] >= a.top_k && before + (e ? c[e - 1] : 0) < a.top_k) L.x_bin = B * tid + e;
    __syncthreads();
    // what lies in the last bin has no weight: without top_k groups before it, the tokens before it are all that count
    const uint32_t bound = min(L.x_bin, RS_BINS - 2);
#pragma unroll
    for (uint32_t e = 0; e < PER; e++)
      if (key[e] && row_bin(a, bv, comp_value((uint64_t)key[e] << 32)) <= bound) chosen[atomicAdd(&L.at, 1u)] = e * RS_T + tid;
    __syncthreads();
    const uint32_t pieces = L.at * 4 * a.steps;  // of four logits
    for (uint32_t i0 = 0; i0 < pieces; i0 += RS_T) {
      const uint32_t i = i0 + tid, j = i < pieces ? chosen[i / (4 * a.steps)] : 0, in = i % (4 * a.steps);
      const uint32_t at = (j / 16) * a.steps * RG_STEP + (in / 4) * RG_STEP + (j % 16) * 16 + (in % 4) * 4;
      const float4 v = i < pieces ? row_load4(a, row, at) : make_float4(NAN, NAN, NAN, NAN);
      const float x[4] = {v.x, v.y, v.z, v.w};
      uint64_t take[4];
      uint32_t n = 0;
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) {
        take[e] = __ballot(finite_f(x[e]) && row_bin(a, bv, x[e]) <= bound);
        n += (uint32_t)__popcll(take[e]);
      }
      if (!n) continue;
      uint32_t to = 0;
      if (lane == 0) to = atomicAdd(&L.nlist, n);
      to = (uint32_t)__builtin_amdgcn_readfirstlane((int)to);
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) {
        const uint32_t place = to + (uint32_t)__popcll(take[e] & ((1ull << lane) - 1));
        if ((take[e] >> lane & 1) && place < RS_CAP) L.list[place] = composite(x[e], at + e);
        to += (uint32_t)__popcll(take[e]);
      }
    }
    __syncthreads();
  }
  const uint32_t nl = L.nlist;
  if (nl > RS_CAP) {  // ties: the row goes through its histogram, formed here
    RowHist &h = a.hist[blockIdx.x];
    uint32_t cnt = 0;
    uint64_t best = 0;
    each_logit<RS_T>(a, row, 0, a.n, [&](bool ok, float v, uint32_t i) {
      cnt += ok;
      if (ok) best = max(best, composite(v, i));
    });
    best = wave_max_u64(best);
    cnt = wave_sum_u32(cnt);
    __syncthreads();
    if (lane == 0) { L.wmass[tid >> 6] = best; L.wcount[tid >> 6] = cnt; }
    __syncthreads();
    uint32_t finite = 0;
    for (uint32_t w = 0; w < RS_T / 64; w++) { best = max(best, L.wmass[w]); finite += L.wcount[w]; }
    row_hist(a, L, h, row, bv);
    const int32_t token = u > 0.0 && u < 1.0 ? pick_row(a, L, h, row, bv, finite, u) : (int32_t)comp_index(best);
    if (tid == 0) a.tokens[blockIdx.x] = token;
    return;
  }
  if (nl <= 64) {
    if (tid >= 64) return;
    const int32_t token = pick_wave(a, L, bv, u, nl);
    if (tid == 0) a.tokens[blockIdx.x] = token;
    return;
  }
  sort_list(a, L, bv);
  int32_t token = (int32_t)comp_index(L.list[0]);
  if (u > 0.0 && u < 1.0) {
    const uint32_t K = a.top_k ? min(a.top_k, nl) : nl;
    const uint64_t S = L.cum[K - 1];
    uint32_t last = K - 1;
    if (a.top_p < 1.0) last = min(last, find_place(L, 0, ~0ull, at_least(a.top_p * (double)S, S)));
    if (a.min_p > 0.0) {  // weights fall along the list
      __syncthreads();
      if (tid == 0) L.at = 0;
      __syncthreads();
      uint32_t kept = 0;
      for (uint32_t j = tid; j <= last; j += RS_T) kept += row_weight(a, bv, comp_value(L.list[j])) >= a.min_p;
      kept = wave_sum_u32(kept);
      if (lane == 0 && kept) atomicAdd(&L.at, kept);
      __syncthreads();
      last = min(last, max(L.at, 1u) - 1);
    }
    const uint64_t R = L.cum[last];
    token = (int32_t)comp_index(L.list[find_place(L, 0, ~0ull, at_least(u * (double)R, R))]);
  }
  if (tid == 0) a.tokens[blockIdx.x] = token;
}

// Steps of a wavefront's part so that a row has at most RS_GROUPS groups: of 16 logits up to 32768, 64 at 128256.
static uint32_t group_steps(uint32_t n) {
  constexpr uint64_t most = RS_GROUPS / 16 * RG_STEP;
  return (uint32_t)((n + most - 1) / most);
}
static uint32_t group_count(uint32_t n) {
  const uint64_t part = (uint64_t)group_steps(n) * RG_STEP;
  return (uint32_t)((n + part - 1) / part) * 16;
}

uint64_t sample_rows_scratch_bytes(const SampleRowsArgs &a) {
  return (uint64_t)std::min(a.rows, RS_ROWS) * (sizeof(RowHist) + sizeof(RowGroups));
}

hipError_t sample_rows(hipStream_t s, const SampleRowsArgs &in) {
  if (!in.rows) return hipSuccess;
  if (!in.n || !in.scratch || in.stride < in.n) return hipErrorInvalidValue;
  RowsK a{};
  a.n = in.n; a.stride = in.stride;
  a.bslice = (std::max(4096u, (in.n + RS_SLICES - 1) / RS_SLICES) + 3) & ~3u;
  a.bslices = (in.n + a.bslice - 1) / a.bslice;
  a.steps = group_steps(in.n); a.ngroups = group_count(in.n);
  a.aligned = (uintptr_t)in.logits % 16 == 0 && in.stride % 4 == 0;
  a.hist = (RowHist *)in.scratch;
  a.groups = (RowGroups *)(a.hist + std::min(in.rows, RS_ROWS));
  a.inv_t = in.temperature > 0.0 ? std::min(1e300, 1.0 / in.temperature) : 0.0;
  a.top_p = in.top_p; a.min_p = in.min_p; a.top_k = in.top_k;
  int log2n = 0;
  while (log2n < 32 && (1ull << log2n) < in.n) log2n++;
  a.unit = std::ldexp(1.0, std::min(51, 62 - log2n));
  // a temperature near 0 has no finite scale: any large one keeps the bins monotonic
  a.bins = in.temperature > 0.0 ? (float)std::min(1e30, RS_BINS / (RS_SPAN * in.temperature)) : 0.f;
  lds_opt_in((const void *)k_rows_topk);
  lds_opt_in((const void *)k_rows_cuts);
  lds_opt_in((const void *)k_rows_last);
  lds_opt_in((const void *)k_rows_few);
  const bool drawn = in.temperature != 0.0 && in.top_k != 1;
  const bool whole = in.n <= RS_CAP, few = drawn && (whole || (in.top_k >= 2 && in.top_k <= RS_FEW && 2 * in.top_k <= a.ngroups));
  for (uint32_t r0 = 0; r0 < in.rows; r0 += RS_ROWS) {
    const uint32_t nr = std::min(RS_ROWS, in.rows - r0);
    a.logits = in.logits + (uint64_t)r0 * in.stride; a.uniforms = in.uniforms + r0; a.tokens = in.tokens + r0;
    if (few) {
      if (!whole) hipLaunchKernelGGL(k_rows_groups, dim3((a.ngroups / 16 + RG_T / 64 - 1) / (RG_T / 64), nr), dim3(RG_T), 0, s, a);
      WGD_HIP(hipGetLastError());
      hipLaunchKernelGGL(k_rows_few, dim3(nr), dim3(RS_T), sizeof(PickLds), s, a);
      WGD_HIP(hipGetLastError());
      continue;
    }
    // slices that give every CU a workgroup; 16384 for all: 33 us in place of 28.5 at one row of 151936, 73 of 59 at 64
    const uint64_t share = (uint64_t)in.n * nr / (uint32_t)device_cu_count();
    a.slice = ((uint32_t)std::min<uint64_t>(std::max<uint64_t>({RS_SLICE, (in.n + RS_SLICES - 1) / RS_SLICES, share}), in.n) + 3) & ~3u;
    const dim3 grid((in.n + a.slice - 1) / a.slice, nr);
    hipLaunchKernelGGL(k_rows_best, dim3(a.bslices, nr), dim3(256), 0, s, a);
    WGD_HIP(hipGetLastError());
    if (drawn) {
      if (in.top_k && in.top_k < in.n) hipLaunchKernelGGL(k_rows_hist<true>, grid, dim3(RS_T), 0, s, a);
      else hipLaunchKernelGGL(k_rows_hist<false>, grid, dim3(RS_T), 0, s, a);
      WGD_HIP(hipGetLastError());
      if (in.top_k && in.top_k < in.n) {
        hipLaunchKernelGGL(k_rows_topk, grid, dim3(RS_T), sizeof(PickLds), s, a);
        WGD_HIP(hipGetLastError());
      }
      hipLaunchKernelGGL(k_rows_cuts, grid, dim3(RS_T), sizeof(PickLds), s, a);
      WGD_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(k_rows_last, dim3(nr), dim3(RS_T), sizeof(PickLds), s, a, drawn ? 1u : 0u);
    WGD_HIP(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace wgd
