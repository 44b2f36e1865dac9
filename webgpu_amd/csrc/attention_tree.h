// attention_tree.h — attention of a tree of drafted tokens over the K/V ring (part of
// attention.hip).
//
// Node i < nodes has the position p_i = start + depth(i) and its key and value in ring slot
// (start + i) % capacity. Its query heads see the cached keys t in (p_i - window, start) and the
// nodes on its path to the root (itself among them) whose positions lie within the window:
//   y = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q . k_t,  m = max s_t.
// The keys are one range [first, start + nodes) in ring order, cached ones first. The rows of a kv
// head are the (node, query head of its group) pairs: they share its keys.
#pragma once

namespace wgd {

constexpr uint32_t TREE_WORDS = WGD_TREE_MAX / 32;

struct TreeK {
  const float *q; const void *k, *v; float *y, *part; const int32_t *parents;
  uint32_t heads, kvh, group, hd, start, window, capacity, nodes, first, nsplit, T;
  float scale;
};

// What a row sees: the first cached key, and the nodes as a bit set. Padding sees nothing.
struct TreeRow { uint32_t begin, valid; uint32_t bits[TREE_WORDS]; };

// The path of `node` to the root over parents in LDS. A parent lies before its child, so the walk
// ends; any parent that does not, or is below -1, leaves the node without keys.
__device__ __forceinline__ void tree_row(TreeRow &r, const int32_t *par, uint32_t node, uint32_t start, uint32_t window) {
  for (uint32_t w = 0; w < TREE_WORDS; w++) r.bits[w] = 0;
  int32_t a = (int32_t)node;
  uint32_t steps = 0;
  while (a >= 0) {
    if (steps < window) r.bits[a >> 5] |= 1u << (a & 31);
    const int32_t p = par[a];
    steps++;
    a = p < a ? p : -2;
  }
  r.valid = a == -1;
  const uint32_t end = start + steps;  // p_i + 1
  r.begin = end - min(end, window);
  if (!r.valid)
    for (uint32_t w = 0; w < TREE_WORDS; w++) r.bits[w] = 0;
}
__device__ __forceinline__ bool tree_sees(const TreeRow &r, uint32_t t, uint32_t start) {
  if (!r.valid) return false;
  if (t < start) return t >= r.begin;
  const uint32_t j = t - start;
  return r.bits[j >> 5] >> (j & 31) & 1;
}

// Any head dim up to 512: a workgroup owns 16 rows of a kv head and a range of keys, in tiles of T
// keys staged in LDS; f32 products one by one. Slots that no row of the workgroup sees are never
// multiplied, so what they hold (NaN too) reaches nothing.
constexpr uint32_t TREE_R = 16;
template <class E>
__global__ __launch_bounds__(256) void k_attn_tree_any(TreeK a) {
  extern __shared__ float lds[];
  __shared__ int32_t par[WGD_TREE_MAX];
  __shared__ TreeRow rows[TREE_R];
  __shared__ float mrow[TREE_R], lrow[TREE_R], corr[TREE_R];
  const uint32_t hd = a.hd, T = a.T, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  float *Ks = lds, *Vs = Ks + T * (hd + 1), *Qs = Vs + T * hd, *S = Qs + TREE_R * hd;
  const uint32_t kv = blockIdx.x, r0 = blockIdx.y * TREE_R, z = blockIdx.z, nrows = a.nodes * a.group;
  const uint32_t end = a.start + a.nodes;
  uint32_t chunk = (end - a.first + a.nsplit - 1) / a.nsplit;
  chunk = (chunk + T - 1) / T * T;
  const uint32_t lo = a.first + min(z * chunk, end - a.first), hi = lo + min(chunk, end - lo);
  auto row_of = [&](uint32_t r) -> uint64_t { return (uint64_t)(r / a.group) * a.heads + kv * a.group + r % a.group; };

  for (uint32_t i = tid; i < a.nodes; i += 256) par[i] = a.parents[i];
  for (uint32_t i = tid; i < TREE_R * hd; i += 256) {
    const uint32_t r = r0 + i / hd;
    Qs[i] = r < nrows ? a.q[row_of(r) * hd + i % hd] : 0.f;
  }
  __syncthreads();
  if (tid < TREE_R) {
    if (r0 + tid < nrows) tree_row(rows[tid], par, (r0 + tid) / a.group, a.start, a.window);
    else rows[tid].valid = 0;
    mrow[tid] = -INFINITY; lrow[tid] = 0.f;
  }
  float o[ATT_MAX_PER_THREAD];
#pragma unroll
  for (int i = 0; i < ATT_MAX_PER_THREAD; i++) o[i] = 0.f;

  for (uint32_t t0 = lo; t0 < hi; t0 += T) {
    __syncthreads();
    for (uint32_t i = tid; i < T * hd; i += 256) {
      const uint32_t j = i / hd, d = i % hd, t = t0 + j;
      float kk = 0.f, vv = 0.f;
      if (t < hi) {
        const uint64_t src = ((uint64_t)(t % a.capacity) * a.kvh + kv) * hd + d;
        kk = kv_get<E>(a.k, src); vv = kv_get<E>(a.v, src);
      }
      Ks[j * (hd + 1) + d] = kk;
      Vs[j * hd + d] = vv;
    }
    __syncthreads();
    for (uint32_t p = tid; p < TREE_R * T; p += 256) {
      const uint32_t r = p / T, j = p % T, t = t0 + j;
      float sc = -INFINITY;
      if (t < hi && tree_sees(rows[r], t, a.start)) {
        const float *qr = Qs + r * hd, *kr = Ks + j * (hd + 1);
        float dot = 0.f;
        for (uint32_t d = 0; d < hd; d++) dot += qr[d] * kr[d];
        sc = dot * a.scale;
      }
      S[p] = sc;
    }
    __syncthreads();
    for (uint32_t r = wv; r < TREE_R; r += 4) {
      float mx = -INFINITY;
      for (uint32_t j = lane; j < T; j += 64) mx = fmaxf(mx, S[r * T + j]);
      mx = wave_max(mx);
      const float m_old = mrow[r], m_new = fmaxf(m_old, mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;  // no finite score yet: exp(-inf) is 0
      float sum = 0.f;
      for (uint32_t j = lane; j < T; j += 64) {
        const float sv = S[r * T + j];
        const bool sees = t0 + j < hi && tree_sees(rows[r], t0 + j, a.start);
        const float pv = sees ? expf(sv - base) : -1.f;  // -1: not seen, not added below
        S[r * T + j] = pv;
        sum += sees ? pv : 0.f;
      }
      sum = wave_sum(sum);
      if (lane == 0) {
        const float c = m_old == -INFINITY ? (m_new == -INFINITY ? 1.f : 0.f) : expf(m_old - m_new);
        corr[r] = c;
        // before the first finite score l is 0 or NaN (a NaN score), which has to stay
        lrow[r] = (m_old == -INFINITY ? lrow[r] : lrow[r] * c) + sum;
        mrow[r] = m_new;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ATT_MAX_PER_THREAD; i++) {
      const uint32_t e = tid + 256 * i;
      if (e >= TREE_R * hd) break;
      const uint32_t r = e / hd, d = e % hd;
      float acc = o[i] * corr[r];
      const float *pr = S + r * T;
      for (uint32_t j = 0; j < T; j++) acc = pr[j] < 0.f ? acc : acc + pr[j] * Vs[j * hd + d];
      o[i] = acc;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ATT_MAX_PER_THREAD; i++) {
    const uint32_t e = tid + 256 * i;
    if (e >= TREE_R * hd) break;
    const uint32_t r = e / hd, d = e % hd;
    if (r0 + r >= nrows) continue;
    const uint64_t row = row_of(r0 + r);
    if (a.nsplit == 1) {
      a.y[row * hd + d] = rows[r].valid ? o[i] / lrow[r] : 0.f;
    } else {
      float *pp = a.part + ((uint64_t)z * a.nodes * a.heads + row) * (hd + 2);
      if (d == 0) { pp[0] = mrow[r]; pp[1] = rows[r].valid ? lrow[r] : -1.f; }
      pp[2 + d] = o[i];
    }
  }
}

// The splits of a row in order: a negative sum marks padding, a sum of zero a split without keys that
// the row sees (or without a finite score, which adds nothing either). A row always sees itself,
// so sums that are all zero mean scores that were all -inf: 0 / 0, as the formula has it.
__global__ __launch_bounds__(128) void k_attn_tree_join(const float *part, float *y, uint32_t rows, uint32_t hd, uint32_t nsplit) {
  const uint64_t row = blockIdx.x, stride = (uint64_t)rows * (hd + 2);
  const float *p = part + row * (hd + 2);
  float M = -INFINITY;
  for (uint32_t z = 0; z < nsplit; z++) M = fmaxf(M, p[z * stride]);
  const bool pad = p[1] < 0.f;
  float L = 0.f;
  for (uint32_t z = 0; z < nsplit; z++) {
    const float l = p[z * stride + 1];
    if (l != 0.f) L += l * expf(p[z * stride] - M);
  }
  for (uint32_t d = threadIdx.x; d < hd; d += blockDim.x) {
    float acc = 0.f;
    for (uint32_t z = 0; z < nsplit; z++)
      if (p[z * stride + 1] != 0.f) acc += p[z * stride + 2 + d] * expf(p[z * stride] - M);
    y[row * hd + d] = pad ? 0.f : acc / L;
  }
}

static uint32_t tree_first(const TreeAttnArgs &in) { return in.start - std::min(in.start, in.window - 1); }

// LDS of k_attn_tree_any: a tile's keys and values, the queries and the scores.
static size_t tree_any_lds(uint32_t hd, uint32_t T) { return sizeof(float) * ((size_t)T * (2 * hd + 1) + TREE_R * hd + TREE_R * T); }

struct TreePlan { uint32_t T, blocks, nsplit; };
static TreePlan tree_plan(const TreeAttnArgs &in) {
  TreePlan p;
  const uint32_t keys = in.start + in.nodes - tree_first(in), group = in.heads / in.kv_heads;
  p.T = tile_keys(in.hd);
  while (tree_any_lds(in.hd, p.T) > 60000) p.T /= 2;  // with the rows' static LDS below 64 KB
  p.blocks = (in.nodes * group + TREE_R - 1) / TREE_R;
  const uint32_t tiles = (keys + p.T - 1) / p.T, wgs = in.kv_heads * p.blocks;
  p.nsplit = std::max(1u, std::min(tiles, 4 * (uint32_t)device_cu_count() / wgs));
  return p;
}

uint64_t attention_tree_scratch_floats(const TreeAttnArgs &in) {
  if (!in.nodes) return 0;
  const uint32_t n = tree_plan(in).nsplit;
  return n > 1 ? (uint64_t)n * in.nodes * in.heads * (in.hd + 2) : 0;
}

hipError_t attention_tree(hipStream_t s, const TreeAttnArgs &in) {
  if (!in.nodes) return hipSuccess;
  if (!in.kv_heads || in.heads % in.kv_heads || !in.hd || in.hd > 512 || !in.window || in.nodes > WGD_TREE_MAX ||
      in.nodes > in.capacity || in.partial_floats < attention_tree_scratch_floats(in))
    return hipErrorInvalidValue;
  const TreePlan p = tree_plan(in);
  TreeK a;
  a.q = in.q; a.k = in.k; a.v = in.v; a.y = in.y; a.part = in.partial; a.parents = in.parents;
  a.heads = in.heads; a.kvh = in.kv_heads; a.group = in.heads / in.kv_heads; a.hd = in.hd; a.start = in.start;
  a.window = in.window; a.capacity = in.capacity; a.nodes = in.nodes; a.first = tree_first(in); a.nsplit = p.nsplit;
  a.T = p.T; a.scale = in.scale;
  const size_t lds = tree_any_lds(in.hd, p.T);
  const dim3 grid(in.kv_heads, p.blocks, p.nsplit);
  if (in.kv16) hipLaunchKernelGGL(k_attn_tree_any<_Float16>, grid, dim3(256), lds, s, a);
  else hipLaunchKernelGGL(k_attn_tree_any<float>, grid, dim3(256), lds, s, a);
  WGD_HIP(hipGetLastError());
  if (p.nsplit > 1) {
    hipLaunchKernelGGL(k_attn_tree_join, dim3(in.nodes * in.heads), dim3(128), 0, s, (const float *)in.partial, in.y,
                       in.nodes * in.heads, in.hd, p.nsplit);
    WGD_HIP(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace wgd
