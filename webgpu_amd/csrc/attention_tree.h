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
constexpr float TREE_LOG2E = 1.44269504088896340736f;

struct TreeK {
  const float *q; const void *k, *v; float *y, *part; const int32_t *parents;
  uint32_t heads, kvh, group, hd, start, window, capacity, nodes, first;
  // a split's keys are `per` blocks of `unit` (k_attn_tree_any: tiles of T)
  uint32_t nsplit, per, T;
  float scale;
};

// Row r of kv head kv among the rows of all heads, as q and y have them.
__device__ __forceinline__ uint64_t tree_row(const TreeK &a, uint32_t kv, uint32_t r) {
  return (uint64_t)(r / a.group) * a.heads + kv * a.group + r % a.group;
}

// The partial outputs of several splits are [split][row][hd], and from an even float on, 8-byte aligned whatever the
// head dim, (max, sum) pairs [split][row].
__host__ __device__ __forceinline__ uint64_t tree_pairs(uint32_t nsplit, uint64_t rows, uint32_t hd) {
  return (nsplit * rows * hd + 1) / 2 * 2;
}

// What the nodes see of each other: bits[i] is i's path to the root (within the window), len[i] its length and
// up[i] -1, or -2 for padding. Formed by doubling the steps of all nodes at once.
struct TreeLds { uint32_t bits[WGD_TREE_MAX][TREE_WORDS]; int32_t up[WGD_TREE_MAX]; uint32_t len[WGD_TREE_MAX]; };

__device__ __forceinline__ int32_t tree_parent(const int32_t *parents, uint32_t i) {
  const int32_t p = parents[i];
  return p < (int32_t)i && p >= -1 ? p : -2;
}

__device__ __forceinline__ void tree_paths(TreeLds &L, const int32_t *parents, uint32_t nodes, uint32_t window) {
  const uint32_t words = (nodes + 31) / 32, i = threadIdx.x;  // at least WGD_TREE_MAX threads
  const bool mine = i < nodes;
  if (mine) {
    L.up[i] = tree_parent(parents, i);
    for (uint32_t w = 0; w < words; w++) L.bits[i][w] = w == i / 32 ? 1u << (i % 32) : 0u;
  }
  __syncthreads();
  for (uint32_t span = 1; span < nodes; span *= 2) {
    uint32_t b[TREE_WORDS];
    int32_t up = -1;
    const bool more = mine && L.up[i] >= 0;
    if (more) {
      const uint32_t a = (uint32_t)L.up[i];
#pragma unroll
      for (uint32_t w = 0; w < TREE_WORDS; w++) b[w] = w < words ? L.bits[a][w] : 0u;
      up = L.up[a];
    }
    if (!__syncthreads_or(more)) break;
    if (more) {
#pragma unroll
      for (uint32_t w = 0; w < TREE_WORDS; w++)
        if (w < words) L.bits[i][w] |= b[w];
      L.up[i] = up;
    }
    __syncthreads();
  }
  if (mine) {
    uint32_t n = 0;
    for (uint32_t w = 0; w < words; w++) n += __popc(L.bits[i][w]);
    L.len[i] = n;
    // parents have lower numbers: the ones beyond the window are the lowest bits
    for (uint32_t w = 0; n > window; w += L.bits[i][w] == 0)
      if (L.bits[i][w]) { L.bits[i][w] &= L.bits[i][w] - 1; n--; }
  }
  __syncthreads();
}

// The same for up to 64 nodes in one wavefront's registers: lane i holds node i.
struct TreeLanes { uint64_t bits; int32_t up; };
__device__ __forceinline__ TreeLanes tree_lanes(const int32_t *parents, uint32_t nodes) {
  const uint32_t lane = threadIdx.x & 63;
  TreeLanes t = {1ull << lane, lane < nodes ? tree_parent(parents, lane) : -1};
  while (__any(t.up >= 0)) {
    const int from = t.up >= 0 ? t.up : (int)lane;
    const uint64_t b = __shfl(t.bits, from, 64);
    const int32_t u = __shfl(t.up, from, 64);
    t.bits |= b;  // a node at its end reads itself
    t.up = u;
  }
  return t;
}

// What one row sees: its first cached key, whether its node is one, and the nodes (`bits` from the
// lanes, the node's row of TreeLds otherwise).
struct TreeSeen { uint32_t node, begin, valid; uint64_t bits; };
__device__ __forceinline__ TreeSeen tree_seen(const TreeLds &L, uint32_t node, uint32_t start, uint32_t window) {
  const uint32_t end = start + L.len[node];  // its position + 1
  return TreeSeen{node, end - min(end, window), L.up[node] == -1, 0};
}
__device__ __forceinline__ TreeSeen tree_seen(const TreeLanes &t, uint32_t node, uint32_t start, uint32_t window) {
  uint64_t bits = __shfl(t.bits, (int)node, 64);
  uint32_t n = (uint32_t)__popcll(bits);
  const uint32_t end = start + n;
  for (; n > window; n--) bits &= bits - 1;
  return TreeSeen{node, end - min(end, window), __shfl(t.up, (int)node, 64) == -1, bits};
}
// Which of the keys t0 .. t0 + 32 (below hi) the row sees, as bits.
template <bool LANES>
__device__ __forceinline__ uint32_t tree_mask(const TreeLds &L, const TreeSeen &s, uint32_t t0, uint32_t hi, uint32_t start, uint32_t nodes) {
  auto below = [](uint32_t n) { return n >= 32 ? ~0u : (1u << n) - 1; };
  if (!s.valid || t0 >= hi) return 0;
  uint32_t m = 0;
  if (t0 < start) {
    m = below(start - t0);
    if (s.begin > t0) m &= ~below(s.begin - t0);
  }
  if (t0 + 32 > start) {
    auto word = [&](uint32_t w) { return LANES ? (uint32_t)(w < 2 ? s.bits >> (32 * w) : 0) : w < (nodes + 31) / 32 ? L.bits[s.node][w] : 0u; };
    if (t0 < start) {
      m |= word(0) << (start - t0);
    } else {
      const uint32_t j = t0 - start, sh = j % 32;
      m |= word(j / 32) >> sh;
      if (sh) m |= word(j / 32 + 1) << (32 - sh);
    }
  }
  return m & below(hi - t0);
}

__device__ __forceinline__ uint32_t tree_sees(const TreeK &a, const TreeLds &L, const TreeSeen &s, uint32_t t0, uint32_t hi) {
  return a.nodes <= 64 ? tree_mask<true>(L, s, t0, hi, a.start, a.nodes) : tree_mask<false>(L, s, t0, hi, a.start, a.nodes);
}

// Rows r0 .. + 16 of kv head kv over the keys [lo, hi), in tiles of T keys staged in LDS (tree_any_lds()
// of it): f32 products one by one, so any head dim up to 512 does, and a key that a row does not see is never
// multiplied with its weight, so what it holds (NaN too) reaches nothing. The output of the rows, or
// with several splits their partial z. Every thread of the NT calls it.
constexpr uint32_t TREE_R = 16;
__host__ __device__ constexpr size_t tree_any_lds(uint32_t hd, uint32_t T) {
  return sizeof(float) * ((size_t)T * (2 * hd + 1) + 2 * TREE_R * hd + TREE_R * T);
}
// Keys of a tile: at most 64, within 50000 bytes (which with the static LDS stay below 64 KB), but 4 at least.
__host__ __device__ constexpr uint32_t tree_any_tile(uint32_t hd) {
  uint32_t T = 64;
  while (T > 4 && tree_any_lds(hd, T) > 50000) T /= 2;
  return T;
}
template <class E, uint32_t NT>
__device__ __forceinline__ void tree_any(const TreeK &a, const TreeLds &L, float *lds, uint32_t T, uint32_t kv, uint32_t r0,
                                         uint32_t z, uint32_t lo, uint32_t hi) {
  __shared__ uint32_t vis[TREE_R][2];
  __shared__ float mrow[TREE_R], lrow[TREE_R], corr[TREE_R];
  const uint32_t hd = a.hd, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, nrows = a.nodes * a.group;
  float *Ks = lds, *Vs = Ks + T * (hd + 1), *Qs = Vs + T * hd, *O = Qs + TREE_R * hd, *S = O + TREE_R * hd;
  __syncthreads();
  for (uint32_t i = tid; i < TREE_R * hd; i += NT) {
    const uint32_t r = r0 + i / hd;
    Qs[i] = r < nrows ? a.q[tree_row(a, kv, r) * hd + i % hd] : 0.f;
    O[i] = 0.f;
  }
  TreeSeen seen = {0, 0, 0, 0};
  if (tid < TREE_R) {
    if (r0 + tid < nrows) seen = tree_seen(L, (r0 + tid) / a.group, a.start, a.window);
    mrow[tid] = -INFINITY; lrow[tid] = 0.f;
  }
#pragma unroll 1
  for (uint32_t t0 = lo; t0 < hi; t0 += T) {
    __syncthreads();
    if (tid < TREE_R) {
      vis[tid][0] = tree_mask<false>(L, seen, t0, min(hi, t0 + T), a.start, a.nodes);
      vis[tid][1] = T > 32 ? tree_mask<false>(L, seen, t0 + 32, min(hi, t0 + T), a.start, a.nodes) : 0;
    }
#pragma unroll 2
    for (uint32_t i = tid; i < T * hd; i += NT) {
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
#pragma unroll 1
    for (uint32_t p = tid; p < TREE_R * T; p += NT) {
      const uint32_t r = p / T, j = p % T;
      float sc = -INFINITY;
      if (vis[r][j / 32] >> (j % 32) & 1) {
        const float *qr = Qs + r * hd, *kr = Ks + j * (hd + 1);
        float dot = 0.f;
#pragma unroll 8
        for (uint32_t d = 0; d < hd; d++) dot += qr[d] * kr[d];
        sc = dot * (a.scale * TREE_LOG2E);
      }
      S[p] = sc;
    }
    __syncthreads();
    for (uint32_t r = wv; r < TREE_R; r += NT / 64) {
      const uint64_t on = (uint64_t)vis[r][1] << 32 | vis[r][0];
      float mx = -INFINITY;
      for (uint32_t j = lane; j < T; j += 64) mx = fmaxf(mx, S[r * T + j]);
      mx = wave_max(mx);
      const float m_old = mrow[r], m_new = fmaxf(m_old, mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;  // no finite score yet: exp(-inf) is 0
      float sum = 0.f;
      for (uint32_t j = lane; j < T; j += 64) {
        const float pv = on >> j & 1 ? exp2f(S[r * T + j] - base) : -1.f;  // -1: not seen, not added below
        S[r * T + j] = pv;
        sum += on >> j & 1 ? pv : 0.f;
      }
      sum = wave_sum(sum);
      if (lane == 0) {
        // before the first finite score the sum is 0 or NaN (a NaN score), which has to stay
        const float f = m_old == -INFINITY ? 1.f : exp2f(m_old - m_new);
        corr[r] = f;
        lrow[r] = lrow[r] * f + sum;
        mrow[r] = m_new;
      }
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = tid; i < TREE_R * hd; i += NT) {
      const uint32_t r = i / hd, d = i % hd;
      float acc = O[i] * corr[r];
      const float *pr = S + r * T;
#pragma unroll 8
      for (uint32_t j = 0; j < T; j++) acc = pr[j] < 0.f ? acc : acc + pr[j] * Vs[j * hd + d];
      O[i] = acc;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (uint32_t i = tid; i < TREE_R * hd; i += NT) {
    const uint32_t r = i / hd, d = i % hd;
    if (r0 + r >= nrows) continue;
    const uint64_t row = tree_row(a, kv, r0 + r), all = (uint64_t)a.nodes * a.heads, at = z * all + row;
    const bool pad = L.up[(r0 + r) / a.group] != -1;
    if (a.nsplit == 1) {
      a.y[row * hd + d] = pad ? 0.f : O[i] / lrow[r];
    } else {
      a.part[at * hd + d] = O[i];
      if (d == 0) *(float2 *)(a.part + tree_pairs(a.nsplit, all, hd) + 2 * at) = make_float2(mrow[r], pad ? -1.f : lrow[r]);
    }
  }
}

template <class E>
__global__ __launch_bounds__(256) void k_attn_tree_any(TreeK a) {
  extern __shared__ float lds[];
  __shared__ TreeLds L;
  const uint32_t z = blockIdx.z, end = a.start + a.nodes, chunk = a.per * a.T;
  const uint32_t lo = a.first + min(z * chunk, end - a.first), hi = lo + min(chunk, end - lo);
  tree_paths(L, a.parents, a.nodes, a.window);
  tree_any<E, 256>(a, L, lds, a.T, blockIdx.x, blockIdx.y * TREE_R, z, lo, hi);
}

// ------------------------------------------------------------------ head dims up to 256, multiples of 8
//
// A wavefront holds a tile of 16 rows of one kv head as matrix operands and walks over its keys in
// blocks of 16 NB, read straight from the ring into registers: no barrier until the end. The
// wavefronts of a workgroup are `rw` groups of rows times key slices (block b of the workgroup's range
// belongs to slice b % slices); the slices merge in LDS, the key ranges of workgroups in
// k_attn_tree_join. Scores come out transposed, S^T = K Q^T: lane (g, c) = (lane / 16, lane % 16)
// holds keys 4 g .. + 4 of row c, whose probabilities are, in the same lane, operand of
// O^T += V^T P^T.
//   f16 rings (v_mfma_f32_16x16x32_f16): K and V are operands as they are, exact. The queries (times
//     scale log2 e) are split into f16 hi + lo with a power of two per row, the probabilities with a
//     factor of 2^11: two products of f16 in place of one of f32, whose rate is an eighth. Each is off by 2^-22 of
//     itself (f32: 2^-24) and by half of f16's least step, 2^-25: below 2^-39 of a row's largest query entry, which
//     lies in [2^14, 2^15), and 2^-36 of its largest weight, 2^11 at least. A weight below 2^-36 of the largest is in the
//     sum, which has them in f32, and not in the outputs: n such keys are n 2^-36 of the largest value at
//     most, where f32 sums of n terms may be off by n 2^-24. Lane (g, c) loads VE values d = VE c of
//     its eight keys and picks the d-th halves of the eight with v_perm: output tile (x, e) is
//     the dims 16 VE x + VE m + e.
//   f32 rings (v_mfma_f32_16x16x4_f32): f32 products and sums.
// The maximum that weights refer to follows lazily: it moves, and sums and outputs with it, only when a score
// lies TREE_LAG above it (in powers of two; weights stay below 2^15, within f16). A row's sum stays
// spread over its four lanes until the end.
// Masks are formed only for blocks that reach into the drafted nodes, past the end or into the
// keys that a window hides from deeper nodes. A masked score's weight is exactly 0; a value that is not
// finite would turn it into NaN, and a split key or query could turn an infinity into NaN: a workgroup
// that ends with anything not finite forms its rows again with tree_any.
// Latency bounds it: a wavefront is 40% of its time at waits for loads and 40% at waits to issue, two to a SIMD. 48
// nodes, 32 heads on 16 of 128, 1071 f32 keys: 18.7 us and 4 to join (the products alone 4.9), 64 nodes over 15000 f32 keys
// of 8 heads 178 us, 88 TFLOP/s of the 153 that f32 matrix products reach. With two tiles a wavefront, which spill, the latter
// takes 163 but shorter rings more.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr float TREE_LAG = 4.f, TREE_BIAS = 11.f;

template <class E> constexpr uint32_t tree_nb() { return sizeof(E) == 2 ? 2 : 1; }
template <uint32_t HD, class E> constexpr uint32_t tree_ve() { return sizeof(E) == 2 && HD >= 128 ? 8 : 4; }

// Threads of a workgroup: as many as their registers allow.
template <uint32_t HD>
constexpr uint32_t tree_threads() { return HD <= 128 ? 512 : 256; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The state of RT tiles of rows: a row's reference maximum m (in powers of two), the lane's share of its sum of
// weights, and outputs: tile (x, e) of o holds the dims 16 VE x + VE m + e in its rows m.
template <uint32_t HD, uint32_t RT, uint32_t NB, uint32_t VE_>
struct TreeRows {
  static constexpr uint32_t KEYS = 16 * NB, VE = VE_, NX = HD / (16 * VE);
  f32x4 o[RT][NX][VE];
  float m[RT], l[RT];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
      m[rt] = -INFINITY; l[rt] = 0.f;
#pragma unroll
      for (uint32_t x = 0; x < NX; x++)
#pragma unroll
        for (uint32_t e = 0; e < VE; e++) o[rt][x][e] = f32x4{0, 0, 0, 0};
    }
  }

  // The weights of a block of keys from its scores over qs (s, in lane order): 2^(s qs + TREE_BIAS - m), with m moved
  // where it lags. `sees`: the keys that the row sees, as bits (all where `masked` is off).
  __device__ __forceinline__ void weigh(uint32_t rt, f32x4 (&s)[NB], float qs, bool masked, uint32_t sees) {
    const uint32_t g = (threadIdx.x & 63) >> 4;
    if (masked) {
#pragma unroll
      for (uint32_t b = 0; b < NB; b++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[b][r] = sees >> (16 * b + 4 * g + r) & 1 ? s[b][r] : -INFINITY;
    }
    const float ref = TREE_BIAS - (m[rt] == -INFINITY ? 0.f : m[rt]);
    f32x4 p[NB];
    float mx = -INFINITY;
#pragma unroll
    for (uint32_t b = 0; b < NB; b++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[b][r] = __builtin_fmaf(s[b][r], qs, ref);
        mx = fmaxf(mx, p[b][r]);
      }
    if (__any(mx > (m[rt] == -INFINITY ? -INFINITY : TREE_BIAS + TREE_LAG))) {
      mx -= ref;
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float to = fmaxf(m[rt], mx);
      // a row without a score so far has nothing to scale but NaN, which stays
      const float f = m[rt] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[rt] - to);
      m[rt] = to;
      l[rt] *= f;
#pragma unroll
      for (uint32_t x = 0; x < NX; x++)
#pragma unroll
        for (uint32_t e = 0; e < VE; e++) o[rt][x][e] *= f;
      const float now = TREE_BIAS - (to == -INFINITY ? 0.f : to);
#pragma unroll
      for (uint32_t b = 0; b < NB; b++)
#pragma unroll
        for (int r = 0; r < 4; r++) p[b][r] = __builtin_fmaf(s[b][r], qs, now);
    }
#pragma unroll
    for (uint32_t b = 0; b < NB; b++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        s[b][r] = __builtin_amdgcn_exp2f(p[b][r]);
        l[rt] += s[b][r];
      }
  }

  __device__ __forceinline__ bool finite() const {
    float t = 0.f;  // stays 0 unless something is not finite
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
      t += 0.f * l[rt];
#pragma unroll
      for (uint32_t x = 0; x < NX; x++)
#pragma unroll
        for (uint32_t e = 0; e < VE; e++)
#pragma unroll
          for (int r = 0; r < 4; r++) t += 0.f * o[rt][x][e][r];
    }
    return t == 0.f;
  }
};

// Weights of two blocks of 16 keys as f16 hi and lo operands.
__device__ __forceinline__ void tree_split(const f32x4 (&p)[2], f16x8 &hi, f16x8 &lo) {
  u32x4 h, l;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const f32x2 v = {p[e / 2][2 * (e % 2)], p[e / 2][2 * (e % 2) + 1]};
    h[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    f32x2 rest;  // v - hi, a half of h[e] each
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rest.x) : "v"(h[e]), "v"(v.x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rest.y) : "v"(h[e]), "v"(v.y));
    l[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, f16x2));
  }
  hi = __builtin_bit_cast(f16x8, h);
  lo = __builtin_bit_cast(f16x8, l);
}

// A row's query times scale log2 e as f16 operands hi and lo of KT steps of 32 dims, over the power of two returned,
// which puts its largest magnitude into [2^14, 2^15). Zero past hd, and where ok is off.
template <uint32_t KT>
__device__ __forceinline__ float tree_query(const float *q, uint32_t hd, float f, bool ok, u32x4 (&hi)[KT], u32x4 (&lo)[KT]) {
  const uint32_t g = (threadIdx.x & 63) >> 4;
  auto four = [&](uint32_t d) { return ok && d < hd ? *(const f32x4 *)(q + d) : f32x4{0, 0, 0, 0}; };
  float v[KT][8];
  uint32_t mx = 0;
#pragma unroll
  for (uint32_t t = 0; t < KT; t++) {
    const f32x4 x = four(32 * t + 8 * g), y = four(32 * t + 8 * g + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[t][e] = x[e] * f;
      v[t][4 + e] = y[e] * f;
      mx = max(mx, max(__float_as_uint(v[t][e]) & 0x7FFFFFFFu, __float_as_uint(v[t][4 + e]) & 0x7FFFFFFFu));
    }
  }
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
  const uint32_t ex = min(max(mx >> 23, 16u), 254u);  // both powers stay normal
  const float inv = __uint_as_float((254u + 14u - ex) << 23);
#pragma unroll
  for (uint32_t t = 0; t < KT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint32_t h, l;
      split2(v[t][2 * e] * inv, v[t][2 * e + 1] * inv, h, l);
      hi[t][e] = h;
      lo[t][e] = l;
    }
  return __uint_as_float((ex - 14u) << 23);
}

// FULL: the head dim is HD itself.
template <uint32_t HD, class E, bool FULL>
struct TreeWave : TreeRows<HD, 1, tree_nb<E>(), tree_ve<HD, E>()> {
  static constexpr bool HALF = sizeof(E) == 2;
  static constexpr uint32_t NB = tree_nb<E>();
  typedef TreeRows<HD, 1, NB, tree_ve<HD, E>()> Rows;
  using Rows::KEYS, Rows::VE, Rows::NX, Rows::o;
  static constexpr uint32_t KT = HALF ? HD / 32 : HD / 16;  // 16-byte pieces of a key per lane
  static constexpr uint32_t VK = 4 * NB;                    // keys per lane of a block of V
  typedef uint32_t vpiece __attribute__((ext_vector_type(VE * sizeof(E) / 4)));

  u32x4 qh[KT], ql[KT];  // f16 hi and lo; f32: qh alone
  float qs;              // the power of two taken out of the row's query
  // the ring: this kv head's K and V, bytes between rows, slots; the end of the keys and the slot of the block's first
  const uint8_t *k, *v;
  uint64_t rowb;
  uint32_t cap, hi, base;
  // lane offsets: pieces of a key row, and of the value rows. Pieces past a head dim below HD read its
  // last one: the query is zero there, and such outputs are not written.
  uint32_t k_piece[KT], v_piece[NX], k_row, v_row;
  u32x4 kr[NB][KT];

  // Byte offset of key t + off of a block with t in slot `base`. Keys past the end read the last one: off stays
  // below cap, so there is one wrap at most.
  __device__ __forceinline__ uint64_t at(uint32_t t, uint32_t off) const {
    const uint32_t s = base + min(off, hi - 1 - t);
    return (uint64_t)min(s, s - cap) * rowb;  // s - cap wraps to a large number below cap
  }
  __device__ __forceinline__ bool whole(uint32_t t) const { return base + KEYS <= cap && t + KEYS <= hi; }
  __device__ __forceinline__ void load_k(uint32_t t) {
    const uint32_t c = threadIdx.x & 15;
    if (whole(t)) {
#pragma unroll
      for (uint32_t b = 0; b < NB; b++) {
        const uint8_t *row = k + (uint64_t)(base + 16 * b) * rowb;
#pragma unroll
        for (uint32_t u = 0; u < KT; u++) kr[b][u] = *(const u32x4 *)(row + (k_row + k_piece[u]));
      }
    } else {
#pragma unroll
      for (uint32_t b = 0; b < NB; b++) {
        const uint8_t *row = k + at(t, 16 * b + c);
#pragma unroll
        for (uint32_t u = 0; u < KT; u++) kr[b][u] = *(const u32x4 *)(row + k_piece[u]);
      }
    }
  }
  // The first block's keys, asked for before anything else.
  __device__ __forceinline__ void begin(const TreeK &a, uint32_t kv, uint32_t t0, uint32_t end) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15, bytes = (FULL ? HD : a.hd) * sizeof(E);
    k = (const uint8_t *)a.k + (uint64_t)kv * bytes;
    v = (const uint8_t *)a.v + (uint64_t)kv * bytes;
    rowb = (uint64_t)a.kvh * bytes;  // below 2^27 (tree_plan)
    cap = a.capacity; hi = end;
    k_row = c * (uint32_t)rowb;
    v_row = 4 * g * (uint32_t)rowb;
#pragma unroll
    for (uint32_t u = 0; u < KT; u++) k_piece[u] = FULL ? 64 * u + 16 * g : min(64 * u + 16 * g, bytes - 16);
#pragma unroll
    for (uint32_t x = 0; x < NX; x++) {
      v_piece[x] = (16 * x + c) * (uint32_t)sizeof(vpiece);
      if (!FULL) v_piece[x] = min(v_piece[x], bytes - (uint32_t)sizeof(vpiece));
    }
    if (t0 >= hi) return;
    base = t0 % cap;
    load_k(t0);
  }

  // The row's query times scale log2 e as operand.
  __device__ __forceinline__ void load_q(const TreeK &a, const float *q, bool ok) {
    const float f = a.scale * TREE_LOG2E;
    if constexpr (!HALF) {
      const uint32_t g = (threadIdx.x & 63) >> 4;
#pragma unroll
      for (uint32_t t = 0; t < KT; t++) {
        const f32x4 x = ok && (FULL || 16 * t + 4 * g < a.hd) ? *(const f32x4 *)(q + 16 * t + 4 * g) : f32x4{0, 0, 0, 0};
        qh[t] = __builtin_bit_cast(u32x4, f32x4{x.x * f, x.y * f, x.z * f, x.w * f});
      }
      qs = 1.f;
    } else {
      qs = tree_query<KT>(q, FULL ? HD : a.hd, f, ok, qh, ql);
    }
  }

  // Keys [t0, ..) in steps of `step` up to hi.
  __device__ __forceinline__ void walk(const TreeK &a, const TreeLds &L, const TreeSeen &seen, uint32_t t0, uint32_t step,
                                       uint32_t masked_below) {
    const uint32_t g = (threadIdx.x & 63) >> 4;
    this->clear();
    for (; t0 < hi; t0 += step) {
      vpiece vr[VK][NX];
      if (whole(t0)) {
#pragma unroll
        for (uint32_t j = 0; j < VK; j++) {
          const uint8_t *row = v + (uint64_t)(base + 16 * (j / 4) + j % 4) * rowb;
#pragma unroll
          for (uint32_t x = 0; x < NX; x++) vr[j][x] = *(const vpiece *)(row + (v_row + v_piece[x]));
        }
      } else {
#pragma unroll
        for (uint32_t j = 0; j < VK; j++) {
          const uint8_t *row = v + at(t0, 16 * (j / 4) + 4 * g + j % 4);
#pragma unroll
          for (uint32_t x = 0; x < NX; x++) vr[j][x] = *(const vpiece *)(row + v_piece[x]);
        }
      }
      // ---- scores
      f32x4 s[NB];
#pragma unroll
      for (uint32_t b = 0; b < NB; b++) {
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t t = 0; t < KT; t++) {
          if constexpr (HALF) {
            const f16x8 kf = __builtin_bit_cast(f16x8, kr[b][t]);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, __builtin_bit_cast(f16x8, qh[t]), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, __builtin_bit_cast(f16x8, ql[t]), acc, 0, 0, 0);
          } else {
            const f32x4 kf = __builtin_bit_cast(f32x4, kr[b][t]), qf = __builtin_bit_cast(f32x4, qh[t]);
#pragma unroll
            for (int u = 0; u < 4; u++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[u], qf[u], acc, 0, 0, 0);
          }
        }
        s[b] = acc;
      }
      base += step;
      if (base >= cap) base %= cap;
      if (t0 + step < hi) load_k(t0 + step);
      // ---- weights, in place of the scores
      const bool masked = t0 + KEYS > min(hi, a.start) || t0 < masked_below;
      this->weigh(0, s, qs, masked, masked ? tree_sees(a, L, seen, t0, hi) : 0);
      // ---- values
      if constexpr (HALF) {
        f16x8 ph, pl;
        tree_split(s, ph, pl);
#pragma unroll
        for (uint32_t x = 0; x < NX; x++)
#pragma unroll
          for (uint32_t e = 0; e < VE; e++) {
            u32x4 f;  // half e of the eight keys
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
              f[i] = __builtin_amdgcn_perm(vr[2 * i + 1][x][e / 2], vr[2 * i][x][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
            const f16x8 vf = __builtin_bit_cast(f16x8, f);
            o[0][x][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o[0][x][e], 0, 0, 0);
            o[0][x][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[0][x][e], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
#pragma unroll
          for (uint32_t x = 0; x < NX; x++)
#pragma unroll
            for (uint32_t e = 0; e < VE; e++)
              o[0][x][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[i][x][e]), s[0][i], o[0][x][e], 0, 0, 0);
      }
    }
  }
};

struct TreeGrid { uint32_t rw, per; };  // row groups of a workgroup; key blocks per split

template <uint32_t HD, uint32_t RT>
constexpr size_t tree_wave_lds() { return sizeof(float) * RT * 16 * (HD + 4 + 2); }

// A workgroup's part of the work: wavefront w has the rows wrow .. + 16 RT and the key blocks of `slice`, of the
// keys [lo, hi); keys below masked_below are hidden from some nodes by the window.
struct TreePart {
  uint32_t kv, z, nrows, wrow, slice, slices, lo, hi, masked_below;
  bool masks;
};
__device__ __forceinline__ TreePart tree_part(const TreeK &a, const TreeGrid &gr, uint32_t RT, uint32_t unit) {
  TreePart p;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), end = a.start + a.nodes;
  p.kv = blockIdx.x; p.z = blockIdx.z; p.nrows = a.nodes * a.group;
  p.slices = (blockDim.x >> 6) / gr.rw; p.slice = w / gr.rw;
  p.wrow = (blockIdx.y * gr.rw + w % gr.rw) * RT * 16;
  p.lo = a.first + min(p.z * gr.per * unit, end - a.first);
  p.hi = p.lo + min(gr.per * unit, end - p.lo);
  p.masked_below = end <= a.window ? 0 : a.first + a.nodes;
  p.masks = p.hi > a.start || p.lo < p.masked_below;
  return p;
}

// The rows of this lane's wavefront, and what they see where the keys need masks.
template <uint32_t RT>
__device__ __forceinline__ void tree_rows(const TreeK &a, TreeLds &L, const TreePart &p, uint32_t (&row)[RT], TreeSeen (&seen)[RT]) {
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
    row[rt] = min(p.wrow + 16 * rt + (threadIdx.x & 15), p.nrows - 1);
    seen[rt] = TreeSeen{row[rt] / a.group, 0, 1, 0};
  }
  if (!p.masks) return;
  if (a.nodes <= 64) {
    const TreeLanes t = tree_lanes(a.parents, a.nodes);
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) seen[rt] = tree_seen(t, seen[rt].node, a.start, a.window);
  } else {
    tree_paths(L, a.parents, a.nodes, a.window);
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) seen[rt] = tree_seen(L, seen[rt].node, a.start, a.window);
  }
}

// The end of a workgroup: the slices of its wavefronts merge in LDS, and the rows go to y, or with several splits
// to their partials. With anything not finite the rows are formed again. Every thread calls it; the LDS
// at `lds` is no longer read by anyone.
template <uint32_t HD, class E, uint32_t RT, uint32_t NT, class Rows>
__device__ __forceinline__ void tree_end(const TreeK &a, const TreeGrid &gr, TreeLds &L, float *lds, const TreePart &p, const Rows &s,
                                         const TreeSeen (&seen)[RT]) {
  constexpr uint32_t VE = Rows::VE, NX = Rows::NX, OS = HD + 4, WS = RT * 16 * (OS + 2);
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  if (__syncthreads_or(!s.finite())) {
    if (!p.masks || a.nodes <= 64) tree_paths(L, a.parents, a.nodes, a.window);
    for (uint32_t i = 0; i < gr.rw * RT; i++) {
      const uint32_t r0 = (blockIdx.y * gr.rw * RT + i) * 16;
      if (r0 < p.nrows) tree_any<E, NT>(a, L, lds, tree_any_tile(HD), p.kv, r0, p.z, p.lo, p.hi);
    }
    return;
  }
  // ---- to LDS: [row] max, sum; [row][HD]
  float *mine = lds + (tid >> 6) * WS;
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
    float l = s.l[rt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) { mine[2 * (16 * rt + c)] = s.m[rt]; mine[2 * (16 * rt + c) + 1] = seen[rt].valid ? l : -1.f; }
    float *row = mine + RT * 32 + (16 * rt + c) * OS;
#pragma unroll
    for (uint32_t x = 0; x < NX; x++) {
      if constexpr (VE == 1) {
        *(f32x4 *)(row + 16 * x + 4 * g) = s.o[rt][x][0];
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (uint32_t e = 0; e < VE; e += 4)
            *(f32x4 *)(row + 16 * VE * x + 4 * VE * g + VE * r + e) =
                f32x4{s.o[rt][x][e][r], s.o[rt][x][e + 1][r], s.o[rt][x][e + 2][r], s.o[rt][x][e + 3][r]};
      }
    }
  }
  __syncthreads();
  // ---- the slices in order, eight dims of a row per thread
  const uint64_t rows = (uint64_t)a.nodes * a.heads;
  for (uint32_t i = tid; i < gr.rw * RT * 16 * (HD / 8); i += NT) {
    const uint32_t d = i % (HD / 8) * 8, lr = i / (HD / 8) % (RT * 16), rg = i / (HD / 8) / (RT * 16);
    const uint32_t r = (blockIdx.y * gr.rw + rg) * RT * 16 + lr;
    if (r >= p.nrows || d >= a.hd) continue;
    float M = -INFINITY, l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t u = 0; u < p.slices; u++) M = fmaxf(M, lds[(u * gr.rw + rg) * WS + 2 * lr]);
    const bool pad = lds[rg * WS + 2 * lr + 1] < 0.f;
    for (uint32_t u = 0; u < p.slices; u++) {
      const float *at = lds + (u * gr.rw + rg) * WS;
      if (at[2 * lr + 1] == 0.f) continue;  // nothing seen
      const float f = at[2 * lr] == M ? 1.f : __builtin_amdgcn_exp2f(at[2 * lr] - M);
      l += at[2 * lr + 1] * f;
      const f32x4 x0 = *(const f32x4 *)(at + RT * 32 + lr * OS + d), x1 = *(const f32x4 *)(at + RT * 32 + lr * OS + d + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) { y[e] += x0[e] * f; y[4 + e] += x1[e] * f; }
    }
    const uint64_t row = tree_row(a, p.kv, r);
    float *to = a.y + row * a.hd + d;
    float inv = 1.f;
    if (a.nsplit > 1) {
      to = a.part + ((uint64_t)p.z * rows + row) * a.hd + d;
      if (d == 0) *(float2 *)(a.part + tree_pairs(a.nsplit, rows, a.hd) + 2 * ((uint64_t)p.z * rows + row)) = make_float2(M - TREE_BIAS, pad ? -1.f : l);
    } else {
      inv = 1.f / l;
    }
    const bool zero = pad && a.nsplit == 1;
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      *(f32x4 *)(to + e) = zero ? f32x4{0, 0, 0, 0} : f32x4{y[e] * inv, y[e + 1] * inv, y[e + 2] * inv, y[e + 3] * inv};
  }
}

template <uint32_t HD, class E, bool FULL>
__global__ __launch_bounds__((tree_threads<HD>())) void k_attn_tree(TreeK a, TreeGrid gr) {
  typedef TreeWave<HD, E, FULL> Wave;
  extern __shared__ float lds[];
  __shared__ TreeLds L;
  const TreePart p = tree_part(a, gr, 1, Wave::KEYS);
  const uint32_t from = p.lo + p.slice * Wave::KEYS;
  Wave s;
  s.begin(a, p.kv, from, p.wrow < p.nrows ? p.hi : 0);
  uint32_t row[1];
  TreeSeen seen[1];
  tree_rows<1>(a, L, p, row, seen);
  s.load_q(a, a.q + tree_row(a, p.kv, row[0]) * a.hd, p.wrow + (threadIdx.x & 15) < p.nrows);
  s.walk(a, L, seen[0], from, p.slices * Wave::KEYS, p.masked_below);
  tree_end<HD, E, 1, tree_threads<HD>()>(a, gr, L, lds, p, s, seen);
}

// ------------------------------------------------------------------ many rows: keys staged in LDS
//
// Where four or more wavefronts have rows of a kv head, each reading the keys from the caches for itself (as
// k_attn_tree's do) is what bounds them: 64 bytes a cycle and CU. Here the workgroup's eight wavefronts load a
// stage of SK keys into LDS once, straight from memory (no registers), while they work on the one before; a
// wavefront's blocks of 32 keys are its slice's. K rows and V rows lie in 16-byte chunks; chunk i of key k
// at place i ^ swizzle(k), so that the 16 keys of a K operand, and the 16-bit transposing reads that make V
// operands (4 keys of one dim per lane), meet all banks evenly. 64 nodes, 32 heads on 8 of 128, 31000 keys: 75 us (k_attn_tree
// 158), 433 TFLOP/s counted once, twice that with the split operands. Matrix products take 36% of the cycles and the issue of
// vector instructions 39%; a wavefront is at waits for LDS, loads and the others of its stage 37% of its life, two to a SIMD.
// Two V operands at LDS addresses `at`: dims in transposing reads of keys 0 .. 4 and, OFF bytes on, 16 .. 20 of each lane
// group. The builtin of this read waits for every load from memory into LDS that is under way, the next
// stage's too, so it is written here with its own wait.
template <uint32_t OFF>
__device__ __forceinline__ void tree_read_values(const uint32_t (&at)[2], u32x4 (&v)[2]) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  u32x2 a, b, c, d;
  asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
               "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d) : "v"(at[0]), "v"(at[1]), "i"(OFF) : "memory");
  v[0] = u32x4{a.x, a.y, b.x, b.y};
  v[1] = u32x4{c.x, c.y, d.x, d.y};
}

template <uint32_t HD, uint32_t RT>
struct TreeStaged : TreeRows<HD, RT, 2, 1> {
  typedef TreeRows<HD, RT, 2, 1> Rows;
  using Rows::NX, Rows::o;
  static constexpr uint32_t KT = HD / 32, CH = HD / 8, ROW = 2 * HD;  // K steps; chunks and bytes of a key
  static constexpr uint32_t VB = 2;  // V operands read at a time

  static __device__ __forceinline__ uint32_t k_swizzle(uint32_t key) { return CH >= 16 ? key & 15 : key >> 1 & 7; }
  static __device__ __forceinline__ uint32_t v_swizzle(uint32_t key) { return CH >= 16 ? 2 * key & 15 : 2 * (key >> 1) & 7; }

  u32x4 qh[RT][KT], ql[RT][KT];
  float qs[RT];

  // A block of 32 keys: its K and V rows in LDS, the first key t0; keys end at hi.
  __device__ __forceinline__ void block(const TreeK &a, const TreeLds &L, const TreeSeen (&seen)[RT], const uint8_t *K, const uint8_t *V,
                                        uint32_t t0, uint32_t hi, uint32_t masked_below) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    f32x4 s[RT][2];
#pragma unroll
    for (uint32_t b = 0; b < 2; b++) {
#pragma unroll
      for (uint32_t rt = 0; rt < RT; rt++) s[rt][b] = f32x4{0, 0, 0, 0};
      f16x8 kf[KT];  // read together, ahead of the products
#pragma unroll
      for (uint32_t t = 0; t < KT; t++) kf[t] = *(const f16x8 *)(K + (16 * b + c) * ROW + ((4 * t + g) ^ k_swizzle(c)) * 16);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (uint32_t t = 0; t < KT; t++)
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) {
          s[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t], __builtin_bit_cast(f16x8, qh[rt][t]), s[rt][b], 0, 0, 0);
          s[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t], __builtin_bit_cast(f16x8, ql[rt][t]), s[rt][b], 0, 0, 0);
        }
    }
    const bool masked = t0 + 32 > min(hi, a.start) || t0 < masked_below;
    f16x8 ph[RT], pl[RT];
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
      this->weigh(rt, s[rt], qs[rt], masked, masked ? tree_sees(a, L, seen[rt], t0, hi) : 0);
      tree_split(s[rt], ph[rt], pl[rt]);
    }
    // lane (g, i) reads dims 4 (i % 4) .. + 4 of key 4 g + i / 4 and receives dim i of keys 4 g .. + 4
    const uint32_t key = 4 * g + c / 4;
    const uint8_t *v0 = V + key * ROW + (c & 1) * 8;
    const uint32_t swz = v_swizzle(key);
#pragma unroll
    for (uint32_t x0 = 0; x0 < NX; x0 += VB) {
      uint32_t at[VB];
#pragma unroll
      for (uint32_t x = 0; x < VB; x++)
        at[x] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)(v0 + ((2 * (x0 + x) + (c >> 1 & 1)) ^ swz) * 16);
      u32x4 vf[VB];
      tree_read_values<16 * ROW>(at, vf);
#pragma unroll
      for (uint32_t x = 0; x < VB; x++)
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) {
          o[rt][x0 + x][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, vf[x]), ph[rt], o[rt][x0 + x][0], 0, 0, 0);
          o[rt][x0 + x][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, vf[x]), pl[rt], o[rt][x0 + x][0], 0, 0, 0);
        }
    }
  }
};

constexpr uint32_t TREE_STAGED_NT = 512;

template <uint32_t HD, uint32_t RT, uint32_t SK>
__global__ __launch_bounds__(TREE_STAGED_NT) void k_attn_tree_staged(TreeK a, TreeGrid gr) {
  typedef TreeStaged<HD, RT> Wave;
  constexpr uint32_t ROW = Wave::ROW, CH = Wave::CH;
  extern __shared__ float lds[];
  __shared__ TreeLds L;
  const TreePart p = tree_part(a, gr, RT, 32);
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6), cap = a.capacity;
  uint8_t *stages = (uint8_t *)lds;
  const uint64_t rowb = (uint64_t)a.kvh * ROW, head = (uint64_t)p.kv * ROW;
  const uint8_t *k = (const uint8_t *)a.k + head, *v = (const uint8_t *)a.v + head;
  // Keys t0 .. + SK (t0 in slot base) into stage s, 64 chunks per wavefront and step; keys past the end read the last one.
  // A step of all wavefronts is STEP keys on, a multiple of the swizzles' period: lane offsets are the same for all.
  constexpr uint32_t STEP = TREE_STAGED_NT / CH;
  static_assert(STEP % 16 == 0, "the swizzles repeat after 16 keys");
  const uint32_t key0 = tid / CH, k_place = (tid % CH ^ Wave::k_swizzle(key0)) * 16, v_place = (tid % CH ^ Wave::v_swizzle(key0)) * 16;
  const uint32_t off = key0 * (uint32_t)rowb, k_off = off + k_place, v_off = off + v_place;  // below 2^32 (tree_plan)
  uint32_t base = p.lo % cap;
  auto load = [&](uint32_t t0, uint32_t s) {
    uint8_t *K = stages + s * 2 * SK * ROW + 1024 * w, *V = K + SK * ROW;
    auto put = [](const uint8_t *from, uint8_t *to) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    };
    if (base + SK <= cap && t0 + SK <= p.hi) {
#pragma unroll
      for (uint32_t n = 0; n < SK / STEP; n++) {
        const uint64_t first = (uint64_t)(base + n * STEP) * rowb;
        put(k + first + k_off, K + n * STEP * ROW);
        put(v + first + v_off, V + n * STEP * ROW);
      }
    } else {
#pragma unroll 1
      for (uint32_t n = 0; n < SK / STEP; n++) {
        const uint32_t at = base + min(key0 + n * STEP, p.hi - 1 - t0);
        const uint64_t row = (uint64_t)min(at, at - cap) * rowb;
        put(k + row + k_place, K + n * STEP * ROW);
        put(v + row + v_place, V + n * STEP * ROW);
      }
    }
    base += SK;
    if (base >= cap) base %= cap;
  };
  if (p.lo < p.hi) load(p.lo, 0);
  uint32_t row[RT];
  TreeSeen seen[RT];
  tree_rows<RT>(a, L, p, row, seen);
  Wave s;
  s.clear();
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++)
    s.qs[rt] = tree_query<Wave::KT>(a.q + tree_row(a, p.kv, row[rt]) * HD, HD, a.scale * TREE_LOG2E,
                                    p.wrow + 16 * rt + (tid & 15) < p.nrows, s.qh[rt], s.ql[rt]);
  uint32_t stage = 0;
  for (uint32_t t0 = p.lo; t0 < p.hi; t0 += SK, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's loads into the stage
    __syncthreads();                                   // everyone's; and the other stage is no longer read
    if (t0 + SK < p.hi) load(t0 + SK, stage ^ 1);
    const uint8_t *K = stages + stage * 2 * SK * ROW, *V = K + SK * ROW;
    if (p.wrow < p.nrows)
      for (uint32_t b = p.slice; b < SK / 32 && t0 + 32 * b < p.hi; b += p.slices)
        s.block(a, L, seen, K + 32 * b * ROW, V + 32 * b * ROW, t0 + 32 * b, p.hi, p.masked_below);
  }
  tree_end<HD, _Float16, RT, TREE_STAGED_NT>(a, gr, L, lds, p, s, seen);
}

// The splits of a row in order, of partial outputs and (max, sum) pairs (tree_pairs), maxima in powers of
// two. A sum of zero is a split without keys that the row sees (or without a finite score, which adds
// nothing either); the last split knows padding, by a negative sum. A row always sees itself, so sums
// that are all zero mean scores that were all -inf: 0 / 0, as the formula has it.
// A wavefront per row: the splits' weights go over its lanes and LDS, then (VEC: hd a power of two of 4 to 256) lane groups
// of hd / 4 (at most 64) lanes take every (64 / group)-th split, 16 bytes a lane and eight loads ahead.
constexpr uint32_t TREE_SPLITS = 256;
template <bool VEC>
__global__ __launch_bounds__(256) void k_attn_tree_join(const float *part, float *y, uint32_t rows, uint32_t hd, uint32_t nsplit) {
  __shared__ float wz[4][TREE_SPLITS];
  const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const uint64_t row = min(blockIdx.x * 4 + wv, rows - 1);
  const float2 *ml = (const float2 *)(part + tree_pairs(nsplit, rows, hd)) + row;
  float2 s[TREE_SPLITS / 64];
  float M = -INFINITY;
#pragma unroll
  for (uint32_t u = 0; u < TREE_SPLITS / 64; u++) {
    const uint32_t z = 64 * u + lane;
    s[u] = z < nsplit ? ml[(uint64_t)z * rows] : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, s[u].x);
  }
  const bool pad = ml[(uint64_t)(nsplit - 1) * rows].y < 0.f;
  M = wave_max(M);
  float sum = 0.f;
#pragma unroll
  for (uint32_t u = 0; u < TREE_SPLITS / 64; u++) {
    const float f = s[u].y == 0.f ? 0.f : s[u].x == M ? 1.f : __builtin_amdgcn_exp2f(s[u].x - M);
    wz[wv][64 * u + lane] = f;
    sum += s[u].y == 0.f ? 0.f : s[u].y * f;
  }
  sum = wave_sum(sum);
  __syncthreads();
  const uint64_t zs = (uint64_t)rows * hd;
  const float *p = part + row * hd;
  const float inv = pad ? 0.f : 1.f / sum;
  if constexpr (VEC) {
    const uint32_t width = min(hd / 4, 64u), groups = 64 / width, zg = lane / width;
    for (uint32_t d = lane % width * 4; d < hd; d += 4 * width) {
      f32x4 acc = {0, 0, 0, 0};
      if (zg < groups)
        for (uint32_t z0 = zg; z0 < nsplit; z0 += 8 * groups) {
          f32x4 v[8];
          float f[8];
#pragma unroll
          for (uint32_t e = 0; e < 8; e++) {
            const uint32_t z = z0 + e * groups;
            f[e] = z < nsplit ? wz[wv][z] : 0.f;
            v[e] = z < nsplit ? *(const f32x4 *)(p + z * zs + d) : f32x4{0, 0, 0, 0};
          }
#pragma unroll
          for (uint32_t e = 0; e < 8; e++)
            if (f[e] != 0.f) acc += v[e] * f[e];
        }
      for (uint32_t o = width; o < groups * width; o *= 2)  // groups is a power of two where there are several
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], o, 64);
      if (zg == 0 && blockIdx.x * 4 + wv < rows)
        *(f32x4 *)(y + row * hd + d) = pad ? f32x4{0, 0, 0, 0} : f32x4{acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    }
  } else {
    for (uint32_t d = lane; d < hd; d += 64) {
      float acc = 0.f;
      for (uint32_t z = 0; z < nsplit; z++)
        if (wz[wv][z] != 0.f) acc += p[z * zs + d] * wz[wv][z];
      if (blockIdx.x * 4 + wv < rows) y[row * hd + d] = pad ? 0.f : acc * inv;
    }
  }
}

static uint32_t tree_first(const TreeAttnArgs &in) { return in.start - std::min(in.start, in.window - 1); }

// mfma: a kernel of matrix products, for head dims that are multiples of 8 up to 256, padded to HD = 64, 128 or 256;
// RT tiles of 16 rows per wavefront (two in the staged kernel up to 128, one else), rw groups of them and `waves`
// wavefronts per workgroup.
struct TreePlan { bool mfma, staged; uint32_t HD, T, RT, rw, waves, per, blocks, nsplit; };
static TreePlan tree_plan(const TreeAttnArgs &in) {
  TreePlan p{};
  const uint32_t keys = in.start + in.nodes - tree_first(in), group = in.heads / in.kv_heads, rows = in.nodes * group;
  const uint32_t cus = (uint32_t)device_cu_count();
  // (a lane's offsets within 16 rows of the ring are 32-bit)
  p.mfma = in.hd % 8 == 0 && in.hd <= 256 && (uint64_t)in.kv_heads * in.hd * 4 < (1u << 27);
  p.HD = in.hd <= 64 ? 64 : in.hd <= 128 ? 128 : 256;
  if (p.mfma) {
    const uint32_t tiles = (rows + 15) / 16, unit = in.kv16 ? 32 : 16;
    // Staged from where its reuse of the keys outweighs its slower start. us, direct against staged, 8 kv heads:
    //   hd 128, 4 tiles, 16000 keys 29.4 / 28.0 (4000: 17.2 / 22.9); 8 tiles, 4000 keys 20.1 / 20.6 (1000: 14.1 / 17.5);
    //   16 tiles, 4000 keys 28.6 / 24.6 (1000: 16.3 / 18.9), 16000 keys 80 / 47; hd 256, 8 tiles, 4000 keys 32.5 / 28.4
    //   (with two row groups: a stage of 64 keys is two blocks then, for four slices, so half of the wavefronts have none).
    p.staged = in.kv16 && in.hd == p.HD && tiles >= 4 && (uint64_t)tiles * keys >= (p.HD == 256 ? 16000 : 32000);
    p.RT = p.staged && p.HD <= 128 ? 2 : 1;
    p.waves = p.staged || p.HD <= 128 ? 8 : 4;
    const uint32_t groups = (tiles + p.RT - 1) / p.RT;
    // Splits, and the row groups of a workgroup, by estimated time (us): a CU has one workgroup at a time; it starts and
    // ends in 4.5 and works 2.1 (f16) or 3.1 (f32) for a block of each slice; the join adds 3.3. hd 128, 8 kv heads, one
    // node: f16 300 keys 8.9 in one split, 11.3 in two; 1000 keys 14.9 and 13.7, 11.9 in four; f32 300 keys 13.2
    // in one, 12.3 in three; f32 1071 keys of 16 kv heads, 6 tiles: 24.4 us with one row group in two splits, 22.7 with two
    // in five. All of it is measured at hd 128 with up to five splits: hd 64 and 256 go by the same figures, a staged block by
    // the direct kernel's, and the join of a few hundred splits takes longer than 3.3 (8 nodes, 8 heads on one of 256, 31000 keys:
    // 243 splits, 50 us in all).
    const uint32_t kb = (keys + unit - 1) / unit;
    const double block = in.kv16 ? 2.1 : 3.1;
    uint32_t want = 1;
    double best = 1e30;
    auto splits = [&](uint32_t rw) {
      const uint32_t blocks = (groups + rw - 1) / rw, wgs = in.kv_heads * blocks, slices = p.waves / rw;
      for (uint32_t n = 1; n <= std::min((kb + slices - 1) / slices, TREE_SPLITS); n++) {
        const uint32_t per = (kb + n - 1) / n, deep = (per + slices - 1) / slices;
        const double t = (double)(((uint64_t)wgs * n + cus - 1) / cus) * (4.5 + block * deep) + (n > 1 ? 3.3 : 0);
        if (t < best) { best = t; want = n; p.rw = rw; p.blocks = blocks; }
      }
    };
    if (p.staged) {
      // four row groups read the keys half as often, but two leave fewer wavefronts without rows and more slices; hd
      // 128, 16 tiles: 31000 keys 80 us with four, 85 with two; 4000 keys 26.2 and 24.6
      splits(keys >= 8000 && (groups >= 8 || (p.HD == 256 && groups >= 4)) ? 4 : 2);
    } else {
      for (uint32_t rw = 1; rw <= 4 && rw <= groups; rw *= 2) splits(rw);
    }
    p.per = (kb + want - 1) / want;
    p.nsplit = (kb + p.per - 1) / p.per;
    return p;
  }
  p.T = tree_any_tile(in.hd);
  p.blocks = (rows + TREE_R - 1) / TREE_R;
  const uint32_t tiles = (keys + p.T - 1) / p.T, wgs = in.kv_heads * p.blocks;
  const uint32_t want = std::max(1u, std::min({tiles, 4 * cus / wgs, TREE_SPLITS}));
  p.per = (tiles + want - 1) / want;
  p.nsplit = (tiles + p.per - 1) / p.per;
  return p;
}

uint64_t attention_tree_scratch_floats(const TreeAttnArgs &in) {
  if (!in.nodes) return 0;
  const uint32_t n = tree_plan(in).nsplit;
  const uint64_t rows = (uint64_t)in.nodes * in.heads;
  return n > 1 ? tree_pairs(n, rows, in.hd) + 2 * n * rows : 0;
}

template <uint32_t HD, class E, bool FULL>
static void launch_tree(hipStream_t s, const TreeK &a, const TreePlan &p) {
  constexpr uint32_t waves = tree_threads<HD>() / 64;
  constexpr size_t lds = std::max(tree_wave_lds<HD, 1>() * waves, tree_any_lds(HD, tree_any_tile(HD)));
  static_assert(lds + sizeof(TreeLds) + 1024 <= LDS_MAX, "the wavefronts' outputs fit LDS");
  lds_opt_in_bytes((const void *)k_attn_tree<HD, E, FULL>, (uint32_t)lds);
  hipLaunchKernelGGL((k_attn_tree<HD, E, FULL>), dim3(a.kvh, p.blocks, p.nsplit), dim3(64 * waves), lds, s, a, TreeGrid{p.rw, p.per});
}
template <uint32_t HD>
static void launch_tree_staged(hipStream_t s, const TreeK &a, const TreePlan &p) {
  constexpr uint32_t RT = HD == 256 ? 1 : 2, SK = HD == 256 ? 64 : 128, waves = TREE_STAGED_NT / 64;
  constexpr size_t lds = std::max({tree_wave_lds<HD, RT>() * waves, tree_any_lds(HD, tree_any_tile(HD)), (size_t)4 * SK * 2 * HD});
  static_assert(lds + sizeof(TreeLds) + 1024 <= LDS_MAX, "two stages, and the wavefronts' outputs, fit LDS");
  lds_opt_in_bytes((const void *)k_attn_tree_staged<HD, RT, SK>, (uint32_t)lds);
  hipLaunchKernelGGL((k_attn_tree_staged<HD, RT, SK>), dim3(a.kvh, p.blocks, p.nsplit), dim3(TREE_STAGED_NT), lds, s, a, TreeGrid{p.rw, p.per});
}
template <uint32_t HD, class E>
static void launch_tree_hd(hipStream_t s, const TreeK &a, const TreePlan &p) {
  if (a.hd < HD) return launch_tree<HD, E, false>(s, a, p);
  if constexpr (sizeof(E) == 2)
    if (p.staged) return launch_tree_staged<HD>(s, a, p);
  launch_tree<HD, E, true>(s, a, p);
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
  a.T = p.T; a.per = p.per; a.scale = in.scale;
  if (p.mfma) {
    if (p.HD == 64) in.kv16 ? launch_tree_hd<64, _Float16>(s, a, p) : launch_tree_hd<64, float>(s, a, p);
    else if (p.HD == 128) in.kv16 ? launch_tree_hd<128, _Float16>(s, a, p) : launch_tree_hd<128, float>(s, a, p);
    else in.kv16 ? launch_tree_hd<256, _Float16>(s, a, p) : launch_tree_hd<256, float>(s, a, p);
  } else {
    const size_t lds = tree_any_lds(in.hd, p.T);
    const dim3 grid(in.kv_heads, p.blocks, p.nsplit);
    if (lds > 50000) lds_opt_in_bytes(in.kv16 ? (const void *)k_attn_tree_any<_Float16> : (const void *)k_attn_tree_any<float>, 100000);
    if (in.kv16) hipLaunchKernelGGL(k_attn_tree_any<_Float16>, grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL(k_attn_tree_any<float>, grid, dim3(256), lds, s, a);
  }
  WGD_HIP(hipGetLastError());
  if (p.nsplit > 1) {
    const uint32_t rows = in.nodes * in.heads;
    const dim3 grid((rows + 3) / 4);
    const bool vec = in.hd >= 4 && in.hd <= 256 && (in.hd & (in.hd - 1)) == 0;  // a power of two of lanes per split
    if (vec) hipLaunchKernelGGL(k_attn_tree_join<true>, grid, dim3(256), 0, s, (const float *)in.partial, in.y, rows, in.hd, p.nsplit);
    else hipLaunchKernelGGL(k_attn_tree_join<false>, grid, dim3(256), 0, s, (const float *)in.partial, in.y, rows, in.hd, p.nsplit);
    WGD_HIP(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace wgd
