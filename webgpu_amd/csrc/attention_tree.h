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

// What the nodes see of each other, in LDS: bits[i] of i's path to the root, by doubling the steps of all
// nodes at once; up[i] ends as -1, or -2 for padding.
struct TreeLds { uint32_t bits[WGD_TREE_MAX][TREE_WORDS]; int32_t up[WGD_TREE_MAX]; int32_t par[WGD_TREE_MAX]; };

__device__ __forceinline__ void tree_paths(TreeLds &L, const int32_t *parents, uint32_t nodes, uint32_t window) {
  const uint32_t words = (nodes + 31) / 32;
  for (uint32_t i = threadIdx.x; i < nodes; i += blockDim.x) {
    const int32_t p = parents[i];
    L.up[i] = L.par[i] = p < (int32_t)i && p >= -1 ? p : -2;
    for (uint32_t w = 0; w < words; w++) L.bits[i][w] = w == i / 32 ? 1u << (i % 32) : 0u;
  }
  __syncthreads();
  for (uint32_t span = 1; span < nodes; span *= 2) {
    // a workgroup has at least nodes threads, or a node has one of two owners: WGD_TREE_MAX / 256 rounds
    uint32_t b[TREE_WORDS];
    int32_t up = -1;
    const uint32_t i = threadIdx.x;
    bool more = false;
    if (i < nodes && L.up[i] >= 0) {
      const uint32_t a = (uint32_t)L.up[i];
      for (uint32_t w = 0; w < TREE_WORDS; w++) b[w] = w < words ? L.bits[a][w] : 0u;
      up = L.up[a];
      more = true;
    }
    if (!__syncthreads_or(more)) break;
    if (more) {
      for (uint32_t w = 0; w < words; w++) L.bits[i][w] |= b[w];
      L.up[i] = up;
    }
    __syncthreads();
  }
}

// Row r of the workgroup's kv head: the node's first cached key, whether it is one, and the node.
struct TreeSeen { uint32_t node, begin, valid; };
__device__ __forceinline__ TreeSeen tree_seen(const TreeLds &L, uint32_t node, uint32_t start, uint32_t nodes, uint32_t window) {
  TreeSeen s;
  s.node = node;
  uint32_t n = 0;
  for (uint32_t w = 0; w < (nodes + 31) / 32; w++) n += __popc(L.bits[node][w]);
  s.valid = L.up[node] == -1;
  const uint32_t end = start + n;  // its position + 1
  s.begin = end - min(end, window);
  return s;
}
// Which of the keys t0 .. t0 + 32 (below hi) the row sees, as bits.
__device__ __forceinline__ uint32_t tree_mask(const TreeLds &L, const TreeSeen &s, uint32_t t0, uint32_t hi, uint32_t start,
                                              uint32_t nodes, uint32_t window) {
  if (!s.valid || t0 >= hi) return 0;
  auto below = [](uint32_t n) { return n >= 32 ? ~0u : (1u << n) - 1; };
  uint32_t m = 0;
  if (t0 < start) {
    m = below(start - t0);
    if (s.begin > t0) m &= ~below(s.begin - t0);
  }
  if (t0 + 32 > start) {
    auto word = [&](uint32_t w) { return w < (nodes + 31) / 32 ? L.bits[s.node][w] : 0u; };
    uint32_t b;
    if (t0 < start) {
      b = word(0) << (start - t0);
    } else {
      const uint32_t j = t0 - start, sh = j % 32;
      b = word(j / 32) >> sh;
      if (sh) b |= word(j / 32 + 1) << (32 - sh);
    }
    if (window < nodes) {  // ancestors beyond the window: those before the window-th one
      int32_t a = (int32_t)s.node;
      for (uint32_t n = 1; n < window && a >= 0; n++) a = L.par[a];
      // nodes below `a` in number are on the path behind it
      if (a > 0) {
        const uint32_t first = start + (uint32_t)a;
        if (first > t0) b &= ~(below(first - t0) & (t0 < start ? ~below(start - t0) : ~0u));
      }
    }
    m |= b;
  }
  return m & below(hi - t0);
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
  TreeSeen seen = {0, 0, 0};
  if (tid < TREE_R) {
    if (r0 + tid < nrows) seen = tree_seen(L, (r0 + tid) / a.group, a.start, a.nodes, a.window);
    mrow[tid] = -INFINITY; lrow[tid] = 0.f;
  }
#pragma unroll 1
  for (uint32_t t0 = lo; t0 < hi; t0 += T) {
    __syncthreads();
    if (tid < TREE_R) {
      vis[tid][0] = tree_mask(L, seen, t0, min(hi, t0 + T), a.start, a.nodes, a.window);
      vis[tid][1] = T > 32 ? tree_mask(L, seen, t0 + 32, min(hi, t0 + T), a.start, a.nodes, a.window) : 0;
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
      if (d == 0) *(float2 *)(a.part + a.nsplit * all * hd + 2 * at) = make_float2(mrow[r], pad ? -1.f : lrow[r]);
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

// ------------------------------------------------------------------ head dims 64, 128 and 256
//
// A wavefront holds RT tiles of 16 rows of one kv head as matrix operands and walks over its keys in
// blocks of 16 NB, read straight from the ring into registers: no barrier until the end. The
// wavefronts of a workgroup are `rw` groups of rows times key slices (block b of the workgroup's range
// belongs to slice b % slices); the slices merge in LDS, the key ranges of workgroups in
// k_attn_tree_join. Scores come out transposed, S^T = K Q^T: lane (g, c) = (lane / 16, lane % 16)
// holds keys 4 g .. + 4 of row c, whose probabilities are, in the same lane, operand of
// O^T += V^T P^T.
//   f16 rings (v_mfma_f32_16x16x32_f16): K and V are operands as they are, exact. The queries (times
//     scale log2 e) are split into f16 hi + lo with a power of two per row, the probabilities with a
//     factor of 2^11: 22 bits each, two products in place of one. Lane (g, c) loads VE values d = VE c of
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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr float TREE_LAG = 4.f, TREE_BIAS = 11.f;

template <class E> constexpr uint32_t tree_nb() { return sizeof(E) == 2 ? 2 : 1; }
template <uint32_t HD, class E> constexpr uint32_t tree_ve() { return sizeof(E) == 2 && HD >= 128 ? 8 : 4; }

// Threads of a workgroup: as many as their registers allow.
template <uint32_t HD, uint32_t RT>
constexpr uint32_t tree_threads() { return RT <= 2 && HD <= 128 ? 512 : 256; }

template <uint32_t HD, class E, uint32_t RT>
struct TreeWave {
  static constexpr bool HALF = sizeof(E) == 2;
  static constexpr uint32_t NB = tree_nb<E>(), KEYS = 16 * NB, VE = tree_ve<HD, E>(), NX = HD / (16 * VE);
  static constexpr uint32_t KT = HALF ? HD / 32 : HD / 16;  // 16-byte pieces of a key per lane
  static constexpr uint32_t VK = 4 * NB;                    // keys per lane of a block of V
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef uint32_t vpiece __attribute__((ext_vector_type(VE * sizeof(E) / 4)));

  u32x4 qh[RT][KT], ql[HALF ? RT : 1][KT];  // f16 hi and lo; f32: qh alone
  float qs[RT];                              // the power of two taken out of the row's query
  f32x4 o[RT][NX][VE];
  float m[RT], l[RT];

  // The row's query times scale log2 e as operand.
  __device__ __forceinline__ void load_q(const TreeK &a, uint32_t rt, const float *q, bool ok, uint32_t g) {
    const float f = a.scale * TREE_LOG2E;
    if constexpr (!HALF) {
#pragma unroll
      for (uint32_t t = 0; t < KT; t++) {
        const f32x4 v = ok ? *(const f32x4 *)(q + 16 * t + 4 * g) : f32x4{0, 0, 0, 0};
        qh[rt][t] = __builtin_bit_cast(u32x4, f32x4{v.x * f, v.y * f, v.z * f, v.w * f});
      }
      qs[rt] = 1.f;
    } else {
      float v[KT][8];
      uint32_t mx = 0;
#pragma unroll
      for (uint32_t t = 0; t < KT; t++) {
        const f32x4 x = ok ? *(const f32x4 *)(q + 32 * t + 8 * g) : f32x4{0, 0, 0, 0};
        const f32x4 y = ok ? *(const f32x4 *)(q + 32 * t + 8 * g + 4) : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[t][e] = x[e] * f;
          v[t][4 + e] = y[e] * f;
          mx = max(mx, max(__float_as_uint(v[t][e]) & 0x7FFFFFFFu, __float_as_uint(v[t][4 + e]) & 0x7FFFFFFFu));
        }
      }
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, 64));
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, 64));
      // the largest magnitude into [2^14, 2^15); both powers stay normal
      const uint32_t ex = min(max(mx >> 23, 16u), 254u);
      const float inv = __uint_as_float((254u + 14u - ex) << 23);
      qs[rt] = __uint_as_float((ex - 14u) << 23);
#pragma unroll
      for (uint32_t t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t h, lo;
          split2(v[t][2 * e] * inv, v[t][2 * e + 1] * inv, h, lo);
          qh[rt][t][e] = h;
          ql[rt][t][e] = lo;
        }
    }
  }

  // Keys [t0, ..) in steps of `step` up to hi, of ring rows `rowb` bytes apart, this kv head at k, v.
  __device__ __forceinline__ void walk(const TreeK &a, const TreeLds &L, const TreeSeen *seen, const uint8_t *k, const uint8_t *v,
                                       uint32_t t0, uint32_t step, uint32_t hi, uint32_t masked_below) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const uint32_t cap = a.capacity;
    const uint64_t rowb = (uint64_t)a.kvh * HD * sizeof(E);
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
      m[rt] = -INFINITY; l[rt] = 0.f;
#pragma unroll
      for (uint32_t x = 0; x < NX; x++)
#pragma unroll
        for (uint32_t e = 0; e < VE; e++) o[rt][x][e] = f32x4{0, 0, 0, 0};
    }
    auto slot = [&](uint32_t base, uint32_t off) {  // (base + off) % cap for base < cap
      const uint32_t s = base + off;
      return cap >= KEYS ? (s >= cap ? s - cap : s) : s % cap;
    };
    u32x4 kr[NB][KT];
    auto load_k = [&](uint32_t base) {
#pragma unroll
      for (uint32_t b = 0; b < NB; b++) {
        const uint8_t *row = k + slot(base, 16 * b + c) * rowb + 16 * g;
#pragma unroll
        for (uint32_t t = 0; t < KT; t++) kr[b][t] = *(const u32x4 *)(row + 64 * t);
      }
    };
    if (t0 >= hi) return;
    uint32_t base = t0 % cap;
    load_k(base);
    for (; t0 < hi; t0 += step) {
      vpiece vr[VK][NX];
#pragma unroll
      for (uint32_t j = 0; j < VK; j++) {
        const uint8_t *row = v + slot(base, 16 * (j / 4) + 4 * g + j % 4) * rowb + VE * sizeof(E) * c;
#pragma unroll
        for (uint32_t x = 0; x < NX; x++) vr[j][x] = *(const vpiece *)(row + 16 * VE * sizeof(E) * x);
      }
      // ---- scores
      f32x4 s[RT][NB];
#pragma unroll
      for (uint32_t rt = 0; rt < RT; rt++)
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) {
          f32x4 acc = {0, 0, 0, 0};
#pragma unroll
          for (uint32_t t = 0; t < KT; t++) {
            if constexpr (HALF) {
              const f16x8 kf = __builtin_bit_cast(f16x8, kr[b][t]);
              acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, __builtin_bit_cast(f16x8, qh[rt][t]), acc, 0, 0, 0);
              acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, __builtin_bit_cast(f16x8, ql[rt][t]), acc, 0, 0, 0);
            } else {
              const f32x4 kf = __builtin_bit_cast(f32x4, kr[b][t]), qf = __builtin_bit_cast(f32x4, qh[rt][t]);
#pragma unroll
              for (int u = 0; u < 4; u++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[u], qf[u], acc, 0, 0, 0);
            }
          }
          s[rt][b] = acc;
        }
      const uint32_t next = (base + step) % cap;
      if (t0 + step < hi) load_k(next);
      // ---- weights
      const bool masked = t0 + KEYS > min(hi, a.start) || t0 < masked_below;
      f32x4 p[RT][NB];
#pragma unroll
      for (uint32_t rt = 0; rt < RT; rt++) {
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) s[rt][b] *= qs[rt];
        if (masked) {
          const uint32_t sees = tree_mask(L, seen[rt], t0, hi, a.start, a.nodes, a.window);
#pragma unroll
          for (uint32_t b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[rt][b][r] = sees >> (16 * b + 4 * g + r) & 1 ? s[rt][b][r] : -INFINITY;
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[rt][b][r]);
        if (__any(mx > (m[rt] == -INFINITY ? -INFINITY : m[rt] + TREE_LAG))) {
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
        }
        const float ref = TREE_BIAS - (m[rt] == -INFINITY ? 0.f : m[rt]);
#pragma unroll
        for (uint32_t b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            p[rt][b][r] = __builtin_amdgcn_exp2f(s[rt][b][r] + ref);
            l[rt] += p[rt][b][r];
          }
      }
      // ---- values
      if (t0 + KEYS > hi) {  // slots past the keys hold anything
#pragma unroll
        for (uint32_t j = 0; j < VK; j++)
          if (t0 + 16 * (j / 4) + 4 * g + j % 4 >= hi)
#pragma unroll
            for (uint32_t x = 0; x < NX; x++) vr[j][x] = vpiece{};
      }
      if constexpr (HALF) {
        f16x8 ph[RT], pl[RT];
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) {
          u32x4 h, lo;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint32_t x, y;
            split2(p[rt][e / 2][2 * (e % 2)], p[rt][e / 2][2 * (e % 2) + 1], x, y);
            h[e] = x;
            lo[e] = y;
          }
          ph[rt] = __builtin_bit_cast(f16x8, h);
          pl[rt] = __builtin_bit_cast(f16x8, lo);
        }
#pragma unroll
        for (uint32_t x = 0; x < NX; x++)
#pragma unroll
          for (uint32_t e = 0; e < VE; e++) {
            u32x4 f;  // half e of the eight keys
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
              f[i] = __builtin_amdgcn_perm(vr[2 * i + 1][x][e / 2], vr[2 * i][x][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
            const f16x8 vf = __builtin_bit_cast(f16x8, f);
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) {
              o[rt][x][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[rt], o[rt][x][e], 0, 0, 0);
              o[rt][x][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[rt], o[rt][x][e], 0, 0, 0);
            }
          }
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
#pragma unroll
          for (uint32_t x = 0; x < NX; x++)
#pragma unroll
            for (uint32_t e = 0; e < VE; e++)
#pragma unroll
              for (uint32_t rt = 0; rt < RT; rt++)
                o[rt][x][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[i][x][e]), p[rt][0][i], o[rt][x][e], 0, 0, 0);
      }
      base = next;
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

struct TreeGrid { uint32_t rw, per; };  // row groups of a workgroup; key blocks per split

template <uint32_t HD, class E, uint32_t RT>
constexpr size_t tree_wave_lds() { return sizeof(float) * RT * 16 * (HD + 4 + 2); }

template <uint32_t HD, class E, uint32_t RT>
__global__ __launch_bounds__((tree_threads<HD, RT>())) void k_attn_tree(TreeK a, TreeGrid gr) {
  typedef TreeWave<HD, E, RT> Wave;
  extern __shared__ float lds[];
  __shared__ TreeLds L;
  constexpr uint32_t VE = Wave::VE, NX = Wave::NX, OS = HD + 4, WS = RT * 16 * (OS + 2);
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6), slices = (blockDim.x >> 6) / gr.rw;
  const uint32_t kv = blockIdx.x, z = blockIdx.z, nrows = a.nodes * a.group, end = a.start + a.nodes;
  const uint32_t wrow = (blockIdx.y * gr.rw + w % gr.rw) * RT * 16, slice = w / gr.rw;
  const uint32_t lo = a.first + min(z * gr.per * Wave::KEYS, end - a.first), hi = lo + min(gr.per * Wave::KEYS, end - lo);
  // keys below this are hidden from some nodes by the window
  const uint32_t masked_below = end <= a.window ? 0 : a.first + a.nodes;
  const bool masks = hi > a.start || lo < masked_below;
  if (masks) tree_paths(L, a.parents, a.nodes, a.window);

  Wave s;
  TreeSeen seen[RT];
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
    const uint32_t r = min(wrow + 16 * rt + c, nrows - 1);
    s.load_q(a, rt, a.q + tree_row(a, kv, r) * HD, wrow + 16 * rt + c < nrows, g);
    seen[rt] = masks ? tree_seen(L, r / a.group, a.start, a.nodes, a.window) : TreeSeen{r / a.group, 0, 1};
  }
  const uint64_t head = (uint64_t)kv * HD * sizeof(E);
  s.walk(a, L, seen, (const uint8_t *)a.k + head, (const uint8_t *)a.v + head, lo + slice * Wave::KEYS, slices * Wave::KEYS,
         wrow < nrows ? hi : 0, masked_below);
  if (__syncthreads_or(!s.finite())) {
    constexpr uint32_t NT = tree_threads<HD, RT>();
    if (!masks) tree_paths(L, a.parents, a.nodes, a.window);
    for (uint32_t i = 0; i < gr.rw * RT; i++) {
      const uint32_t r0 = (blockIdx.y * gr.rw * RT + i) * 16;
      if (r0 < nrows) tree_any<E, NT>(a, L, lds, tree_any_tile(HD), kv, r0, z, lo, hi);
    }
    return;
  }

  // ---- to LDS: [row] max, sum; [row][HD]
  __syncthreads();
  float *mine = lds + w * WS;
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
    float l = s.l[rt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) { mine[2 * (16 * rt + c)] = s.m[rt]; mine[2 * (16 * rt + c) + 1] = seen[rt].valid ? l : -1.f; }
    float *row = mine + RT * 32 + (16 * rt + c) * OS;
#pragma unroll
    for (uint32_t x = 0; x < NX; x++)
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (uint32_t e = 0; e < VE; e += 4)
          *(f32x4 *)(row + 16 * VE * x + 4 * VE * g + VE * r + e) =
              f32x4{s.o[rt][x][e][r], s.o[rt][x][e + 1][r], s.o[rt][x][e + 2][r], s.o[rt][x][e + 3][r]};
  }
  __syncthreads();
  // ---- the slices in order, eight dims of a row per thread
  const uint64_t rows = (uint64_t)a.nodes * a.heads;
  for (uint32_t i = tid; i < gr.rw * RT * 16 * (HD / 8); i += blockDim.x) {
    const uint32_t d = i % (HD / 8) * 8, lr = i / (HD / 8) % (RT * 16), rg = i / (HD / 8) / (RT * 16);
    const uint32_t r = (blockIdx.y * gr.rw + rg) * RT * 16 + lr;
    if (r >= nrows) continue;
    float M = -INFINITY, l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t u = 0; u < slices; u++) M = fmaxf(M, lds[(u * gr.rw + rg) * WS + 2 * lr]);
    const bool pad = lds[rg * WS + 2 * lr + 1] < 0.f;
    for (uint32_t u = 0; u < slices; u++) {
      const float *p = lds + (u * gr.rw + rg) * WS;
      if (p[2 * lr + 1] == 0.f) continue;  // nothing seen (all NaN: the sum is NaN)
      const float f = p[2 * lr] == M ? 1.f : __builtin_amdgcn_exp2f(p[2 * lr] - M);
      l += p[2 * lr + 1] * f;
      const f32x4 x0 = *(const f32x4 *)(p + RT * 32 + lr * OS + d), x1 = *(const f32x4 *)(p + RT * 32 + lr * OS + d + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) { y[e] += x0[e] * f; y[4 + e] += x1[e] * f; }
    }
    const uint64_t row = tree_row(a, kv, r);
    float *to_row = a.y + row * HD + d;
    float inv = 1.f;
    if (a.nsplit > 1) {
      to_row = a.part + ((uint64_t)z * rows + row) * HD + d;
      if (d == 0) *(float2 *)(a.part + (uint64_t)a.nsplit * rows * HD + 2 * ((uint64_t)z * rows + row)) = make_float2(M - TREE_BIAS, pad ? -1.f : l);
    } else {
      inv = 1.f / l;
    }
    const bool zero = pad && a.nsplit == 1;
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      *(f32x4 *)(to_row + e) = zero ? f32x4{0, 0, 0, 0} : f32x4{y[e] * inv, y[e + 1] * inv, y[e + 2] * inv, y[e + 3] * inv};
  }
}

// The splits of a row in order, of partial outputs [split][row][hd] and behind them (max, sum) pairs
// [split][row], maxima in powers of two. A sum of zero is a split without keys that the row sees (or
// without a finite score, which adds nothing either); the last split knows padding, by a negative sum. A row
// always sees itself, so sums that are all zero mean scores that were all -inf: 0 / 0, as the
// formula has it.
__global__ __launch_bounds__(128) void k_attn_tree_join(const float *part, float *y, uint32_t rows, uint32_t hd, uint32_t nsplit) {
  const uint64_t row = blockIdx.x;
  const float2 *ml = (const float2 *)(part + (uint64_t)nsplit * rows * hd) + row;
  float M = -INFINITY;
  for (uint32_t z = 0; z < nsplit; z++) M = fmaxf(M, ml[(uint64_t)z * rows].x);
  const bool pad = ml[(uint64_t)(nsplit - 1) * rows].y < 0.f;
  float L = 0.f;
  for (uint32_t z = 0; z < nsplit; z++) {
    const float2 s = ml[(uint64_t)z * rows];
    if (s.y != 0.f) L += s.y * (s.x == M ? 1.f : exp2f(s.x - M));
  }
  for (uint32_t d = threadIdx.x; d < hd; d += blockDim.x) {
    float acc = 0.f;
    for (uint32_t z = 0; z < nsplit; z++) {
      const float2 s = ml[(uint64_t)z * rows];
      if (s.y != 0.f) acc += part[((uint64_t)z * rows + row) * hd + d] * (s.x == M ? 1.f : exp2f(s.x - M));
    }
    y[row * hd + d] = pad ? 0.f : acc / L;
  }
}

static uint32_t tree_first(const TreeAttnArgs &in) { return in.start - std::min(in.start, in.window - 1); }

// mfma: the kernel for head dims 64, 128 and 256; RT tiles of 16 rows per wavefront, rw groups of them
// and `waves` wavefronts per workgroup.
struct TreePlan { bool mfma; uint32_t T, RT, rw, waves, per, blocks, nsplit; };
static TreePlan tree_plan(const TreeAttnArgs &in) {
  TreePlan p{};
  const uint32_t keys = in.start + in.nodes - tree_first(in), group = in.heads / in.kv_heads, rows = in.nodes * group;
  const uint32_t cus = (uint32_t)device_cu_count();
  p.mfma = in.hd == 64 || in.hd == 128 || in.hd == 256;
  if (p.mfma) {
    const uint32_t tiles = (rows + 15) / 16, unit = in.kv16 ? 32 : 16;
    p.RT = tiles > 1 ? 2 : 1;
    if (in.kv16 && in.hd == 64 && tiles > 2) p.RT = 4;
    if (in.hd == 256) p.RT = 1;
    p.waves = p.RT == 4 || in.hd == 256 ? 4 : 8;
    const uint32_t groups = (tiles + p.RT - 1) / p.RT;
    p.rw = groups >= 4 && p.waves >= 4 ? 4 : groups >= 2 ? 2 : 1;
    const uint32_t slices = p.waves / p.rw, kb = (keys + unit - 1) / unit;
    p.blocks = (groups + p.rw - 1) / p.rw;
    const uint32_t wgs = in.kv_heads * p.blocks;
    const uint32_t want = std::max(1u, std::min((kb + slices - 1) / slices, (cus + wgs - 1) / wgs));
    p.per = (kb + want - 1) / want;
    p.nsplit = (kb + p.per - 1) / p.per;
    return p;
  }
  p.T = tree_any_tile(in.hd);
  p.blocks = (rows + TREE_R - 1) / TREE_R;
  const uint32_t tiles = (keys + p.T - 1) / p.T, wgs = in.kv_heads * p.blocks;
  const uint32_t want = std::max(1u, std::min(tiles, 4 * cus / wgs));
  p.per = (tiles + want - 1) / want;
  p.nsplit = (tiles + p.per - 1) / p.per;
  return p;
}

uint64_t attention_tree_scratch_floats(const TreeAttnArgs &in) {
  if (!in.nodes) return 0;
  const uint32_t n = tree_plan(in).nsplit;
  return n > 1 ? (uint64_t)n * in.nodes * in.heads * (in.hd + 2) : 0;
}

template <uint32_t HD, class E, uint32_t RT>
static void launch_tree(hipStream_t s, const TreeK &a, const TreePlan &p) {
  constexpr uint32_t waves = tree_threads<HD, RT>() / 64;
  constexpr size_t lds = std::max(tree_wave_lds<HD, E, RT>() * waves, tree_any_lds(HD, tree_any_tile(HD)));
  static_assert(lds + sizeof(TreeLds) + 1024 <= LDS_MAX, "the wavefronts' outputs fit LDS");
  lds_opt_in_bytes((const void *)k_attn_tree<HD, E, RT>, (uint32_t)lds);
  hipLaunchKernelGGL((k_attn_tree<HD, E, RT>), dim3(a.kvh, p.blocks, p.nsplit), dim3(64 * waves), lds, s, a, TreeGrid{p.rw, p.per});
}
template <uint32_t HD, class E>
static void launch_tree_rt(hipStream_t s, const TreeK &a, const TreePlan &p) {
  if (p.RT == 1) launch_tree<HD, E, 1>(s, a, p);
  if constexpr (HD <= 128)
    if (p.RT == 2) launch_tree<HD, E, 2>(s, a, p);
  if constexpr (HD <= 128 && sizeof(E) == 2)
    if (p.RT == 4) launch_tree<HD, E, 4>(s, a, p);
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
    if (in.hd == 64) in.kv16 ? launch_tree_rt<64, _Float16>(s, a, p) : launch_tree_rt<64, float>(s, a, p);
    else if (in.hd == 128) in.kv16 ? launch_tree_rt<128, _Float16>(s, a, p) : launch_tree_rt<128, float>(s, a, p);
    else in.kv16 ? launch_tree_rt<256, _Float16>(s, a, p) : launch_tree_rt<256, float>(s, a, p);
  } else {
    const size_t lds = tree_any_lds(in.hd, p.T);
    const dim3 grid(in.kv_heads, p.blocks, p.nsplit);
    if (lds > 50000) lds_opt_in_bytes(in.kv16 ? (const void *)k_attn_tree_any<_Float16> : (const void *)k_attn_tree_any<float>, 100000);
    if (in.kv16) hipLaunchKernelGGL(k_attn_tree_any<_Float16>, grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL(k_attn_tree_any<float>, grid, dim3(256), lds, s, a);
  }
  WGD_HIP(hipGetLastError());
  if (p.nsplit > 1) {
    hipLaunchKernelGGL(k_attn_tree_join, dim3(in.nodes * in.heads), dim3(128), 0, s, (const float *)in.partial, in.y,
                       in.nodes * in.heads, in.hd, p.nsplit);
    WGD_HIP(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace wgd
