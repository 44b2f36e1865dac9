// attention_pages.h — attention of a batch of requests over K/V pages (part of attention.hip).
//
// Request r has lengths[r] tokens in the pages that its row of the table names, the last n_r of them (counts[r], at
// most `tokens`) with a query each: query t has the position p = lengths[r] - n_r + t and sees the keys (p - window, p]:
//   y = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m),  s_k = scale q . k_k,  m = max s_k.
// The lengths are on the device, so the work is shared out there: every wavefront forms the same plan from them.
// A request's keys are cut into chunks of the same length for all, about `target` of them together; a workgroup has one
// chunk, one kv head and some of the rows, the (query, head of the group) pairs that share the head's keys.
// Requests whose first `shared` tokens are the owner's have these computed together: the rows of all of them
// against the owner's keys, in `nprefix` parts. The parts of a row meet in k_pages_join, as (max, sum, weighted values).
#pragma once

namespace wgd {

struct PagesK {
  const float *q; const void *k, *v; float *y, *part; const int32_t *table, *lengths, *counts;
  uint32_t heads, kvh, group, hd, window, shift, max_pages, pages, requests, tokens, shared, owner;
  uint32_t unit, least, target, slots;  // keys of a unit; least units of a chunk; chunks wanted, and at most
  uint32_t nprefix, per;                // parts of the prefix, keys of each
  uint32_t blocks;                      // row blocks of a request (of all of them, in the prefix)
  float scale;
};

// The parts of the rows: [slot][token][head][hd] of the requests' own chunks, [part][request][token][head][hd] of the prefix, then from
// an even float on (max, sum) pairs in the same order. A sum below 0: the row sees nothing of the part.
__host__ __device__ __forceinline__ uint64_t pages_part_rows(uint32_t slots, uint32_t nprefix, uint32_t requests, uint64_t rows) {
  return ((uint64_t)slots + (uint64_t)nprefix * requests) * rows;
}
__host__ __device__ __forceinline__ uint64_t pages_pairs(uint64_t part_rows, uint32_t hd) { return (part_rows * hd + 1) / 2 * 2; }

// What lane-wide plans say of one request.
struct PagesRequest { uint32_t len, n, lo; bool shares; };  // its keys start at lo where it shares nothing
__device__ __forceinline__ PagesRequest pages_request(const PagesK &a, uint32_t r) {
  PagesRequest q = {0, 0, 0, false};
  if (r >= a.requests) return q;
  q.len = min((uint32_t)max(a.lengths[r], 0), a.max_pages << a.shift);
  q.n = min(q.len, a.counts ? (uint32_t)min(max(a.counts[r], 0), (int32_t)a.tokens) : a.tokens);
  const uint32_t first = q.len - q.n + 1;  // keys up to the first query's own
  q.lo = first > a.window ? first - a.window : 0;
  if (a.shared) {
    const uint32_t c = (a.shared >> a.shift) - 1;
    const bool owned = min((uint32_t)max(a.lengths[a.owner], 0), a.max_pages << a.shift) >= a.shared;
    q.shares = owned && q.n && q.len - q.n >= a.shared && q.len <= a.window &&
               a.table[(uint64_t)r * a.max_pages + c] == a.table[(uint64_t)a.owner * a.max_pages + c];
  }
  return q;
}
__device__ __forceinline__ uint32_t pages_units(const PagesK &a, const PagesRequest &q, bool sharing) {
  const uint32_t lo = sharing && q.shares ? a.shared : q.lo;
  return q.n ? (q.len - lo + a.unit - 1) / a.unit : 0;
}

// The plan of all requests: whether a prefix is shared (by two or more), and the units of a chunk.
struct PagesPlan { bool sharing; uint32_t chunk; };
__device__ __forceinline__ PagesPlan pages_plan(const PagesK &a) {
  const uint32_t lane = threadIdx.x & 63;
  uint64_t alone = 0, apart = 0;
  uint32_t sharers = 0;
  for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
    const PagesRequest q = pages_request(a, r0 + lane);
    alone += pages_units(a, q, false);
    apart += pages_units(a, q, true);
    sharers += (uint32_t)__popcll(__ballot(q.shares));
  }
  const bool sharing = sharers > 1;
  uint64_t sum = sharing ? apart : alone;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor((unsigned long long)sum, o, 64);
  const uint64_t even = (sum + a.target - 1) / a.target;
  const uint32_t whole = 0x7FFFFFFFu / a.unit + 1;  // the longest request
  return PagesPlan{sharing, max(even < whole ? (uint32_t)even : whole, a.least)};
}

// One request in the plan: the slot of its first chunk, their number, its keys [lo, len). It is the one that has the slot `find`,
// or with BY_REQUEST the request `find` itself. The same in all lanes.
struct PagesChunks { uint32_t r, first, count, lo, len, n; bool shares; };
template <bool BY_REQUEST>
__device__ __forceinline__ PagesChunks pages_chunks(const PagesK &a, const PagesPlan &plan, uint32_t find) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
    const PagesRequest q = pages_request(a, r0 + lane);
    const uint32_t units = pages_units(a, q, plan.sharing);
    const uint32_t mine = r0 + lane < a.requests ? max(1u, (units + plan.chunk - 1) / plan.chunk) : 0;
    uint32_t s = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const uint32_t u = (uint32_t)__shfl_up((int)s, o, 64);
      if (lane >= (uint32_t)o) s += u;
    }
    const uint64_t here = __ballot(BY_REQUEST ? r0 + lane == find : mine && find >= before + s - mine && find < before + s);
    if (here) {
      const int at = (int)__ffsll((unsigned long long)here) - 1;
      const bool shares = plan.sharing && q.shares;
      return PagesChunks{r0 + (uint32_t)at, before + (uint32_t)__shfl((int)(s - mine), at, 64), (uint32_t)__shfl((int)mine, at, 64),
                         (uint32_t)__shfl((int)(shares ? a.shared : q.lo), at, 64), (uint32_t)__shfl((int)q.len, at, 64),
                         (uint32_t)__shfl((int)q.n, at, 64), (bool)__shfl((int)shares, at, 64)};
    }
    before += (uint32_t)__shfl((int)s, 63, 64);
  }
  return PagesChunks{0xFFFFFFFFu, 0, 0, 0, 0, 0, false};
}

// A workgroup's part of the work: rows of kv head kv against the keys [lo, hi) of one row of the table. Row i of the part is
// (request, query, head): of one request, or of those that share the prefix (`list`, in LDS).
struct PagesPart {
  uint32_t kv, row0, nrows, lo, hi;
  uint32_t r, n, end0;       // own chunks: the request, its queries, lengths - n + 1 (what query 0 sees of it)
  const int32_t *table;
  const uint16_t *list;      // the prefix: null otherwise
  bool direct;               // the only part of its rows: to y
  uint64_t part;             // else the first row of its part
};
struct PagesRow { bool valid; uint64_t row; uint32_t request, query, begin, end; };  // row of q and y; keys [begin, end)
__device__ __forceinline__ PagesRow pages_row(const PagesK &a, const PagesPart &p, uint32_t i) {
  PagesRow w = {i < p.nrows, 0, p.r, 0, 0, 0};
  if (!w.valid) return w;
  uint32_t t = i / a.group;
  if (p.list) {
    w.request = p.list[t / a.tokens];
    t %= a.tokens;
    w.end = p.hi;
    w.valid = !a.counts || (int32_t)t < a.counts[w.request];
  } else {
    w.end = min(p.hi, p.end0 + t);
    w.begin = p.end0 + t > a.window ? p.end0 + t - a.window : 0;
    w.valid = t < p.n;
  }
  w.query = t;
  w.row = ((uint64_t)w.request * a.tokens + t) * a.heads + p.kv * a.group + i % a.group;
  return w;
}
// Where a part keeps row w: own parts have the rows of one request, those of the prefix all of them.
__device__ __forceinline__ uint64_t pages_at(const PagesK &a, const PagesPart &p, const PagesRow &w) {
  return p.part + (p.list ? w.row : w.row - (uint64_t)p.r * a.tokens * a.heads);
}

// ------------------------------------------------------------------ any head dim up to 512
// 16 rows in tiles of T keys staged in LDS (tree_any_lds() of it): f32 products one by one, and a key that a row does not see, or on a
// page that is none, is never multiplied with its weight, so what it holds (NaN too) reaches nothing. Every thread of the NT calls it.
template <class E, uint32_t NT>
__device__ __forceinline__ void pages_any(const PagesK &a, float *lds, uint32_t T, const PagesPart &p, uint32_t r0) {
  __shared__ uint64_t vis[TREE_R];
  __shared__ uint32_t there[2];
  __shared__ float mrow[TREE_R], lrow[TREE_R], corr[TREE_R];
  __shared__ uint32_t any[TREE_R];
  const uint32_t hd = a.hd, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, pg = (1u << a.shift) - 1;
  float *Ks = lds, *Vs = Ks + T * (hd + 1), *Qs = Vs + T * hd, *O = Qs + TREE_R * hd, *S = O + TREE_R * hd;
  __syncthreads();
  for (uint32_t i = tid; i < TREE_R * hd; i += NT) {
    const PagesRow w = pages_row(a, p, r0 + i / hd);
    Qs[i] = w.valid ? a.q[w.row * hd + i % hd] : 0.f;
    O[i] = 0.f;
  }
  PagesRow mine = {false, 0, 0, 0, 0, 0};
  if (tid < TREE_R) {
    mine = pages_row(a, p, r0 + tid);
    mrow[tid] = -INFINITY; lrow[tid] = 0.f; any[tid] = 0;
  }
  auto page = [&](uint32_t t) { const int32_t id = p.table[t >> a.shift]; return id >= 0 && (uint32_t)id < a.pages ? id : -1; };
#pragma unroll 1
  for (uint32_t t0 = p.lo; t0 < p.hi; t0 += T) {
    __syncthreads();
    if (tid < 64) {
      const uint64_t m = __ballot(lane < T && t0 + lane < p.hi && page(t0 + lane) >= 0);
      if (tid < TREE_R) {
        auto below = [&](uint32_t t) { return t <= t0 ? 0ull : t - t0 >= 64 ? ~0ull : (1ull << (t - t0)) - 1; };
        const uint64_t sees = mine.valid ? m & below(mine.end) & ~below(mine.begin) : 0;
        vis[tid] = sees;
        any[tid] |= sees != 0;
      }
    }
#pragma unroll 2
    for (uint32_t i = tid; i < T * hd; i += NT) {
      const uint32_t j = i / hd, d = i % hd, t = t0 + j;
      const int32_t id = t < p.hi ? page(t) : -1;
      float kk = 0.f, vv = 0.f;
      if (id >= 0) {
        const uint64_t src = ((((uint64_t)id << a.shift) + (t & pg)) * a.kvh + p.kv) * hd + d;
        kk = kv_get<E>(a.k, src); vv = kv_get<E>(a.v, src);
      }
      Ks[j * (hd + 1) + d] = kk;
      Vs[j * hd + d] = vv;
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = tid; i < TREE_R * T; i += NT) {
      const uint32_t r = i / T, j = i % T;
      float sc = -INFINITY;
      if (vis[r] >> j & 1) {
        const float *qr = Qs + r * hd, *kr = Ks + j * (hd + 1);
        float dot = 0.f;
#pragma unroll 8
        for (uint32_t d = 0; d < hd; d++) dot += qr[d] * kr[d];
        sc = dot * (a.scale * TREE_LOG2E);
      }
      S[i] = sc;
    }
    __syncthreads();
    for (uint32_t r = wv; r < TREE_R; r += NT / 64) {
      const uint64_t on = vis[r];
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
    const PagesRow w = pages_row(a, p, r0 + r);
    if (!w.valid) continue;
    if (p.direct) {
      a.y[w.row * hd + d] = any[r] ? O[i] / lrow[r] : 0.f;
    } else {
      const uint64_t at = pages_at(a, p, w);
      a.part[at * hd + d] = O[i];
      if (d == 0) {
        const uint64_t pairs = pages_pairs(pages_part_rows(a.slots, a.nprefix, a.requests, (uint64_t)a.tokens * a.heads), hd);
        *(float2 *)(a.part + pairs + 2 * at) = make_float2(mrow[r], any[r] ? lrow[r] : -1.f);
      }
    }
  }
}

// The workgroup's part; false where it has none. PREFIX: blockIdx.y is a part of the prefix, else a slot. `list` has WGD_REQUESTS_MAX
// places in LDS. Queries that a request does not have get zeros here, from its first chunk's workgroups of `rows` rows each.
template <bool PREFIX, uint32_t NT>
__device__ __forceinline__ bool pages_part(const PagesK &a, uint32_t rows, uint16_t *list, PagesPart &p) {
  const PagesPlan plan = pages_plan(a);
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint64_t all = (uint64_t)a.tokens * a.heads;
  p.kv = blockIdx.x % a.kvh;
  p.row0 = blockIdx.x / a.kvh * rows;
  if constexpr (PREFIX) {
    if (!plan.sharing) return false;
    uint32_t n = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 64) {
      const bool shares = pages_request(a, r0 + lane).shares;
      const uint64_t m = __ballot(shares);
      if (tid < 64 && shares) list[n + (uint32_t)__popcll(m & ((1ull << lane) - 1))] = (uint16_t)(r0 + lane);
      n += (uint32_t)__popcll(m);
    }
    p.nrows = n * a.tokens * a.group;
    p.lo = min(blockIdx.y * a.per, a.shared);
    p.hi = min(p.lo + a.per, a.shared);
    p.r = a.owner; p.n = a.tokens; p.end0 = 0;
    p.table = a.table + (uint64_t)a.owner * a.max_pages;
    p.list = list;
    p.direct = false;
    p.part = a.slots * all + (uint64_t)blockIdx.y * a.requests * all;
    if (p.row0 >= p.nrows) return false;
    __syncthreads();
    return true;
  } else {
    const PagesChunks c = pages_chunks<false>(a, plan, blockIdx.y);
    if (c.r == 0xFFFFFFFFu) return false;
    const uint32_t at = blockIdx.y - c.first, keys = plan.chunk * a.unit;  // (chunks behind the first have keys: at * keys < len)
    p.nrows = c.n * a.group;
    p.lo = c.lo + at * keys;
    p.hi = c.len - p.lo < keys ? c.len : p.lo + keys;
    p.r = c.r; p.n = c.n; p.end0 = c.len - c.n + 1;
    p.table = a.table + (uint64_t)c.r * a.max_pages;
    p.list = nullptr;
    p.direct = c.count == 1 && !c.shares;
    p.part = blockIdx.y * all;
    if (at == 0) {  // rows of queries that are not there
      const uint32_t last = min(p.row0 + rows, a.tokens * a.group);
      for (uint32_t i = max(p.row0, p.nrows); i < last; i++)
        for (uint32_t d = tid; d < a.hd; d += NT)
          a.y[(((uint64_t)c.r * a.tokens + i / a.group) * a.heads + p.kv * a.group + i % a.group) * a.hd + d] = 0.f;
    }
    return p.row0 < p.nrows;
  }
}

template <class E, bool PREFIX>
__global__ __launch_bounds__(256) void k_pages_any(PagesK a, uint32_t T) {
  extern __shared__ float lds[];
  __shared__ uint16_t list[PREFIX ? WGD_REQUESTS_MAX : 1];
  PagesPart p;
  if (!pages_part<PREFIX, 256>(a, TREE_R, list, p)) return;
  pages_any<E, 256>(a, lds, T, p, p.row0);
}

// ------------------------------------------------------------------ the parts of a row
// A wavefront per row: the weights of its parts go over the lanes and LDS, then lanes take the dims.
constexpr uint32_t PAGES_TARGET = 512, PAGES_PREFIX = 256, PAGES_PARTS = PAGES_TARGET + 1 + PAGES_PREFIX;
__global__ __launch_bounds__(256) void k_pages_join(PagesK a) {
  __shared__ float weight[4][PAGES_PARTS];
  const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const uint64_t all = (uint64_t)a.tokens * a.heads, row = blockIdx.x * 4ull + wv;
  if (row >= a.requests * all) return;  // (no barriers below)
  const uint32_t r = (uint32_t)(row / all);
  const PagesPlan plan = pages_plan(a);
  const PagesChunks c = pages_chunks<true>(a, plan, r);
  if (row % all / a.heads >= c.n || (c.count == 1 && !c.shares)) return;
  const uint64_t pairs = pages_pairs(pages_part_rows(a.slots, a.nprefix, a.requests, all), a.hd);
  const uint32_t np = c.shares ? a.nprefix : 0, n = np + c.count;
  auto at = [&](uint32_t i) { return i < np ? a.slots * all + (uint64_t)i * a.requests * all + row : (c.first + i - np) * all + row % all; };
  float M = -INFINITY;
  bool seen = false;
  for (uint32_t i = lane; i < n; i += 64) {
    const float2 s = *(const float2 *)(a.part + pairs + 2 * at(i));
    if (!(s.y < 0.f)) { M = fmaxf(M, s.x); seen = true; }
  }
  M = wave_max(M);
  float sum = 0.f;
  for (uint32_t i = lane; i < n; i += 64) {
    const float2 s = *(const float2 *)(a.part + pairs + 2 * at(i));
    // (a sum of 0 is a part without a finite score: it adds nothing, and its values may be NaN)
    const float f = s.y < 0.f || s.y == 0.f ? 0.f : s.x == M ? 1.f : exp2f(s.x - M);
    weight[wv][i] = f;
    sum += s.y < 0.f || s.y == 0.f ? 0.f : s.y * f;
  }
  sum = wave_sum(sum);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const bool none = !__any(seen);
  for (uint32_t d = lane; d < a.hd; d += 64) {
    float acc = 0.f;
    for (uint32_t i = 0; i < n; i++)
      if (weight[wv][i] != 0.f) acc += a.part[at(i) * a.hd + d] * weight[wv][i];
    a.y[row * a.hd + d] = none ? 0.f : acc / sum;
  }
}

struct PagesLaunch { uint32_t T, rows, blocks, pblocks, unit, least, target, slots, nprefix, per; };
static PagesLaunch pages_launch(const PagesAttnArgs &in) {
  PagesLaunch p{};
  const uint32_t group = in.heads / in.kv_heads, cus = (uint32_t)device_cu_count();
  p.T = tree_any_tile(in.hd);
  p.rows = TREE_R;
  p.unit = p.T; p.least = 4;
  p.blocks = (in.tokens * group + p.rows - 1) / p.rows;
  const uint64_t longest = (uint64_t)in.max_pages << in.shift;
  const uint32_t wgs = in.kv_heads * p.blocks;
  p.target = std::max(1u, std::min(4 * cus / std::max(1u, wgs), PAGES_TARGET));
  // no request is cut where the longest is one chunk
  const uint64_t chunks = std::min<uint64_t>(p.target, (uint64_t)in.requests * ((longest + p.unit * p.least - 1) / (p.unit * p.least)));
  p.slots = (uint32_t)chunks + in.requests;
  if (in.shared && in.requests > 1) {
    p.pblocks = (uint32_t)(((uint64_t)in.requests * in.tokens * group + p.rows - 1) / p.rows);
    const uint32_t want = std::max(1u, std::min({4 * cus / std::max(1u, in.kv_heads * p.pblocks), in.shared / (p.unit * p.least) + 1, PAGES_PREFIX}));
    p.per = ((in.shared + want - 1) / want + p.unit - 1) / p.unit * p.unit;
    p.nprefix = (in.shared + p.per - 1) / p.per;
  }
  return p;
}
// Whether some row may have several parts.
static bool pages_joins(const PagesAttnArgs &in, const PagesLaunch &p) {
  return p.nprefix || ((uint64_t)in.max_pages << in.shift) > (uint64_t)p.unit * p.least;
}

uint64_t attention_pages_scratch_floats(const PagesAttnArgs &in) {
  if (!in.requests) return 0;
  const PagesLaunch p = pages_launch(in);
  if (!pages_joins(in, p)) return 0;
  const uint64_t rows = pages_part_rows(p.slots, p.nprefix, in.requests, (uint64_t)in.tokens * in.heads);
  return pages_pairs(rows, in.hd) + 2 * rows;
}

hipError_t attention_pages(hipStream_t s, const PagesAttnArgs &in) {
  if (!in.requests) return hipSuccess;
  if (!in.kv_heads || in.heads % in.kv_heads || !in.hd || in.hd > 512 || !in.window || !in.tokens || in.requests > WGD_REQUESTS_MAX ||
      in.partial_floats < attention_pages_scratch_floats(in))
    return hipErrorInvalidValue;
  const PagesLaunch p = pages_launch(in);
  PagesK a;
  a.q = in.q; a.k = in.k; a.v = in.v; a.y = in.y; a.part = in.partial; a.table = in.table; a.lengths = in.lengths; a.counts = in.counts;
  a.heads = in.heads; a.kvh = in.kv_heads; a.group = in.heads / in.kv_heads; a.hd = in.hd; a.window = in.window; a.shift = in.shift;
  a.max_pages = in.max_pages; a.pages = in.pages; a.requests = in.requests; a.tokens = in.tokens;
  a.shared = p.nprefix ? in.shared : 0; a.owner = in.owner;
  a.unit = p.unit; a.least = p.least; a.target = p.target; a.slots = p.slots; a.nprefix = p.nprefix; a.per = p.per; a.blocks = p.blocks;
  a.scale = in.scale;
  const size_t lds = tree_any_lds(in.hd, p.T);
  auto any = [&](auto kernel, uint32_t x, uint32_t y) {
    if (lds > 50000) lds_opt_in_bytes((const void *)kernel, 100000);
    hipLaunchKernelGGL(kernel, dim3(x, y), dim3(256), lds, s, a, p.T);
  };
  if (p.nprefix) {
    if (in.kv16) any(k_pages_any<_Float16, true>, in.kv_heads * p.pblocks, p.nprefix);
    else any(k_pages_any<float, true>, in.kv_heads * p.pblocks, p.nprefix);
    WGD_HIP(hipGetLastError());
  }
  if (in.kv16) any(k_pages_any<_Float16, false>, in.kv_heads * p.blocks, p.slots);
  else any(k_pages_any<float, false>, in.kv_heads * p.blocks, p.slots);
  WGD_HIP(hipGetLastError());
  if (!pages_joins(in, p)) return hipSuccess;
  const uint64_t rows = (uint64_t)in.requests * in.tokens * in.heads;
  hipLaunchKernelGGL(k_pages_join, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace wgd
