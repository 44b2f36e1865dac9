// attention_pages.h — attention of a batch of requests over K/V pages (part of attention.hip).
//
// Request r has lengths[r] tokens in the pages that its row of the table names, the last n_r of them (counts[r], at
// most `tokens`) with a query each: query t has the position p = lengths[r] - n_r + t and sees the keys (p - window, p]:
//   y = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m),  s_k = scale q . k_k,  m = max s_k.
// The lengths are on the device, so the work is shared out there: every wavefront forms the same plan from them.
// The keys of the requests are cut into about `target` chunks of similar length; a workgroup has one chunk, one kv head and
// some of the rows, the (query, head of the group) pairs that share the head's keys.
// Requests whose first `shared` tokens are the owner's have these computed together: the rows of all of them
// against the owner's keys, in `nprefix` parts. The parts of a row meet in k_pages_join, as (max, sum, weighted values).
#pragma once

namespace wgd {

struct PagesK {
  const float *q; const void *k, *v; float *y, *part; const int32_t *table, *lengths, *counts;
  uint32_t heads, kvh, group, hd, window, shift, max_pages, pages, requests, tokens, shared, owner;
  uint32_t unit, least, slots;          // keys of a unit (1 << unit); least units of a chunk; chunks at most
  float per_target;                     // 1 / the chunks wanted, rounded up
  uint32_t nprefix, per;                // parts of the prefix, keys of each
  float scale;
};

// The parts of the rows: [slot][token][head][hd] of the requests' own chunks, [part][request][token][head][hd] of the prefix, then from
// an even float on (max, sum) pairs in the same order. A sum below 0: the row sees nothing of the part.
__host__ __device__ __forceinline__ uint64_t pages_part_rows(uint32_t slots, uint32_t nprefix, uint32_t requests, uint64_t rows) {
  return ((uint64_t)slots + (uint64_t)nprefix * requests) * rows;
}
__host__ __device__ __forceinline__ uint64_t pages_pairs(uint64_t part_rows, uint32_t hd) { return (part_rows * hd + 1) / 2 * 2; }

// What lane-wide plans say of one request: its keys start at lo where it shares nothing.
struct PagesRequest { uint32_t len, n, lo; bool shares; };
struct PagesRaw { int32_t len, count, page; };      // as they are in memory
struct PagesOwner { uint32_t len; int32_t page; };  // of the prefix: its last page
__device__ __forceinline__ PagesRaw pages_raw(const PagesK &a, uint32_t r) {
  const uint32_t at = min(r, a.requests - 1);
  return PagesRaw{a.lengths[at], a.counts ? a.counts[at] : (int32_t)a.tokens, a.shared ? a.table[(uint64_t)at * a.max_pages + (a.shared >> a.shift) - 1] : 0};
}
__device__ __forceinline__ PagesOwner pages_owner(const PagesK &a) {
  if (!a.shared) return PagesOwner{0, 0};
  return PagesOwner{min((uint32_t)max(a.lengths[a.owner], 0), a.max_pages << a.shift), a.table[(uint64_t)a.owner * a.max_pages + (a.shared >> a.shift) - 1]};
}
__device__ __forceinline__ PagesRequest pages_request(const PagesK &a, const PagesOwner &o, const PagesRaw &raw, uint32_t r) {
  PagesRequest q = {0, 0, 0, false};
  if (r >= a.requests) return q;
  q.len = min((uint32_t)max(raw.len, 0), a.max_pages << a.shift);
  q.n = min(q.len, (uint32_t)min(max(raw.count, 0), (int32_t)a.tokens));
  const uint32_t first = q.len - q.n + 1;  // keys up to the first query's own
  q.lo = first > a.window ? first - a.window : 0;
  if (a.shift >= 4) q.lo &= ~15u;  // whole halves of blocks, on the same page; nothing before the first key is read
  q.shares = a.shared && o.len >= a.shared && q.n && q.len - q.n >= a.shared && q.len <= a.window && raw.page == o.page && o.page >= 0 && (uint32_t)o.page < a.pages;
  return q;
}
__device__ __forceinline__ uint32_t pages_units(const PagesK &a, const PagesRequest &q, bool sharing) {
  const uint32_t lo = sharing && q.shares ? a.shared : q.lo;
  return q.n ? (q.len - lo + (1u << a.unit) - 1) >> a.unit : 0;
}
// Sums over the lanes up to this one.
__device__ __forceinline__ uint32_t pages_sums(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast15 into rows 1 and 3
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // row_bcast31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ uint32_t pages_lane(uint32_t v, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane); }

// The plan of all requests: whether a prefix is shared (by two or more), and the units of a chunk. The first 64 PAGES_HELD requests
// are held in registers, their loads all under way at once; the others are loaded wherever they are asked for.
constexpr uint32_t PAGES_HELD = 1;  // (two or four, 128 or 256 requests, made every workgroup's plan 1 us longer)
struct PagesPlan { bool sharing; uint32_t chunk; PagesOwner owner; PagesRequest held[PAGES_HELD]; };
// what(r0, requests r0 .. + 64) for all, as long as it returns false.
template <class F> __device__ __forceinline__ void pages_each(const PagesK &a, const PagesPlan &p, F &&what) {
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (uint32_t e = 0; e < PAGES_HELD; e++) {
    if (64 * e >= a.requests) return;
    if (what(64 * e, p.held[e])) return;
  }
  for (uint32_t r0 = 64 * PAGES_HELD; r0 < a.requests; r0 += 64)
    if (what(r0, pages_request(a, p.owner, pages_raw(a, r0 + lane), r0 + lane))) return;
}
__device__ __forceinline__ PagesPlan pages_plan(const PagesK &a) {
  const uint32_t lane = threadIdx.x & 63;
  PagesPlan p;
  PagesRaw raw[PAGES_HELD];
#pragma unroll
  for (uint32_t e = 0; e < PAGES_HELD; e++)
    if (e == 0 || 64 * e < a.requests) raw[e] = pages_raw(a, 64 * e + lane);
  p.owner = pages_owner(a);
#pragma unroll
  for (uint32_t e = 0; e < PAGES_HELD; e++)
    if (e == 0 || 64 * e < a.requests) p.held[e] = pages_request(a, p.owner, raw[e], 64 * e + lane);
  float alone = 0.f, apart = 0.f;  // units; below 2^-19 off, which per_target makes up for
  uint32_t sharers = 0;
  pages_each(a, p, [&](uint32_t, const PagesRequest &q) {
    alone += wave_total((float)pages_units(a, q, false));
    if (a.shared) {
      apart += wave_total((float)pages_units(a, q, true));
      sharers += (uint32_t)__popcll(__ballot(q.shares));
    }
    return false;
  });
  p.sharing = sharers > 1;
  // rounded up, so that there are no more chunks than wanted, and one for each request
  const float even = ceilf((p.sharing ? apart : alone) * a.per_target);
  p.chunk = (uint32_t)__builtin_amdgcn_readfirstlane((int)max((uint32_t)fminf(even, 0x1p30f), a.least));
  return p;
}

// One request in the plan: the slot of its first chunk, their number, its keys [lo, len). It is the one that has the slot `find`,
// or with BY_REQUEST the request `find` itself. The same in all lanes.
struct PagesChunks { uint32_t r, first, count, lo, len, n; bool shares; };
template <bool BY_REQUEST>
__device__ __forceinline__ PagesChunks pages_chunks(const PagesK &a, const PagesPlan &plan, uint32_t find) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t before = 0;
  PagesChunks c = {0xFFFFFFFFu, 0, 0, 0, 0, 0, false};
  pages_each(a, plan, [&](uint32_t r0, const PagesRequest &q) {
    const uint32_t units = pages_units(a, q, plan.sharing);
    const uint32_t mine = r0 + lane < a.requests ? max(1u, (units + plan.chunk - 1) / plan.chunk) : 0;
    const uint32_t s = pages_sums(mine) + before;
    before = pages_lane(s, 63);
    const uint64_t here = __ballot(BY_REQUEST ? r0 + lane == find : find < s);  // the first of these
    if (!here) return false;
    const uint32_t at = (uint32_t)__ffsll((unsigned long long)here) - 1;
    c.r = r0 + at;
    c.count = pages_lane(mine, at);
    c.first = pages_lane(s, at) - c.count;
    c.shares = plan.sharing && (__ballot(q.shares) >> at & 1);
    c.lo = c.shares ? a.shared : pages_lane(q.lo, at);
    c.len = pages_lane(q.len, at);
    c.n = pages_lane(q.n, at);
    return true;
  });
  return c;
}

// A workgroup's part of the work: rows of kv head kv against the keys [lo, hi) of one row of the table. Row i of the part is
// (request, query, head): of one request, or of those that share the prefix (`list`, in LDS).
struct PagesPart {
  uint32_t kv, row0, nrows, lo, hi, seen;  // seen: the first key that a row sees, if that lies behind lo
  uint32_t r, n, end0;       // own chunks: the request, its queries, lengths - n + 1 (what query 0 sees of it)
  const int32_t *table;
  const uint16_t *list;      // the prefix: null otherwise
  bool direct;               // the only part of its rows: to y
  uint64_t part;             // else the first row of its part
};
// i / d by its reciprocal, for i <= 2^25 and d <= 2^20: the first estimate is off by 2^25 2^-22 at most, the second by one.
__device__ __forceinline__ uint32_t pages_div(uint32_t i, uint32_t d) {
  if (d == 1) return i;
  const float inv = __builtin_amdgcn_rcpf((float)d);
  uint32_t q = (uint32_t)((float)i * inv);
  q += (uint32_t)(int32_t)floorf((float)(int32_t)(i - q * d) * inv);
  q -= (int32_t)(i - q * d) < 0;
  return q + ((int32_t)(i - q * d) >= (int32_t)d);
}
struct PagesRow { bool valid; uint64_t row; uint32_t request, query, begin, end; };  // row of q and y; keys [begin, end)
__device__ __forceinline__ PagesRow pages_row(const PagesK &a, const PagesPart &p, uint32_t i) {
  PagesRow w = {i < p.nrows, 0, p.r, 0, 0, 0};
  if (!w.valid) return w;
  const uint32_t at = !p.list && a.tokens == 1 ? 0 : pages_div(i, a.group), head = i - at * a.group;
  uint32_t t = at;
  if (p.list) {
    const uint32_t u = pages_div(at, a.tokens);
    w.request = p.list[u];
    t = at - u * a.tokens;
    w.end = p.hi;
    w.valid = !a.counts || (int32_t)t < a.counts[w.request];
  } else {
    w.end = min(p.hi, p.end0 + t);
    w.begin = p.end0 + t > a.window ? p.end0 + t - a.window : 0;
    w.valid = t < p.n;
  }
  w.query = t;
  w.row = ((uint64_t)w.request * a.tokens + t) * a.heads + p.kv * a.group + head;
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

// The workgroup's part; false where it has none. PREFIX: (kv head, part) and the block of rows, else (kv head, block of rows) and a slot. `list` has WGD_REQUESTS_MAX
// places in LDS. Queries that a request does not have get zeros here, from its first chunk's workgroups of `rows` rows each.
template <bool PREFIX, uint32_t NT>
__device__ __forceinline__ bool pages_part(const PagesK &a, uint32_t rows, uint16_t *list, PagesPart &p) {
  const PagesPlan plan = pages_plan(a);
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint64_t all = (uint64_t)a.tokens * a.heads;
  // (row blocks of the prefix go last: a last one without rows would hold up others where they are dealt out)
  p.kv = blockIdx.x % a.kvh;
  p.row0 = (PREFIX ? blockIdx.y : blockIdx.x / a.kvh) * rows;
  if constexpr (PREFIX) {
    const uint32_t part = blockIdx.x / a.kvh;
    if (!plan.sharing) return false;
    uint32_t n = 0;
    pages_each(a, plan, [&](uint32_t r0, const PagesRequest &q) {
      const uint64_t m = __ballot(q.shares);
      if (tid < 64 && q.shares) list[n + (uint32_t)__popcll(m & ((1ull << lane) - 1))] = (uint16_t)(r0 + lane);
      n += (uint32_t)__popcll(m);
      return false;
    });
    p.nrows = n * a.tokens * a.group;
    p.lo = min(part * a.per, a.shared);
    p.hi = min(p.lo + a.per, a.shared);
    p.r = a.owner; p.n = a.tokens; p.end0 = 0; p.seen = 0;
    p.table = a.table + (uint64_t)a.owner * a.max_pages;
    p.list = list;
    p.direct = false;
    p.part = a.slots * all + (uint64_t)part * a.requests * all;
    if (p.row0 >= p.nrows) return false;
    __syncthreads();
    return true;
  } else {
    const PagesChunks c = pages_chunks<false>(a, plan, blockIdx.y);
    if (c.r == 0xFFFFFFFFu) return false;
    const uint32_t at = blockIdx.y - c.first, units = c.n ? (c.len - c.lo + (1u << a.unit) - 1) >> a.unit : 0;  // no fewer than chunks, or 0
    const uint32_t each = units / c.count, more = units - each * c.count;  // the first `more` chunks have one unit more
    p.nrows = c.n * a.group;
    p.lo = c.lo + ((at * each + min(at, more)) << a.unit);
    p.hi = at + 1 == c.count ? c.len : c.lo + (((at + 1) * each + min(at + 1, more)) << a.unit);
    p.r = c.r; p.n = c.n; p.end0 = c.len - c.n + 1;
    p.seen = p.end0 > a.window ? p.end0 - a.window : 0;
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

// ------------------------------------------------------------------ head dims up to 256, multiples of 8
//
// The page numbers of a workgroup's keys lie in LDS, PAGES_IDS at a time; blocks of keys go from the pages straight into matrix
// operands, as those of k_attn_tree do from a ring, each wavefront with its tile of 16 rows and every slices-th block. Pages
// of 16 tokens or more have the 16 keys of a half block one behind the other (all ranges begin at a multiple of 16 there): one
// number, a scalar, for the lot.
// A masked key's weight is exactly 0, but 0 times what is not finite is NaN, and the split operands turn infinities into it: a workgroup that
// ends with anything not finite, or that has a page that is none, forms its rows again with pages_any.
// What bounds k_pages: long caches, the bytes of the keys and values. 31 requests of 100 to 4000 keys, 32 heads on 8 of 128, f16 (271 MB): 61 us,
// 4.4 TB/s where a large copy has 4.8; 46% of a wavefront's life waits for loads, matrix products are at work for 6% of the cycles. Short
// ones, latency: 9 us for four requests of 40 to 500 f32 keys. A workgroup there has the plan for 2.8 us (lengths, then the sums over lanes), the
// page numbers for 1.1, and ends in 2.9.
constexpr uint32_t PAGES_IDS = 1024, PAGES_WG = 256;

// Which of the keys t0 .. + 32 (below hi) a row sees, as bits.
__device__ __forceinline__ uint32_t pages_mask(uint32_t begin, uint32_t end, uint32_t t0) {
  auto below = [&](uint32_t t) { return t <= t0 ? 0u : t - t0 >= 32 ? ~0u : (1u << (t - t0)) - 1; };
  return below(end) & ~below(begin);
}

// The numbers of the pages of [k0, k1) into ids; true in all threads if one of them is none.
template <uint32_t NT>
__device__ __forceinline__ bool pages_ids(const PagesK &a, const PagesPart &p, uint32_t *ids, uint32_t k0, uint32_t k1) {
  const uint32_t first = k0 >> a.shift, n = ((k1 - 1) >> a.shift) + 1 - first;
  int32_t id[PAGES_IDS / NT];
#pragma unroll
  for (uint32_t e = 0; e < PAGES_IDS / NT; e++)
    if (e == 0 || e * NT < n) id[e] = p.table[first + min(threadIdx.x + e * NT, n - 1)];
  bool none = false;
#pragma unroll
  for (uint32_t e = 0; e < PAGES_IDS / NT; e++)
    if (threadIdx.x + e * NT < n) {
      const bool ok = id[e] >= 0 && (uint32_t)id[e] < a.pages;
      none |= !ok;
      ids[threadIdx.x + e * NT] = ok ? (uint32_t)id[e] : 0;
    }
  return __syncthreads_or(none);
}

template <uint32_t HD, class E, bool FULL>
struct PagesWave : TreeWave<HD, E, FULL> {
  typedef TreeWave<HD, E, FULL> Wave;
  using Wave::NB, Wave::KT, Wave::VK, Wave::KEYS, Wave::NX, Wave::k, Wave::v, Wave::rowb, Wave::hi, Wave::k_piece, Wave::v_piece, Wave::k_row,
      Wave::v_row, Wave::kr;
  typedef typename Wave::vpiece vpiece;
  const uint32_t *ids;  // from page `first` on
  uint32_t first, shift, seen;
  vpiece vr[VK][NX];

  __device__ __forceinline__ uint64_t at(uint32_t t) const {  // of one key, the nearest of [seen, hi)
    t = min(max(t, seen), hi - 1);
    return (((uint64_t)ids[(t >> shift) - first] << shift) + (t & ((1u << shift) - 1))) * rowb;
  }
  __device__ __forceinline__ uint64_t half(uint32_t t) const {  // of 16 keys side by side
    const uint32_t id = __builtin_amdgcn_readfirstlane(ids[(t >> shift) - first]);
    return (((uint64_t)id << shift) + (t & ((1u << shift) - 1))) * rowb;
  }
  // Blocks of keys one behind the other, all there: 16 keys at a time on one page.
  __device__ __forceinline__ void load_k(uint32_t t) {
#pragma unroll
    for (uint32_t b = 0; b < NB; b++) {
      const uint8_t *row = k + half(t + 16 * b);
#pragma unroll
      for (uint32_t u = 0; u < KT; u++) kr[b][u] = *(const u32x4 *)(row + (k_row + k_piece[u]));
    }
  }
  __device__ __forceinline__ void load_v(uint32_t t) {
#pragma unroll
    for (uint32_t b = 0; b < NB; b++) {
      const uint8_t *rows = v + half(t + 16 * b);
#pragma unroll
      for (uint32_t j = 0; j < 4; j++)
#pragma unroll
        for (uint32_t x = 0; x < NX; x++) vr[4 * b + j][x] = *(const vpiece *)(rows + j * rowb + (v_row + v_piece[x]));
    }
  }
  // A block of any keys.
  __device__ __forceinline__ void load_any(uint32_t t) {
    const uint32_t c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (uint32_t b = 0; b < NB; b++) {
      const uint8_t *row = k + at(t + 16 * b + c);
#pragma unroll
      for (uint32_t u = 0; u < KT; u++) kr[b][u] = *(const u32x4 *)(row + k_piece[u]);
    }
#pragma unroll
    for (uint32_t j = 0; j < VK; j++) {
      const uint8_t *row = v + at(t + 16 * (j / 4) + 4 * g + j % 4);
#pragma unroll
      for (uint32_t x = 0; x < NX; x++) vr[j][x] = *(const vpiece *)(row + v_piece[x]);
    }
  }
  // A query's dims as the operands need them, zero where ok is off (the place is there all the same).
  static constexpr uint32_t QN = Wave::HALF ? 2 * KT : KT;
  __device__ __forceinline__ void ask_q(const float *q, uint32_t hd, f32x4 (&x)[QN]) const {
    const uint32_t g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (uint32_t t = 0; t < QN; t++) x[t] = *(const f32x4 *)(q + piece(t, g, FULL ? HD : hd));
  }
  static __device__ __forceinline__ uint32_t piece(uint32_t t, uint32_t g, uint32_t hd) {
    const uint32_t d = Wave::HALF ? 32 * (t / 2) + 8 * g + 4 * (t % 2) : 16 * t + 4 * g;
    return FULL ? d : min(d, hd - 4);
  }
  __device__ __forceinline__ void take_q(f32x4 (&x)[QN], float scale, uint32_t hd, bool ok) {
    const uint32_t g = (threadIdx.x & 63) >> 4;
    const float f = scale * TREE_LOG2E;
#pragma unroll
    for (uint32_t t = 0; t < QN; t++) {
      const bool there = ok && (FULL || piece(t, g, hd) == (Wave::HALF ? 32 * (t / 2) + 8 * g + 4 * (t % 2) : 16 * t + 4 * g));
      x[t] = there ? x[t] : f32x4{0, 0, 0, 0};
    }
    if constexpr (Wave::HALF) {
      this->qs = tree_query_of<KT>(x, f, this->qh, this->ql);
    } else {
#pragma unroll
      for (uint32_t t = 0; t < KT; t++) this->qh[t] = __builtin_bit_cast(u32x4, f32x4{x[t].x * f, x[t].y * f, x[t].z * f, x[t].w * f});
      this->qs = 1.f;
    }
  }
  __device__ __forceinline__ bool whole(uint32_t t) const { return shift >= 4 && t >= seen && t + KEYS <= hi; }
  // Asks for the block at t0.
  __device__ __forceinline__ void start(uint32_t t0) {
    if (whole(t0)) {
      load_k(t0);
      load_v(t0);
    } else {
      load_any(t0);
    }
  }
  // Keys [t0, hi) in steps of `step`; the row sees [begin, end), all rows of the wavefront [all_begin, all_end).
  // The keys and values of a block are asked for while the one before is at work, with no load behind a branch: what waits for one
  // would wait for all.
  __device__ __forceinline__ void walk(uint32_t t0, uint32_t step, uint32_t begin, uint32_t end, uint32_t all_begin, uint32_t all_end) {
    f32x4 s[NB];
    auto weights = [&](uint32_t t) {
      const bool masked = t + KEYS > min(hi, all_end) || t < all_begin;
      this->weigh(0, s, this->qs, masked, masked ? pages_mask(begin, min(end, hi), t) : 0);
    };
    while (t0 < hi) {
      start(t0);
      const uint32_t last = whole(t0) ? t0 + (hi - KEYS - t0) / step * step : t0;
      for (; t0 < last; t0 += step) {
        this->scores(s);
        load_k(t0 + step);
        weights(t0);
        this->values(vr, s);
        load_v(t0 + step);
      }
      this->scores(s);
      weights(t0);
      this->values(vr, s);
      t0 += step;
    }
  }
};

// The end of a workgroup: the slices of its wavefronts merge in LDS, and the rows go to y or to their parts. wave w has the rows row0 + (w % rw) *
// 16 RT .. and the slice w / rw. With anything not finite, or `again`, the rows are formed again.
template <uint32_t HD, class E, uint32_t RT, uint32_t NT, class Rows>
__device__ __forceinline__ void pages_end(const PagesK &a, uint32_t rw, float *lds, const PagesPart &p, const Rows &s, bool again) {
  constexpr uint32_t VE = Rows::VE, NX = Rows::NX, OS = HD + 4, WS = RT * 16 * (OS + 2);
  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15, slices = NT / 64 / rw;
  if (__syncthreads_or(again || !s.finite())) {
    for (uint32_t i = 0; i < rw * RT; i++)
      if (p.row0 + 16 * i < p.nrows) pages_any<E, NT>(a, lds, tree_any_tile(HD), p, p.row0 + 16 * i);
    return;
  }
  // ---- to LDS: where the rows go (in floats; ~0: nowhere), and whether they see anything; [row] max, sum; [row][HD]
  __shared__ uint64_t place[128];
  __shared__ uint32_t sees_any[4];
  const uint32_t rows = rw * RT * 16;
  if (tid < 128) {
    const PagesRow w = pages_row(a, p, p.row0 + tid);
    const bool ok = tid < rows && w.valid;
    place[tid] = ok ? (p.direct ? w.row : pages_at(a, p, w)) : ~0ull;
    const uint64_t m = __ballot(ok && w.begin < p.hi && w.end > p.lo);
    if (lane == 0) { sees_any[tid / 32] = (uint32_t)m; sees_any[tid / 32 + 1] = (uint32_t)(m >> 32); }
  }
  float *mine = lds + (tid >> 6) * WS;
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
    float l = s.l[rt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) { mine[2 * (16 * rt + c)] = s.m[rt]; mine[2 * (16 * rt + c) + 1] = l; }
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
  const uint64_t pairs = pages_pairs(pages_part_rows(a.slots, a.nprefix, a.requests, (uint64_t)a.tokens * a.heads), a.hd);
  for (uint32_t i = tid; i < rows * (HD / 8); i += NT) {
    const uint32_t d = i % (HD / 8) * 8, at_row = i / (HD / 8), lr = at_row % (RT * 16), rg = at_row / (RT * 16);
    const uint64_t go = place[at_row];
    if (go == ~0ull || d >= a.hd) continue;
    float M = -INFINITY, l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t u = 0; u < slices; u++) M = fmaxf(M, lds[(u * rw + rg) * WS + 2 * lr]);
    for (uint32_t u = 0; u < slices; u++) {
      const float *at = lds + (u * rw + rg) * WS;
      if (at[2 * lr + 1] == 0.f) continue;  // nothing seen
      const float f = at[2 * lr] == M ? 1.f : __builtin_amdgcn_exp2f(at[2 * lr] - M);
      l += at[2 * lr + 1] * f;
      const f32x4 x0 = *(const f32x4 *)(at + RT * 32 + lr * OS + d), x1 = *(const f32x4 *)(at + RT * 32 + lr * OS + d + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) { y[e] += x0[e] * f; y[4 + e] += x1[e] * f; }
    }
    float *to = (p.direct ? a.y : a.part) + go * a.hd + d;
    const float inv = p.direct ? 1.f / l : 1.f;  // (a row sees its own key at least)
    if (!p.direct && d == 0)
      *(float2 *)(a.part + pairs + 2 * go) = make_float2(M - TREE_BIAS, sees_any[at_row / 32] >> (at_row % 32) & 1 ? l : -1.f);
#pragma unroll
    for (int e = 0; e < 8; e += 4) *(f32x4 *)(to + e) = f32x4{y[e] * inv, y[e + 1] * inv, y[e + 2] * inv, y[e + 3] * inv};
  }
}

// What a lane's row sees, and all rows of its wavefront.
struct PagesSees { uint32_t begin, end, all_begin, all_end; };
__device__ __forceinline__ PagesSees pages_sees(const PagesRow &w) {
  PagesSees s = {w.valid ? w.begin : 0u, w.valid ? w.end : 0u, w.valid ? w.begin : 0u, w.valid ? w.end : ~0u};
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    s.all_begin = max(s.all_begin, (uint32_t)__shfl_xor((int)s.all_begin, o, 64));
    s.all_end = min(s.all_end, (uint32_t)__shfl_xor((int)s.all_end, o, 64));
  }
  s.all_begin = __builtin_amdgcn_readfirstlane(s.all_begin);
  s.all_end = __builtin_amdgcn_readfirstlane(s.all_end);
  return s;
}

template <uint32_t HD, class E, bool FULL, bool PREFIX>
__global__ __launch_bounds__(PAGES_WG, HD == 256 ? 1 : 2) void k_pages(PagesK a, uint32_t rw) {
  constexpr uint32_t NT = PAGES_WG;
  typedef PagesWave<HD, E, FULL> Wave;
  extern __shared__ float lds[];
  __shared__ uint16_t list[PREFIX ? WGD_REQUESTS_MAX : 1];
  __shared__ uint32_t ids[PAGES_IDS];
  PagesPart p;
  if (!pages_part<PREFIX, NT>(a, 16 * rw, list, p)) return;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slice = w / rw, wrow = p.row0 + w % rw * 16;
  const PagesRow row = pages_row(a, p, wrow + (threadIdx.x & 15));
  const PagesSees sees = pages_sees(row);
  Wave s;
  f32x4 q[Wave::QN];
  s.ask_q(a.q + row.row * a.hd, a.hd, q);
  s.place(a.k, a.v, a.kvh, a.hd, p.kv);
  s.clear();
  s.ids = ids; s.shift = a.shift; s.seen = p.seen;
  const uint32_t step = NT / 64 / rw * Wave::KEYS;
  auto numbers = [&](uint32_t k0) {
    s.first = k0 >> a.shift;
    s.hi = min((uint64_t)p.hi, (uint64_t)(s.first + PAGES_IDS) << a.shift);
    return pages_ids<NT>(a, p, ids, k0, s.hi);
  };
  bool none = numbers(p.lo);
  s.take_q(q, a.scale, a.hd, row.valid);
  auto walk = [&](uint32_t k0) {
    if (wrow < p.nrows) s.walk(k0 + slice * Wave::KEYS, step, sees.begin, sees.end, sees.all_begin, sees.all_end);
  };
  if constexpr (PREFIX) {  // (the numbers of a part fit, pages_launch())
    if (!none) walk(p.lo);
  } else {
    for (uint32_t k0 = p.lo; !none;) {
      walk(k0);
      k0 = s.hi;
      if (k0 >= p.hi) break;
      __syncthreads();
      none = numbers(k0);
    }
  }
  pages_end<HD, E, 1, NT>(a, rw, lds, p, s, none);
}

// ------------------------------------------------------------------ many rows over halves: keys staged in LDS
// As k_attn_tree_staged: eight wavefronts load stages of SK keys into LDS while they work on the one before. For 128 rows of a kv head
// and more, whose workgroups would each read all keys again. What bounds it: a prefix of 8192 keys under 64 requests, 32 heads on 8 of 128, takes
// 36 us, 480 TFLOP/s with both products of the split operands; a workgroup's stage of 128 keys takes 4.4 us (two fifths of it matrix products, then the
// weights and their split, LDS, the barrier), what comes before its first stage 10 and the end 7.
template <uint32_t HD, uint32_t RT, uint32_t SK, bool PREFIX>
__global__ __launch_bounds__(TREE_STAGED_NT) void k_pages_staged(PagesK a, uint32_t rw) {
  typedef TreeStaged<HD, RT> Wave;
  constexpr uint32_t ROW = Wave::ROW, CH = Wave::CH, NT = TREE_STAGED_NT, STEP = NT / CH;
  extern __shared__ float lds[];
  __shared__ uint16_t list[PREFIX ? WGD_REQUESTS_MAX : 1];
  __shared__ uint32_t ids[PAGES_IDS];
  PagesPart p;
  if (!pages_part<PREFIX, NT>(a, 16 * RT * rw, list, p)) return;
  const uint32_t tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), slice = w / rw, slices = NT / 64 / rw;
  const uint32_t wrow = p.row0 + w % rw * 16 * RT, pg = (1u << a.shift) - 1;
  uint8_t *stages = (uint8_t *)lds;
  const uint64_t rowb = (uint64_t)a.kvh * ROW, head = (uint64_t)p.kv * ROW;
  const uint8_t *k = (const uint8_t *)a.k + head, *v = (const uint8_t *)a.v + head;
  const uint32_t key0 = tid / CH, k_place = (tid % CH ^ Wave::k_swizzle(key0)) * 16, v_place = (tid % CH ^ Wave::v_swizzle(key0)) * 16;
  static_assert(STEP % 16 == 0, "the swizzles repeat after 16 keys");
  uint32_t first = 0, hi = 0;
  auto load = [&](uint32_t t0, uint32_t s) {
    uint8_t *K = stages + s * 2 * SK * ROW + 1024 * w, *V = K + SK * ROW;
    auto put = [](const uint8_t *from, uint8_t *to) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    };
    uint64_t at[SK / STEP];
#pragma unroll
    for (uint32_t n = 0; n < SK / STEP; n++) {
      const uint32_t t = min(max(t0 + key0 + n * STEP, p.seen), hi - 1);
      at[n] = (((uint64_t)ids[(t >> a.shift) - first] << a.shift) + (t & pg)) * rowb;
    }
#pragma unroll
    for (uint32_t n = 0; n < SK / STEP; n++) {
      put(k + at[n] + k_place, K + n * STEP * ROW);
      put(v + at[n] + v_place, V + n * STEP * ROW);
    }
  };
  PagesSees sees[RT];
  Wave s;
  s.clear();
  f32x4 q[RT][2 * Wave::KT];
  bool valid[RT];
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
    const PagesRow row = pages_row(a, p, wrow + 16 * rt + (tid & 15));
    sees[rt] = pages_sees(row);
    valid[rt] = row.valid;
#pragma unroll
    for (uint32_t t = 0; t < 2 * Wave::KT; t++) q[rt][t] = *(const f32x4 *)(a.q + row.row * HD + 32 * (t / 2) + 8 * ((tid & 63) >> 4) + 4 * (t % 2));
  }
  uint32_t all_begin = 0, all_end = ~0u;
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) { all_begin = max(all_begin, sees[rt].all_begin); all_end = min(all_end, sees[rt].all_end); }
  auto numbers = [&](uint32_t k0) {
    first = k0 >> a.shift;
    hi = min((uint64_t)p.hi, (uint64_t)(first + PAGES_IDS) << a.shift);
    return pages_ids<NT>(a, p, ids, k0, hi);
  };
  bool none = numbers(p.lo);
#pragma unroll
  for (uint32_t rt = 0; rt < RT; rt++) {
#pragma unroll
    for (uint32_t t = 0; t < 2 * Wave::KT; t++) q[rt][t] = valid[rt] ? q[rt][t] : f32x4{0, 0, 0, 0};
    s.qs[rt] = tree_query_of<Wave::KT>(q[rt], a.scale * TREE_LOG2E, s.qh[rt], s.ql[rt]);
  }
  auto walk = [&](uint32_t k0) {
    load(k0, 0);
    uint32_t stage = 0;
    for (uint32_t t0 = k0; t0 < hi; t0 += SK, stage ^= 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's loads into the stage
      __syncthreads();                                   // everyone's; and the other stage is no longer read
      if (t0 + SK < hi) load(t0 + SK, stage ^ 1);
      const uint8_t *K = stages + stage * 2 * SK * ROW, *V = K + SK * ROW;
      if (wrow < p.nrows)
        for (uint32_t b = slice; b < SK / 32 && t0 + 32 * b < hi; b += slices) {
          const uint32_t t = t0 + 32 * b;
          s.block(K + 32 * b * ROW, V + 32 * b * ROW, t + 32 > min(hi, all_end) || t < all_begin,
                  [&](uint32_t rt) { return pages_mask(sees[rt].begin, min(sees[rt].end, hi), t); });
        }
    }
  };
  if constexpr (PREFIX) {  // (the numbers of a part fit, pages_launch())
    if (!none) walk(p.lo);
  } else {
    for (uint32_t k0 = p.lo; !none;) {
      walk(k0);
      k0 = hi;
      if (k0 >= p.hi) break;
      __syncthreads();  // the numbers and both stages are no longer read
      none = numbers(k0);
    }
  }
  pages_end<HD, _Float16, RT, NT>(a, rw, lds, p, s, none);
}

// ------------------------------------------------------------------ the parts of a row
// A wavefront per row: the weights of its parts go over the lanes and LDS, then lane groups of hd / 4 (VEC: hd a power of two from 4) take every
// (64 / group)-th part, 16 bytes a lane and four loads ahead. Bound by latency: the plan, the pairs, the values. 4.3 us for 64 rows of 128 and for 1024,
// 7.9 for 2112 with 16 to 20 parts each.
constexpr uint32_t PAGES_TARGET = 512, PAGES_PREFIX = 256, PAGES_PARTS = PAGES_TARGET + 1 + PAGES_PREFIX;
template <bool VEC>
__global__ __launch_bounds__(256) void k_pages_join(PagesK a) {
  __shared__ float weight[4][PAGES_PARTS];
  const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const uint32_t all = a.tokens * a.heads, row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wv);
  if (row >= a.requests * all) return;  // (no barriers below)
  const uint32_t r = row / all, within = row - r * all;
  const PagesPlan plan = pages_plan(a);
  const PagesChunks c = pages_chunks<true>(a, plan, r);
  if (within >= c.n * a.heads || (c.count == 1 && !c.shares)) return;
  const uint64_t pairs = pages_pairs(pages_part_rows(a.slots, a.nprefix, a.requests, all), a.hd);
  const uint32_t np = c.shares ? a.nprefix : 0, n = np + c.count;
  auto at = [&](uint32_t i) { return i < np ? (uint64_t)a.slots * all + (uint64_t)i * a.requests * all + row : (uint64_t)(c.first + i - np) * all + within; };
  float2 mine = make_float2(-INFINITY, -1.f);
  if (lane < n) mine = *(const float2 *)(a.part + pairs + 2 * at(lane));
  auto pair = [&](uint32_t i) { return i < 64 ? mine : *(const float2 *)(a.part + pairs + 2 * at(i)); };
  float M = -INFINITY;
  bool seen = false;
  for (uint32_t i = lane; i < n; i += 64) {
    const float2 s = pair(i);
    if (!(s.y < 0.f)) { M = fmaxf(M, s.x); seen = true; }
  }
  M = wave_max(M);
  float sum = 0.f;
  for (uint32_t i = lane; i < n; i += 64) {
    const float2 s = pair(i);
    // (a part that the row sees nothing of has zeros; a weight of 0 is multiplied as any other, so that values that are not finite stay so)
    const float f = s.y < 0.f ? 0.f : s.x == M ? 1.f : exp2f(s.x - M);
    weight[wv][i] = f;
    sum += s.y < 0.f ? 0.f : s.y * f;
  }
  sum = wave_sum(sum);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const bool none = !__any(seen);
  if constexpr (VEC) {
    const uint32_t width = a.hd / 4, groups = width < 64 ? 64 / width : 1, per = 64 / groups, z0 = lane / per, d0 = lane % per;  // groups: a power of two
    for (uint32_t d = 4 * d0; d < a.hd; d += 4 * per) {
      f32x4 acc = {0, 0, 0, 0};
      for (uint32_t i0 = z0; i0 < n; i0 += 4 * groups) {
        f32x4 v[4];
        float f[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const uint32_t i = i0 + e * groups;
          f[e] = i < n ? weight[wv][i] : 0.f;
          v[e] = *(const f32x4 *)(a.part + at(min(i, n - 1)) * a.hd + d);
        }
#pragma unroll
        for (uint32_t e = 0; e < 4; e++)
          if (i0 + e * groups < n) acc += v[e] * f[e];
      }
      for (uint32_t o = per; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], o, 64);
      if (z0 == 0) *(f32x4 *)(a.y + (uint64_t)row * a.hd + d) = none ? f32x4{0, 0, 0, 0} : f32x4{acc.x / sum, acc.y / sum, acc.z / sum, acc.w / sum};
    }
  } else {
    for (uint32_t d = lane; d < a.hd; d += 64) {
      float acc = 0.f;
      for (uint32_t i = 0; i < n; i++) acc += a.part[at(i) * a.hd + d] * weight[wv][i];
      a.y[(uint64_t)row * a.hd + d] = none ? 0.f : acc / sum;
    }
  }
}

// The kernels of a call. mfma: matrix products; HD: the head dim padded to 64, 128 or 256; rows: of a workgroup, blocks and pblocks how
// many that makes of a request and of all of them together.
struct PagesLaunch { bool mfma, staged, pstaged; uint32_t HD, T, rw, prw, rows, prows, blocks, pblocks, unit, least, target, slots, nprefix, per; };  // unit: keys
static PagesLaunch pages_launch(const PagesAttnArgs &in) {
  PagesLaunch p{};
  const uint32_t group = in.heads / in.kv_heads, cus = (uint32_t)device_cu_count(), nrows = in.tokens * group;
  const uint64_t longest = (uint64_t)in.max_pages << in.shift, prows = (uint64_t)in.requests * nrows;
  // (a lane's offsets within 16 rows of a page are 32-bit)
  p.mfma = in.hd % 8 == 0 && in.hd <= 256 && (uint64_t)in.kv_heads * in.hd * 4 < (1u << 27);
  p.HD = in.hd <= 64 ? 64 : in.hd <= 128 ? 128 : 256;
  const bool can_stage = p.mfma && in.kv16 && in.hd == p.HD;
  auto shape = [&](uint64_t n, bool &staged, uint32_t &rw, uint32_t &rows) {
    if (!p.mfma) { rows = TREE_R; rw = 1; return; }
    const uint64_t tiles = (n + 15) / 16;
    staged = can_stage && tiles >= 8;
    const uint32_t RT = staged && p.HD <= 128 ? 2 : 1;
    const uint64_t groups = (tiles + RT - 1) / RT;
    rw = groups >= 4 ? 4 : groups >= 2 ? 2 : 1;
    rows = 16 * RT * rw;
  };
  shape(nrows, p.staged, p.rw, p.rows);
  p.blocks = (nrows + p.rows - 1) / p.rows;
  p.T = tree_any_tile(in.hd);
  // Chunks: about four workgroups a CU (two are there at a time), of one step of all wavefronts at least. us, 31 requests of 100 to 4000 keys,
  // 32 heads on 8 of 128, f16, by workgroups wanted a CU: 1: 73, 2: 66, 3: 63, 4: 61, 8: 62; with workgroups of 512 threads 70 to 77, of 128 the
  // same. Four requests of 40 to 500 f32 keys, 8 kv heads: chunks of one step 9.0, two 10.8, four 13.
  p.unit = !p.mfma ? p.T : p.staged ? 128 : (in.kv16 ? 32 : 16) * (PAGES_WG / 64 / p.rw);
  p.least = p.mfma ? 1 : 4;
  const uint32_t wgs = in.kv_heads * p.blocks;
  // Staged workgroups have a CU to themselves: all of them at once where the requests are few enough for that (every one rounds its
  // chunks up, by half of one on average). us, times as many as CUs in all, 1: 2: the rule; 32 heads on 8 of 128, 128 tokens of 1 request, 4000 keys,
  // 36, 51, 36; 4 requests of up to 4000 77, 77, 68; 64 tokens of 8 of up to 8000 142, 140, 116. 128 of 16 of up to 2000 131, 127, 127.
  const uint32_t at_once = cus / std::max(1u, wgs);
  if (p.staged) p.target = in.requests <= at_once ? at_once - in.requests / 2 : 2 * cus / std::max(1u, wgs);
  else p.target = (p.HD == 256 ? 2 : 4) * cus / std::max(1u, wgs);
  p.target = std::max(1u, std::min(p.target, PAGES_TARGET));
  // no request is cut where the longest is one chunk
  const uint64_t chunks = std::min<uint64_t>(p.target, (uint64_t)in.requests * ((longest + p.unit * p.least - 1) / (p.unit * p.least)));
  p.slots = (uint32_t)chunks + in.requests;
  if (in.shared && in.requests > 1) {
    shape(prows, p.pstaged, p.prw, p.prows);
    p.pblocks = (uint32_t)((prows + p.prows - 1) / p.prows);
    // Parts by estimated time, us: a workgroup starts and ends in 4.5 and works 2.1 (f16) or 3.1 (f32) for a block of each slice; a part is
    // written and read once more. A last block of rows that may have few of them counts as none. 64 of 66 requests, 32 heads on 8 of 128, 8192
    // keys: 4 parts 75, 8 49, 10 46, 16 36 us (as many workgroups as CUs), 32 73.
    const uint32_t unit = std::max(!p.mfma ? p.T : p.pstaged ? 128 : (in.kv16 ? 32 : 16) * (PAGES_WG / 64 / p.prw), 1u << in.shift);
    const uint32_t slices = p.pstaged ? 8 / p.prw : PAGES_WG / 64 / p.prw, block = in.kv16 ? 32 : 16;
    const uint64_t wgs = in.kv_heads * std::max<uint64_t>(1, (prows + p.prows / 4) / p.prows);
    const double held = (double)in.requests * in.tokens * in.heads * in.hd * 8 / 4e6;
    double best = 1e30;
    // (a launch has at most 65535 blocks of rows along y, and fewer than 2^32 threads along x)
    const uint64_t threads = (uint64_t)in.kv_heads * (p.pstaged ? TREE_STAGED_NT : PAGES_WG);
    for (uint32_t n = 1; p.pblocks <= 65535 && n <= PAGES_PREFIX && threads * n <= 0xFFFFFFFFull && (uint64_t)(n - 1) * unit < in.shared; n++) {
      const uint32_t per = ((in.shared + n - 1) / n + unit - 1) / unit * unit, parts = (in.shared + per - 1) / per;
      if (parts < n || (p.mfma && per >> in.shift >= PAGES_IDS)) continue;  // (too many parts for that: computed apart)
      const double work = p.mfma ? (in.kv16 ? 2.1 : 3.1) * ((per + block * slices - 1) / (block * slices)) : 0.5 * per;
      const double t = (double)((wgs * n + (p.pstaged ? 1 : 2) * cus - 1) / ((p.pstaged ? 1 : 2) * cus)) * (4.5 + work) + held * n;
      if (t < best) { best = t; p.per = per; p.nprefix = parts; }
    }
  }
  return p;
}
// Whether some row may have several parts: with one chunk wanted each request is one (pages_plan() rounds up).
static bool pages_joins(const PagesAttnArgs &in, const PagesLaunch &p) {
  return p.nprefix || (p.target > 1 && ((uint64_t)in.max_pages << in.shift) > (uint64_t)p.unit * p.least);
}

uint64_t attention_pages_scratch_floats(const PagesAttnArgs &in) {
  if (!in.requests) return 0;
  const PagesLaunch p = pages_launch(in);
  if (!pages_joins(in, p)) return 0;
  const uint64_t rows = pages_part_rows(p.slots, p.nprefix, in.requests, (uint64_t)in.tokens * in.heads);
  return pages_pairs(rows, in.hd) + 2 * rows;
}

template <bool PREFIX> static dim3 pages_grid(const PagesK &a, const PagesLaunch &p) {
  return PREFIX ? dim3(a.kvh * p.nprefix, p.pblocks) : dim3(a.kvh * p.blocks, p.slots);
}
template <bool PREFIX, class E>
static void launch_pages_any(hipStream_t s, const PagesK &a, const PagesLaunch &p) {
  const size_t lds = tree_any_lds(a.hd, p.T);
  if (lds > 50000) lds_opt_in_bytes((const void *)k_pages_any<E, PREFIX>, 100000);
  hipLaunchKernelGGL((k_pages_any<E, PREFIX>), pages_grid<PREFIX>(a, p), dim3(256), lds, s, a, p.T);
}
template <uint32_t HD, class E, bool FULL, bool PREFIX>
static void launch_pages_direct(hipStream_t s, const PagesK &a, const PagesLaunch &p) {
  constexpr uint32_t waves = PAGES_WG / 64;
  constexpr size_t lds = std::max(tree_wave_lds<HD, 1>() * waves, tree_any_lds(HD, tree_any_tile(HD)));
  static_assert(lds + 4 * PAGES_IDS + 2 * WGD_REQUESTS_MAX + 1024 <= LDS_MAX, "the wavefronts' outputs fit LDS");
  lds_opt_in_bytes((const void *)k_pages<HD, E, FULL, PREFIX>, (uint32_t)lds);
  hipLaunchKernelGGL((k_pages<HD, E, FULL, PREFIX>), pages_grid<PREFIX>(a, p), dim3(64 * waves), lds, s,
                     a, PREFIX ? p.prw : p.rw);
}
template <uint32_t HD, bool PREFIX>
static void launch_pages_staged(hipStream_t s, const PagesK &a, const PagesLaunch &p) {
  constexpr uint32_t RT = HD == 256 ? 1 : 2, SK = HD == 256 ? 64 : 128, waves = TREE_STAGED_NT / 64;
  constexpr size_t lds = std::max({tree_wave_lds<HD, RT>() * waves, tree_any_lds(HD, tree_any_tile(HD)), (size_t)4 * SK * 2 * HD});
  static_assert(lds + 4 * PAGES_IDS + 2 * WGD_REQUESTS_MAX + 1024 <= LDS_MAX, "two stages, and the wavefronts' outputs, fit LDS");
  lds_opt_in_bytes((const void *)k_pages_staged<HD, RT, SK, PREFIX>, (uint32_t)lds);
  hipLaunchKernelGGL((k_pages_staged<HD, RT, SK, PREFIX>), pages_grid<PREFIX>(a, p), dim3(TREE_STAGED_NT),
                     lds, s, a, PREFIX ? p.prw : p.rw);
}
template <uint32_t HD, class E, bool PREFIX>
static void launch_pages_hd(hipStream_t s, const PagesK &a, const PagesLaunch &p) {
  if (a.hd < HD) return launch_pages_direct<HD, E, false, PREFIX>(s, a, p);
  if constexpr (sizeof(E) == 2)
    if (PREFIX ? p.pstaged : p.staged) return launch_pages_staged<HD, PREFIX>(s, a, p);
  launch_pages_direct<HD, E, true, PREFIX>(s, a, p);
}
template <class E, bool PREFIX>
static void launch_pages(hipStream_t s, const PagesK &a, const PagesLaunch &p) {
  if (!p.mfma) launch_pages_any<PREFIX, E>(s, a, p);
  else if (p.HD == 64) launch_pages_hd<64, E, PREFIX>(s, a, p);
  else if (p.HD == 128) launch_pages_hd<128, E, PREFIX>(s, a, p);
  else launch_pages_hd<256, E, PREFIX>(s, a, p);
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
  a.unit = (uint32_t)__builtin_ctz(p.unit); a.least = p.least; a.slots = p.slots; a.nprefix = p.nprefix; a.per = p.per;
  a.per_target = (float)((1.0 + 0x1p-18) / p.target);
  a.scale = in.scale;
  if (p.nprefix) {
    in.kv16 ? launch_pages<_Float16, true>(s, a, p) : launch_pages<float, true>(s, a, p);
    WGD_HIP(hipGetLastError());
  }
  in.kv16 ? launch_pages<_Float16, false>(s, a, p) : launch_pages<float, false>(s, a, p);
  WGD_HIP(hipGetLastError());
  if (!pages_joins(in, p)) return hipSuccess;
  const uint64_t rows = (uint64_t)in.requests * in.tokens * in.heads;
  const dim3 grid((uint32_t)((rows + 3) / 4));
  if (in.hd >= 4 && (in.hd & (in.hd - 1)) == 0) hipLaunchKernelGGL(k_pages_join<true>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_pages_join<false>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace wgd
