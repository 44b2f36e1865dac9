// pages.h — K/V caches in pages that requests share: places for new tokens, forks, compaction, and the moves of pages
// and rows that these ask for (part of ops.hip; include/wgd.h, "many requests").
//
// The state is three int32 arrays: table[request][column] names the page of a request's tokens column * page .. + page,
// lengths[request] its tokens, refs[page] the rows of the table (and the caller's own lists) that hold a page; 0 and
// below is free. All choices go by the lowest number, so the result does not depend on the order of threads: the
// counts are changed by integer atomics, whose sum has no order.
// What bounds the three that change the state is latency: loads that depend on one another, scans, barriers.
#pragma once

namespace wgd {

constexpr uint32_t PAGES_NT = 1024;  // threads of the workgroup that sees all requests
static_assert(WGD_REQUESTS_MAX <= PAGES_NT, "a thread per request");

// Exclusive sum over the PAGES_NT threads of a workgroup; `lds` holds PAGES_NT / 64 + 1 words.
__device__ __forceinline__ uint32_t pages_scan(uint32_t v, uint32_t *lds, uint32_t &total) {
  const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint32_t u = (uint32_t)__shfl_up((int)s, o, 64);
    if (lane >= (uint32_t)o) s += u;
  }
  __syncthreads();
  if (lane == 63) lds[wv] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < PAGES_NT / 64; w++) {
    before += w < wv ? lds[w] : 0;
    all += lds[w];
  }
  total = all;
  return before + s - v;
}

// Pages of a thread at a time: 1, 4 or 16, so that all threads have some; a thread goes through its own one after another.
__device__ __forceinline__ uint32_t pages_per(uint32_t pages) { return pages <= PAGES_NT ? 1 : pages <= 4 * PAGES_NT ? 4 : 16; }
// Which of the `per` pages p0 .. have `test`, as bits.
template <class F> __device__ __forceinline__ uint32_t pages_bits(const int32_t *refs, uint32_t pages, uint32_t p0, uint32_t per, F &&test) {
  auto four = [&](uint32_t e) {
    const int4 v = *(const int4 *)(refs + p0 + e);
    return ((test(v.x) ? 1u : 0u) | (test(v.y) ? 2u : 0u) | (test(v.z) ? 4u : 0u) | (test(v.w) ? 8u : 0u)) << e;
  };
  uint32_t m = 0;
  if (per == 16 && p0 + 16 <= pages) {
#pragma unroll
    for (uint32_t e = 0; e < 16; e += 4) m |= four(e);
  } else if (per == 4 && p0 + 4 <= pages) {
    m = four(0);
  } else {
    for (uint32_t e = 0; e < per && p0 + e < pages; e++) m |= (test(refs[p0 + e]) ? 1u : 0u) << e;
  }
  return m;
}

// The `want` lowest free pages: give(rank, page) where GIVE is on. Returns their number, less than want where there are
// fewer. Every thread calls it.
template <bool GIVE, class F>
__device__ __forceinline__ uint32_t pages_free(const int32_t *refs, uint32_t pages, uint32_t want, uint32_t *lds, F &&give) {
  uint32_t found = 0;
  const uint32_t per = pages_per(pages);
  for (uint32_t base = 0; base < pages && found < want; base += per * PAGES_NT) {
    const uint32_t p0 = base + per * threadIdx.x;
    uint32_t m = pages_bits(refs, pages, p0, per, [](int32_t n) { return n <= 0; }), total;
    uint32_t rank = found + pages_scan(__popc(m), lds, total);
    if constexpr (GIVE)
      for (; m && rank < want; m &= m - 1, rank++) give(rank, p0 + __ffs(m) - 1);
    found += total;
  }
  return min(found, want);
}

// ------------------------------------------------------------------ places for new tokens
// A thread per request: what it needs, the sum before it; then the free pages go to the requests in order. Where pages run short one thread goes through the requests. 4.6 us for 4 tokens of 8 requests and 700 pages, 7.0 for 512 tokens of each.
struct ExtendLds { uint32_t scan[PAGES_NT / 64 + 1]; uint32_t start[PAGES_NT + 1]; int32_t len[PAGES_NT], added[PAGES_NT]; };

__device__ __forceinline__ void extend_place(const PagesExtendArgs &a, uint32_t i, int32_t before, int32_t added) {
  const uint32_t r = i / a.tokens, t = i % a.tokens;
  int32_t pos = -1, slot = -1;
  if ((int32_t)t < added) {
    pos = before + (int32_t)t;
    const int32_t id = a.table[(uint64_t)r * a.max_pages + ((uint32_t)pos >> a.shift)];
    if (id >= 0 && (uint32_t)id < a.pages) slot = (int32_t)((uint32_t)id << a.shift | ((uint32_t)pos & ((1u << a.shift) - 1)));
  }
  a.positions[i] = pos;
  a.slots[i] = slot;
}

__global__ __launch_bounds__(PAGES_NT) void k_pages_extend(PagesExtendArgs a, bool places) {
  __shared__ ExtendLds L;
  const uint32_t r = threadIdx.x, cap = a.max_pages << a.shift, pg = (1u << a.shift) - 1;
  int32_t len = 0, n = -1;
  uint32_t have = 0, need = 0;
  if (r < a.requests) {
    len = a.lengths[r];
    n = a.counts ? a.counts[r] : (int32_t)a.tokens;
    if (n < 0 || n > (int32_t)a.tokens || len < 0 || (uint32_t)len > cap || (uint32_t)n > cap - (uint32_t)len) n = -1;
    if (n > 0) {
      have = ((uint32_t)len + pg) >> a.shift;
      need = (((uint32_t)(len + n) + pg) >> a.shift) - have;
    }
  }
  uint32_t want;
  uint32_t start = pages_scan(need, L.scan, want);
  if (want) {
    const uint32_t found = pages_free<false>(a.refs, a.pages, want, L.scan, [](uint32_t, uint32_t) {});
    if (found < want) {  // one after another: who fits what is left
      L.start[r] = need;
      __syncthreads();
      if (r == 0) {
        uint32_t left = found;
        for (uint32_t i = 0; i < a.requests; i++) {
          const uint32_t w = L.start[i];
          if (w > left) L.start[i] = 0xFFFFFFFFu;
          else left -= w;
        }
      }
      __syncthreads();
      if (L.start[r] == 0xFFFFFFFFu) { n = -1; need = 0; }
      start = pages_scan(need, L.scan, want);
    }
    __syncthreads();
    L.start[r] = start;
    L.len[r] = (int32_t)have;
    __syncthreads();
    pages_free<true>(a.refs, a.pages, want, L.scan, [&](uint32_t rank, uint32_t p) {
      uint32_t lo = 0, hi = a.requests - 1;  // the last request whose pages start at `rank` or before
      while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (L.start[mid] <= rank) lo = mid;
        else hi = mid - 1;
      }
      a.table[(uint64_t)lo * a.max_pages + L.len[lo] + (rank - L.start[lo])] = (int32_t)p;
      a.refs[p] = 1;
    });
    __syncthreads();
  }
  if (r < a.requests) {
    if (n > 0) a.lengths[r] = len + n;
    a.added[r] = n;
    L.len[r] = len;
    L.added[r] = n;
  }
  if (!places) return;
  __syncthreads();
  for (uint32_t i = r; i < a.requests * a.tokens; i += PAGES_NT) extend_place(a, i, L.len[i / a.tokens], L.added[i / a.tokens]);
}

__global__ __launch_bounds__(256) void k_pages_places(PagesExtendArgs a) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.requests * a.tokens) return;
  const int32_t added = a.added[i / a.tokens];
  extend_place(a, i, a.lengths[i / a.tokens] - max(added, 0), added);
}

hipError_t pages_extend(hipStream_t s, const PagesExtendArgs &a) {
  if (!a.requests || !a.tokens) return hipSuccess;
  const bool inside = (uint64_t)a.requests * a.tokens <= 4096;
  hipLaunchKernelGGL(k_pages_extend, dim3(1), dim3(PAGES_NT), 0, s, a, inside);
  WGD_HIP(hipGetLastError());
  if (!inside) hipLaunchKernelGGL(k_pages_places, dim3((a.requests * a.tokens + 255) / 256), dim3(256), 0, s, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------ forks
// Three steps over the rows that change, an element of the table per thread: their old pages are let go, the full pages
// of their new rows held, and the new rows set down in scratch; then the last pages that are not full are given to one
// row each, or copied; then the new rows go to the table. Without enough pages the last step takes the first one back.
// 6.5 us in one launch for 8 requests of 64 pages; in three 3.6 + 6.8 + 2.5 for 64 requests of 256.
struct ForkRow { bool changed; uint32_t from, held, kept; };  // pages that the row held; tokens that it keeps

__device__ __forceinline__ uint32_t fork_length(const PagesForkArgs &a, uint32_t r) {
  return min((uint32_t)max(a.lengths[r], 0), a.max_pages << a.shift);
}
__device__ __forceinline__ ForkRow fork_row(const PagesForkArgs &a, uint32_t r) {
  const int32_t from = a.origin[r];
  const uint32_t len = fork_length(a, r);
  ForkRow f = {true, 0, (len + (1u << a.shift) - 1) >> a.shift, 0};
  if (from >= 0 && (uint32_t)from < a.requests) {
    f.from = (uint32_t)from;
    f.kept = (uint32_t)from == r ? len : fork_length(a, f.from);
    if (a.keep) f.kept = min(f.kept, (uint32_t)max(a.keep[r], 0));
    f.changed = f.from != r || f.kept < len;
  }
  return f;
}
__device__ __forceinline__ bool fork_page(const PagesForkArgs &a, int32_t id) { return id >= 0 && (uint32_t)id < a.pages; }

// Column c of row r: its old page loses a holder, its new one, if full, gains one; BACK the other way round.
template <bool BACK> __device__ __forceinline__ void fork_hold(const PagesForkArgs &a, uint32_t r, uint32_t c) {
  const ForkRow f = fork_row(a, r);
  if (!f.changed) return;
  const uint64_t at = (uint64_t)r * a.max_pages + c;
  int32_t id = -1;
  if (c < f.held) {
    id = a.table[at];
    if (fork_page(a, id)) atomicAdd(a.refs + id, BACK ? 1 : -1);
  }
  if (c << a.shift < f.kept) {
    id = a.table[(uint64_t)f.from * a.max_pages + c];
    if ((c + 1) << a.shift <= f.kept && fork_page(a, id)) atomicAdd(a.refs + id, BACK ? -1 : 1);
    if (!BACK) a.rows[at] = id;
  } else if (!BACK) {
    a.rows[at] = -1;
  }
}

// The last pages: thread r has row r's. One that nobody else holds stays with the first row that has it last.
struct ForkLds { uint32_t scan[PAGES_NT / 64 + 1]; int32_t last[PAGES_NT]; uint32_t to[PAGES_NT]; };
__device__ __forceinline__ void fork_settle(const PagesForkArgs &a, ForkLds &L) {
  const uint32_t r = threadIdx.x;
  ForkRow f = {false, 0, 0, 0};
  int32_t p = -1;
  if (r < a.requests) {
    f = fork_row(a, r);
    if (f.changed && (f.kept & ((1u << a.shift) - 1))) p = a.rows[(uint64_t)r * a.max_pages + (f.kept >> a.shift)];
    if (!fork_page(a, p)) p = -1;
  }
  L.last[r] = p;
  const int32_t others = p >= 0 ? a.refs[p] : 0;
  __syncthreads();
  bool stays = p >= 0 && others <= 0;
  if (stays)
    for (uint32_t i = 0; i < r; i++)
      if (L.last[i] == p) { stays = false; break; }
  if (stays) a.refs[p] = 1;
  const bool copied = p >= 0 && !stays;
  uint32_t want;
  const uint32_t rank = pages_scan(copied, L.scan, want);
  __syncthreads();
  bool enough = true;
  if (want) {
    enough = pages_free<false>(a.refs, a.pages, want, L.scan, [](uint32_t, uint32_t) {}) == want;
    if (enough) pages_free<true>(a.refs, a.pages, want, L.scan, [&](uint32_t k, uint32_t page) { L.to[k] = page; a.refs[page] = 1; });
    __syncthreads();
    if (enough && copied) {
      a.rows[(uint64_t)r * a.max_pages + (f.kept >> a.shift)] = (int32_t)L.to[rank];
      a.copies[1 + 2 * rank] = p;
      a.copies[2 + 2 * rank] = (int32_t)L.to[rank];
    }
    if (!enough && stays) a.refs[p] = others;
  }
  if (r < a.requests) {
    if (!enough || r >= want) a.copies[1 + 2 * r] = a.copies[2 + 2 * r] = -1;
    // 1: the row of the table takes the new one, 0: it stays, -1: the counts go back
    a.settled[r] = !f.changed ? 0 : enough ? 1 : -1;
    if (enough && f.changed) a.lengths[r] = (int32_t)f.kept;
  }
  if (r == 0) a.copies[0] = enough ? (int32_t)want : -1;
}

__device__ __forceinline__ void fork_write(const PagesForkArgs &a, uint32_t r, uint32_t c) {
  const int32_t s = a.settled[r];
  const uint64_t at = (uint64_t)r * a.max_pages + c;
  if (s > 0) a.table[at] = a.rows[at];
  else if (s < 0) fork_hold<true>(a, r, c);
}

// The three steps in one workgroup, for small tables: two launches less, which the host would take 4 us each for.
constexpr uint32_t FORK_SMALL = 4096;
__global__ __launch_bounds__(PAGES_NT) void k_pages_fork(PagesForkArgs a) {
  __shared__ ForkLds L;
  const uint32_t n = a.requests * a.max_pages;
  for (uint32_t i = threadIdx.x; i < n; i += PAGES_NT) fork_hold<false>(a, i / a.max_pages, i % a.max_pages);
  __syncthreads();
  fork_settle(a, L);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += PAGES_NT) fork_write(a, i / a.max_pages, i % a.max_pages);
}
__global__ __launch_bounds__(256) void k_pages_hold(PagesForkArgs a) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c < a.max_pages) fork_hold<false>(a, blockIdx.y, c);
}
__global__ __launch_bounds__(PAGES_NT) void k_pages_settle(PagesForkArgs a) {
  __shared__ ForkLds L;
  fork_settle(a, L);
}
__global__ __launch_bounds__(256) void k_pages_write(PagesForkArgs a) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c < a.max_pages) fork_write(a, blockIdx.y, c);
}

uint64_t pages_fork_scratch_bytes(const PagesForkArgs &a) { return ((uint64_t)a.requests * a.max_pages + a.requests) * 4; }

hipError_t pages_fork(hipStream_t s, const PagesForkArgs &in) {
  if (!in.requests) return hipSuccess;
  PagesForkArgs a = in;
  a.settled = a.rows + (uint64_t)a.requests * a.max_pages;
  if ((uint64_t)a.requests * a.max_pages <= FORK_SMALL) {
    hipLaunchKernelGGL(k_pages_fork, dim3(1), dim3(PAGES_NT), 0, s, a);
    return hipGetLastError();
  }
  const dim3 grid((a.max_pages + 255) / 256, a.requests);
  hipLaunchKernelGGL(k_pages_hold, grid, dim3(256), 0, s, a);
  WGD_HIP(hipGetLastError());
  hipLaunchKernelGGL(k_pages_settle, dim3(1), dim3(PAGES_NT), 0, s, a);
  WGD_HIP(hipGetLastError());
  hipLaunchKernelGGL(k_pages_write, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------ compaction
// With `used` pages in use, the free ones below `used` are as many as the used ones from there on: the j-th of
// these moves to the j-th of those. One workgroup goes through the pages twice, to count and to pair; a hole comes before
// the page that moves there, so its number is listed when it is asked for. 3.4 us for 128 pages, 8.1 for 4000: loads, scans,
// and four pages a thread one after another (16: 7.8 and 13.9).
struct CompactLds { uint32_t scan[PAGES_NT / 64 + 1]; };
__global__ __launch_bounds__(PAGES_NT) void k_pages_compact(PagesCompactArgs a) {
  __shared__ CompactLds L;
  const uint32_t tid = threadIdx.x, per = pages_per(a.pages);
  auto bits = [&](uint32_t p0) { return p0 < a.pages ? pages_bits(a.refs, a.pages, p0, per, [](int32_t n) { return n > 0; }) : 0; };
  uint32_t total;
  const uint32_t on0 = bits(per * tid);  // (they are read once where that is all)
  uint32_t used = __popc(on0);
  for (uint32_t p0 = per * (tid + PAGES_NT); p0 < a.pages; p0 += per * PAGES_NT) used += __popc(bits(p0));
  pages_scan(used, L.scan, total);
  used = total;
  uint32_t holes = 0, moves = 0;
  for (uint32_t base = 0; base < a.pages; base += per * PAGES_NT) {
    const uint32_t p0 = base + per * tid, n = p0 < a.pages ? min(per, a.pages - p0) : 0;
    const uint32_t on = base ? bits(p0) : on0;
    const uint32_t low = used > p0 ? (1u << min(used - p0, n)) - 1 : 0;  // of those that are there
    uint32_t hole = ~on & low, move = on & ~low;
    uint32_t h = holes + pages_scan(__popc(hole), L.scan, total);
    holes += total;
    for (; hole; hole &= hole - 1, h++) a.copies[2 + 2 * h] = (int32_t)(p0 + __ffs(hole) - 1);
    uint32_t m = moves + pages_scan(__popc(move), L.scan, total);  // its barriers come after the holes' stores
    moves += total;
    for (uint32_t e = 0; e < n; e++) {
      const uint32_t p = p0 + e;
      int32_t to = on >> e & 1 ? (int32_t)p : -1;
      if (move >> e & 1) {
        to = a.copies[2 + 2 * m];
        a.copies[1 + 2 * m] = (int32_t)p;
        m++;
        a.refs_to[to] = a.refs[p];
        a.refs_to[p] = 0;
      } else if (to >= 0 || p >= used) {
        a.refs_to[p] = a.refs[p];
      }
      a.moved[p] = to;
    }
  }
  if (tid == 0) a.copies[0] = (int32_t)moves;
  for (uint32_t i = moves + tid; i < a.pages / 2; i += PAGES_NT) a.copies[1 + 2 * i] = a.copies[2 + 2 * i] = -1;
}

__global__ __launch_bounds__(256) void k_pages_remap(const int32_t *table, int32_t *to, const int32_t *moved, uint64_t n, uint32_t pages) {
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
    const int32_t id = table[i];
    to[i] = id >= 0 && (uint32_t)id < pages ? moved[id] : id;
  }
}

hipError_t pages_compact(hipStream_t s, const PagesCompactArgs &a) {
  hipLaunchKernelGGL(k_pages_compact, dim3(1), dim3(PAGES_NT), 0, s, a);
  WGD_HIP(hipGetLastError());
  const uint64_t n = (uint64_t)a.requests * a.max_pages;
  if (!n) return hipSuccess;
  hipLaunchKernelGGL(k_pages_remap, dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 2048)), dim3(256), 0, s, a.table, a.table_to, a.moved, n,
                     a.pages);
  return hipGetLastError();
}

// ------------------------------------------------------------------ pages from place to place
// A workgroup has 256 COPY_AHEAD units of a page, every gridDim.y-th pair and one pool; its loads go ahead of its stores. Bound by the
// bytes: 1000 moves of 64 KB in two pools, 262 MB read and written, 53 us (4.9 TB/s).
constexpr uint32_t COPY_POOLS = 64, COPY_AHEAD = 4;
struct CopyPools { void *p[COPY_POOLS]; };
typedef uint32_t copy16 __attribute__((ext_vector_type(4)));

template <class U>
__global__ __launch_bounds__(256) void k_pages_copy(CopyPools pools, const int32_t *copies, uint32_t most, uint64_t units, uint32_t pages) {
  const uint32_t count = min((uint32_t)max(copies[0], 0), most);
  const uint64_t u0 = (uint64_t)blockIdx.x * 256 * COPY_AHEAD + threadIdx.x;
  U *pool = (U *)pools.p[blockIdx.z];
  for (uint32_t i = blockIdx.y; i < count; i += gridDim.y) {
    const int32_t from = copies[1 + 2 * i], to = copies[2 + 2 * i];
    if (from < 0 || to < 0 || (uint32_t)from >= pages || (uint32_t)to >= pages) continue;
    const U *src = pool + (uint64_t)from * units;
    U *dst = pool + (uint64_t)to * units;
    U v[COPY_AHEAD];
#pragma unroll
    for (uint32_t e = 0; e < COPY_AHEAD; e++)
      if (u0 + 256 * e < units) v[e] = src[u0 + 256 * e];
#pragma unroll
    for (uint32_t e = 0; e < COPY_AHEAD; e++)
      if (u0 + 256 * e < units) dst[u0 + 256 * e] = v[e];
  }
}

hipError_t pages_copy(hipStream_t s, void *const *pools, uint32_t count, const int32_t *copies, uint32_t most, uint64_t page_bytes,
                      uint32_t pages) {
  if (!most) return hipSuccess;
  const uint32_t unit = page_bytes % 16 == 0 ? 16 : page_bytes % 4 == 0 ? 4 : 2;
  const uint64_t units = page_bytes / unit;
  const uint32_t blocks = (uint32_t)((units + 256 * COPY_AHEAD - 1) / (256 * COPY_AHEAD));
  for (uint32_t p0 = 0; p0 < count; p0 += COPY_POOLS) {
    const uint32_t n = std::min(count - p0, COPY_POOLS);
    CopyPools c{};
    for (uint32_t i = 0; i < n; i++) c.p[i] = pools[p0 + i];
    const dim3 grid(blocks, std::min(most, std::max(1u, 8192 / std::max(1u, std::min(blocks * n, 8192u)))), n);
    if (unit == 16) hipLaunchKernelGGL(k_pages_copy<copy16>, grid, dim3(256), 0, s, c, copies, most, units, pages);
    else if (unit == 4) hipLaunchKernelGGL(k_pages_copy<uint32_t>, grid, dim3(256), 0, s, c, copies, most, units, pages);
    else hipLaunchKernelGGL(k_pages_copy<uint16_t>, grid, dim3(256), 0, s, c, copies, most, units, pages);
    WGD_HIP(hipGetLastError());
  }
  return hipSuccess;
}

// ------------------------------------------------------------------ K/V rows into their slots
// A row has `per` threads (a power of two), so that short rows share a workgroup. VEC: four elements a thread, where rows,
// strides and offsets are whole multiples of four. Bound by the bytes: 2400 rows of 1024 f32 values of K and V each into halves, 30 MB, 7.5 us.
template <class E, bool VEC>
__global__ __launch_bounds__(256) void k_pages_store(PagesStoreArgs a, uint32_t per) {
  constexpr uint32_t W = VEC ? 4 : 1;
  const float *src = blockIdx.y ? a.v : a.k;
  void *pool = blockIdx.y ? a.v_pool : a.k_pool;
  const uint32_t at = 256 / per, e0 = threadIdx.x % per * W;
  for (uint64_t t = (uint64_t)blockIdx.x * at + threadIdx.x / per; t < a.rows; t += (uint64_t)gridDim.x * at) {
    const int32_t slot = a.slots[t];
    if (slot < 0 || (uint32_t)slot >= a.slots_in_pool) continue;
    const float *from = src + t * a.stride;
    const uint64_t to = (uint64_t)slot * a.row;
    for (uint64_t e = e0; e < a.row; e += per * W) {
      if constexpr (VEC) kv_put4<E>(pool, to + e, *(const float4 *)(from + e));
      else kv_put(pool, to + e, from[e], sizeof(E) == 2);
    }
  }
}

hipError_t pages_store(hipStream_t s, const PagesStoreArgs &a) {
  if (!a.rows || !a.row) return hipSuccess;
  const bool vec = a.row % 4 == 0 && a.stride % 4 == 0 && ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0;
  const uint32_t units = vec ? a.row / 4 : a.row;
  uint32_t per = 1;
  while (per < 256 && per < units) per *= 2;
  const dim3 grid(std::min((a.rows - 1) / (256 / per) + 1, 1u << 16), 2);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, per); };
  if (a.kv16) vec ? go(k_pages_store<_Float16, true>) : go(k_pages_store<_Float16, false>);
  else vec ? go(k_pages_store<float, true>) : go(k_pages_store<float, false>);
  return hipGetLastError();
}

}  // namespace wgd
