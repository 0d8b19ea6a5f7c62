// Pages of a paged cache on gfx950: copied, shared between sequences (fork), handed out
// (reserve), given back (free) and moved together (compact), and the rows of accepted drafted
// tokens moved up in the last pages (keep).
//
// The state is three int32 arrays: refs [num_pages], how many block-table entries name a page
// (0: free); table [R, P], the pages of every sequence row; lens [R], its tokens.  Entry i of a
// row is in use for i < ceil(len / page).  Free pages are handed out lowest first, to the rows
// in order, so that a result does not depend on how a launch ran: what is added up by atomics
// is whole numbers.
//
// Fork, reserve and the plan of a compaction run as one work-group, pass after pass with a barrier between
// them.  For the tables of a serving batch (a few kilobytes) the latency of these passes bounds them: a fork
// of four rows to sixteen 10 us (targets, sources, the entries' check, a prefix sum, the free pages' count,
// the moves, the hand-out, the entries' sharing, the lengths), its growth 4.5, the plan 3 to 5.  Their time
// grows with the entries and the pages, 1,024 lanes at a time: rows of 100 pages forked, 16 of them 11 us,
// 128 44, 1,024 302, 4,096 1,198; grown, 16 rows 6 us, 1,024 (of a pool of 110,656 pages) 62, 4,096 (of
// 442,432) 255.  Freeing takes a work-group a row, 3.1 us for twenty.  The copies are bound by HBM: 16 bytes a
// lane, several loads in flight before the first store.

#include "dash_common.h"

namespace dash {

constexpr int kKvThreads = 1024;
constexpr int kKvMaxRows = 8192;      // rows of a table (prefix sums in LDS)
constexpr int kKvMaxCaches = 32;      // caches per launch (kernel argument space)

// One cache: page p of layer l starts at base + l * layer + p * page bytes; a page holds
// n1 x n2 pieces of seg bytes at strides s1 and s2.  For rows, s1 is the stride of a token and a row
// holds n2 pieces.
struct KvCache {
  char* base;
  int64_t layer, page, s1, s2;
  int64_t units;                      // of a layer's page (or row)
  int32_t n2, segu;                   // segu: units of a piece (0: the page, or row, in one piece)
  int32_t per;                        // tasks of a layer's page (or row)
  int32_t task0;                      // first task of the cache
};
struct KvCaches {
  KvCache c[kKvMaxCaches];
  int n;
};

// The cache that task t belongs to.
__device__ __forceinline__ const KvCache& kv_cache_of(const KvCaches& a, int t) {
  int i = 0;
  while (i + 1 < a.n && t >= a.c[i + 1].task0) ++i;
  return a.c[i];
}

typedef uint32_t KvVec __attribute__((ext_vector_type(4)));   // 16 bytes
constexpr int kCpThreads = 256, kCpUnroll = 4;
constexpr int kCpPairs = 65535;       // of a launch's grid

// One work-group per (task, pair), pairs past the grid's kCpPairs in a loop; a task is kCpThreads *
// kCpUnroll units of one layer's page.  Bound by HBM: 730 MB read and written in 138 to 145 us, 5.0 to 5.3
// TB/s; 149 us where the loads and stores leave their lines in the L2 (a page is not read again here), 225
// with eight units a lane in flight instead of four.  A pair without pages costs its work-groups' launch:
// 5,280 of them 3.1 us.
template <typename U>
__global__ __launch_bounds__(kCpThreads) void copy_pages_kernel(KvCaches a, const int32_t* frm,
                                                                const int32_t* to, int pairs,
                                                                int num_pages) {
  for (int64_t pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
    const int f = frm[pair], d = to[pair];
    if (f < 0 || d < 0 || f >= num_pages || d >= num_pages || f == d) continue;
    const KvCache& c = kv_cache_of(a, blockIdx.x);
    const int rel = blockIdx.x - c.task0;
    const int l = rel / c.per, ch = rel % c.per;
    char* const lb = c.base + l * c.layer;
    const char* const sp = lb + f * c.page;
    char* const dp = lb + d * c.page;
    const int64_t units = c.units;
    const int64_t u0 = (int64_t)ch * (kCpThreads * kCpUnroll) + threadIdx.x;
    U x[kCpUnroll];
    int64_t off[kCpUnroll];
#pragma unroll
    for (int k = 0; k < kCpUnroll; ++k) {
      const int64_t u = u0 + k * kCpThreads;
      if (c.segu == 0) {
        off[k] = u * (int)sizeof(U);
      } else {
        const int64_t piece = u / c.segu;
        off[k] = (piece / c.n2) * c.s1 + (piece % c.n2) * c.s2 + (u - piece * c.segu) * (int)sizeof(U);
      }
      if (u < units) x[k] = __builtin_nontemporal_load((const U*)(sp + off[k]));
    }
#pragma unroll
    for (int k = 0; k < kCpUnroll; ++k)
      if (u0 + k * kCpThreads < units) __builtin_nontemporal_store(x[k], (U*)(dp + off[k]));
  }
}

// Rows ctx + path[i] -> ctx + i, 1 <= i < count, of one sequence and one unit column of one
// cache and layer per lane.  Parents come before their children, so path is strictly
// increasing and path[i] >= i: the source of a row is never a place that an earlier row moved
// to, and ascending order needs no copy kept aside.  Latency: 5.5 us for 8 sequences of 24 caches, 3.8 MB.
constexpr int kKeepRows = 8;
template <typename U>
__global__ __launch_bounds__(kWave) void keep_rows_kernel(KvCaches a, const int32_t* path,
                                                          int64_t path_st, const int32_t* count,
                                                          const int32_t* ctx, const int32_t* table,
                                                          int64_t table_st, int P, int page,
                                                          int num_pages, int max_n) {
  const int b = blockIdx.y, lane = threadIdx.x;
  const int n = min(count[b], max_n);
  const int c0 = ctx[b];
  if (n <= 0 || c0 < 0) return;
  const KvCache& c = kv_cache_of(a, blockIdx.x);
  const int units = (int)c.units;
  const int rel = blockIdx.x - c.task0;
  const int l = rel / c.per, u = (rel % c.per) * kWave + lane;
  char* const lb = c.base + l * c.layer;
  const int64_t col = c.segu == 0 ? (int64_t)u * (int)sizeof(U)
                                  : (int64_t)(u / c.segu) * c.s2 + (int64_t)(u % c.segu) * (int)sizeof(U);
  const int32_t* tr = table + (int64_t)b * table_st;
  // byte offset of a slot's row in this layer, -1 where there is none
  auto row_of = [&](int64_t s) -> int64_t {
    if (s < 0 || s >= (int64_t)P * page) return -1;
    const int p = tr[s / page];
    if (p < 0 || p >= num_pages) return -1;
    return p * c.page + (int64_t)(s % page) * c.s1;
  };
  for (int r0 = 0; r0 < n; r0 += kWave) {
    // this lane's row of the next 64
    int64_t so = -1, dn = -1;
    if (r0 + lane < n) {
      const int p = path[b * path_st + r0 + lane];
      if (p > r0 + lane) {
        so = row_of((int64_t)c0 + p);
        dn = row_of((int64_t)c0 + r0 + lane);
      }
    }
    uint64_t todo = __ballot(so >= 0 && dn >= 0);
    while (todo) {
      U x[kKeepRows];
      int64_t d[kKeepRows];
#pragma unroll
      for (int k = 0; k < kKeepRows; ++k) {
        const int s = todo ? __builtin_ctzll(todo) : -1;
        d[k] = s >= 0 ? __shfl(dn, s, kWave) : -1;
        const int64_t f = s >= 0 ? __shfl(so, s, kWave) : -1;
        if (f >= 0 && u < units) x[k] = *(const U*)(lb + f + col);
        if (todo) todo &= todo - 1;
      }
#pragma unroll
      for (int k = 0; k < kKeepRows; ++k)
        if (d[k] >= 0 && u < units) *(U*)(lb + d[k] + col) = x[k];
    }
  }
}

// What a step leaves of every row: its accepted nodes stand where the row holds the slot of the last of
// them, which is the highest (path is strictly increasing), and none does where it does not, as after a
// reserve that was refused.  stand: how many stand; kept: the row's tokens; context: its context;
// summed: the tokens whose block summaries changed (0: none).  One lane a row; 1.7 us, two trips to memory.
__global__ __launch_bounds__(256) void keep_lens_kernel(const int32_t* path, int64_t path_st,
                                                        const int32_t* count, const int32_t* ctx,
                                                        const int32_t* lens, int B, int max_n,
                                                        int32_t* stand, int32_t* kept,
                                                        int32_t* context, int32_t* summed) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int n = min(count[b], max_n), c = ctx[b], len = lens[b];
  bool ok = false;
  if (n > 0 && c >= 0) {
    const int p = path[b * path_st + n - 1];
    ok = p >= n - 1 && (int64_t)c + p < len;
  }
  stand[b] = ok ? n : 0;
  kept[b] = ok ? c + n : len;
  context[b] = ok ? c + n : c;
  summed[b] = ok ? c + n : 0;
}

// Sum of v over the work-group's earlier threads; `total` gets the sum over all.
__device__ __forceinline__ int block_exclusive(int v, int* sW, int& total) {
  const int lane = wave_lane(), wv = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) {
    const int y = __shfl_up(x, s, kWave);
    if (lane >= s) x += y;
  }
  __syncthreads();
  if (lane == kWave - 1) sW[wv] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kKvThreads / kWave; ++w) {
    const int t = sW[w];
    if (w < wv) before += t;
    total += t;
  }
  return before + x - v;
}

// (no sum that could pass 32 bits: a length that is no length must not look short)
__device__ __forceinline__ int kv_blocks(int len, int page) { return len / page + (len % page > 0); }

__device__ __forceinline__ int kv_count_free(const int32_t* refs, int num_pages, int* sW) {
  int mine = 0, total;
  for (int p = threadIdx.x; p < num_pages; p += kKvThreads) mine += refs[p] == 0;
  block_exclusive(mine, sW, total);
  return total;
}

// Hands the lowest free pages out: want[i] .. want[i + 1] - 1 are the ranks of item i;
// give(item, k, page) takes the k-th page of an item.
template <typename Give>
__device__ __forceinline__ void kv_hand_out(int32_t* refs, int num_pages, const int* want, int items,
                                            int total, int* sW, Give give) {
  int given = 0;
  for (int p0 = 0; p0 < num_pages && given < total; p0 += kKvThreads) {
    const int p = p0 + threadIdx.x;
    const bool is_free = p < num_pages && refs[p] == 0;
    int got;
    const int rank = given + block_exclusive(is_free ? 1 : 0, sW, got);
    if (is_free && rank < total) {
      int lo = 0, hi = items;              // the last item with want[item] <= rank
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (want[mid] <= rank) lo = mid; else hi = mid;
      }
      refs[p] = 1;
      give(lo, rank - want[lo], p);
    }
    given += got;
  }
}

// Prefix sums of n values value(i) into want [n + 1] in LDS.
template <typename Value>
__device__ __forceinline__ int kv_prefix(int n, int* want, int* sW, Value value) {
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kKvThreads) {
    const int i = i0 + threadIdx.x;
    int total;
    const int before = block_exclusive(i < n ? value(i) : 0, sW, total);
    if (i < n) want[i] = base + before;
    base += total;
  }
  if (threadIdx.x == 0) want[n] = base;
  __syncthreads();
  return base;
}

// take(i, k, tokens, page) for every entry k of the rows src[i] (entries past a row's tokens too), four
// of a thread's loads in flight: one row after another took 20 us for 16 rows.
template <typename Take>
__device__ __forceinline__ void kv_entries(const int32_t* table, int64_t table_st, int P,
                                           const int32_t* src, const int32_t* lens, int n, Take take) {
  const int64_t all = (int64_t)n * P;
  for (int64_t e0 = threadIdx.x; e0 < all; e0 += 4 * kKvThreads) {
    int i[4], k[4], len[4], p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t e = min(e0 + u * kKvThreads, all - 1);
      i[u] = (int)(e / P);
      k[u] = (int)(e - (int64_t)i[u] * P);
      const int s = src[i[u]];
      len[u] = lens[s];
      p[u] = table[(int64_t)s * table_st + k[u]];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (e0 + u * kKvThreads < all) take(i[u], k[u], len[u], p[u]);
  }
}

// Row dst[i] becomes row src[i]: its whole pages shared, its last, partly filled one a page of
// its own, to be copied (frm[i] -> to[i]; -1 where there is none).  All pairs or none: ok is 0
// and nothing changes where a row is out of range or named wrongly (a filled or repeated target, a
// source that is a target, a table entry that is no page) or the free pages do not suffice.
__global__ __launch_bounds__(kKvThreads) void fork_pages_kernel(
    int32_t* refs, int num_pages, int32_t* table, int64_t table_st, int R, int P, int32_t* lens,
    const int32_t* src, const int32_t* dst, int n, int page, int32_t* ok, int32_t* frm, int32_t* to) {
  __shared__ int sW[kKvThreads / kWave];
  __shared__ int sWant[kKvMaxRows + 1];
  __shared__ uint32_t sDst[kKvMaxRows / 32];
  const int tid = threadIdx.x;
  for (int i = tid; i < kKvMaxRows / 32; i += kKvThreads) sDst[i] = 0u;
  __syncthreads();
  bool bad = false;
  for (int i = tid; i < n; i += kKvThreads) {
    const int d = dst[i];
    if (d < 0 || d >= R || lens[d] != 0) { bad = true; continue; }
    bad |= (atomicOr(&sDst[d >> 5], 1u << (d & 31)) >> (d & 31)) & 1u;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kKvThreads) {
    const int s = src[i];
    if (s < 0 || s >= R || (sDst[s >> 5] >> (s & 31)) & 1u || lens[s] < 0 ||
        kv_blocks(lens[s], page) > P)
      bad = true;
  }
  if (__syncthreads_or(bad)) {
    for (int i = tid; i < n; i += kKvThreads) frm[i] = to[i] = -1;
    if (tid == 0) *ok = 0;
    return;
  }
  // every entry that is shared or copied names a page
  kv_entries(table, table_st, P, src, lens, n, [&](int, int k, int len, int p) {
    if (k * (int64_t)page < len) bad |= p < 0 || p >= num_pages;
  });
  const int total = kv_prefix(n, sWant, sW, [&](int i) { return lens[src[i]] % page != 0 ? 1 : 0; });
  const int n_free = kv_count_free(refs, num_pages, sW);
  if (__syncthreads_or(bad || total > n_free)) {
    for (int i = tid; i < n; i += kKvThreads) frm[i] = to[i] = -1;
    if (tid == 0) *ok = 0;
    return;
  }
  for (int i = tid; i < n; i += kKvThreads) {
    const int s = src[i], len = lens[s];
    frm[i] = len % page != 0 ? table[(int64_t)s * table_st + len / page] : -1;
    if (len % page == 0) to[i] = -1;
  }
  kv_hand_out(refs, num_pages, sWant, n, total, sW, [&](int i, int, int p) {
    // an item without a page has an empty range, and the last of equal starts is taken
    to[i] = p;
    table[(int64_t)dst[i] * table_st + lens[src[i]] / page] = p;
  });
  __syncthreads();
  kv_entries(table, table_st, P, src, lens, n, [&](int i, int k, int len, int p) {
    if ((k + 1) * (int64_t)page > len) return;
    table[(int64_t)dst[i] * table_st + k] = p;
    atomicAdd(&refs[p], 1);
  });
  __syncthreads();
  for (int i = tid; i < n; i += kKvThreads) lens[dst[i]] = lens[src[i]];
  if (tid == 0) *ok = 1;
}

// Rows grow to new_lens (shorter ones stay): new pages for the blocks they lack, and a page of
// its own for a partly filled last page that another row shares, to be copied (frm[r] -> to[r]).
// All rows or none, as above.
__global__ __launch_bounds__(kKvThreads) void reserve_pages_kernel(
    int32_t* refs, int num_pages, int32_t* table, int64_t table_st, int R, int P, int32_t* lens,
    const int32_t* new_lens, int page, int32_t* ok, int32_t* frm, int32_t* to) {
  __shared__ int sW[kKvThreads / kWave];
  __shared__ int sWant[kKvMaxRows + 1];
  const int tid = threadIdx.x;
  bool bad = false;
  for (int r = tid; r < R; r += kKvThreads) {
    const int len = lens[r], want = new_lens[r];
    frm[r] = to[r] = -1;
    if (len < 0 || kv_blocks(len, page) > P) { bad = true; continue; }
    if (want <= len) continue;
    if (want > (int64_t)P * page) { bad = true; continue; }
    if (len % page != 0) {
      const int p = table[(int64_t)r * table_st + len / page];
      if (p < 0 || p >= num_pages) bad = true;
      else if (refs[p] > 1) frm[r] = p;
    }
  }
  // each row was read and written by its own thread alone; the barrier in the prefix orders
  // these before the loops of other threads
  if (__syncthreads_or(bad)) {
    for (int r = tid; r < R; r += kKvThreads) frm[r] = -1;
    if (tid == 0) *ok = 0;
    return;
  }
  const int total = kv_prefix(R, sWant, sW, [&](int r) {
    const int len = lens[r], want = new_lens[r];
    return want <= len ? 0 : kv_blocks(want, page) - kv_blocks(len, page) + (frm[r] >= 0 ? 1 : 0);
  });
  const int n_free = kv_count_free(refs, num_pages, sW);
  if (total > n_free) {
    __syncthreads();
    for (int r = tid; r < R; r += kKvThreads) frm[r] = -1;
    if (tid == 0) *ok = 0;
    return;
  }
  // several rows may leave one shared page: all of them get a page of their own but, where no
  // other row keeps it, the page loses its last name here and is free again
  kv_hand_out(refs, num_pages, sWant, R, total, sW, [&](int r, int k, int p) {
    const int have = kv_blocks(lens[r], page);
    int at = have + k;
    if (frm[r] >= 0) {
      at -= 1;
      if (k == 0) to[r] = p;
    }
    table[(int64_t)r * table_st + at] = p;
  });
  __syncthreads();
  for (int r = tid; r < R; r += kKvThreads) {
    if (frm[r] >= 0) atomicSub(&refs[frm[r]], 1);
    if (new_lens[r] > lens[r]) lens[r] = new_lens[r];
  }
  if (tid == 0) *ok = 1;
}

// Rows are cut to keep[r] tokens (longer ones; below 0 counts as 0) and the pages above given up.
__global__ __launch_bounds__(256) void free_pages_kernel(int32_t* refs, int num_pages, int32_t* table,
                                                         int64_t table_st, int P, int32_t* lens,
                                                         const int32_t* keep, int page) {
  const int r = blockIdx.x;
  const int len = lens[r], k = max(keep[r], 0);
  if (k >= len) return;
  const int b1 = (int)min((int64_t)P, ((int64_t)len + page - 1) / page);
  for (int i = kv_blocks(k, page) + threadIdx.x; i < b1; i += 256) {
    const int p = table[(int64_t)r * table_st + i];
    if (p >= 0 && p < num_pages) atomicSub(&refs[p], 1);
    table[(int64_t)r * table_st + i] = -1;
  }
  __syncthreads();                          // every thread read the length
  if (threadIdx.x == 0) lens[r] = k;
}

// The live pages move to the lowest places: with `live` of them, the i-th live page at or above
// `live` goes to the i-th free page below it.  new_refs and the moves (frm, to; -1 past them);
// place [num_pages]: where each page went.
__global__ __launch_bounds__(kKvThreads) void compact_plan_kernel(const int32_t* refs, int num_pages,
                                                                  int32_t* new_refs, int32_t* frm,
                                                                  int32_t* to, int32_t* place) {
  __shared__ int sW[kKvThreads / kWave];
  const int tid = threadIdx.x;
  const int live = num_pages - kv_count_free(refs, num_pages, sW);
  int highs = 0, lows = 0;
  for (int p0 = 0; p0 < num_pages; p0 += kKvThreads) {
    const int p = p0 + tid;
    const int rc = p < num_pages ? refs[p] : 0;
    const bool in = p < num_pages;
    const bool low = in && rc == 0 && p < live, high = in && rc != 0 && p >= live;
    // at most 1024 of each: both counts in one scan
    int both;
    const int before = block_exclusive((low ? 1 : 0) | (high ? 1 << 16 : 0), sW, both);
    if (low) to[lows + (before & 0xffff)] = p;
    if (high) frm[highs + (before >> 16)] = p;
    if (in) {
      new_refs[p] = p < live ? rc : 0;
      place[p] = p;
    }
    lows += both & 0xffff;
    highs += both >> 16;
  }
  __syncthreads();
  for (int i = tid; i < num_pages / 2; i += kKvThreads) {
    if (i < highs) {
      const int f = frm[i], t = to[i];
      new_refs[t] = refs[f];
      place[f] = t;
    } else {
      frm[i] = to[i] = -1;
    }
  }
}

__global__ __launch_bounds__(256) void compact_table_kernel(const int32_t* table, int64_t table_st,
                                                            int R, int P, const int32_t* lens,
                                                            int page, const int32_t* place,
                                                            int num_pages, int32_t* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)R * P) return;
  const int r = (int)(i / P), k = (int)(i % P);
  const int p = table[(int64_t)r * table_st + k];
  // entries past a row's pages, and those that name no page, come out as -1
  out[i] = (int64_t)k * page < lens[r] && p >= 0 && p < num_pages ? place[p] : -1;
}

static int kv_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}

// The caches of one launch: descriptors first .. first + n - 1 of desc [.., 8] (layers, layer
// stride, page stride, n1, s1, n2, s2, seg; bytes), tasks of `task_units` units of a layer's page
// (or row).  Returns the unit's bytes, 0 if a number does not fit.
static int kv_fill(KvCaches& a, void* const* base, const int64_t* desc, int n, bool rows,
                   int task_units, int64_t* tasks) {
  int unit = 16;
  for (int i = 0; i < n; ++i) {
    const int64_t* d = desc + 8 * i;
    const int64_t m = (int64_t)(uintptr_t)base[i] | d[1] | d[2] | d[4] | d[6] | d[7];
    while (m % unit) unit >>= 1;
  }
  if (unit == 8) unit = 4;
  a.n = n;
  int64_t t = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t* d = desc + 8 * i;
    if (!base[i] || d[0] < 0 || d[3] < 1 || d[5] < 1 || d[7] < 1 || d[0] > INT32_MAX ||
        d[3] > INT32_MAX || d[5] > INT32_MAX || d[7] > INT32_MAX || d[1] < 0 || d[2] < 0)
      return 0;
    const int64_t pieces = (rows ? 1 : d[3]) * d[5], segu = d[7] / unit, units = pieces * segu;
    const int64_t per = (units + task_units - 1) / task_units;
    if (d[5] * segu > INT32_MAX - 64 || per > INT32_MAX) return 0;
    a.c[i] = KvCache{(char*)base[i], d[1], d[2], d[4], d[6], units, (int)d[5],
                     pieces == 1 ? 0 : (int)segu, (int)per, (int)t};
    t += d[0] * per;
    if (t > INT32_MAX) return 0;
  }
  *tasks = t;
  return unit;
}

// Launches Op over (tasks, count) of the caches, 32 at a time: units of 16 bytes where every address
// and size allows it, else the largest that does.
template <template <typename> class Op, typename... Args>
static int kv_launches(void* const* base, const int64_t* desc, int num, int64_t count, void* stream,
                       Args... args) {
  hipStream_t st = (hipStream_t)stream;
  KvCaches a;
  int64_t tasks = 0;
  if (num > kKvMaxCaches)                  // all of them or none
    for (int c0 = 0; c0 < num; c0 += kKvMaxCaches) {
      if (!kv_fill(a, base + c0, desc + 8 * c0, std::min(kKvMaxCaches, num - c0), Op<KvVec>::kRows,
                   Op<KvVec>::kTask, &tasks))
        return kErrInvalid;
      if (!fits_grid(tasks, Op<KvVec>::kThreads)) return kErrUnsupported;
    }
  for (int c0 = 0; c0 < num; c0 += kKvMaxCaches) {
    const int unit = kv_fill(a, base + c0, desc + 8 * c0, std::min(kKvMaxCaches, num - c0), Op<KvVec>::kRows,
                             Op<KvVec>::kTask, &tasks);
    if (unit == 0) return kErrInvalid;
    if (tasks == 0) continue;
    if (!fits_grid(tasks, Op<KvVec>::kThreads)) return kErrUnsupported;
    if (unit == 16) Op<KvVec>::launch(a, tasks, count, st, args...);
    else if (unit == 4) Op<uint32_t>::launch(a, tasks, count, st, args...);
    else if (unit == 2) Op<uint16_t>::launch(a, tasks, count, st, args...);
    else Op<uint8_t>::launch(a, tasks, count, st, args...);
    const int s = kv_status();
    if (s != kOk) return s;
  }
  return kOk;
}

template <typename U>
struct CopyOp {
  static constexpr bool kRows = false;
  static constexpr int kThreads = kCpThreads, kTask = kCpThreads * kCpUnroll;
  static void launch(const KvCaches& a, int64_t tasks, int64_t pairs, hipStream_t st, const int32_t* frm,
                     const int32_t* to, int num_pages) {
    hipLaunchKernelGGL(copy_pages_kernel<U>,
                       dim3((unsigned)tasks, (unsigned)std::min<int64_t>(pairs, kCpPairs)),
                       dim3(kCpThreads), 0, st, a, frm, to, (int)pairs, num_pages);
  }
};
template <typename U>
struct KeepOp {
  static constexpr bool kRows = true;
  static constexpr int kThreads = kWave, kTask = kWave;
  static void launch(const KvCaches& a, int64_t tasks, int64_t B, hipStream_t st, const int32_t* path,
                     int64_t path_st, const int32_t* count, const int32_t* ctx, const int32_t* table,
                     int64_t table_st, int P, int page, int num_pages, int max_n) {
    hipLaunchKernelGGL(keep_rows_kernel<U>, dim3((unsigned)tasks, (unsigned)B), dim3(kWave), 0, st, a,
                       path, path_st, count, ctx, table, table_st, P, page, num_pages, max_n);
  }
};

}  // namespace dash

extern "C" int dash_copy_pages(int num_caches, void* const* caches, const int64_t* desc,
                               const int32_t* from_pages, const int32_t* to_pages, int num_pairs,
                               int num_pages, void* stream) {
  using namespace dash;
  if (num_caches < 0 || num_pairs < 0 || num_pages < 0) return kErrInvalid;
  if (num_caches == 0 || num_pairs == 0 || num_pages == 0) return kOk;
  if (!caches || !desc || !from_pages || !to_pages) return kErrInvalid;
  return kv_launches<CopyOp>(caches, desc, num_caches, num_pairs, stream, from_pages, to_pages, num_pages);
}

extern "C" int dash_keep_rows(int num_caches, void* const* caches, const int64_t* desc,
                              const int32_t* path, int64_t path_stride, const int32_t* count,
                              const int32_t* context_lens, const int32_t* block_table,
                              int64_t table_stride, int B, int P, int page_size, int num_pages,
                              int max_query_len, void* stream) {
  using namespace dash;
  if (num_caches < 0 || B < 0 || P < 0 || page_size <= 0 || num_pages < 0 || max_query_len < 0)
    return kErrInvalid;
  if (num_caches == 0 || B == 0 || P == 0 || num_pages == 0 || max_query_len == 0) return kOk;
  if (!caches || !desc || !path || !count || !context_lens || !block_table) return kErrInvalid;
  if (B > 65535) return kErrUnsupported;
  return kv_launches<KeepOp>(caches, desc, num_caches, B, stream, path, path_stride, count,
                             context_lens, block_table, table_stride, P, page_size, num_pages,
                             max_query_len);
}

extern "C" int dash_keep_lens(const int32_t* path, int64_t path_stride, const int32_t* count,
                              const int32_t* context_lens, const int32_t* lens, int B,
                              int max_query_len, int32_t* stand, int32_t* kept,
                              int32_t* new_context, int32_t* summed, void* stream) {
  using namespace dash;
  if (B < 0 || max_query_len < 0) return kErrInvalid;
  if (B == 0) return kOk;
  if ((max_query_len > 0 && !path) || !count || !context_lens || !lens || !stand || !kept ||
      !new_context || !summed)
    return kErrInvalid;
  hipLaunchKernelGGL(keep_lens_kernel, dim3(B / 256 + 1), dim3(256), 0, (hipStream_t)stream, path,
                     path_stride, count, context_lens, lens, B, max_query_len, stand, kept,
                     new_context, summed);
  return kv_status();
}

extern "C" int dash_fork_pages(int32_t* refs, int num_pages, int32_t* block_table,
                               int64_t table_stride, int R, int P, int32_t* lens,
                               const int32_t* src_rows, const int32_t* dst_rows, int n,
                               int page_size, int32_t* ok, int32_t* from_pages, int32_t* to_pages,
                               void* stream) {
  using namespace dash;
  if (!refs || !block_table || !lens || !ok || num_pages < 0 || R < 0 || P < 0 || n < 0 ||
      page_size <= 0)
    return kErrInvalid;
  if (n > 0 && (!src_rows || !dst_rows || !from_pages || !to_pages)) return kErrInvalid;
  if (R > kKvMaxRows || n > kKvMaxRows) return kErrUnsupported;
  hipLaunchKernelGGL(fork_pages_kernel, dim3(1), dim3(kKvThreads), 0, (hipStream_t)stream, refs,
                     num_pages, block_table, table_stride, R, P, lens, src_rows, dst_rows, n,
                     page_size, ok, from_pages, to_pages);
  return kv_status();
}

extern "C" int dash_reserve_pages(int32_t* refs, int num_pages, int32_t* block_table,
                                  int64_t table_stride, int R, int P, int32_t* lens,
                                  const int32_t* new_lens, int page_size, int32_t* ok,
                                  int32_t* from_pages, int32_t* to_pages, void* stream) {
  using namespace dash;
  if (!refs || !block_table || !lens || !new_lens || !ok || !from_pages || !to_pages ||
      num_pages < 0 || R < 0 || P < 0 || page_size <= 0)
    return kErrInvalid;
  // (the pages that all rows want, at most R * P, are added up in 32 bits)
  if (R > kKvMaxRows || (int64_t)R * P > INT32_MAX) return kErrUnsupported;
  hipLaunchKernelGGL(reserve_pages_kernel, dim3(1), dim3(kKvThreads), 0, (hipStream_t)stream, refs,
                     num_pages, block_table, table_stride, R, P, lens, new_lens, page_size, ok,
                     from_pages, to_pages);
  return kv_status();
}

extern "C" int dash_free_pages(int32_t* refs, int num_pages, int32_t* block_table,
                               int64_t table_stride, int R, int P, int32_t* lens,
                               const int32_t* keep_lens, int page_size, void* stream) {
  using namespace dash;
  if (!refs || !block_table || !lens || !keep_lens || num_pages < 0 || R < 0 || P < 0 ||
      page_size <= 0)
    return kErrInvalid;
  if (R > kKvMaxRows) return kErrUnsupported;
  if (R == 0) return kOk;
  hipLaunchKernelGGL(free_pages_kernel, dim3(R), dim3(256), 0, (hipStream_t)stream, refs, num_pages,
                     block_table, table_stride, P, lens, keep_lens, page_size);
  return kv_status();
}

extern "C" int dash_compact_pages(const int32_t* refs, int num_pages, const int32_t* block_table,
                                  int64_t table_stride, int R, int P, const int32_t* lens,
                                  int page_size, int32_t* new_refs, int32_t* new_table,
                                  int32_t* from_pages, int32_t* to_pages, int32_t* place,
                                  void* stream) {
  using namespace dash;
  if (num_pages < 0 || R < 0 || P < 0 || page_size <= 0) return kErrInvalid;
  if (num_pages > 0 && (!refs || !new_refs || !from_pages || !to_pages || !place)) return kErrInvalid;
  const int64_t entries = (int64_t)R * P;
  if (entries > 0 && (!block_table || !lens || !new_table || (num_pages > 0 && !place)))
    return kErrInvalid;
  if (R > kKvMaxRows || !fits_grid((entries + 255) / 256, 256)) return kErrUnsupported;
  hipStream_t st = (hipStream_t)stream;
  if (num_pages > 0)
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kKvThreads), 0, st, refs, num_pages,
                       new_refs, from_pages, to_pages, place);
  if (entries > 0)
    hipLaunchKernelGGL(compact_table_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, st,
                       block_table, table_stride, R, P, lens, page_size, place, num_pages, new_table);
  return kv_status();
}
