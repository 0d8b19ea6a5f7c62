// Full attention of a batch whose sequences share prompts, over a paged cache.  Included by
// dash_prefill.hip, whose tile helpers it uses.
//
// Row r = cu[b] + i is new token i of sequence b, at position t = ctx[b] + i, and sees the keys j <= t.
// The keys below prefix[g] of the sequences of group g (cu_groups[g] <= b < cu_groups[g + 1]) are read
// through one block-table row, once for all rows of the group: that of the first sequence that has rows and holds the
// prefix (an answer that left holds nothing), or the most of it.  The others are read through the sequence's own row.
// So there are G + B segments: rows of a group with the keys [0, prefix), and rows of a sequence with the keys
// [prefix, ctx + n).  A row's result is the sum of two segments'.
//
// The lengths lie on the device, and a launch's grid cannot depend on them: a plan adds up the
// segments' work in units of 64 keys and one tile of rows, the same for every key head, and each of the W
// work-groups of a head takes the same number of units, one after another, over as many segments as that
// reaches.  Each run of units within a (segment, row tile) leaves an unnormalised fp32 partial per row, and
// the merge kernel adds a row's partials up.  Neighbouring work-groups take the heads of the same keys, whose
// rows lie side by side in memory (each head's keys by work-groups of their own: 124 us for the 32 answers below, 95).
//
// Up to 64 sequences and groups, every work-group makes the plan for itself (1.5 us more of the attention, where a
// launch before it takes 5: 4 answers 22.0 us and 19.4, 32 answers 100.4 and 97.8); more need the plan kernel.
//
// Bound by HBM where the cache is long: 32 answers to 4 prompts, 10 heads of 128, a call 98 us: attention 92.5, 475 MB
// fetched (every key once, a prompt's for all its answers) at 5.1 TB/s, merge 6.6.  64 answers to one prompt 82 us, 314
// MB at 3.9 TB/s in 81, merge 6.4: of its 1,011 units a head 585 are own keys, one row of a tile of 64, whose second
// row tile's wavefronts leave at once, and a CU's two work-groups wait for a unit's keys, sums and barriers in turn
// (matrix cores busy 14 % of the time, vector units 27 %; of the 32 answers 13 and 23).  Few keys are bound by the
// chain lengths, pages, keys, sums, merge: 4 answers 13.4 + 6.6 us.
//
// A prompt itself: every row tile of a sequence takes the keys up to the last row's, and half of the units of one
// without a context hold none that the tile sees: they are fetched, and left at once.  8,190 tokens of 10 heads 651 us
// (2,730: 125).
#pragma once

namespace dash {

constexpr int kShMaxSeqs = 8192;
constexpr int kShMaxKeys = INT32_MAX - 127;      // (a tile's end past the last key is a number of 32 bits still)
constexpr int kShThreads = 256;           // of the plan kernel
constexpr int kShFew = 64;                // sequences, and groups, whose plan every work-group makes for itself

struct SharedSeg {
  int32_t r0, rows;                       // first packed row; rows times query heads of a key head
  int32_t k0, k1;                         // keys
  int32_t table_row, group;               // group: of a sequence's segment, -1 none
  int32_t base, tiles;                    // partial rows of a head of the segments before; row tiles
  int32_t lo, unused[3];                  // keys below it are seen by every row
};

struct SharedArgs {
  const bf16* q; int64_t q_st, q_sh;
  const bf16* k; int64_t k_sp, k_st, k_sh;
  const bf16* v; int64_t v_sp, v_st, v_sh;
  const int32_t* table; int64_t table_stride; int page, num_pages;
  const int32_t* ctx; const int32_t* cu;
  const int32_t* cu_groups; const int32_t* prefix;
  void* out; int out_bf16; int64_t o_st, o_sh;
  float* lse; int64_t lse_st, lse_sh;
  int B, G, H, Hkv, S, tile_rows;
  int W;                                  // work-groups of a key head
  int64_t T, parts;                       // partial rows of a key head
  float scale_log2e;
  // workspace
  int64_t* head;                          // units in all, units of a work-group
  int64_t* starts;                        // [G + B] units of the segments before
  SharedSeg* seg;                         // [G + B]
  int32_t* row_seq; int32_t* row_pos;     // [T]
  float2* part_ml;                        // base-2 reference and weight sum
  float* part_o;                          // [.., 128]
};

__device__ __forceinline__ int sh_cu(const SharedArgs& a, int b) {
  return (int)min(max((int64_t)a.cu[b], (int64_t)0), a.T);
}

// a / b rounded down, of numbers of 53 bits at most (a product of the two is none: the quotient of the
// doubles does not reach the next whole number).
__device__ __forceinline__ int64_t sh_div(int64_t a, int64_t b) { return (int64_t)((double)a / (double)b); }

// Units of a work-group.  Of larger tiles at least two: a run's partials are as many bytes as a unit's keys and more (128
// rows: 64 KB; three groups of three sequences 28.3 us with one, 24.6 with two, 27.8 with four; 32 rows: 19.4 and 21.4).
__device__ __forceinline__ int64_t sh_per(const SharedArgs& a, int64_t all) {
  return max(sh_div(all + a.W - 1, a.W), (int64_t)(a.tile_rows > 32 ? 2 : 1));
}

// Sum over the work-group's earlier threads, and over all.
__device__ __forceinline__ int64_t sh_before(int64_t v, int64_t* sW, int64_t& total) {
  const int lane = wave_lane(), wv = threadIdx.x / kWave;
  int64_t x = v;
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) {
    const int64_t y = __shfl_up(x, s, kWave);
    if (lane >= s) x += y;
  }
  __syncthreads();
  if (lane == kWave - 1) sW[wv] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kShThreads / kWave; ++w) {
    if (w < wv) before += sW[w];
    total += sW[w];
  }
  return before + x - v;
}

// The segment of a group of sequences from .. to - 1, whose rows start at cu(b); of sequence b with rows r0 .. r1 - 1, in
// a batch of groups that start at cu_groups.
template <typename Cu>
__device__ __forceinline__ SharedSeg sh_group(const SharedArgs& a, int from, int to, int prefix, Cu cu) {
  SharedSeg g = {0, 0, 0, 0, 0, -1, 0, 0, INT32_MAX, {0, 0, 0}};
  const int b0 = min(max(from, 0), a.B), b1 = min(max(to, b0), a.B);
  g.r0 = cu(b0);
  g.rows = b1 > b0 ? max(cu(b1) - g.r0, 0) * (a.H / a.Hkv) : 0;
  g.k1 = min(max(prefix, 0), a.S);
  return g;
}
__device__ __forceinline__ SharedSeg sh_sequence(const SharedArgs& a, int b, int r0, int r1, int ctx,
                                                 const int* cu_groups, const int* prefix) {
  SharedSeg g = {0, 0, 0, 0, 0, -1, 0, 0, 0, {0, 0, 0}};
  const int n = max(r1 - r0, 0);
  g.r0 = r0;
  g.rows = n * (a.H / a.Hkv);
  int lo = -1, hi = a.G;                  // the last group that starts at or before b
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_groups[mid] <= b) lo = mid; else hi = mid;
  }
  if (lo >= 0 && b < cu_groups[lo + 1]) {
    g.group = lo;
    g.k0 = min(max(prefix[lo], 0), a.S);
  }
  ctx = min(max(ctx, 0), a.S);
  g.k1 = (int)min((int64_t)ctx + n, (int64_t)a.S);
  g.lo = ctx + 1;
  g.table_row = b;
  return g;
}
// How much of its group's prefix a sequence holds.
__device__ __forceinline__ int sh_holds(const SharedSeg& g) { return min(g.k0, g.k1); }

// With the partial rows before it, of groups or of sequences (those of sequences lie behind those of groups); its units.
// Groups, or sequences, whose prefix sums are none could have more rows than the workspace holds.
__device__ __forceinline__ int64_t sh_place(const SharedArgs& a, SharedSeg& g, bool group, int64_t before) {
  const int64_t room = a.T * (a.H / a.Hkv);
  if (before + g.rows > room) g.rows = 0;
  g.base = (int)min(group ? before : room + before, 2 * room);
  g.tiles = (g.rows + a.tile_rows - 1) / a.tile_rows;
  return (int64_t)g.tiles * ((max(g.k1 - g.k0, 0) + 63) / 64);
}
// Row r's sequence and position, of sequences whose rows start at cu.
__device__ __forceinline__ int2 sh_row(const SharedArgs& a, int64_t r, const int* cu, const int* ctx) {
  if (r < cu[0] || r >= cu[a.B]) return make_int2(-1, -1);
  int lo = 0, hi = a.B;                   // cu[lo] <= r < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= r) lo = mid; else hi = mid;
  }
  return make_int2(lo, (int)min((int64_t)min(max(ctx[lo], 0), a.S) + (r - cu[lo]), (int64_t)INT32_MAX - 1));
}

// Work-group 0: the segments and their units.  The others: the sequence and position of every row.
__global__ __launch_bounds__(kShThreads) void shared_plan_kernel(SharedArgs a) {
  __shared__ int sCu[kShMaxSeqs + 1], sLo[kShMaxSeqs];
  __shared__ unsigned long long sFrom[kShMaxSeqs];      // the most of a prefix that is held, and the first to hold it
  __shared__ int64_t sW[kShThreads / kWave];
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (int b = tid; b <= a.B; b += kShThreads) sCu[b] = sh_cu(a, b);
    __syncthreads();
    const int64_t r = (int64_t)(blockIdx.x - 1) * kShThreads + tid;
    if (r >= a.T) return;
    const int2 at = sh_row(a, r, sCu, a.ctx);
    a.row_seq[r] = at.x;
    a.row_pos[r] = at.y;
    return;
  }
  int64_t units_before = 0, rows_before = 0, own_before = 0;
  const int ns = a.G + a.B;
  for (int g = tid; g <= a.G && a.G > 0; g += kShThreads) {
    sCu[g] = a.cu_groups[g];
    if (g < a.G) { sLo[g] = INT32_MAX; sFrom[g] = 0; }
  }
  __syncthreads();
  for (int s0 = 0; s0 < ns; s0 += kShThreads) {
    const int s = s0 + tid;
    SharedSeg g = {0, 0, 0, 0, 0, -1, 0, 0, 0, {0, 0, 0}};
    const bool group = s < a.G;
    if (group) {
      g = sh_group(a, sCu[s], sCu[s + 1], a.prefix[s], [&](int b) { return sh_cu(a, b); });
    } else if (s < ns) {
      const int b = s - a.G;
      g = sh_sequence(a, b, sh_cu(a, b), sh_cu(a, b + 1), a.ctx[b], sCu, a.prefix);
      if (g.group >= 0 && g.rows > 0) {
        atomicMin(&sLo[g.group], g.lo);
        atomicMax(&sFrom[g.group], (unsigned long long)sh_holds(g) << 32 | (uint32_t)~g.table_row);
      }
    }
    int64_t total, own_total;
    // (groups come first: of a group's thread, rows of groups)
    const int64_t rows = sh_before(g.rows, sW, total) + rows_before;
    const int64_t own = sh_before(group ? 0 : g.rows, sW, own_total) + own_before;
    rows_before += total;
    own_before += own_total;
    const int64_t units = sh_place(a, g, group, group ? rows : own);
    const int64_t before = sh_before(units, sW, total);
    if (s < ns) {
      a.starts[s] = units_before + before;
      a.seg[s] = g;
    }
    units_before += total;
  }
  if (tid == 0) {
    a.head[0] = units_before;
    a.head[1] = sh_per(a, units_before);
  }
  __syncthreads();
  for (int g = tid; g < a.G; g += kShThreads) {
    a.seg[g].lo = sLo[g];
    a.seg[g].table_row = sFrom[g] ? (int)~(uint32_t)sFrom[g] : 0;     // (0: of a group without rows no key is read)
  }
}

// The same of up to kShFew sequences and groups, by one wavefront, a lane for a group and for a sequence; every
// work-group of the attention makes it for itself.  A segment's partial rows start where its packed rows do.  Returns
// the units in all.
struct SharedFew {
  int64_t starts[2 * kShFew];
  SharedSeg seg[2 * kShFew];
  int most[kShFew], from[kShFew], lo[kShFew], prefix[kShFew], cu_groups[kShFew + 1];
};
__device__ __forceinline__ int64_t sh_plan_few(const SharedArgs& a, int* sCu, int* sCtx, SharedFew* few) {
  const int lane = wave_lane(), Gq = a.H / a.Hkv;
  {                                       // (every load before the first wait)
    const int32_t* groups = a.G > 0 ? a.cu_groups : a.cu;
    const int32_t* prefix = a.G > 0 ? a.prefix : a.cu;
    const int c = sh_cu(a, min(lane, a.B)), c_last = sh_cu(a, a.B), x = a.ctx[min(lane, a.B - 1)];
    const int g = groups[min(lane, a.G)], g_last = groups[a.G], pre = prefix[min(lane, max(a.G - 1, 0))];
    few->lo[lane] = INT32_MAX;
    few->most[lane] = 0;
    few->from[lane] = INT32_MAX;
    sCtx[lane] = x;
    few->prefix[lane] = pre;
    sCu[lane] = c;
    few->cu_groups[lane] = g;
    if (lane == 0) { sCu[kShFew] = c_last; few->cu_groups[kShFew] = g_last; }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  SharedSeg g = {0, 0, 0, 0, 0, -1, 0, 0, 0, {0, 0, 0}}, q = g;
  if (lane < a.G)
    g = sh_group(a, few->cu_groups[lane], few->cu_groups[lane + 1], few->prefix[lane], [&](int b) { return sCu[b]; });
  if (lane < a.B) q = sh_sequence(a, lane, sCu[lane], sCu[lane + 1], sCtx[lane], few->cu_groups, few->prefix);
  if (q.group >= 0 && q.rows > 0) {
    atomicMin(&few->lo[q.group], q.lo);
    atomicMax(&few->most[q.group], sh_holds(q));
  }
  g.base = g.r0 * Gq;
  q.base = ((int)a.T + q.r0) * Gq;
  g.tiles = (g.rows + a.tile_rows - 1) / a.tile_rows;
  q.tiles = (q.rows + a.tile_rows - 1) / a.tile_rows;
  const int64_t gu = (int64_t)g.tiles * ((max(g.k1 - g.k0, 0) + 63) / 64);
  const int64_t qu = (int64_t)q.tiles * ((max(q.k1 - q.k0, 0) + 63) / 64);
  int64_t gs = gu, qs = qu;
#pragma unroll 1
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t x = __shfl_up((long long)gs, d, kWave), y = __shfl_up((long long)qs, d, kWave);
    gs += lane >= d ? x : 0;
    qs += lane >= d ? y : 0;
  }
  const int64_t g_units = __shfl((long long)gs, kWave - 1, kWave), units = g_units + __shfl((long long)qs, kWave - 1, kWave);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  // (in two steps of 32 bits: one of 64, as in the plan kernel, costs the attention three registers that it lacks)
  if (q.group >= 0 && q.rows > 0 && few->most[q.group] == sh_holds(q)) atomicMin(&few->from[q.group], lane);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (lane < a.G) {
    g.lo = few->lo[lane];
    g.table_row = min(few->from[lane], a.B - 1);
    few->seg[lane] = g;
    few->starts[lane] = gs - gu;
  }
  if (lane < a.B) {
    few->seg[a.G + lane] = q;
    few->starts[a.G + lane] = g_units + qs - qu;
  }
  return units;
}

// The last segment that starts at or before unit u, over the wavefront.
__device__ __forceinline__ int sh_find(const SharedArgs& a, const int64_t* starts, int64_t u) {
  const int lane = wave_lane();
  int lo = 0, n = a.G + a.B;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const int i = lane * step;
    const bool at = i < n && starts[lo + i] <= u;
    const int c = max(__popcll(__ballot(at)) - 1, 0) * step;
    lo += c;
    n = min(step, n - c);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// What a unit is: seg, first row, first key, end of the segment's keys; table row, end of the keys that every row of
// the tile sees, whether its run starts or ends with it, rows of the segment; first packed row, partial rows before,
// end of the keys that the first row sees.
struct SharedUnit { int4 a, b, c; };
constexpr int kShUnits = 64;              // made at a time, a lane each

// Units u .. of the work-group's u0 .. u_end - 1, by one wavefront: the segments that begin among them are met one
// after another.
__device__ __forceinline__ void sh_units(const SharedArgs& a, const int64_t* starts, const SharedSeg* segs,
                                         int64_t u0, int64_t u, int64_t u_end, int tr, SharedUnit* sU) {
  const int lane = wave_lane(), ns = a.G + a.B, Gq = a.H / a.Hkv;
  const int n = (int)min((int64_t)kShUnits, u_end - u);
  const int64_t mine = u + min(lane, n - 1);
  const int s0 = sh_find(a, starts, u);
  int s = s0;
  for (int k0 = s0 + 1; k0 < ns; k0 += kWave) {
    const int64_t next = k0 + lane < ns ? starts[k0 + lane] : INT64_MAX;
    uint64_t some = __ballot(next < u + n);
    const bool more = some == ~0ull;
    for (; some; some &= some - 1) {
      const int l = __builtin_ctzll(some);
      if (__shfl((long long)next, l, kWave) <= mine) s = k0 + l;
    }
    if (!more) break;
  }
  const SharedSeg g = segs[s];
  const int items = max((g.k1 - g.k0 + 63) / 64, 1);
  const int64_t rel = mine - starts[s];
  const int tile = (int)sh_div(rel, items), i = (int)(rel - (int64_t)tile * items), rb = tile * tr;
  const int j0 = g.k0 + 64 * i;
  const int seen = min(s >= a.G ? (int)min((int64_t)g.lo + rb / Gq, (int64_t)INT32_MAX) : g.lo, g.k1);
  const int ends = (i == 0 || mine == u0 ? 1 : 0) | (i == items - 1 || mine == u_end - 1 ? 2 : 0);
  if (lane < n) {
    sU[lane].a = make_int4(s, rb, j0, g.k1);
    sU[lane].b = make_int4(g.table_row, seen, ends, g.rows);
    sU[lane].c = make_int4(g.r0, g.base, g.lo, 0);
  }
}

// RT row tiles of 32 rows are the columns of S^T = K Q^T (v_mfma_f32_32x32x16_bf16); with KG = 2 two
// wavefronts share a row tile, one half of 64 keys each, and meet at the end of a run.  Weights enter
// the second product as three bf16 parts (24 bits), so that a bf16 output is the fp32 one rounded once.
// A work-group's units form one pipeline whatever runs they belong to: the next unit's keys and values are on their
// way to LDS (two stages) and the pages of the units after looked up while one is multiplied.
// FEW: the plan is made here.
template <int RT, int KG, bool FEW>
__global__ __launch_bounds__(64 * RT * KG, 2) void shared_attn_kernel(SharedArgs a) {
  constexpr int D = 128, NW = RT * KG, TH = 64 * NW, TR = 32 * RT;
  constexpr int NH = 2 / KG;              // halves of 64 keys that a wavefront takes
  constexpr int PARTS = 3;                // of a weight
  constexpr int CH = RT == 1 ? 2 : 4;     // units whose rows' offsets are laid out at a time
  constexpr int PER = 64 * CH / TH;       // offsets of a thread
  constexpr int ST = RT == 1 ? 1 : 2;     // stages
  constexpr int NG = 16 / NW;             // groups of four key rows that a wavefront loads
  constexpr int kAux = RT == 4 ? 0 : 2;   // past the caches, but where tiles of the same keys share them (112, 100 us)
  __shared__ __attribute__((aligned(16))) bf16 sK0[64 * D];
  __shared__ __attribute__((aligned(16))) bf16 sK1[ST == 2 ? 64 * D : 8];
  __shared__ __attribute__((aligned(16))) bf16 sV0[64 * D];
  __shared__ __attribute__((aligned(16))) bf16 sV1[ST == 2 ? 64 * D : 8];
  __shared__ SharedUnit sU[kShUnits];
  __shared__ longlong2 sOff[2][64 * CH];  // offsets of a key row in K and V
  __shared__ uint32_t sBad[2][NW];
  __shared__ float2 sMl[32 * RT];
  __shared__ int sCu[FEW ? kShFew + 1 : 1], sCtx[FEW ? kShFew : 1];
  __shared__ int64_t sAll;
  const int tid = threadIdx.x, lane = wave_lane();
  const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int rt = wv % RT, kg = wv / RT;
  const int hl = lane >> 5, col = lane & 31;
  const int Gq = a.H / a.Hkv;
  const int hk = blockIdx.x % a.Hkv, turn = blockIdx.x / a.Hkv;
  // (the plan of a few lies where keys will)
  static_assert(sizeof(SharedFew) <= sizeof(sK0), "its room");
  SharedFew* const few = (SharedFew*)sK0;
  int64_t u0 = 0, u_end = 0;
  auto mine = [&](int64_t all, int64_t per) { u0 = turn * per; u_end = min(u0 + per, all); };
  if (!FEW) {
    mine(a.head[0], a.head[1]);
    if (u0 >= u_end) return;
  }
  const uint32_t kl0 = k_lane_off(col, hl), vl0 = v_lane_off(lane);
  const float csc = a.scale_log2e;
  const bf16* const kb = a.k + hk * a.k_sh;
  const bf16* const vb = a.v + hk * a.v_sh;

  // the run at hand
  int rr = 0, end = 0, e_min = 0;         // this lane's row; keys below `end` are seen, below e_min by the wavefront's
  bool rvalid = false;
  bf16x8 qop[D / 16];
  floatx16 acc_o[D / 32];
  float m_run = -INFINITY, l_run = 0.f;

  auto begin = [&](int x) __attribute__((always_inline)) {
    const int4 ua = sU[x].a, ub = sU[x].b, uc = sU[x].c;
    const int rows = ub.w, r = ua.y + rt * 32 + col;
    rvalid = r < rows;
    rr = min(r, rows - 1);
    const int64_t row = uc.x + rr / Gq;
    const int h = hk * Gq + rr % Gq;
    end = ua.x >= a.G ? (int)min((int64_t)uc.z + rr / Gq, (int64_t)INT32_MAX)
                      : (FEW ? sh_row(a, row, sCu, sCtx).y : a.row_pos[row]) + 1;
    const bf16* qb = a.q + row * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) qop[kk] = *(const bf16x8*)(qb + kk * 16 + hl * 8);
    end = min(end, ua.w);
    int e = rvalid ? end : INT32_MAX;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) e = min(e, __shfl_xor(e, m, kWave));
    e_min = __builtin_amdgcn_readfirstlane(e);
    m_run = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int n = 0; n < 16; ++n) acc_o[dt][n] = 0.f;
  };
  // The table entries of units CH c .. of the batch; their offsets, once they have come.
  int page_of[PER];
  auto key_of = [&](int y, int c, int nu) {
    const int x = min(CH * c + y / 64, nu - 1);
    return min(sU[x].a.z + (y & 63), sU[x].a.w - 1);
  };
  auto look_up = [&](int c, int nu) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int y = n * TH + tid, x = min(CH * c + y / 64, nu - 1);
      page_of[n] = a.table[(int64_t)sU[x].b.x * a.table_stride + key_of(y, c, nu) / a.page];
    }
  };
  auto put = [&](int c, int nu) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int y = n * TH + tid, jp = key_of(y, c, nu) % a.page;
      const int p = min(max(page_of[n], 0), a.num_pages - 1);
      sOff[c & 1][y] = make_longlong2((int64_t)p * a.k_sp + (int64_t)jp * a.k_st,
                                      (int64_t)p * a.v_sp + (int64_t)jp * a.v_st);
    }
  };
  auto fetch = [&](int x, bf16* sKn, bf16* sVn) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int grp = NW * n + wv, r = 4 * grp + (lane >> 4);
      const longlong2 o = sOff[x / CH & 1][64 * (x % CH) + r];
      __builtin_amdgcn_global_load_lds((const void*)(kb + o.x + k_slot(r, lane & 15) * 8),
          (__attribute__((address_space(3))) void*)(sKn + grp * 4 * D), 16, 0, kAux);
      __builtin_amdgcn_global_load_lds((const void*)(vb + o.y + v_slot(r, lane & 15) * 8),
          (__attribute__((address_space(3))) void*)(sVn + grp * 4 * D), 16, 0, kAux);
    }
  };
  // V values that are not finite would reach, through weights of 0, rows that do not see their keys.
  // Where some row does not see every key, each wavefront clears them in the rows it loaded, and notes
  // their groups: item() adds them to the rows that see them.
  auto clear = [&](int x, bf16* sVn, uint32_t* bad_of) __attribute__((always_inline)) {
    uint32_t bad = 0;
    if (__builtin_amdgcn_readfirstlane(sU[x].a.z) + 64 > __builtin_amdgcn_readfirstlane(sU[x].b.y)) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        uint4* p = (uint4*)(sVn + (NW * n + wv) * 4 * D) + lane;
        uint4 y = *p;
        bool is = false;
        auto fix = [&](uint32_t& w) {
          if ((w & 0x7f80u) == 0x7f80u) { w &= 0xffff0000u; is = true; }
          if ((w & 0x7f800000u) == 0x7f800000u) { w &= 0xffffu; is = true; }
        };
        fix(y.x); fix(y.y); fix(y.z); fix(y.w);
        if (is) *p = y;
        if (__any(is)) bad |= 1u << n;
      }
    }
    if (lane == 0) bad_of[wv] = bad;
  };
  // unit x: this wavefront's halves
  auto item = [&](int x0, const bf16* sKc, const bf16* sVc,
                  const uint32_t* bad_of) __attribute__((always_inline)) {
    const int j0 = __builtin_amdgcn_readfirstlane(sU[x0].a.z);
    uint32_t vis[NH];
    bool any = false;
    auto below = [](int y) -> uint32_t { return y >= 32 ? ~0u : y <= 0 ? 0u : (1u << y) - 1u; };
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      const int j = j0 + 32 * (KG == 2 ? kg : x);
      vis[x] = rvalid ? (j + 32 <= e_min ? ~0u : below(end - j)) : 0u;
      any = any || vis[x] != 0u;
    }
    if (!__any(any)) return;
    floatx16 sc[NH];
    float mloc = -INFINITY;
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      const int hf = KG == 2 ? kg : x;
      bf16x8 kf[D / 16];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) kf[kk] = k_frag_at(sKc, kl0, hf, kk);
      floatx16 t;                       // two chains: a product need not wait for the one before it
#pragma unroll
      for (int r = 0; r < 16; ++r) { sc[x][r] = 0.f; t[r] = 0.f; }
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2) {
        sc[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk], qop[kk], sc[x], 0, 0, 0);
        t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk + 1], qop[kk + 1], t, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[x][r] += t[r];
      if (__all(vis[x] == 0u || vis[x] == ~0u)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[x][r] = vis[x] ? sc[x][r] : -INFINITY;
      } else {
        const uint32_t vb = vis[x] >> (4 * hl);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sc[x][r] = (vb >> (8 * (r >> 2) + (r & 3))) & 1u ? sc[x][r] : -INFINITY;
      }
      float mraw = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mraw = fmaxf(mraw, sc[x][r]);
      mloc = fmaxf(mloc, mraw * csc);
    }
    mloc = xor32_max(mloc);
    // the reference moves only when a row's maximum exceeds it by more than 8
    const bool up = mloc > m_run + 8.f;
    if (__any(up)) {
      const float alpha = up ? fast_exp2(m_run - mloc) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc_o[dt][r] *= alpha;
      m_run = up ? mloc : m_run;
    }
    const float off = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      const int hf = KG == 2 ? kg : x;
      bf16x8 vop[4][2];                 // V in registers before the weights are ready
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const char* vp = (const char*)sVc + (32 * hf + 16 * jj) * 256 + (vl0 ^ (uint32_t)(dt << 6));
          const bf16x4 l4 = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_short4*)(__attribute__((address_space(3))) void*)vp));
          const bf16x4 h4 = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_short4*)(__attribute__((address_space(3))) void*)(vp + 2048)));
#pragma unroll
          for (int e = 0; e < 4; ++e) { vop[dt][jj][e] = l4[e]; vop[dt][jj][e + 4] = h4[e]; }
        }
      uint32_t part[PARTS][2][4];
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(sc[x][8 * jj + e], csc, off));
        l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int n = 0; n < PARTS; ++n) {
            bf16x2 y;
            y[0] = (bf16)p[2 * e];
            y[1] = (bf16)p[2 * e + 1];
            const uint32_t w = __builtin_bit_cast(uint32_t, y);
            part[n][jj][e] = w;
            p[2 * e] -= __uint_as_float(w << 16);
            p[2 * e + 1] -= __uint_as_float(w & 0xffff0000u);
          }
      }
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int n = PARTS - 1; n >= 0; --n) {       // smallest parts first
          const bf16x8 w = __builtin_bit_cast(bf16x8, *(uint4*)part[n][jj]);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
            acc_o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vop[dt][jj], w, acc_o[dt], 0, 0, 0);
        }
    }
    if (j0 + 64 <= __builtin_amdgcn_readfirstlane(sU[x0].b.y)) return;
    for (int w = 0; w < NW; ++w)
      for (uint32_t todo = bad_of[w]; todo; todo &= todo - 1)
        for (int q4 = 0; q4 < 4; ++q4) {
          const int r = 4 * (NW * __builtin_ctz(todo) + w) + q4;
          if (j0 + r >= sU[x0].a.w || (KG == 2 && r / 32 != kg)) continue;   // a repeated row
          const bool sees = (vis[KG == 2 ? 0 : r / 32] >> (r & 31)) & 1u;
          const bf16* vp = vb + sOff[x0 / CH & 1][64 * (x0 % CH) + r].y + 4 * hl;
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const bf16x4 y = *(const bf16x4*)(vp + 32 * dt + 8 * n);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float f = (float)y[e];
                if (sees && !(fabsf(f) <= 3.402823466e38f)) acc_o[dt][4 * n + e] += f;
              }
            }
        }
  };
  // the end of a run; the stage of its last unit is free once every wavefront has left it
  auto finish = [&](int x, bf16* sKc, bf16* sVc) __attribute__((always_inline)) {
    float l_tot = xor32_sum(l_run);
    if (KG == 2) {
      // the second half's wavefronts hand their sums to the first's
      __syncthreads();
      float* so = (float*)(rt ? sVc : sKc);
      if (kg == 1) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) so[(16 * dt + r) * 64 + lane] = acc_o[dt][r];
        if (hl == 0) sMl[rt * 32 + col] = make_float2(m_run, l_tot);
      }
      __syncthreads();
      if (kg == 0) {
        const float2 ml = sMl[rt * 32 + col];
        const float mn = fmaxf(m_run, ml.x), mu = mn == -INFINITY ? 0.f : mn;
        const float al = fast_exp2(m_run - mu), be = fast_exp2(ml.x - mu);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc_o[dt][r] = acc_o[dt][r] * al + so[(16 * dt + r) * 64 + lane] * be;
        l_tot = l_tot * al + ml.y * be;
        m_run = mn;
      }
    }
    if (kg == 0 && rvalid) {
      const int64_t at = hk * a.parts + sU[x].c.y + rr + (int64_t)turn * TR;
      float* po = a.part_o + at * D + 4 * hl;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          *(float4*)(po + dt * 32 + 8 * n) = make_float4(acc_o[dt][4 * n], acc_o[dt][4 * n + 1],
                                                         acc_o[dt][4 * n + 2], acc_o[dt][4 * n + 3]);
      if (hl == 0) a.part_ml[at] = make_float2(m_run, l_tot);
    }
  };

  bool planned = !FEW;
  for (int64_t u = u0; !planned || u < u_end; u += kShUnits) {
    __syncthreads();                      // every wavefront left the batch before
    SharedArgs b = a;
    if (FEW) {
      // (read again here: held from the start, the arguments would cost the loop registers)
      auto* args = (const __attribute__((address_space(4))) SharedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+s"(args));
      b.cu = args->cu; b.ctx = args->ctx; b.cu_groups = args->cu_groups; b.prefix = args->prefix;
      b.B = args->B; b.G = args->G; b.H = args->H; b.Hkv = args->Hkv; b.S = args->S; b.tile_rows = args->tile_rows;
      b.W = args->W; b.T = args->T;
      b.head = args->head; b.starts = args->starts; b.seg = args->seg; b.row_seq = args->row_seq;
      if (wv == 0) {
        const int64_t all = sh_plan_few(b, sCu, sCtx, few);
        if (lane == 0) sAll = all;
      }
      __syncthreads();
    }
    if (FEW && !planned) {
      const int64_t all = sAll, per = sh_per(b, all);
      mine(all, per);
      // what the merge needs of it
      if (blockIdx.x == 0) {
        if (tid == 0) { b.head[0] = all; b.head[1] = per; }
        for (int s = tid; s < b.G + b.B; s += TH) { b.starts[s] = few->starts[s]; b.seg[s] = few->seg[s]; }
      }
      for (int64_t r = (int64_t)blockIdx.x * TH + tid; r < b.T; r += (int64_t)gridDim.x * TH)
        b.row_seq[r] = sh_row(b, r, sCu, sCtx).x;
      if (u0 >= u_end) return;
      u = u0;
      planned = true;
    }
    const int nu = (int)min((int64_t)kShUnits, u_end - u), chunks = (nu + CH - 1) / CH;
    if (wv == 0) sh_units(b, FEW ? few->starts : a.starts, FEW ? few->seg : a.seg, u0, u, u_end, TR, sU);
    __syncthreads();
    look_up(0, nu);
    put(0, nu);
    __syncthreads();
    if (ST == 2) fetch(0, sK0, sV0);
    auto step = [&](int x, auto par) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      bf16* const sKc = P ? sK1 : sK0;
      bf16* const sVc = P ? sV1 : sV0;
      const int ends = __builtin_amdgcn_readfirstlane(sU[x].b.z), c = x / CH;
      const bool ahead = x % CH == 0 && c + 1 < chunks;
      if (ST == 1) {
        __syncthreads();                  // every wavefront left unit x - 1
        fetch(x, sKc, sVc);
        if (ahead) look_up(c + 1, nu);
      }
      if (ends & 1) begin(x);
      __builtin_amdgcn_s_waitcnt(0);      // unit x landed, and what was looked up
      if (ST == 1 ? ahead : x % CH == 1 && c + 1 < chunks) put(c + 1, nu);
      clear(x, sVc, sBad[P]);
      __syncthreads();                    // every wavefront's part of it; and they left unit x - 1
      if (ST == 2) {
        if (x + 1 < nu) fetch(x + 1, P ? sK0 : sK1, P ? sV0 : sV1);
        if (ahead) look_up(c + 1, nu);
      }
      item(x, sKc, sVc, sBad[P]);
      if (ends & 2) finish(x, sKc, sVc);
    };
    for (int x = 0; x < nu; x += ST) {
      step(x, std::integral_constant<int, 0>{});
      if (ST == 2 && x + 1 < nu) step(x + 1, std::integral_constant<int, 1>{});
    }
  }
}

// One wavefront per (row, head): the partials of the row's two segments, a lane for the (maximum, sum) of each,
// 64 at a time; half a wavefront reads a partial, four dims a lane, and sixteen are in flight.
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a) {
  constexpr int D = 128, U = 8;
  const int64_t rh = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (rh >= a.T * a.H) return;
  const int lane = wave_lane(), hl = lane >> 5, Gq = a.H / a.Hkv;
  const int64_t row = rh / a.H;
  const int h = (int)(rh - row * a.H), hk = h / Gq;
  const int b = a.row_seq[row];
  // runs [first, first + n) of work-groups, and the row's place in the first one's partials
  int64_t at[2] = {0, 0};
  int n[2] = {0, 0};
  if (b >= 0) {
    const int64_t per = a.head[1];
    int s = a.G + b;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const SharedSeg g = a.seg[s];
      const int items = (max(g.k1 - g.k0, 0) + 63) / 64;
      const int64_t rr = (row - g.r0) * Gq + h % Gq;
      if (items > 0 && rr >= 0 && rr < g.rows) {
        const int64_t u0 = a.starts[s] + rr / a.tile_rows * items;
        const int64_t first = sh_div(u0, per);
        n[x] = (int)(sh_div(u0 + items - 1, per) - first) + 1;
        at[x] = hk * a.parts + g.base + rr + first * a.tile_rows;
      }
      if (g.group < 0) break;
      s = g.group;
    }
  }
  float M = -INFINITY, L = 0.f;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  bool any = false;
  const int all = n[0] + n[1];
  for (int e0 = 0; e0 < all; e0 += kWave) {
    const int e = e0 + lane;
    const bool in = e < all;
    const int64_t p = e < n[0] ? at[0] + (int64_t)e * a.tile_rows
                               : at[1] + (int64_t)(in ? e - n[0] : 0) * a.tile_rows;
    const float2 ml = in ? a.part_ml[p] : make_float2(-INFINITY, 0.f);
    // NaN in a score leaves the maximum and comes in through the sums
    const bool seen = in && !(ml.x == -INFINITY && ml.y == 0.f);
    const float Mn = fmaxf(M, wave_max(ml.x)), Mu = Mn == -INFINITY ? 0.f : Mn;
    const float al = fast_exp2(M - Mu), w = seen ? fast_exp2(ml.x - Mu) : 0.f;
    M = Mn;
    L = L * al + wave_sum(seen ? ml.y * w : 0.f);
    acc *= al;
    const uint64_t live = __ballot(seen);
    any = any || live != 0;
    const int m = min(kWave, all - e0);
    for (int i0 = 0; i0 < m; i0 += 2 * U) {
      floatx4 x[U];
      float f[U];
      bool in_sum[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int l = i0 + 2 * i + hl;
        const int64_t pl = __shfl(p, min(l, m - 1), kWave);
        f[i] = __shfl(w, min(l, m - 1), kWave);
        in_sum[i] = l < m && (live >> l) & 1u;
        x[i] = *(const floatx4*)(a.part_o + pl * D + 4 * (lane & 31));
      }
      // (every run that saw a key: where its weight is 0 its values need not be finite)
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (in_sum[i]) acc += f[i] * x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = xor32_sum(acc[i]);
  const float inv = any ? 1.f / L : 0.f;
  acc *= inv;
  const int64_t to = row * a.o_st + (int64_t)h * a.o_sh + 4 * lane;
  if (hl == 0) {
    if (a.out_bf16) {
      bf16x4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = (bf16)acc[i];
      *(bf16x4*)((bf16*)a.out + to) = r;
    } else {
      *(floatx4*)((float*)a.out + to) = acc;
    }
  }
  if (a.lse && lane == 0)
    a.lse[row * a.lse_st + (int64_t)h * a.lse_sh] = any ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

// Row tiles of a work-group by the rows that share a key head, and its work-groups: four a CU of the one-stage kernel,
// two of the others.  The rows are a group's on average, all that the host knows: one group beside many sequences of no
// group counts them as its own, which makes the tiles of their single rows larger than they need.
struct SharedPlan { int rt, W; int64_t parts, head, starts, seg, rows, ml, o, total; };
inline SharedPlan shared_plan(int B, int G, int H, int Hkv, int64_t T) {
  SharedPlan p;
  const int64_t rows = T * (H / Hkv) / std::max(1, G > 0 ? G : B);
  p.rt = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.W = std::max(1, (p.rt == 1 ? 1024 : 512) / Hkv);
  p.parts = 2 * T * (H / Hkv) + (int64_t)p.W * 32 * p.rt;
  const int64_t parts = p.parts * Hkv;
  auto align = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t o = 0;
  p.head = o; o += 256;
  p.starts = o; o = align(o + ((int64_t)G + B) * 8);
  p.seg = o; o = align(o + ((int64_t)G + B) * (int64_t)sizeof(SharedSeg));
  p.rows = o; o = align(o + 2 * T * 4);
  p.ml = o; o = align(o + parts * 8);
  p.o = o; o = align(o + parts * 128 * 4);
  p.total = o;
  return p;
}

// Sizes whose rows, partial rows and grids 32 bits hold (and whose workspace 64 do).
inline bool shared_takes(int B, int G, int H, int Hkv, int64_t T) {
  return H % Hkv == 0 && B <= kShMaxSeqs && G <= kShMaxSeqs && T <= INT32_MAX - kShThreads && 2 * T * H <= INT32_MAX &&
         fits_grid((T * H + 3) / 4, 256) && fits_grid((int64_t)shared_plan(B, G, H, Hkv, T).W * Hkv, 256);
}

}  // namespace dash

extern "C" int dash_attn_shared_workspace_size(int B, int G, int H, int Hkv, int64_t T, int64_t* bytes) {
  using namespace dash;
  if (!bytes || B < 0 || G < 0 || H <= 0 || Hkv <= 0 || T < 0) return kErrInvalid;
  if (!shared_takes(B, G, H, Hkv, T)) return kErrUnsupported;
  *bytes = shared_plan(B, G, H, Hkv, T).total;
  return kOk;
}

extern "C" int dash_attn_shared(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sp,
                                int64_t k_st, int64_t k_sh, const void* v, int64_t v_sp, int64_t v_st,
                                int64_t v_sh, const int32_t* block_table, int64_t table_stride, int P,
                                int page_size, int num_pages, const int32_t* context_lens,
                                const int32_t* cu_seqlens_q, const int32_t* cu_groups,
                                const int32_t* prefix_lens, void* out, int out_bf16, int64_t o_st,
                                int64_t o_sh, float* lse, int64_t lse_st, int64_t lse_sh, int B, int G, int H,
                                int Hkv, int64_t T, int D, float scale, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  using namespace dash;
  if (B < 0 || G < 0 || H <= 0 || Hkv <= 0 || T < 0 || P < 0 || page_size <= 0 || num_pages < 0)
    return kErrInvalid;
  if (T == 0) return kOk;
  if (!q || !out || !cu_seqlens_q || (B > 0 && !context_lens) || (G > 0 && (!cu_groups || !prefix_lens)))
    return kErrInvalid;
  if (B > 0 && P > 0 && !block_table) return kErrInvalid;
  if (num_pages > 0 && (!k || !v)) return kErrInvalid;
  if (D != 128 || !(scale > 0.f) || (int64_t)P * page_size > kShMaxKeys || !shared_takes(B, G, H, Hkv, T))
    return kErrUnsupported;
  const int64_t strides[] = {q_st, q_sh, k_sp, k_st, k_sh, v_sp, v_st, v_sh};
  for (int64_t s : strides)
    if (s % 8 != 0) return kErrUnsupported;
  const void* ptrs[] = {q, k, v};
  for (const void* x : ptrs)
    if ((uintptr_t)x % 16 != 0) return kErrUnsupported;
  const SharedPlan p = shared_plan(B, G, H, Hkv, T);
  if (!workspace || workspace_bytes < p.total || (uintptr_t)workspace % 256 != 0) return kErrWorkspace;
  char* w = (char*)workspace;
  SharedArgs a = {};
  a.q = (const bf16*)q; a.q_st = q_st; a.q_sh = q_sh;
  a.k = (const bf16*)k; a.k_sp = k_sp; a.k_st = k_st; a.k_sh = k_sh;
  a.v = (const bf16*)v; a.v_sp = v_sp; a.v_st = v_st; a.v_sh = v_sh;
  a.table = block_table; a.table_stride = table_stride; a.page = page_size; a.num_pages = num_pages;
  a.ctx = context_lens; a.cu = cu_seqlens_q; a.cu_groups = cu_groups; a.prefix = prefix_lens;
  a.out = out; a.out_bf16 = out_bf16; a.o_st = o_st; a.o_sh = o_sh;
  a.lse = lse; a.lse_st = lse_st; a.lse_sh = lse_sh;
  a.B = B; a.G = B > 0 ? G : 0; a.H = H; a.Hkv = Hkv; a.T = T;
  a.S = num_pages > 0 ? P * page_size : 0;
  a.W = p.W; a.parts = p.parts; a.tile_rows = 32 * p.rt; a.scale_log2e = scale * 1.4426950408889634f;
  a.head = (int64_t*)(w + p.head); a.starts = (int64_t*)(w + p.starts);
  a.seg = (SharedSeg*)(w + p.seg); a.row_seq = (int32_t*)(w + p.rows); a.row_pos = a.row_seq + T;
  a.part_ml = (float2*)(w + p.ml); a.part_o = (float*)(w + p.o);
  hipStream_t st = (hipStream_t)stream;
  const bool few = a.S > 0 && B > 0 && B <= kShFew && G <= kShFew;
  if (!few)
    hipLaunchKernelGGL(shared_plan_kernel, dim3((unsigned)(1 + (T + kShThreads - 1) / kShThreads)),
                       dim3(kShThreads), 0, st, a);
  if (a.S > 0) {
    const dim3 grid((unsigned)(p.W * Hkv)), block(p.rt == 1 ? 128 : 256);
    auto* const kernel = p.rt == 1 ? few ? shared_attn_kernel<1, 2, true> : shared_attn_kernel<1, 2, false>
                         : p.rt == 2 ? few ? shared_attn_kernel<2, 2, true> : shared_attn_kernel<2, 2, false>
                                     : few ? shared_attn_kernel<4, 1, true> : shared_attn_kernel<4, 1, false>;
    hipLaunchKernelGGL(kernel, grid, block, 0, st, a);
  }
  hipLaunchKernelGGL(shared_merge_kernel, dim3((unsigned)((T * H + 3) / 4)), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
