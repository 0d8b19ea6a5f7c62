// Attention of a tree of drafted tokens over a cache, and the trees' masks.  Included by
// dash_prefill.hip, whose tile helpers it uses.
//
// Row r = cu[b] + i is node i of sequence b, whose first ctx[b] keys are committed; the key and
// value of node m lie in the cache at slot ctx[b] + m.  With depth d the row's position is
// t = ctx[b] + d and its window starts at w = t - LW + 1.  It sees
//   committed keys j >= w                                       bias 0
//   committed keys j < w of its routed blocks (valid, first slot of a block wins)  bias b(r, c)
//   the drafted keys m whose bit is set in its mask             bias 0
// and a row that sees no key gives 0 (log-sum-exp -inf).
#pragma once

namespace dash {

constexpr int kTrMaxNodes = 256;
constexpr int64_t kTrTarget = 1024;       // work-groups a call aims at

struct TreeArgs {
  const bf16* q; int64_t q_st, q_sh;
  const bf16* k; int64_t k_sb, k_sh, k_st;     // sb: page (or sequence) stride
  const bf16* v; int64_t v_sb, v_sh, v_st;
  const int32_t* table; int64_t table_stride; int page, num_pages;   // null: contiguous
  const int32_t* ctx; const int32_t* cu;
  const int32_t* idx; const uint8_t* valid; const float* bias; int K;
  const uint64_t* mask; int words; const int32_t* depth;
  void* out; int out_bf16; int64_t o_st, o_sh;
  float* lse; int64_t lse_st, lse_sh;
  int B, H, Hkv, S, bs, lw, max_n;
  int groups, nsplit, slot_cap;                // slot_cap: slots of a row group
  float* part_o;                               // [T, H, nsplit, 128], not normalised
  float2* part_ml;                             // [T, H, nsplit] base-2 reference and weight sum
  int64_t T;
  float scale_log2e;
};

__device__ __forceinline__ int tree_ctx(const TreeArgs& a, int b) {
  return min(max(a.ctx[b], 0), a.S);
}

// A table entry that names no page is read as the nearest: no address leaves the cache.
__device__ __forceinline__ int tree_page(const TreeArgs& a, int p) {
  return min(max(p, 0), a.num_pages - 1);
}

// The masks and depths of the trees: one work-group per sequence, one lane per node, which
// climbs to the root (parents come before their children, so it ends).  Latency: two trips to memory
// (the prefix sums, then the parents: 1.4 us where the L2 of the work-group's XCD holds them, 2 to 3 more
// where it does not, as for 8 trees of up to 32 nodes, 3.7, and 32 of up to 64, 4.8) and 65 ns in LDS per
// level of the deepest node (a chain of 32 nodes 3.5 us, of 256 18).
__global__ __launch_bounds__(kTrMaxNodes) void tree_masks_kernel(const int32_t* parents,
                                                                 const int32_t* cu, int64_t T,
                                                                 int words, int max_n, uint64_t* mask,
                                                                 int32_t* depth) {
  __shared__ int sPar[kTrMaxNodes];
  const int b = blockIdx.x, i = threadIdx.x;
  int64_t r0;
  const int n = packed_rows(cu, b, T, max_n, r0);
  if (i < n) {
    const int p = parents[r0 + i];
    sPar[i] = p >= 0 && p < i ? p : -1;
  }
  __syncthreads();
  if (i >= n) return;
  uint64_t m[kTrMaxNodes / 64] = {0, 0, 0, 0};
  int d = -1;
  for (int j = i; j >= 0; j = sPar[j], ++d) {
#pragma unroll
    for (int w = 0; w < kTrMaxNodes / 64; ++w)
      if (j >> 6 == w) m[w] |= 1ull << (j & 63);
  }
#pragma unroll
  for (int w = 0; w < kTrMaxNodes / 64; ++w)
    if (w < words) mask[(r0 + i) * words + w] = m[w];
  depth[r0 + i] = d;
}

// ---------------------------------------------------------------------------
// One work-group per (sequence, key head, 32 RT rows, split).  The rows of a key head are
// (node, query head of its group) pairs, node first.  Keys come in halves of 32: the band from
// the root's window to the last drafted key, then the blocks that the rows name, in ascending
// order; an item is two halves, 64 keys of K and V in a double-buffered LDS stage filled by
// direct loads.  The items of a (sequence, head) are divided evenly among its splits, each of which
// writes an unnormalised fp32 partial that tree_merge_kernel adds up (one split writes the result).
//
// RT row tiles of 32 rows are the columns of S^T = K Q^T (v_mfma_f32_32x32x16_bf16); with KG = 2
// two wavefronts share a row tile, one half of every item each, and meet at the end.  A half's
// visible keys are 32 bits per row, so the band's edges, the drafted keys' mask and the routed
// blocks of rows that do not name them are one test.  A weight enters the second product as three
// bf16 parts (24 bits: it is not rounded), as in the extend kernels, whatever the output's type: a bf16
// output is the fp32 one rounded once.  Two parts (17 bits) changed the last bit of one bf16 output in
// 400; the third is a third of the matrix work and a quarter of the vector work, which an item's loads
// hide in all but the largest batches (8 trees of 16 to 32 nodes: 42.8 and 43.3 us, 32 trees of 24 to 64
// over 2,730 to 27,300 tokens: 119 and 124).
//
// Bound by HBM and the work on the weights together where there are many trees: those 32 fetch 500 MB
// (counted; every key once) and write 22 MB of partials in 119 to 123 us, 4.3 TB/s, where a read alone
// reaches 5.9.  Eight trees over 27,300 tokens fetch 127 MB in 37 us.  One tree of eight nodes takes 12 us for
// 8 MB: the rows, their slots, the page table, the keys and the partials are trips to memory that wait for
// each other.  More than 64 rows a key head, over 27,300 tokens: 64 nodes of 10 heads on one key head, one
// tree 19 us, eight 44 (16 MB of keys, which the five groups of rows fetch as 74, and 70 MB of partials);
// 256 nodes of 10 heads of their own, one tree 54 and eight 133 (293 MB fetched for 147: two groups of rows).
// ---------------------------------------------------------------------------
constexpr uint32_t kTrNotNamed = 0xffffffffu;

template <int RT, int KG>
__global__ __launch_bounds__(64 * RT * KG, 2) void tree_attn_kernel(TreeArgs a) {
  constexpr int D = 128, NW = RT * KG, TH = 64 * NW;
  constexpr int NH = 2 / KG;              // halves of an item that a wavefront takes
  constexpr int PARTS = 3;                // of a weight
  constexpr int CH = 8;                   // items laid out at a time
  constexpr int ST = RT == 1 ? 1 : 2;     // stages
  // arrays of their own: the compiler waits for direct loads before it reads an array they may write
  __shared__ __attribute__((aligned(16))) bf16 sK0[64 * D];
  __shared__ __attribute__((aligned(16))) bf16 sK1[ST == 2 ? 64 * D : 8];
  __shared__ __attribute__((aligned(16))) bf16 sV0[64 * D];
  __shared__ __attribute__((aligned(16))) bf16 sV1[ST == 2 ? 64 * D : 8];
  __shared__ uint32_t sBits[kPfMaxBlocks / 32];       // the blocks that the rows name
  __shared__ int sPref[kPfMaxBlocks / 32 + 1];        // set bits before each word
  // halves of the items laid out: first key, place among the laid out blocks (-1: the band, -2: no
  // keys), last row to load (later ones repeat it); the offsets of row 0 in K and V
  __shared__ int4 sHalf[2 * CH];
  __shared__ longlong2 sOff[2 * CH];
  // (block, node): the bits of the log2 bias; kTrNotNamed where the node does not name the block
  __shared__ uint32_t sBias[2 * CH][32 * RT];
  __shared__ uint32_t sBad[NW];
  __shared__ float2 sMl[32 * RT];
  // [nodes, K]: the bias of every slot (up to 64 rows; above, it would cost the second work-group of
  // a CU), then its block, -1 where it is not used
  extern __shared__ float dyn[];
  float* const sSlotBias = dyn;
  int16_t* const slots = (int16_t*)(dyn + (RT == 4 ? 0 : a.slot_cap));
  const int tid = threadIdx.x, lane = wave_lane();
  const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);   // scalar: so are the stages' addresses
  const int rt = wv % RT, kg = wv / RT;
  int id = blockIdx.x;
  const int hk = id % a.Hkv; id /= a.Hkv;
  const int split = id % a.nsplit; id /= a.nsplit;
  const int rg = id % a.groups, b = id / a.groups;
  const int G = a.H / a.Hkv;
  int64_t r0;
  const int nn = packed_rows(a.cu, b, a.T, a.max_n, r0);  // nodes
  const int ctx = tree_ctx(a, b);
  const int n = min(nn, a.S - ctx);                       // with a slot in the cache
  const int R = nn * G, rb = rg * RT * 32;
  if (rb >= R) return;
  const int node0 = rb / G, node1 = min(nn, (rb + RT * 32 - 1) / G + 1);
  const int nblk = (a.S + a.bs - 1) / a.bs;

  // this lane's row
  const int hl = lane >> 5, col = lane & 31;
  const int rr = min(rb + rt * 32 + col, R - 1);
  const bool rvalid = rb + rt * 32 + col < R;
  const int node = rr / G;
  const int64_t row = r0 + node;
  const int h = hk * G + rr % G;
  const int w_row = ctx + a.depth[row] - a.lw + 1;
  const int top = min(w_row, ctx);
  const uint64_t mask0 = a.mask[row * a.words];
  // over the wavefront's rows: the last window to start, the first end of the keys below one
  int w_last = rvalid ? w_row : INT32_MIN, top_first = rvalid ? top : INT32_MAX;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    w_last = max(w_last, __shfl_xor(w_last, m, kWave));
    top_first = min(top_first, __shfl_xor(top_first, m, kWave));
  }
  w_last = __builtin_amdgcn_readfirstlane(w_last);
  top_first = __builtin_amdgcn_readfirstlane(top_first);
  bf16x8 qop[D / 16];
  {
    const bf16* qb = a.q + row * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) qop[kk] = *(const bf16x8*)(qb + kk * 16 + hl * 8);
  }

  // the blocks that the rows name: a bit each, and every slot's block in LDS
  const int n_slots = (node1 - node0) * a.K;
  const int64_t s0 = (r0 + node0) * a.K;
  int n_blocks = 0;
  if (n_slots > 0) {
    for (int i = tid; i < kPfMaxBlocks / 32; i += TH) sBits[i] = 0u;
    __syncthreads();
    for (int i0 = 0; i0 < n_slots; i0 += 4 * TH) {
      int c[4], d[4];
      float x[4];
      bool ok[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {       // every load before the first store to LDS
        const int i = min(i0 + u * TH + tid, n_slots - 1);
        c[u] = a.idx[s0 + i];
        ok[u] = !a.valid || a.valid[s0 + i];
        d[u] = a.depth[r0 + node0 + i / a.K];
        x[u] = RT == 4 ? 0.f : a.bias[s0 + i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * TH + tid;
        if (i >= n_slots) break;
        const bool use = ok[u] && c[u] >= 0 && c[u] < nblk && c[u] * a.bs < min(ctx + d[u] - a.lw + 1, ctx);
        slots[i] = (int16_t)(use ? c[u] : -1);
        if (RT != 4) sSlotBias[i] = x[u];
        if (use) atomicOr(&sBits[c[u] >> 5], 1u << (c[u] & 31));
      }
    }
    __syncthreads();
    if (wv == 0) {
      int x = __popc(sBits[lane]);
#pragma unroll
      for (int s = 1; s < kWave; s <<= 1) {
        const int y = __shfl_up(x, s, kWave);
        if (lane >= s) x += y;
      }
      sPref[lane + 1] = x;
      if (lane == 0) sPref[0] = 0;
    }
    __syncthreads();
    n_blocks = sPref[kPfMaxBlocks / 32];
  }

  // items: the band's, then the blocks'
  const int hpb = a.bs / 32;              // halves of a block
  const int jw0 = max(ctx - a.lw + 1, 0) & ~31;
  const int jend = ctx + n;
  const int n_wi = (jend - jw0 + 63) / 64;
  const int n_items = n_wi + (n_blocks * hpb + 1) / 2;
  const int i_first = (int)((int64_t)n_items * split / a.nsplit);
  const int i_last = (int)((int64_t)n_items * (split + 1) / a.nsplit);
  if (i_first == i_last && a.nsplit > 1) {         // nothing for this split: no partial to read
    if (kg == 0 && hl == 0 && rvalid)
      a.part_ml[(row * a.H + h) * a.nsplit + split] = make_float2(-INFINITY, 0.f);
    return;
  }

  // Lays out items c0 .. c1 - 1 (at most CH): every wavefront has left the items before.
  auto lay_out = [&](int c0, int c1) {
    const int x0 = max(2 * (c0 - n_wi), 0), x1 = min(2 * (c1 - n_wi), n_blocks * hpb);
    const int l0 = x0 / hpb, l1 = x1 > x0 ? (x1 - 1) / hpb + 1 : l0;   // their blocks' places
    for (int x = tid; x < (l1 - l0) * 32 * RT; x += TH) (&sBias[0][0])[x] = kTrNotNamed;
    if (tid < 2 * (c1 - c0)) {
      const int i = c0 + (tid >> 1);
      int j, at;
      if (i < n_wi) {
        j = jw0 + 64 * i + 32 * (tid & 1);
        at = -1;
        if (j >= jend) { at = -2; j -= 32; }
      } else {
        int x = 2 * (i - n_wi) + (tid & 1);
        const bool none = x >= n_blocks * hpb;
        if (none) --x;
        const int l = x / hpb;
        int lo = 0, hi = kPfMaxBlocks / 32;        // the word of the l-th block
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (sPref[mid] <= l) lo = mid; else hi = mid;
        }
        uint32_t w = sBits[lo];
        for (int u = sPref[lo]; u < l; ++u) w &= w - 1u;
        j = (32 * lo + (int)__builtin_ctz(w)) * a.bs + x % hpb * 32;
        at = none ? -2 : l - l0;
      }
      const int pg = a.table ? tree_page(a, a.table[(int64_t)b * a.table_stride + j / a.page]) : b;
      // (a block's second half may lie past the last key as a whole)
      const int last = (i < n_wi ? jend : ctx) - 1 - j;
      const int jp = (a.table ? j % a.page : j) + min(last, 0);
      sHalf[tid] = make_int4(j, at, min(max(last, 0), 31), 0);
      sOff[tid] = make_longlong2((int64_t)pg * a.k_sb + (int64_t)jp * a.k_st + (int64_t)hk * a.k_sh,
                                 (int64_t)pg * a.v_sb + (int64_t)jp * a.v_st + (int64_t)hk * a.v_sh);
    }
    if (l1 > l0) {
      // a block's first slot in a row wins: the smallest slot first, then its bias in its place (a
      // bias whose bits could be a slot's number counts as 0, and a NaN is one whose bits are not
      // kTrNotNamed)
      auto place_of = [&](int c) {
        return c < 0 ? -1 : sPref[c >> 5] + __popc(sBits[c >> 5] & ((1u << (c & 31)) - 1u)) - l0;
      };
      __syncthreads();
      for (int i = tid; i < n_slots; i += TH) {
        const int l = place_of(slots[i]);
        if (l >= 0 && l < l1 - l0) atomicMin(&sBias[l][i / a.K], (uint32_t)(i % a.K));
      }
      __syncthreads();
      for (int i = tid; i < n_slots; i += TH) {
        const int l = place_of(slots[i]);
        if (l < 0 || l >= l1 - l0) continue;
        uint32_t& to = sBias[l][i / a.K];
        if (to != (uint32_t)(i % a.K)) continue;
        const float x = (RT == 4 ? a.bias[s0 + i] : sSlotBias[i]) * 1.4426950408889634f;
        to = x != x ? 0x7fc00000u : __float_as_uint(fabsf(x) < 1e-30f ? 0.f : x);
      }
    }
    __syncthreads();
  };
  // Direct loads of laid out item x into a stage: a half's rows at a scalar base plus 32-bit offsets.
  uint32_t ko[8 / NW], vo[8 / NW];
#pragma unroll
  for (int u = 0; u < 8 / NW; ++u) {
    const int r = 4 * (NW * u + wv) + (lane >> 4);        // four rows a wavefront
    ko[u] = 2u * (uint32_t)(r * a.k_st + k_slot(r, lane & 15) * 8);
    vo[u] = 2u * (uint32_t)(r * a.v_st + v_slot(r, lane & 15) * 8);
  }
  // Up to 64 rows every key is read once: non-temporal (the 32 trees 131 -> 125 us); more rows are
  // several work-groups, which share the lines in the L2.
  constexpr int kAux = RT == 4 ? 0 : 2;
  auto fetch = [&](int x, bf16* sKn, bf16* sVn) __attribute__((always_inline)) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int4 o = *(const int4*)&sOff[2 * x + hf];
      const int last = __builtin_amdgcn_readfirstlane(sHalf[2 * x + hf].z);
      auto wide = [](int lo, int hi) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(lo) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(hi) << 32);
      };
      const char* kb = (const char*)(a.k + wide(o.x, o.y));
      const char* vb = (const char*)(a.v + wide(o.z, o.w));
#pragma unroll
      for (int u = 0; u < 8 / NW; ++u) {
        const int grp = NW * u + wv;
        uint32_t kx = ko[u], vx = vo[u];
        if (last < 31) {
          const int r = 4 * grp + (lane >> 4), rc = min(r, last);
          kx = 2u * (uint32_t)(rc * a.k_st + k_slot(r, lane & 15) * 8);
          vx = 2u * (uint32_t)(rc * a.v_st + v_slot(r, lane & 15) * 8);
        }
        asm volatile("" : "+v"(kx), "+v"(vx));    // one load for both: a scalar base, a 32-bit offset
        __builtin_amdgcn_global_load_lds((const void*)(kb + kx),
            (__attribute__((address_space(3))) void*)(sKn + (hf * 32 + grp * 4) * D), 16, 0, kAux);
        __builtin_amdgcn_global_load_lds((const void*)(vb + vx),
            (__attribute__((address_space(3))) void*)(sVn + (hf * 32 + grp * 4) * D), 16, 0, kAux);
      }
    }
  };
  // the keys of half hf of laid out item x that this lane's row sees, a bit each, and their log2 bias
  auto visible = [&](int x, int hf, float& blog) -> uint32_t {
    const int2 d = *(const int2*)&sHalf[2 * x + hf];
    const int j = __builtin_amdgcn_readfirstlane(d.x), at = __builtin_amdgcn_readfirstlane(d.y);
    blog = 0.f;
    if (at == -2) return 0u;
    auto below = [](int y) -> uint32_t { return y >= 32 ? ~0u : y <= 0 ? 0u : (1u << y) - 1u; };
    if (at == -1 && j >= w_last && j + 32 <= ctx) return rvalid ? ~0u : 0u;   // inside every window
    if (at >= 0) {
      const uint32_t bits = sBias[at][node - node0];
      const bool sees = rvalid && bits != kTrNotNamed;
      blog = sees ? __uint_as_float(bits) : 0.f;
      if (j + 32 <= top_first) return sees ? ~0u : 0u;
      return sees ? below(top - j) : 0u;
    }
    if (!rvalid) return 0u;
    uint32_t v = below(ctx - j) & ~below(w_row - j);
    const int m0 = j - ctx;
    if (m0 > -32) {
      uint64_t m;
      if (m0 < 0) {
        m = mask0 << -m0;
      } else {
        const int wd = m0 >> 6, sh = m0 & 63;
        m = (wd ? a.mask[row * a.words + wd] : mask0) >> sh;
        if (sh > 32 && wd + 1 < a.words) m |= a.mask[row * a.words + wd + 1] << (64 - sh);
      }
      v |= (uint32_t)m & below(jend - j) & ~below(ctx - j);
    }
    return v;
  };

  floatx16 acc_o[D / 32];
  float m_run, l_run;
  auto reset = [&] {
    m_run = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc_o[dt][r] = 0.f;
  };
  const uint32_t kl0 = k_lane_off(col, hl), vl0 = v_lane_off(lane);
  const float csc = a.scale_log2e;

  // this wavefront's halves of laid out item i
  auto item = [&](int i, const bf16* sKc, const bf16* sVc,
                  uint32_t (&vis)[NH]) __attribute__((always_inline)) {
    float blog[NH];
    bool any = false;
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      vis[x] = visible(i, KG == 2 ? kg : x, blog[x]);
      any = any || vis[x] != 0u;
    }
    if (!__any(any)) return;
    floatx16 s[NH];
    float mloc = -INFINITY;
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      const int hf = KG == 2 ? kg : x;
      bf16x8 kf[D / 16];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) kf[kk] = k_frag_at(sKc, kl0, hf, kk);
      // two chains: a product need not wait for the one before it
      floatx16 t;
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[x][r] = 0.f; t[r] = 0.f; }
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2) {
        s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk], qop[kk], s[x], 0, 0, 0);
        t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk + 1], qop[kk + 1], t, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[x][r] += t[r];
      float mraw = -INFINITY;
      // a half that every row sees whole or not at all, as inside the band and the blocks
      if (__all(vis[x] == 0u || vis[x] == ~0u)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[x][r] = vis[x] ? s[x][r] : -INFINITY;
      } else {
        const uint32_t vb = vis[x] >> (4 * hl);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[x][r] = (vb >> (8 * (r >> 2) + (r & 3))) & 1u ? s[x][r] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) mraw = fmaxf(mraw, s[x][r]);
      mloc = fmaxf(mloc, fmaf(mraw, csc, blog[x]));
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
#pragma unroll
    for (int x = 0; x < NH; ++x) {
      const int hf = KG == 2 ? kg : x;
      // V in registers before the weights are ready
      bf16x8 vop[4][2];
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const char* vp = (const char*)sVc + (32 * hf + 16 * jj) * 256 + (vl0 ^ (uint32_t)(dt << 6));
          const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_short4*)(__attribute__((address_space(3))) void*)vp);
          const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_short4*)(__attribute__((address_space(3))) void*)(vp + 2048));
          const bf16x4 l4 = __builtin_bit_cast(bf16x4, lo);
          const bf16x4 h4 = __builtin_bit_cast(bf16x4, hi);
#pragma unroll
          for (int e = 0; e < 4; ++e) { vop[dt][jj][e] = l4[e]; vop[dt][jj][e + 4] = h4[e]; }
        }
      const float off = blog[x] - (m_run == -INFINITY ? 0.f : m_run);
      uint32_t part[PARTS][2][4];
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(s[x][8 * jj + e], csc, off));
        l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < PARTS; ++i) {
            bf16x2 y;
            y[0] = (bf16)p[2 * e];
            y[1] = (bf16)p[2 * e + 1];
            const uint32_t w = __builtin_bit_cast(uint32_t, y);
            part[i][jj][e] = w;
            p[2 * e] -= __uint_as_float(w << 16);
            p[2 * e + 1] -= __uint_as_float(w & 0xffff0000u);
          }
      }
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) {       // smallest parts first
          const bf16x8 w = __builtin_bit_cast(bf16x8, *(uint4*)part[i][jj]);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
            acc_o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vop[dt][jj], w, acc_o[dt], 0, 0, 0);
        }
    }
  };

  reset();
  uint32_t vis[NH];
  for (int c0 = i_first; c0 < i_last; c0 += CH) {
    const int c1 = min(c0 + CH, i_last);
    if (c0 > i_first) __syncthreads();    // every wavefront left the items before
    lay_out(c0, c1);
    if (ST == 1) {
      for (int i = c0; i < c1; ++i) {
        if (i > c0) __syncthreads();      // every wavefront left item i - 1
        fetch(i - c0, sK0, sV0);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();                  // item i landed
        item(i - c0, sK0, sV0, vis);
      }
      continue;
    }
    fetch(0, sK0, sV0);
    auto step = [&](int i, auto par) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();                    // item i landed; every wavefront left item i - 1
      if (i + 1 < c1) fetch(i + 1 - c0, P ? sK0 : sK1, P ? sV0 : sV1);
      item(i - c0, P ? sK1 : sK0, P ? sV1 : sV0, vis);
    };
    for (int i = c0; i < c1; i += 2) {
      step(i, std::integral_constant<int, 0>{});
      if (i + 1 < c1) step(i + 1, std::integral_constant<int, 1>{});
    }
  }

  // V values that are not finite reached every row of the tile through masked weights: the items
  // again, with V's finite values in the products and the others for the rows that see them
  float z = 0.f;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = fmaf(acc_o[dt][r], 0.f, z);
  if (__syncthreads_or(z != 0.f)) {
    reset();
    for (int i = i_first; i < i_last; ++i) {
      const int x0 = (i - i_first) % CH;
      if (x0 == 0) {
        __syncthreads();
        lay_out(i, min(i + CH, i_last));
      }
      __syncthreads();                    // every wavefront left the stage
      fetch(x0, sK0, sV0);
      __builtin_amdgcn_s_waitcnt(0);
      // each wavefront clears the rows it loaded; bit 8 hf + u: its group u of half hf holds some
      uint32_t bad = 0;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int u = 0; u < 8 / NW; ++u) {
          uint4* p = (uint4*)(sV0 + (hf * 32 + (NW * u + wv) * 4) * D) + lane;
          uint4 x = *p;
          bool is = false;
          auto fix = [&](uint32_t& w) {
            if ((w & 0x7f80u) == 0x7f80u) { w &= 0xffff0000u; is = true; }
            if ((w & 0x7f800000u) == 0x7f800000u) { w &= 0xffffu; is = true; }
          };
          fix(x.x); fix(x.y); fix(x.z); fix(x.w);
          if (is) *p = x;
          if (__any(is)) bad |= 1u << (8 * hf + u);
        }
      if (lane == 0) sBad[wv] = bad;
      __syncthreads();
#pragma unroll
      for (int y = 0; y < NH; ++y) vis[y] = 0u;
      item(x0, sK0, sV0, vis);
#pragma unroll
      for (int y = 0; y < NH; ++y) {
        const int hf = KG == 2 ? kg : y;
        const int last = sHalf[2 * x0 + hf].z;
        const bf16* vh = a.v + sOff[2 * x0 + hf].y + 4 * hl;
        for (int w = 0; w < NW; ++w)
          for (uint32_t todo = (sBad[w] >> (8 * hf)) & 0xffu; todo; todo &= todo - 1)
            for (int q4 = 0; q4 < 4; ++q4) {
              const int r = 4 * (NW * __builtin_ctz(todo) + w) + q4;
              if (r > last) continue;              // a repeated row
              const bool sees = (vis[y] >> r) & 1u;
              const bf16* vp = vh + (int64_t)r * a.v_st;
#pragma unroll
              for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const bf16x4 x = *(const bf16x4*)(vp + 32 * dt + 8 * q);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float f = (float)x[e];
                    if (sees && !(fabsf(f) <= 3.402823466e38f)) acc_o[dt][4 * q + e] += f;
                  }
                }
            }
      }
    }
  }
  float l_tot = xor32_sum(l_run);
  if (KG == 2) {
    // the second half's wavefronts hand their sums to the first's
    __syncthreads();
    float* so = (float*)(rt ? sK1 : sK0);
    if (kg == 1) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) so[(16 * dt + r) * 64 + lane] = acc_o[dt][r];
      if (hl == 0) sMl[rt * 32 + col] = make_float2(m_run, l_tot);
    }
    __syncthreads();
    if (kg == 1) return;
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
  if (!rvalid) return;
  const int64_t rh = row * a.H + h;
  if (a.nsplit > 1) {
    float* po = a.part_o + (rh * a.nsplit + split) * D + 4 * hl;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(float4*)(po + dt * 32 + 8 * q) = make_float4(acc_o[dt][4 * q], acc_o[dt][4 * q + 1],
                                                       acc_o[dt][4 * q + 2], acc_o[dt][4 * q + 3]);
    if (hl == 0) a.part_ml[rh * a.nsplit + split] = make_float2(m_run, l_tot);
    return;
  }
  const bool none = m_run == -INFINITY && l_tot == 0.f;     // (a NaN score leaves m as it was)
  const float inv = none ? 0.f : 1.f / l_tot;
  const int64_t at = row * a.o_st + (int64_t)h * a.o_sh + 4 * hl;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x[4] = {acc_o[dt][4 * q] * inv, acc_o[dt][4 * q + 1] * inv, acc_o[dt][4 * q + 2] * inv,
                          acc_o[dt][4 * q + 3] * inv};
      if (a.out_bf16) {
        bf16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (bf16)x[e];
        *(bf16x4*)((bf16*)a.out + at + 32 * dt + 8 * q) = y;
      } else {
        *(float4*)((float*)a.out + at + 32 * dt + 8 * q) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
  if (a.lse && hl == 0)
    a.lse[row * a.lse_st + (int64_t)h * a.lse_sh] =
        none ? -INFINITY : (m_run + log2f(l_tot)) * 0.6931471805599453f;
}

// One wavefront per (row, head), two dims a lane; lane s holds the weight of split s (at most 64),
// and eight partials are in flight (13,480 rows and heads of 3 splits: 7 us; 80 of 41: 4).  A split that
// saw no key wrote m = -inf and is not read.
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  constexpr int D = 128;
  const int64_t rh = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (rh >= a.T * a.H) return;
  const int lane = wave_lane();
  const float2 ml = lane < a.nsplit ? a.part_ml[rh * a.nsplit + lane] : make_float2(-INFINITY, 0.f);
  const float M = wave_max(ml.x);
  // NaN in a score leaves the maximum and comes in through the sums
  const bool seen = lane < a.nsplit && !(ml.x == -INFINITY && ml.y == 0.f);
  const float w = seen ? fast_exp2(ml.x - (M == -INFINITY ? 0.f : M)) : 0.f;
  const float L = wave_sum(seen ? ml.y * w : 0.f);
  const float* po = a.part_o + rh * a.nsplit * D + 2 * lane;
  float2 acc = make_float2(0.f, 0.f);
  uint64_t todo = __ballot(seen);
  const bool any = todo != 0;
  while (todo) {
    float2 x[8];
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = todo ? __builtin_ctzll(todo) : 0;
      u[i] = todo ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s)) : 0.f;
      x[i] = make_float2(0.f, 0.f);
      if (todo) x[i] = *(const float2*)(po + s * D);
      todo &= todo - 1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc.x = fmaf(u[i], x[i].x, acc.x);
      acc.y = fmaf(u[i], x[i].y, acc.y);
    }
  }
  const float inv = any ? 1.f / L : 0.f;
  const int64_t row = rh / a.H;
  const int h = (int)(rh % a.H);
  const int64_t at = row * a.o_st + (int64_t)h * a.o_sh + 2 * lane;
  if (a.out_bf16) {
    bf16x2 r;
    r[0] = (bf16)(acc.x * inv);
    r[1] = (bf16)(acc.y * inv);
    *(bf16x2*)((bf16*)a.out + at) = r;
  } else {
    *(float2*)((float*)a.out + at) = make_float2(acc.x * inv, acc.y * inv);
  }
  if (a.lse && lane == 0)
    a.lse[row * a.lse_st + (int64_t)h * a.lse_sh] = any ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

// Rows of a work-group, row groups and splits of a call: 32 rows per wavefront pair up to 64, then
// 128 rows; splits until the grid is about two rounds of two work-groups per CU (640, 768, 1,536 or 2,048
// work-groups instead of 1,024: slower by 3 to 20 % on one side or the other).
struct TreePlan { int rt, groups, nsplit, nodes; };
inline TreePlan tree_plan(int B, int H, int Hkv, int max_n, int K, int S, int bs, int lw) {
  TreePlan p;
  const int64_t rows = (int64_t)max_n * (H / Hkv);
  p.rt = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.groups = (int)((rows + 32 * p.rt - 1) / (32 * p.rt));
  const int64_t nodes = std::min<int64_t>(max_n, (32 * p.rt - 1) / (H / Hkv) + 2);
  p.nodes = (int)nodes;                   // at most, of a row group
  // the nodes of a tree name much the same blocks: splits for four times a row's (where they name
  // more, a split takes more items)
  const int64_t blocks = std::min<int64_t>({(S + bs - 1) / bs, nodes * K, 4 * K});
  const int64_t items = (std::min<int64_t>(S, (int64_t)lw + max_n) + 95) / 64 + (blocks * (bs / 32) + 1) / 2;
  const int64_t streams = std::max<int64_t>(1, (int64_t)B * Hkv * p.groups);
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({64, items, kTrTarget / streams}));
  return p;
}
inline int64_t tree_workspace(const TreePlan& p, int64_t T, int H) {
  return p.nsplit > 1 ? T * H * p.nsplit * (128 * 4 + 8) : 0;
}

}  // namespace dash

extern "C" int dash_tree_masks(const int32_t* parents, const int32_t* cu_seqlens_q, int B, int64_t T,
                               int max_query_len, int words, int64_t* mask, int32_t* depth,
                               void* stream) {
  using namespace dash;
  if (B < 0 || T < 0 || max_query_len < 0) return kErrInvalid;
  if (B == 0 || T == 0) return kOk;
  if (!parents || !cu_seqlens_q || !mask || !depth || max_query_len == 0) return kErrInvalid;
  if (max_query_len > kTrMaxNodes || words != (max_query_len + 63) / 64 || !fits_grid(B, kTrMaxNodes))
    return kErrUnsupported;
  hipLaunchKernelGGL(tree_masks_kernel, dim3(B), dim3(kTrMaxNodes), 0, (hipStream_t)stream, parents,
                     cu_seqlens_q, T, words, max_query_len, (uint64_t*)mask, depth);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}

extern "C" int dash_attn_tree_workspace_size(int B, int H, int Hkv, int64_t T, int max_query_len,
                                             int K, int S, int block_size, int local_window,
                                             int64_t* bytes) {
  using namespace dash;
  if (!bytes || B < 0 || H <= 0 || Hkv <= 0 || T < 0 || max_query_len < 0 || K < 0 || S < 0)
    return kErrInvalid;
  if (H % Hkv != 0 || block_size < 32 || local_window < 1) return kErrUnsupported;
  *bytes = tree_workspace(tree_plan(B, H, Hkv, max_query_len, K, S, block_size, local_window), T, H);
  return kOk;
}

extern "C" int dash_attn_tree(
    const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st,
    const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, const int32_t* block_table,
    int64_t table_stride, int page_size, int num_pages, const int32_t* context_lens,
    const int32_t* cu_seqlens_q,
    const int32_t* idx, const uint8_t* valid, const float* bias, int K, const int64_t* mask, int words,
    const int32_t* depth, void* out, int out_bf16, int64_t o_st, int64_t o_sh, float* lse,
    int64_t lse_st, int64_t lse_sh, int B, int H, int Hkv, int64_t T, int max_query_len, int S, int D,
    int block_size, int local_window, float scale, void* workspace, int64_t workspace_bytes,
    void* stream) {
  using namespace dash;
  if (B < 0 || H <= 0 || Hkv <= 0 || T < 0 || max_query_len < 0 || S < 0 || K < 0 || local_window < 1)
    return kErrInvalid;
  if (B == 0 || T == 0) return kOk;
  if (!q || !k || !v || !out || !context_lens || !cu_seqlens_q || !mask || !depth) return kErrInvalid;
  if (K > 0 && (!idx || !bias)) return kErrInvalid;
  if (max_query_len == 0 || S == 0) return kErrInvalid;
  if (D != 128 || H % Hkv != 0 || K > kPfMaxSlots || max_query_len > kTrMaxNodes ||
      words != (max_query_len + 63) / 64 || block_size <= 0 ||
      (block_size != 32 && block_size % 64 != 0) || !(scale > 0.f))
    return kErrUnsupported;
  if ((S + block_size - 1) / block_size > kPfMaxBlocks) return kErrUnsupported;
  if (block_table && num_pages <= 0) return kErrInvalid;
  if (block_table && (page_size <= 0 || page_size % block_size != 0)) return kErrUnsupported;
  const int64_t strides[] = {q_st, q_sh, k_sb, k_sh, k_st, v_sb, v_sh, v_st};
  for (int64_t s : strides)
    if (s % 8 != 0) return kErrUnsupported;
  if (k_st > kMaxKeyRowStride || v_st > kMaxKeyRowStride || k_st < 0 || v_st < 0) return kErrUnsupported;
  const void* ptrs[] = {q, k, v};
  for (const void* x : ptrs)
    if ((uintptr_t)x % 16 != 0) return kErrUnsupported;
  TreeArgs a = {};
  a.q = (const bf16*)q; a.q_st = q_st; a.q_sh = q_sh;
  a.k = (const bf16*)k; a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v = (const bf16*)v; a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  a.table = block_table; a.table_stride = table_stride; a.page = page_size;
  a.num_pages = num_pages;
  a.ctx = context_lens; a.cu = cu_seqlens_q;
  a.idx = idx; a.valid = valid; a.bias = bias; a.K = K;
  a.mask = (const uint64_t*)mask; a.words = words; a.depth = depth;
  a.out = out; a.out_bf16 = out_bf16; a.o_st = o_st; a.o_sh = o_sh;
  a.lse = lse; a.lse_st = lse_st; a.lse_sh = lse_sh;
  a.B = B; a.H = H; a.Hkv = Hkv; a.S = S; a.bs = block_size; a.lw = local_window;
  a.max_n = max_query_len; a.T = T;
  a.scale_log2e = scale * 1.4426950408889634f;
  const TreePlan p = tree_plan(B, H, Hkv, max_query_len, K, S, block_size, local_window);
  a.groups = p.groups; a.nsplit = p.nsplit;
  const int64_t wgs = (int64_t)B * Hkv * p.groups * p.nsplit;
  if (T > INT32_MAX || !fits_grid(wgs, 64 * (p.rt == 1 ? 2 : 4)) || T * H > INT32_MAX ||
      (p.nsplit > 1 && !fits_grid((T * H + 3) / 4, 256)))
    return kErrUnsupported;
  if (p.nsplit > 1) {
    if (!workspace || workspace_bytes < tree_workspace(p, T, H) || (uintptr_t)workspace % 16 != 0)
      return kErrWorkspace;
    a.part_o = (float*)workspace;
    a.part_ml = (float2*)(a.part_o + T * H * p.nsplit * 128);
  }
  hipStream_t st = (hipStream_t)stream;
  a.slot_cap = p.nodes * K;
  const unsigned lds = (unsigned)((a.slot_cap * (p.rt == 4 ? 2 : 6) + 15) / 16 * 16);
  const dim3 grid((unsigned)wgs);
  if (p.rt == 1) {
    hipLaunchKernelGGL((tree_attn_kernel<1, 2>), grid, dim3(128), lds, st, a);
  } else if (p.rt == 2) {
    hipLaunchKernelGGL((tree_attn_kernel<2, 2>), grid, dim3(256), lds, st, a);
  } else {
    hipLaunchKernelGGL((tree_attn_kernel<4, 1>), grid, dim3(256), lds, st, a);
  }
  if (p.nsplit > 1)
    hipLaunchKernelGGL(tree_merge_kernel, dim3((unsigned)((T * H + 3) / 4)), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
