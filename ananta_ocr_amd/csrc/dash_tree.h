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
// climbs to the root (parents come before their children, so it ends).
__global__ __launch_bounds__(kTrMaxNodes) void tree_masks_kernel(const int32_t* parents,
                                                                 const int32_t* cu, int words,
                                                                 int max_n, uint64_t* mask,
                                                                 int32_t* depth) {
  __shared__ int sPar[kTrMaxNodes];
  const int b = blockIdx.x, i = threadIdx.x;
  const int64_t r0 = cu[b];
  const int n = min((int)(cu[b + 1] - r0), max_n);
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

// One wavefront per (row, head): 16 lanes per key row, four keys per load.
__global__ __launch_bounds__(kWave) void tree_rows_kernel(TreeArgs a) {
  constexpr int D = 128;
  const int h = blockIdx.x, lane = threadIdx.x;
  const int64_t row = blockIdx.y;
  int b = 0;
  {
    int hi = a.B;
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (a.cu[mid] <= row) b = mid; else hi = mid;
    }
  }
  const int ctx = tree_ctx(a, b);
  const int n = min(min((int)(a.cu[b + 1] - a.cu[b]), a.max_n), a.S - ctx);
  const int hk = h / (a.H / a.Hkv);
  const int w0 = ctx + a.depth[row] - a.lw + 1;
  const int g = lane >> 4, dl = (lane & 15) * 8;
  const bf16x8 q = *(const bf16x8*)(a.q + row * a.q_st + (int64_t)h * a.q_sh + dl);
  float m = -INFINITY, l = 0.f, o[8];
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  // keys j0 .. j1 - 1; sees(j) the mask, blog the log2 bias
  auto keys = [&](int j0, int j1, float blog, auto sees) {
    for (int j = j0; j < j1; j += 4) {
      const int key = min(j + g, j1 - 1);
      int64_t kr, vr;
      if (a.table) {
        const int p = tree_page(a, a.table[(int64_t)b * a.table_stride + key / a.page]);
        kr = (int64_t)p * a.k_sb + (int64_t)(key % a.page) * a.k_st;
        vr = (int64_t)p * a.v_sb + (int64_t)(key % a.page) * a.v_st;
      } else {
        kr = (int64_t)b * a.k_sb + (int64_t)key * a.k_st;
        vr = (int64_t)b * a.v_sb + (int64_t)key * a.v_st;
      }
      const bf16x8 kx = *(const bf16x8*)(a.k + kr + (int64_t)hk * a.k_sh + dl);
      const bf16x8 vx = *(const bf16x8*)(a.v + vr + (int64_t)hk * a.v_sh + dl);
      float s = 0.f;
      for (int e = 0; e < 8; ++e) s += (float)q[e] * (float)kx[e];
      for (int x = 1; x < 16; x <<= 1) s += __shfl_xor(s, x, kWave);
      const bool ok = j + g < j1 && sees(key);
      s = ok ? s * a.scale_log2e + blog : -INFINITY;
      const float mn = fmaxf(m, s);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float al = fast_exp2(m - mu), p = fast_exp2(s - mu);
      l = l * al + p;
      for (int e = 0; e < 8; ++e) o[e] = o[e] * al + (ok ? p * (float)vx[e] : 0.f);
      m = mn;
    }
  };
  keys(max(w0, 0), ctx, 0.f, [](int) { return true; });
  keys(ctx, ctx + n, 0.f, [&](int j) {
    const int x = j - ctx;
    return ((a.mask[row * a.words + (x >> 6)] >> (x & 63)) & 1ull) != 0;
  });
  const int top = min(w0, ctx);             // routed keys lie below it
  for (int s = 0; s < a.K; ++s) {
    auto usable = [&](int x) {
      const int c = a.idx[row * a.K + x];
      return c >= 0 && c < (a.S + a.bs - 1) / a.bs && c * a.bs < top && (!a.valid || a.valid[row * a.K + x]);
    };
    if (!usable(s)) continue;
    const int c = a.idx[row * a.K + s];
    bool first = true;
    for (int x = 0; x < s; ++x) first = first && !(a.idx[row * a.K + x] == c && usable(x));
    if (first)
      keys(c * a.bs, min((c + 1) * a.bs, top), a.bias[row * a.K + s] * 1.4426950408889634f,
           [](int) { return true; });
  }
  // the four lane groups
  for (int x = 16; x <= 32; x <<= 1) {
    const float m2 = __shfl_xor(m, x, kWave), l2 = __shfl_xor(l, x, kWave);
    const float mn = fmaxf(m, m2), mu = mn == -INFINITY ? 0.f : mn;
    const float al = fast_exp2(m - mu), be = fast_exp2(m2 - mu);
    for (int e = 0; e < 8; ++e) o[e] = o[e] * al + __shfl_xor(o[e], x, kWave) * be;
    l = l * al + l2 * be;
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (g == 0) {
    const int64_t at = row * a.o_st + (int64_t)h * a.o_sh + dl;
    for (int e = 0; e < 8; ++e) {
      if (a.out_bf16) ((bf16*)a.out)[at + e] = (bf16)(o[e] * inv);
      else ((float*)a.out)[at + e] = o[e] * inv;
    }
  }
  if (a.lse && lane == 0)
    a.lse[row * a.lse_st + (int64_t)h * a.lse_sh] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace dash

extern "C" int dash_tree_masks(const int32_t* parents, const int32_t* cu_seqlens_q, int B, int64_t T,
                               int max_query_len, int words, int64_t* mask, int32_t* depth,
                               void* stream) {
  using namespace dash;
  if (B < 0 || T < 0 || max_query_len < 0) return kErrInvalid;
  if (B == 0 || T == 0) return kOk;
  if (!parents || !cu_seqlens_q || !mask || !depth || max_query_len == 0) return kErrInvalid;
  if (max_query_len > kTrMaxNodes || words != (max_query_len + 63) / 64) return kErrUnsupported;
  hipLaunchKernelGGL(tree_masks_kernel, dim3(B), dim3(kTrMaxNodes), 0, (hipStream_t)stream, parents,
                     cu_seqlens_q, words, max_query_len, (uint64_t*)mask, depth);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}

extern "C" int dash_attn_tree_workspace_size(int B, int H, int Hkv, int64_t T, int max_query_len,
                                             int K, int S, int block_size, int local_window,
                                             int64_t* bytes) {
  using namespace dash;
  if (!bytes || B < 0 || H <= 0 || Hkv <= 0 || T < 0 || max_query_len < 0 || K < 0 || S < 0)
    return kErrInvalid;
  *bytes = 0;
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
      (block_size != 32 && block_size % 64 != 0) || !(scale > 0.f) || B > 65535 || T > 65535)
    return kErrUnsupported;
  if ((S + block_size - 1) / block_size > kPfMaxBlocks) return kErrUnsupported;
  if (block_table && num_pages <= 0) return kErrInvalid;
  if (block_table && (page_size <= 0 || page_size % block_size != 0)) return kErrUnsupported;
  const int64_t strides[] = {q_st, q_sh, k_sb, k_sh, k_st, v_sb, v_sh, v_st};
  for (int64_t s : strides)
    if (s % 8 != 0) return kErrUnsupported;
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
  hipLaunchKernelGGL(tree_rows_kernel, dim3(H, (unsigned)T), dim3(kWave), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
