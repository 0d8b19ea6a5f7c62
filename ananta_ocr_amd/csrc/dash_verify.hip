// Verification of drafted tokens on gfx950: which nodes of a sequence's tree the target's
// distribution accepts, from given random numbers, and the token that follows the last of them.
//
// Row r = cu[b] + i is node i of sequence b; node 0 is the root (the newest sampled token), and
// p[r] the target's distribution of the token after it.  At a node, its children are tried in
// order.  With draft probabilities q (the children were drawn from q[node], each by itself) what is
// left of p after some rejections is max(p - a q, 0) for one number a: taking max(x - Z q, 0) of
// x = max(p - a q, 0) gives max(p - (a + Z) q, 0).  So with a = 0 and Z = 1 at first, child x is
// accepted if u Z q(x) < max(p(x) - a q(x), 0), and a rejection sets a += Z and
// Z = sum_v max(p - a q, 0).  Without draft probabilities a child is a certain proposal: accepted
// if u Z < p(x), else its token's probability leaves p and Z.  The root's number draws the next
// token from what is left at the last accepted node, in order of the token ids.  Greedy: a
// child that is the row's best token (the lowest of equals) is accepted.
//
// Sums and products are taken in 64 bits: products of 32-bit inputs are then exact, and a
// different order of a sum moves a border by 1e-16 of the row's mass, not by the 1e-7 that would
// change a drawn token in every few thousandth row of 131,072 tokens.
//
// Probabilities that are not above 0 (NaN too) count as 0, and so do random numbers below it.

#include <hip/hip_fp16.h>

#include "dash_common.h"

namespace dash {

constexpr int kVfMaxNodes = 256;      // nodes of a sequence
constexpr int kVfChunk = 4096;        // tokens per work-group of the sums
constexpr int kVfThreads = 256;
constexpr uint64_t kVfUnset = ~0ull;  // of a sum that is not there yet (no sum has these bits: a NaN)

struct VerifyArgs {
  const void* p; int64_t p_st;
  const void* q; int64_t q_st;          // null: certain proposals
  const void* tok; int tok64;
  const int32_t* parents; const int32_t* cu;
  const float* u;                       // null: greedy
  int B, V, max_n, chunks;              // chunks of a row (sums, or greedy partials)
  int chunk;                            // tokens of a greedy partial
  int64_t T;
  int32_t* count; int32_t* path; int64_t path_st; int64_t* token;
  // workspace
  int32_t* stop;                        // [B] the last accepted node
  double* gone;                         // [B] a at that node
  uint64_t* sums;                       // [B, chunks, 2] bits of (what is left, the row itself)
  int32_t* done;                        // [B] chunks that have arrived (the walk clears it)
  float* best_v; int32_t* best_i;       // [T, chunks] greedy partials
};

// Sixteen bytes of a row, at any element's boundary (global loads need no more).
typedef uint32_t VfBytes __attribute__((ext_vector_type(4), aligned(1)));
template <typename T> struct VfVec {
  static constexpr int kN = 16 / sizeof(T);
  union { VfBytes b; T e[kN]; };
};

template <typename T> __device__ __forceinline__ float vf_load(const T* x) { return (float)*x; }
template <> __device__ __forceinline__ float vf_load<__half>(const __half* x) { return __half2float(*x); }

__device__ __forceinline__ int64_t vf_token(const VerifyArgs& a, int64_t row) {
  return a.tok64 ? ((const int64_t*)a.tok)[row] : ((const int32_t*)a.tok)[row];
}

// What is left of probability p where the draft's is q (maxima take what is no number to 0; with q and
// gone at least 0, a p below 0 ends there too).
__device__ __forceinline__ double vf_rest(float p, float q, double gone) {
  return fmax(fma(-gone, (double)fmaxf(q, 0.f), (double)p), 0.0);
}
__device__ __forceinline__ double vf_left(float p, float q, double gone) {
  return gone == 0.0 ? (double)fmaxf(p, 0.f) : vf_rest(p, q, gone);
}

// Sum over the work-group, the same on every thread.
template <int THREADS>
__device__ __forceinline__ double vf_block_sum(double v, double* sD) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  __syncthreads();
  if (wave_lane() == 0) sD[threadIdx.x / kWave] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) s += sD[w];
  return s;
}

// Greedy: the best token of a piece of a row; the lowest of equals, NaN never.  Bound by HBM: 1,156
// rows of 131,072 bf16 tokens in 46 us, 6.6 TB/s (54 us where the loads leave their lines in the L2).
template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_best_kernel(VerifyArgs a) {
  __shared__ float sV[kVfThreads / kWave];
  __shared__ int sI[kVfThreads / kWave];
  const int64_t row = blockIdx.x / a.chunks;
  const int ch = blockIdx.x % a.chunks, tid = threadIdx.x;
  const int v0 = ch * a.chunk, v1 = (int)min((int64_t)a.V, (int64_t)v0 + a.chunk);
  const T* p = (const T*)a.p + row * a.p_st;
  float best = -INFINITY;
  int at = INT32_MAX;
  constexpr int E = VfVec<T>::kN, U = 4;
  int v = v0;
  for (; v + kVfThreads * E * U <= v1; v += kVfThreads * E * U) {
    VfVec<T> x[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      x[k].b = __builtin_nontemporal_load((const VfBytes*)(p + v + (k * kVfThreads + tid) * E));
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float f = vf_load(&x[k].e[j]);
        if (f > best) { best = f; at = v + (k * kVfThreads + tid) * E + j; }
      }
  }
  for (int w = v + tid; w < v1; w += kVfThreads) {
    const float f = vf_load(p + w);
    if (f > best) { best = f; at = w; }
  }
  auto take = [&](float f, int i) {
    if (f > best || (f == best && i < at)) { best = f; at = i; }
  };
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) take(__shfl_xor(best, m, kWave), __shfl_xor(at, m, kWave));
  if (wave_lane() == 0) { sV[tid / kWave] = best; sI[tid / kWave] = at; }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kVfThreads / kWave; ++w) take(sV[w], sI[w]);
    a.best_v[blockIdx.x] = best;
    a.best_i[blockIdx.x] = at;
  }
}

// The walk from the root.  Every wavefront walks by itself on the same values in LDS; the draft
// and target probabilities of every drafted token are gathered first, in one round trip.  Only a
// rejected child that has a later sibling, with draft probabilities, needs a pass over a row: 8.5 us for
// 100,003 fp32 tokens (0.8 MB), the rate of one CU's reads.  Without such a pass 3 to 5 us, of latency.
template <typename T, int MODE, int THREADS>   // MODE 0 greedy, 1 certain proposals, 2 drawn ones
__global__ __launch_bounds__(THREADS) void verify_walk_kernel(VerifyArgs a) {
  __shared__ int sPar[kVfMaxNodes];
  __shared__ int64_t sTok[kVfMaxNodes];
  __shared__ float sP[kVfMaxNodes], sQ[kVfMaxNodes], sU[kVfMaxNodes];
  __shared__ int sBest[MODE == 0 ? kVfMaxNodes : 1];
  __shared__ int sPath[kVfMaxNodes];
  __shared__ double sD[THREADS / kWave];
  const int b = blockIdx.x, tid = threadIdx.x, lane = wave_lane();
  int64_t r0;
  const int n = packed_rows(a.cu, b, a.T, a.max_n, r0);
  if (n <= 0) {
    for (int i = tid; i < a.max_n; i += THREADS) a.path[b * a.path_st + i] = -1;
    if (tid == 0) { a.count[b] = 0; a.token[b] = -1; if (MODE != 0) a.stop[b] = -1; }
    return;
  }
  for (int i = tid; i < n; i += THREADS) {
    int par = a.parents[r0 + i];
    if (i == 0 || par < 0 || par >= i) par = -1;
    const int64_t t = vf_token(a, r0 + i);
    sPar[i] = par;
    sTok[i] = t;
    if (MODE != 0) {
      const bool in = par >= 0 && t >= 0 && t < a.V;
      sP[i] = in ? vf_load((const T*)a.p + (r0 + par) * a.p_st + t) : 0.f;
      sQ[i] = MODE == 2 && in ? fmaxf(vf_load((const T*)a.q + (r0 + par) * a.q_st + t), 0.f) : 1.f;
      sU[i] = fmaxf(a.u[r0 + i], 0.f);
    }
  }
  if (MODE == 0) {
    for (int i = tid; i < n; i += THREADS) {
      float best = -INFINITY;
      int at = INT32_MAX;
      for (int c = 0; c < a.chunks; ++c) {
        const float f = a.best_v[(r0 + i) * a.chunks + c];
        if (f > best) { best = f; at = a.best_i[(r0 + i) * a.chunks + c]; }
      }
      sBest[i] = at == INT32_MAX ? 0 : at;
    }
  }
  __syncthreads();
  int s = 0, cnt = 1;
  double gone = 0.0;
  if (tid == 0) sPath[0] = 0;
  for (;;) {
    int found = -1;
    double Z = 1.0;
    gone = 0.0;
    for (int w = 0; w < n && found < 0; w += kWave) {
      uint64_t kids = __ballot(w + lane < n && sPar[min(w + lane, n - 1)] == s);
      while (kids) {
        const int i = w + __builtin_ctzll(kids);
        kids &= kids - 1;
        if (MODE == 0) {
          if (sTok[i] == sBest[s]) { found = i; break; }
        } else if (MODE == 1) {
          // a token that an earlier sibling named is no longer in p
          bool again = false;
          for (int k = 0; k <= w; k += kWave)
            again |= __any(k + lane < i && sPar[min(k + lane, n - 1)] == s &&
                           sTok[min(k + lane, n - 1)] == sTok[i]);
          const double e = again ? 0.0 : vf_left(sP[i], 0.f, 0.0);
          if ((double)sU[i] * Z < e) { found = i; break; }
          Z -= e;
        } else {
          const double e = vf_left(sP[i], sQ[i], gone);
          if ((double)sU[i] * Z * (double)sQ[i] < e) { found = i; break; }
          gone += Z;
          bool more = kids != 0;
          for (int k = w + kWave; k < n && !more; k += kWave)
            more = __any(k + lane < n && sPar[min(k + lane, n - 1)] == s);
          if (more) {
            const T* p = (const T*)a.p + (r0 + s) * a.p_st;
            const T* q = (const T*)a.q + (r0 + s) * a.q_st;
            // one work-group's reads in flight: 16 tokens a lane of each row, 64 or 128 KB (32 tokens:
            // 36 us for the passes of 16 trees, 16: 34.5; the next 8 loaded while 8 are added up: 40)
            constexpr int E = VfVec<T>::kN, U = 16 / E;
            double mine = 0.0, odd = 0.0;
            int v = 0;
            for (; v + THREADS * E * U <= a.V; v += THREADS * E * U) {
              VfVec<T> x[U], y[U];
#pragma unroll
              for (int k = 0; k < U; ++k) {
                x[k].b = *(const VfBytes*)(p + v + (k * THREADS + tid) * E);
                y[k].b = *(const VfBytes*)(q + v + (k * THREADS + tid) * E);
              }
#pragma unroll
              for (int k = 0; k < U; ++k)
#pragma unroll
                for (int j = 0; j < E; j += 2) {
                  mine += vf_rest(vf_load(&x[k].e[j]), vf_load(&y[k].e[j]), gone);
                  odd += vf_rest(vf_load(&x[k].e[j + 1]), vf_load(&y[k].e[j + 1]), gone);
                }
            }
#pragma unroll 4
            for (int w2 = v + tid; w2 < a.V; w2 += THREADS)
              mine += vf_rest(vf_load(p + w2), vf_load(q + w2), gone);
            Z = vf_block_sum<THREADS>(mine + odd, sD);
          }
        }
      }
    }
    if (found < 0) break;
    s = found;
    if (tid == 0) sPath[cnt] = s;
    ++cnt;
  }
  __syncthreads();
  for (int i = tid; i < a.max_n; i += THREADS) a.path[b * a.path_st + i] = i < cnt ? sPath[i] : -1;
  if (MODE != 0)
    for (int i = tid; i < 2 * a.chunks; i += THREADS) a.sums[(int64_t)b * 2 * a.chunks + i] = kVfUnset;
  if (tid == 0) {
    a.count[b] = cnt;
    if (MODE == 0) {
      a.token[b] = sBest[s];
    } else {
      a.stop[b] = s;
      a.gone[b] = gone;
      a.done[b] = 0;
    }
  }
}

// The token of this thread's node where it is a child of node s, -1 else (certain proposals).
__device__ __forceinline__ int64_t vf_child(const VerifyArgs& a, int64_t r0, int n, int s) {
  static_assert(kVfMaxNodes <= kVfThreads, "a thread per node");
  const int i = threadIdx.x;
  if (i < 1 || i >= n) return -1;
  const int par = a.parents[r0 + i];
  const int64_t t = vf_token(a, r0 + i);
  return par == s && par < i ? t : -1;
}

// The children's tokens that lie in chunk v0, a bit each.
__device__ __forceinline__ void vf_named(int64_t child, int v0, uint32_t* sBits) {
  for (int i = threadIdx.x; i < kVfChunk / 32; i += kVfThreads) sBits[i] = 0u;
  __syncthreads();
  const int64_t t = child - v0;
  if (child >= 0 && t >= 0 && t < kVfChunk) atomicOr(&sBits[t >> 5], 1u << (t & 31));
  __syncthreads();
}

constexpr int kVfPer = kVfChunk / kVfThreads;      // tokens of a thread, one after another

// This thread's tokens of chunk v0 of the last node's row (zeros past the row's end) ...
template <typename T, bool DRAFT>
struct VfTokens {
  static constexpr int E = VfVec<T>::kN, N = kVfPer / E;
  VfVec<T> x[N], y[DRAFT ? N : 1];
  __device__ __forceinline__ void load(const VerifyArgs& a, int64_t row, int v0) {
    const int e0 = threadIdx.x * kVfPer, m = min(a.V - v0 - e0, kVfPer);
    const T* p = (const T*)a.p + row * a.p_st + v0 + e0;
    const T* q = DRAFT ? (const T*)a.q + row * a.q_st + v0 + e0 : nullptr;
    if (m == kVfPer) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[k].b = ((const VfBytes*)p)[k];
        if (DRAFT) y[k].b = ((const VfBytes*)q)[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[k].b = VfBytes{0u, 0u, 0u, 0u};
        if (DRAFT) y[k].b = VfBytes{0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (k * E + j < m) {
            x[k].e[j] = p[k * E + j];
            if (DRAFT) y[k].e[j] = q[k * E + j];
          }
      }
    }
  }
  // ... what is left of token i, and the row itself.
  __device__ __forceinline__ double2 at(int i, double gone, uint32_t named) const {
    const float f = vf_load(&x[i / E].e[i % E]);
    const double whole = vf_left(f, 0.f, 0.0);
    if (DRAFT) return make_double2(vf_left(f, vf_load(&y[i / E].e[i % E]), gone), whole);
    return make_double2((named >> i) & 1u ? 0.0 : whole, whole);
  }
};

// The bits of this thread's tokens.
__device__ __forceinline__ uint32_t vf_bits(const uint32_t* sBits) {
  const int e0 = threadIdx.x * kVfPer;
  return (sBits[e0 >> 5] >> (e0 & 31)) & ((1u << kVfPer) - 1u);
}

// Sum over the work-group's earlier threads, and over all.
__device__ __forceinline__ double vf_before(double v, double* sD, double& total) {
  const int lane = wave_lane(), wv = threadIdx.x / kWave;
  double x = v;
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) {
    const double y = __shfl_up(x, s, kWave);
    if (lane >= s) x += y;
  }
  double own = __shfl_up(x, 1, kWave);
  if (lane == 0) own = 0.0;
  __syncthreads();
  if (lane == kWave - 1) sD[wv] = x;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int w = 0; w < kVfThreads / kWave; ++w) {
    if (w < wv) before += sD[w];
    total += sD[w];
  }
  return before + own;
}

// The smallest `first` and the largest `last` over the work-group.
__device__ __forceinline__ void vf_ends(int& first, int& last, int2* sE) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    first = min(first, __shfl_xor(first, m, kWave));
    last = max(last, __shfl_xor(last, m, kWave));
  }
  __syncthreads();
  if (wave_lane() == 0) sE[threadIdx.x / kWave] = make_int2(first, last);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVfThreads / kWave; ++w) {
    first = min(first, sE[w].x);
    last = max(last, sE[w].y);
  }
}

// The next token: every work-group sums a chunk of the last node's row, and the one that arrives
// last finds the chunk that the root's number falls into, then the token within it.  Whichever that
// is adds the same sums in the same order.  Bound by latency: a chunk's loads, the arrival, and the
// chosen chunk again (a row is 0.26 to 0.8 MB, read by a tenth of the chip): 10 us for 8 rows of 131,072
// bf16 tokens, 13 for 16 of 100,003 fp32 ones with draft values, 8.6 for one of 32,000.
template <typename T, bool DRAFT>
__global__ __launch_bounds__(kVfThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ uint32_t sBits[kVfChunk / 32];
  __shared__ double sD[kVfThreads / kWave];
  __shared__ int2 sE[kVfThreads / kWave];
  __shared__ double sBase;
  __shared__ int sTurn;
  const int b = blockIdx.y, tid = threadIdx.x;
  int64_t r0;
  const int n = packed_rows(a.cu, b, a.T, a.max_n, r0);
  const int s = a.stop[b];
  if (s < 0) return;
  const int64_t row = r0 + s;
  const double gone = a.gone[b];
  const double u = (double)fmaxf(a.u[r0], 0.f);
  const int64_t child = DRAFT ? -1 : vf_child(a, r0, n, s);
  uint64_t* sums = a.sums + (int64_t)b * 2 * a.chunks;
  VfTokens<T, DRAFT> tk;
  uint32_t named = 0u;
  {
    const int v0 = blockIdx.x * kVfChunk;
    tk.load(a, row, v0);
    if (!DRAFT) {
      vf_named(child, v0, sBits);
      named = vf_bits(sBits);
    }
    double x = 0.0, y = 0.0;
#pragma unroll
    for (int k = 0; k < kVfPer; ++k) {
      const double2 z = tk.at(k, gone, named);
      x += z.x;
      y += z.y;
    }
    x = vf_block_sum<kVfThreads>(x, sD);
    y = vf_block_sum<kVfThreads>(y, sD);
    if (tid == 0) {
      // agent scope: the work-group that adds them up may run on another XCD.  No release, which
      // would write the whole L2 back (2 us of a call's 12): a sum tells by its bits that it is there
      __hip_atomic_store(&sums[2 * blockIdx.x], __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&sums[2 * blockIdx.x + 1], __builtin_bit_cast(uint64_t, y), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      __builtin_amdgcn_s_waitcnt(0);
      sTurn = __hip_atomic_fetch_add(&a.done[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (sTurn != a.chunks - 1) return;
  }
  // each thread's run of chunks, the first of them in registers
  const int per = (a.chunks + kVfThreads - 1) / kVfThreads;
  const int c0 = min(tid * per, a.chunks), c1 = min(c0 + per, a.chunks);
  // every sum was stored before its work-group counted itself in: none stays unset (two calls at once on
  // one workspace, which is no use of it, could clear one for good: the wait ends all the same)
  auto one = [&](int i) {
    uint64_t w = kVfUnset;
    for (int k = 0; k < 65536 && w == kVfUnset; ++k)
      w = __hip_atomic_load(&sums[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return __builtin_bit_cast(double, w);
  };
  auto read = [&](int c) { return make_double2(one(2 * c), one(2 * c + 1)); };
  const double2 sum0 = c0 < c1 ? read(c0) : make_double2(0.0, 0.0);
  auto sum_of = [&](int c) { return c == c0 ? sum0 : read(c); };
  double mine = 0.0, mine_w = 0.0, total, total_w;
  for (int c = c0; c < c1; ++c) {
    const double2 x = sum_of(c);
    mine += x.x;
    mine_w += x.y;
  }
  double before = vf_before(mine, sD, total);
  const double before_w = vf_before(mine_w, sD, total_w);
  const bool rest = total > 0.0;            // nothing left by rounding: the row itself
  if (!rest) { before = before_w; total = total_w; }
  if (!(total > 0.0)) {
    if (tid == 0) a.token[b] = -1;
    return;
  }
  // a number of 1 is exceeded by no running sum, however its additions were grouped
  const double want = u < 1.0 ? u * total : (double)INFINITY;
  int first = INT32_MAX, last = -1;
  {
    double x = before;
    for (int c = c0; c < c1; ++c) {
      const double2 z = sum_of(c);
      const double y = rest ? z.x : z.y;
      x += y;
      if (y > 0.0) {                          // (a chunk without anything holds no token to draw)
        last = c;
        if (x > want) { first = c; break; }
      }
    }
  }
  vf_ends(first, last, sE);
  const int at = first == INT32_MAX ? last : first;
  const int v0 = at * kVfChunk;
  tk.load(a, row, v0);
  if (at >= c0 && at < c1) {
    double x = before;
    for (int c = c0; c < at; ++c) { const double2 z = sum_of(c); x += rest ? z.x : z.y; }
    sBase = x;
  }
  if (!DRAFT) {
    vf_named(child, v0, sBits);
    named = vf_bits(sBits);
  }
  double run = 0.0;
#pragma unroll
  for (int k = 0; k < kVfPer; ++k) {
    const double2 z = tk.at(k, gone, named);
    run += rest ? z.x : z.y;
  }
  double x = vf_before(run, sD, total);     // (its barriers order sBase)
  x += sBase;
  first = INT32_MAX;
  last = -1;
#pragma unroll
  for (int k = 0; k < kVfPer; ++k) {
    const double2 z = tk.at(k, gone, named);
    const double y = rest ? z.x : z.y;
    x += y;
    if (y > 0.0) {
      last = tid * kVfPer + k;
      if (x > want && first == INT32_MAX) first = last;
    }
  }
  vf_ends(first, last, sE);
  if (tid == 0) a.token[b] = v0 + (first == INT32_MAX ? last : first);
}

static int verify_chunks(int64_t T, int V, bool greedy, int& chunk) {
  if (!greedy) {
    chunk = kVfChunk;
    return (V + kVfChunk - 1) / kVfChunk;
  }
  // work-groups for two rounds of eight on every CU, a piece of a row of 8,192 tokens at least (1,156 rows
  // whole: 53 us, in four pieces: 51)
  const int64_t per_row = (4096 + T - 1) / std::max<int64_t>(T, 1);
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(per_row, (V + 8191) / 8192));
  chunk = (int)(((V + pieces - 1) / pieces + 63) / 64 * 64);
  return (V + chunk - 1) / chunk;
}

struct VerifyLayout { int64_t stop, done, gone, sums, best_v, best_i, total; int chunks, chunk; };
static VerifyLayout verify_layout(int B, int64_t T, int V, bool greedy) {
  VerifyLayout L;
  L.chunks = verify_chunks(T, V, greedy, L.chunk);
  auto align = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t o = 0;
  L.stop = o; o = align(o + (int64_t)B * 4);
  L.done = o; o = align(o + (int64_t)B * 4);
  L.gone = o; o = align(o + (int64_t)B * 8);
  L.sums = o; if (!greedy) o = align(o + (int64_t)B * L.chunks * 16);
  L.best_v = o; if (greedy) o = align(o + T * L.chunks * 4);
  L.best_i = o; if (greedy) o = align(o + T * L.chunks * 4);
  L.total = o;
  return L;
}

template <typename T>
static void verify_launch(const VerifyArgs& a, hipStream_t st) {
  if (!a.u) {
    if (a.T > 0)
      hipLaunchKernelGGL(verify_best_kernel<T>, dim3((unsigned)(a.T * a.chunks)), dim3(kVfThreads), 0, st, a);
    hipLaunchKernelGGL((verify_walk_kernel<T, 0, 256>), dim3(a.B), dim3(256), 0, st, a);
    return;
  }
  const dim3 grid(a.chunks, a.B);
  if (a.q) {
    hipLaunchKernelGGL((verify_walk_kernel<T, 2, 1024>), dim3(a.B), dim3(1024), 0, st, a);
    hipLaunchKernelGGL((verify_draw_kernel<T, true>), grid, dim3(kVfThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL((verify_walk_kernel<T, 1, 256>), dim3(a.B), dim3(256), 0, st, a);
    hipLaunchKernelGGL((verify_draw_kernel<T, false>), grid, dim3(kVfThreads), 0, st, a);
  }
}

}  // namespace dash

extern "C" int dash_verify_tree_workspace_size(int B, int64_t T, int V, int greedy, int64_t* bytes) {
  using namespace dash;
  if (!bytes || B < 0 || T < 0 || V <= 0) return kErrInvalid;
  *bytes = verify_layout(B, T, V, greedy != 0).total;
  return kOk;
}

extern "C" int dash_verify_tree(const void* target, int64_t target_stride, const void* draft,
                                int64_t draft_stride, int dtype, const void* tokens, int tokens_int64,
                                const int32_t* parents, const int32_t* cu_seqlens_q,
                                const float* uniforms, int B, int64_t T, int V, int max_query_len,
                                int32_t* count, int32_t* path, int64_t path_stride,
                                int64_t* next_token, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  using namespace dash;
  if (B < 0 || T < 0 || V <= 0 || max_query_len < 0 || dtype < 0 || dtype > 2) return kErrInvalid;
  if (B == 0) return kOk;
  if (!cu_seqlens_q || !count || !next_token) return kErrInvalid;
  if (T > 0 && (!target || !tokens || !parents)) return kErrInvalid;
  if (max_query_len > 0 && !path) return kErrInvalid;
  if (draft && !uniforms) return kErrInvalid;
  if (max_query_len > kVfMaxNodes || B > 65535 || V > (1 << 30)) return kErrUnsupported;
  const VerifyLayout L = verify_layout(B, T, V, !uniforms);
  if (!uniforms && (T > INT32_MAX || !fits_grid(T * L.chunks, kVfThreads))) return kErrUnsupported;
  if (!workspace || workspace_bytes < L.total || (uintptr_t)workspace % 256 != 0) return kErrWorkspace;
  char* w = (char*)workspace;
  VerifyArgs a = {};
  a.p = target; a.p_st = target_stride; a.q = draft; a.q_st = draft_stride;
  a.tok = tokens; a.tok64 = tokens_int64; a.parents = parents; a.cu = cu_seqlens_q; a.u = uniforms;
  a.B = B; a.V = V; a.max_n = max_query_len; a.chunks = L.chunks; a.chunk = L.chunk; a.T = T;
  a.count = count; a.path = path; a.path_st = path_stride; a.token = next_token;
  a.stop = (int32_t*)(w + L.stop); a.done = (int32_t*)(w + L.done);
  a.gone = (double*)(w + L.gone); a.sums = (uint64_t*)(w + L.sums);
  a.best_v = (float*)(w + L.best_v); a.best_i = (int32_t*)(w + L.best_i);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) verify_launch<float>(a, st);
  else if (dtype == 1) verify_launch<bf16>(a, st);
  else verify_launch<__half>(a, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
