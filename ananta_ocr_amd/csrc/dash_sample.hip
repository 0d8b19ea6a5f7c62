// Sampling on gfx950: the next token of every row of logits, from given random numbers, after
// temperature, top-k, top-p and min-p, and the probabilities that are left.
//
// Token v of a row has the weight w_v = exp((x_v - M) / T), M the row's largest logit.  In the order of
// falling logits (of equals, the lower id first) the first k tokens stay; of those, the ones whose
// predecessors hold less than p of the first k's weight; of those, the ones with w >= min_p.  The first
// always does.  The random number u draws the first id whose running sum of what stays exceeds u times the
// whole.
//
// Weights are whole numbers of 2^-s of the largest, s = 62 - log2 V (at most 51), taken from a 64-bit
// exponential: the sums are exact, so no token depends on the order in which work-groups, wavefronts or
// atomics add them up, and a border lies where the 64-bit weights put it but for 2^-46 of the
// best token's weight a token.  A token below half of 2^-s is never drawn and counts as none.
//
// A row is cut into S chunks of a work-group each; a chunk's tiles are 4,096 tokens, four in a row a thread:
//   sample_max    the best token and the lowest logit of every chunk
//   sample_bins   count and weight of a chunk's tokens in kSmBins bins of equal width in M - x, from M down
//   sample_pick   the bins in which the k-th token and the border of p lie (every work-group by itself from
//                 the chunks' sums), their tokens listed; the weight of what surely stays, tile by tile
//   sample_draw   the borders within the listed tokens, by their (logit, id); the tile and then the token
//                 that u falls into; the probabilities
// Rows that need no border skip the bins.  A list that would be too long (many tokens of one logit) is
// not made: its work-group reads the row again instead, as often as the border needs.
#include <hip/hip_fp16.h>

#include "dash_common.h"

namespace dash {

constexpr int kSmThreads = 1024;
constexpr int kSmTile = 4 * kSmThreads;   // tokens
constexpr int kSmBins = 512;
constexpr int kSmMaxChunks = 16;
constexpr int kSmList = 2048;             // tokens listed of a row
constexpr int kSmMaxV = 1 << 20;
constexpr int kSmTiles = kSmMaxV / kSmTile;
constexpr int kSmRows = 2048;             // rows of a pass
constexpr int kSmWaves = kSmThreads / kWave;

struct SampleState {                      // of a row, from sample_pick
  uint64_t k_mass, k_whole;               // weight of the bins before the k-th token's; of the first k if exact
  uint64_t p_mass;                        // weight of the bins before the border of p's
  int32_t k_count, k_bin;                 // tokens of the bins before; -1: no border of k
  int32_t p_lo, p_hi;                     // bins that may hold the border of p; p_lo -1: none
  int32_t sure;                           // bins below it stay
  int32_t listed;                         // tokens listed, -1: too many
};

struct SampleArgs {
  const void* x; int64_t x_st;
  const float* u;                         // null: no draw
  const float* t; const int32_t* k; const float* p; const float* m;    // null: the number below
  float t0; int32_t k0; float p0, m0;
  int V, S, chunk, tiles;                 // tiles of a row
  int bits;                               // s
  int64_t* token; void* probs; int64_t p_st;
  // workspace
  uint64_t* best;                         // [R, S] key and inverted id of a chunk's best token
  uint32_t* low;                          // [R, S] lowest live key
  uint32_t* cnt; uint64_t* mass;          // [R, S, kSmBins]
  SampleState* state;                     // [R]
  int32_t* n_list;                        // [R]
  uint64_t* list;                         // [R, kSmList]
  uint64_t* tile;                         // [R, tiles] weight of what surely stays
};

__device__ __forceinline__ float sm_in(float x) { return x; }
__device__ __forceinline__ float sm_in(bf16 x) { return (float)x; }
__device__ __forceinline__ float sm_in(__half x) { return __half2float(x); }
__device__ __forceinline__ void sm_out(float x, float& y) { y = x; }
__device__ __forceinline__ void sm_out(float x, bf16& y) { y = (bf16)x; }
__device__ __forceinline__ void sm_out(float x, __half& y) { y = __float2half_rn(x); }

// Four tokens from v on (masked, -inf, past v1).
template <typename T>
__device__ __forceinline__ void sm_load(const T* row, int v, int v1, float (&x)[4]) {
  typedef uint32_t V __attribute__((ext_vector_type(sizeof(T)), aligned(2)));
  if (v + 4 <= v1) {
    union { V b; T e[4]; } y;
    y.b = *(const V*)(row + v);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = sm_in(y.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = v + j < v1 ? sm_in(row[v + j]) : -INFINITY;
  }
}

// Keys order the logits; 0: masked (-inf) or no number.  -0 is 0.
__device__ __forceinline__ uint32_t sm_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_logit(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// A token's place in the order: larger is earlier.
__device__ __forceinline__ uint64_t sm_place(uint32_t key, int v) {
  return (uint64_t)key << 32 | (uint32_t)~v;
}

// What a row's tokens are measured by.
struct SampleRow {
  float top, bin_scale;
  double c, scale;                        // log2(e) / T; 2^s
  float min_p;
  int k; float p;
  bool any, greedy, filter;
  int best_id;
};

template <typename A>
__device__ __forceinline__ SampleRow sm_row(const A& a, int64_t r, uint64_t best, uint32_t low) {
  SampleRow w;
  const float t = a.t ? a.t[r] : a.t0;
  w.k = a.k ? a.k[r] : a.k0;
  w.p = a.p ? a.p[r] : a.p0;
  const float m = a.m ? a.m[r] : a.m0;
  w.min_p = m > 0.f ? fminf(m, 1.f) : 0.f;
  const uint32_t key = (uint32_t)(best >> 32);
  w.any = key != 0;
  w.best_id = (int)~(uint32_t)best;
  w.greedy = !(t > 0.f);
  w.top = sm_logit(key);
  w.c = 1.4426950408889634 / (double)t;
  w.scale = __builtin_bit_cast(double, (uint64_t)(1023 + a.bits) << 52);
  if (w.k >= a.V) w.k = 0;
  w.filter = w.any && !w.greedy && (w.k > 0 || w.p < 1.f);
  // past (s + 1) ln 2 T from the top a weight is none
  const float range = fminf(w.top - sm_logit(low), (float)(a.bits + 1) * 0.6931472f * t);
  w.bin_scale = range > 1e-30f ? (float)kSmBins / range : 0.f;
  return w;
}
// The best token of a row and its lowest logit, from its chunks.
template <typename A>
__device__ __forceinline__ SampleRow sm_row_of(const A& a, int64_t r) {
  uint64_t best = 0;
  uint32_t low = ~0u;
  for (int c = 0; c < a.S; ++c) {
    best = max(best, a.best[r * a.S + c]);
    low = min(low, a.low[r * a.S + c]);
  }
  return sm_row(a, r, best, low);
}

// exp((x - top) / T).  2^y = 2^n 2^f with |f| <= 1/2, 2^f by the exponential's series up to the 12th power
// of f ln 2, whose next term is below 1.7e-16.
__device__ __forceinline__ double sm_weight(const SampleRow& w, float x) {
  if (x == w.top) return 1.0;
  const double y = ((double)x - (double)w.top) * w.c;
  if (!(y > -60.0)) return 0.0;
  const double n = __builtin_rint(y), f = (y - n) * 0.6931471805599453;
  double s = 1.0 / 479001600.0;
  s = fma(s, f, 1.0 / 39916800.0);
  s = fma(s, f, 1.0 / 3628800.0);
  s = fma(s, f, 1.0 / 362880.0);
  s = fma(s, f, 1.0 / 40320.0);
  s = fma(s, f, 1.0 / 5040.0);
  s = fma(s, f, 1.0 / 720.0);
  s = fma(s, f, 1.0 / 120.0);
  s = fma(s, f, 1.0 / 24.0);
  s = fma(s, f, 1.0 / 6.0);
  s = fma(s, f, 0.5);
  s = fma(s, f, 1.0);
  s = fma(s, f, 1.0);
  return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, s) + ((uint64_t)(int64_t)(int)n << 52));
}
// The weight as a whole number of 2^-s, to the nearest: added to 2^52 it stands in the last bits.
__device__ __forceinline__ uint64_t sm_whole(const SampleRow& w, double e) {
  return __builtin_bit_cast(uint64_t, fma(e, w.scale, 4503599627370496.0)) - 0x4330000000000000ull;
}
__device__ __forceinline__ int sm_bin(const SampleRow& w, float x) {
  return x == w.top ? 0 : (int)fminf((w.top - x) * w.bin_scale, (float)(kSmBins - 1));
}

// Sum over the work-group's earlier threads; total: over all.
__device__ __forceinline__ uint64_t sm_before(uint64_t v, uint64_t* sW, uint64_t& total) {
  const int lane = wave_lane(), wv = threadIdx.x / kWave;
  uint64_t x = v;
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) {
    const uint64_t y = __shfl_up(x, s, kWave);
    if (lane >= s) x += y;
  }
  __syncthreads();
  if (lane == kWave - 1) sW[wv] = x;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSmWaves; ++w) {
    if (w < wv) before += sW[w];
    total += sW[w];
  }
  return before + x - v;
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ uint64_t sB[kSmWaves];
  __shared__ uint32_t sL[kSmWaves];
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x, tid = threadIdx.x;
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  const T* row = (const T*)a.x + r * a.x_st;
  uint64_t best = 0;
  uint32_t low = ~0u;
  for (int v = v0 + 4 * tid; v < v1; v += kSmTile) {
    float x[4];
    sm_load(row, v, v1, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = sm_key(x[j]);
      if (key == 0) continue;
      best = max(best, sm_place(key, v + j));
      low = min(low, key);
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, m, kWave));
    low = min(low, (uint32_t)__shfl_xor(low, m, kWave));
  }
  if (wave_lane() == 0) { sB[tid / kWave] = best; sL[tid / kWave] = low; }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kSmWaves; ++w) {
      best = max(best, sB[w]);
      low = min(low, sL[w]);
    }
    a.best[r * a.S + c] = best;
    a.low[r * a.S + c] = low;
    if (c == 0) a.n_list[r] = 0;
  }
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_bins_kernel(SampleArgs a) {
  __shared__ uint32_t sCnt[kSmBins];
  __shared__ unsigned long long sMass[kSmBins];
  const int64_t r = blockIdx.y;
  const SampleRow w = sm_row_of(a, r);
  if (!w.filter) return;
  const int c = blockIdx.x, tid = threadIdx.x;
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  const T* row = (const T*)a.x + r * a.x_st;
  if (tid < kSmBins) { sCnt[tid] = 0; sMass[tid] = 0; }
  __syncthreads();
  for (int v = v0 + 4 * tid; v < v1; v += kSmTile) {
    float x[4];
    sm_load(row, v, v1, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (sm_key(x[j]) == 0) continue;
      const uint64_t e = sm_whole(w, sm_weight(w, x[j]));
      if (e == 0) continue;
      const int b = sm_bin(w, x[j]);
      atomicAdd(&sCnt[b], 1u);
      atomicAdd(&sMass[b], (unsigned long long)e);
    }
  }
  __syncthreads();
  if (tid < kSmBins) {
    const int64_t at = (r * a.S + c) * kSmBins + tid;
    a.cnt[at] = sCnt[tid];
    a.mass[at] = sMass[tid];
  }
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_pick_kernel(SampleArgs a) {
  __shared__ uint64_t sW[kSmWaves];
  __shared__ uint32_t sBefore[kSmBins + 1];         // tokens of the bins before
  __shared__ SampleState sSt;
  __shared__ uint64_t sKMass, sAll;
  __shared__ unsigned long long sTile[kSmTiles];
  const int64_t r = blockIdx.y;
  const SampleRow w = sm_row_of(a, r);
  if (!w.any || w.greedy) return;
  const int c = blockIdx.x, tid = threadIdx.x;
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  if (tid == 0) sSt = SampleState{0, 0, 0, 0, -1, -1, -1, kSmBins, 0};
  if (w.filter) {
    uint32_t cnt = 0;
    uint64_t mass = 0;
    if (tid < kSmBins)
      for (int i = 0; i < a.S; ++i) {
        cnt += a.cnt[(r * a.S + i) * kSmBins + tid];
        mass += a.mass[(r * a.S + i) * kSmBins + tid];
      }
    uint64_t live, all;
    const uint64_t cb = sm_before(cnt, sW, live), mb = sm_before(mass, sW, all);
    if (tid <= kSmBins) sBefore[tid] = (uint32_t)cb;
    if (tid == 0) sAll = all;
    const bool k_on = w.k > 0 && (uint64_t)w.k < live;
    if (k_on && cb < (uint64_t)w.k && cb + cnt >= (uint64_t)w.k) {
      sSt.k_bin = tid;
      sSt.k_count = (int)cb;
      sSt.k_mass = mb;
      sKMass = mass;
      if (cb + cnt == (uint64_t)w.k) sSt.k_whole = mb + mass;
    }
    __syncthreads();
    const int kb = sSt.k_bin;
    const bool part = kb >= 0 && sSt.k_whole == 0;  // the k-th token is not its bin's last
    if (w.p < 1.f) {
      const double hi = (double)w.p * (double)(kb >= 0 ? sSt.k_mass + sKMass : all);
      const double lo = part ? (double)w.p * (double)sSt.k_mass : hi;
      if (mass > 0) {
        // the bin in which the weight reaches p of the first k's, whatever that is between lo and hi
        if ((lo <= 0.0 && tid == 0) || ((double)mb < lo && (double)(mb + mass) >= lo)) {
          sSt.p_lo = tid;
          sSt.p_mass = mb;
        }
        if ((hi <= 0.0 && tid == 0) || ((double)mb < hi && (double)(mb + mass) >= hi)) sSt.p_hi = tid;
      }
    }
    __syncthreads();
    if (tid == 0) {
      SampleState st = sSt;
      int n = part ? sBefore[kb + 1] - sBefore[kb] : 0;
      st.sure = kb < 0 ? kSmBins : part ? kb : kb + 1;
      if (st.p_lo >= 0) {
        if (kb >= 0) st.p_hi = min(st.p_hi, kb);
        st.sure = st.p_lo;
        n += sBefore[st.p_hi + 1] - sBefore[st.p_lo];
        if (part && kb >= st.p_lo && kb <= st.p_hi) n -= sBefore[kb + 1] - sBefore[kb];
      }
      st.listed = n <= kSmList ? n : -1;
      sSt = st;
    }
  }
  __syncthreads();
  const SampleState st = sSt;
  const bool part = st.k_bin >= 0 && st.k_whole == 0;
  if (c == 0 && tid == 0) a.state[r] = st;
  const int t0 = v0 / kSmTile, nt = (v1 - v0 + kSmTile - 1) / kSmTile;
  if (tid < nt) sTile[tid] = 0;
  __syncthreads();
  const T* row = (const T*)a.x + r * a.x_st;
  for (int i = 0; i < nt; ++i) {
    const int v = v0 + i * kSmTile + 4 * tid;
    float x[4];
    if (v < v1) {
      sm_load(row, v, v1, x);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = -INFINITY;
    }
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = sm_key(x[j]);
      if (key == 0) continue;
      const int b = sm_bin(w, x[j]);
      const bool sure = b < st.sure;
      const bool take = st.listed > 0 && ((part && b == st.k_bin) || (b >= st.p_lo && b <= st.p_hi && st.p_lo >= 0));
      if (!sure && !take) continue;
      const double e = sm_weight(w, x[j]);
      const uint64_t whole = sm_whole(w, e);
      if (sure && e >= (double)w.min_p) sum += whole;
      if (take && whole > 0) {
        const int at = atomicAdd(&a.n_list[r], 1);
        if (at < kSmList) a.list[r * kSmList + at] = sm_place(key, v + j);
      }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor((unsigned long long)sum, m, kWave);
    if (wave_lane() == 0 && sum > 0) atomicAdd(&sTile[i], (unsigned long long)sum);
  }
  __syncthreads();
  if (tid < nt) a.tile[r * a.tiles + t0 + tid] = sTile[tid];
}

// The last token (by its place) of those in [lo, hi] that the rule keeps: with `need` > 0 the need-th,
// else the last whose predecessors' weight, `mass` of them outside, is below `target` (the first if none
// is).  for_each(f) calls f(place, key) for the tokens of the source.  mass: with the token found added.
struct SampleCut { uint64_t place, mass; };
template <typename Each>
__device__ SampleCut sm_cut(const SampleRow& w, Each for_each, int need, double target, uint64_t mass,
                            uint64_t lo, uint64_t hi, uint32_t* sCnt, unsigned long long* sMass, uint64_t* sW,
                            unsigned long long* sEnds, int* sAt) {
  const int tid = threadIdx.x;
  // the ends of what there is
  __syncthreads();
  if (tid == 0) { sEnds[0] = ~0ull; sEnds[1] = 0; }
  __syncthreads();
  {
    uint64_t mn = ~0ull, mx = 0;
    for_each([&](uint64_t place, float) {
      if (place < lo || place > hi) return;
      mn = min(mn, place);
      mx = max(mx, place);
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      mn = min(mn, (uint64_t)__shfl_xor((unsigned long long)mn, m, kWave));
      mx = max(mx, (uint64_t)__shfl_xor((unsigned long long)mx, m, kWave));
    }
    if (wave_lane() == 0 && mx > 0) { atomicMin(&sEnds[0], (unsigned long long)mn); atomicMax(&sEnds[1], (unsigned long long)mx); }
  }
  __syncthreads();
  lo = sEnds[0];
  hi = sEnds[1];
  while (lo < hi) {                       // 256 steps a pass: at most eight passes
    const int top = 64 - __clzll(hi - lo), shift = max(top - 8, 0);
    __syncthreads();
    if (tid < 256) { sCnt[tid] = 0; sMass[tid] = 0; }
    if (tid == 0) *sAt = 0;
    __syncthreads();
    for_each([&](uint64_t place, float x) {
      if (place < lo || place > hi) return;
      const int b = (int)((hi - place) >> shift);
      atomicAdd(&sCnt[b], 1u);
      atomicAdd(&sMass[b], (unsigned long long)sm_whole(w, sm_weight(w, x)));
    });
    __syncthreads();
    const uint32_t cnt = tid < 256 ? sCnt[tid] : 0;
    const uint64_t mine = tid < 256 ? sMass[tid] : 0;
    uint64_t total;
    const uint64_t cb = sm_before(cnt, sW, total), mb = mass + sm_before(mine, sW, total);
    if (cnt > 0) {
      if (need > 0 ? cb < (uint64_t)need : cb == 0 || (double)mb < target) atomicMax(sAt, tid);
    }
    __syncthreads();
    const int b = *sAt;
    if (tid == b) { sEnds[0] = cb; sEnds[1] = mb; }
    __syncthreads();
    if (need > 0) need -= (int)sEnds[0];
    mass = sEnds[1];
    hi -= (uint64_t)b << shift;
    const uint64_t width = (1ull << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    if (sCnt[b] == 1 && shift > 0) {      // one token: where it is
      __syncthreads();
      for_each([&](uint64_t place, float) {
        if (place >= lo && place <= hi) sEnds[0] = place;
      });
      __syncthreads();
      lo = hi = sEnds[0];
    }
  }
  __syncthreads();
  return SampleCut{hi, mass + sm_whole(w, sm_weight(w, sm_logit((uint32_t)(hi >> 32))))};
}

template <typename T, typename P>
__global__ __launch_bounds__(kSmThreads) void sample_draw_kernel(SampleArgs a) {
  __shared__ uint64_t sList[kSmList];
  __shared__ uint32_t sCnt[256];
  __shared__ unsigned long long sMass[256];
  __shared__ uint64_t sW[kSmWaves];
  __shared__ unsigned long long sEnds[2];
  __shared__ int sAt[2];
  __shared__ unsigned long long sTile[kSmTiles];
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x, tid = threadIdx.x;
  const SampleRow w = sm_row_of(a, r);
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  P* const probs = a.probs ? (P*)a.probs + r * a.p_st : nullptr;
  if (!w.any || w.greedy) {
    if (c == 0 && tid == 0 && a.token) a.token[r] = w.any ? w.best_id : -1;
    if (probs)
      for (int v = v0 + tid; v < v1; v += kSmThreads) sm_out(w.any && v == w.best_id ? 1.f : 0.f, probs[v]);
    return;
  }
  const T* row = (const T*)a.x + r * a.x_st;
  const SampleState st = a.state[r];
  const bool part = st.k_bin >= 0 && st.k_whole == 0;
  for (int i = tid; i < st.listed; i += kSmThreads) sList[i] = a.list[r * kSmList + i];
  for (int i = tid; i < a.tiles; i += kSmThreads) sTile[i] = a.tile[r * a.tiles + i];
  __syncthreads();
  // the tokens of bins b0 .. b1
  auto tokens = [&](int b0, int b1) {
    return [&, b0, b1](auto f) {
      if (st.listed >= 0) {
        for (int i = tid; i < st.listed; i += kSmThreads) {
          const float x = sm_logit((uint32_t)(sList[i] >> 32));
          const int b = sm_bin(w, x);
          if (b >= b0 && b <= b1) f(sList[i], x);
        }
        return;
      }
      for (int v = 4 * tid; v < a.V; v += kSmTile) {
        float x[4];
        sm_load(row, v, a.V, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t key = sm_key(x[j]);
          if (key == 0) continue;
          const int b = sm_bin(w, x[j]);
          if (b >= b0 && b <= b1 && sm_whole(w, sm_weight(w, x[j])) > 0) f(sm_place(key, v + j), x[j] + 0.f);
        }
      }
    };
  };
  uint64_t last = ~0ull;                  // the last place that stays past the sure bins
  uint64_t k_place = 0, k_mass = st.k_whole;
  if (part) {
    const SampleCut z = sm_cut(w, tokens(st.k_bin, st.k_bin), w.k - st.k_count, 0.0, st.k_mass, 0, ~0ull, sCnt,
                               sMass, sW, sEnds, sAt);
    last = k_place = z.place;
    k_mass = z.mass;
  }
  if (st.p_lo >= 0) {
    if (st.k_bin < 0) {                   // of the whole row
      uint64_t all = 0;
      if (tid < kSmBins)
        for (int i = 0; i < a.S; ++i) all += a.mass[(r * a.S + i) * kSmBins + tid];
      sm_before(all, sW, k_mass);
    }
    last = sm_cut(w, tokens(st.p_lo, st.p_hi), 0, (double)w.p * (double)k_mass, st.p_mass, k_place, ~0ull, sCnt,
                  sMass, sW, sEnds, sAt).place;
  }
  if (st.sure < kSmBins)
    tokens(st.sure, kSmBins - 1)([&](uint64_t place, float x) {
      if (place < last) return;
      const double e = sm_weight(w, x);
      if (e >= (double)w.min_p)
        atomicAdd(&sTile[(int)~(uint32_t)place / kSmTile], (unsigned long long)sm_whole(w, e));
    });
  auto stays = [&](float x, int v, double& e) {
    const uint32_t key = sm_key(x);
    if (key == 0 || (sm_bin(w, x) >= st.sure && sm_place(key, v) < last)) return false;
    e = sm_weight(w, x);
    return e >= (double)w.min_p;
  };
  // the tile that the number falls into
  __syncthreads();
  uint64_t total;
  const uint64_t mine = tid < a.tiles ? sTile[tid] : 0;
  const uint64_t before = sm_before(mine, sW, total);
  if (c == 0 && a.u) {
    const float u = fmaxf(a.u[r], 0.f);
    // a number of 1 is exceeded by no running sum: the last token that stays
    const double want = u < 1.f ? (double)u * (double)total : (double)INFINITY;
    if (tid == 0) { sAt[0] = INT32_MAX; sAt[1] = 0; }
    __syncthreads();
    if (mine > 0) {
      if ((double)(before + mine) > want) atomicMin(&sAt[0], tid);
      atomicMax(&sAt[1], tid);
    }
    __syncthreads();
    const int t = sAt[0] == INT32_MAX ? sAt[1] : sAt[0];
    if (tid == t) sEnds[0] = before;
    __syncthreads();
    if (tid == 0) { sAt[0] = INT32_MAX; sAt[1] = 0; }
    const int v = t * kSmTile + 4 * tid;
    float x[4];
    if (v < a.V) {
      sm_load(row, v, a.V, x);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = -INFINITY;
    }
    uint64_t e[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      double f;
      e[j] = stays(x[j], v + j, f) ? sm_whole(w, f) : 0;
      sum += e[j];
    }
    uint64_t tile;
    uint64_t run = sEnds[0] + sm_before(sum, sW, tile);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      run += e[j];
      if (e[j] > 0) {
        if ((double)run > want) atomicMin(&sAt[0], v + j);
        atomicMax(&sAt[1], v + j);
      }
    }
    __syncthreads();
    if (tid == 0) a.token[r] = sAt[0] == INT32_MAX ? sAt[1] : sAt[0];
  }
  if (!probs) return;
  const double inv = w.scale / (double)total;
  for (int v = v0 + 4 * tid; v < v1; v += kSmTile) {
    float x[4];
    sm_load(row, v, v1, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      double e;
      const bool is = stays(x[j], v + j, e) && sm_whole(w, e) > 0;
      if (v + j < v1) sm_out(is ? (float)(e * inv) : 0.f, probs[v + j]);
    }
  }
}

// Chunks of a row: work-groups for two a CU in all, a tile each at least.
struct SampleLayout {
  int S, chunk, tiles;
  int64_t best, low, cnt, mass, state, n_list, list, tile, total;
};
static SampleLayout sample_layout(int64_t R, int V) {
  SampleLayout L;
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(R, kSmRows));
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kSmMaxChunks, 512 / rows));
  L.chunk = (int)(((V + want - 1) / want + kSmTile - 1) / kSmTile * kSmTile);
  L.S = (V + L.chunk - 1) / L.chunk;
  L.tiles = (V + kSmTile - 1) / kSmTile;
  auto align = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t o = 0;
  L.best = o; o = align(o + rows * L.S * 8);
  L.low = o; o = align(o + rows * L.S * 4);
  L.cnt = o; o = align(o + rows * L.S * kSmBins * 4);
  L.mass = o; o = align(o + rows * L.S * kSmBins * 8);
  L.state = o; o = align(o + rows * (int64_t)sizeof(SampleState));
  L.n_list = o; o = align(o + rows * 4);
  L.list = o; o = align(o + rows * kSmList * 8);
  L.tile = o; o = align(o + rows * L.tiles * 8);
  L.total = o;
  return L;
}

template <typename T>
static void sample_launch(const SampleArgs& a, int rows, int p_dtype, bool filter, hipStream_t st) {
  const dim3 grid(a.S, rows), block(kSmThreads);
  hipLaunchKernelGGL(sample_max_kernel<T>, grid, block, 0, st, a);
  if (filter) hipLaunchKernelGGL(sample_bins_kernel<T>, grid, block, 0, st, a);
  hipLaunchKernelGGL(sample_pick_kernel<T>, grid, block, 0, st, a);
  const dim3 draw(a.probs ? a.S : 1, rows);
  if (p_dtype == 1) hipLaunchKernelGGL((sample_draw_kernel<T, bf16>), draw, block, 0, st, a);
  else if (p_dtype == 2) hipLaunchKernelGGL((sample_draw_kernel<T, __half>), draw, block, 0, st, a);
  else hipLaunchKernelGGL((sample_draw_kernel<T, float>), draw, block, 0, st, a);
}

}  // namespace dash

extern "C" int dash_sample_workspace_size(int64_t R, int V, int64_t* bytes) {
  using namespace dash;
  if (!bytes || R < 0 || V <= 0) return kErrInvalid;
  if (V > kSmMaxV) return kErrUnsupported;
  *bytes = sample_layout(R, V).total;
  return kOk;
}

extern "C" int dash_sample(const void* logits, int64_t row_stride, int dtype, const float* uniforms,
                           const float* temperature, float temperature0, const int32_t* top_k, int top_k0,
                           const float* top_p, float top_p0, const float* min_p, float min_p0, int64_t R, int V,
                           int64_t* tokens, void* probs, int64_t probs_stride, int probs_dtype, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  using namespace dash;
  if (R < 0 || V <= 0 || dtype < 0 || dtype > 2 || probs_dtype < 0 || probs_dtype > 2) return kErrInvalid;
  if (R == 0) return kOk;
  if (!logits || (!uniforms != !tokens) || (!tokens && !probs)) return kErrInvalid;
  if (V > kSmMaxV) return kErrUnsupported;
  const SampleLayout L = sample_layout(R, V);
  if (!workspace || workspace_bytes < L.total || (uintptr_t)workspace % 256 != 0) return kErrWorkspace;
  char* ws = (char*)workspace;
  hipStream_t st = (hipStream_t)stream;
  const int size = dtype == 0 ? 4 : 2, p_size = probs_dtype == 0 ? 4 : 2;
  for (int64_t r0 = 0; r0 < R; r0 += kSmRows) {
    const int rows = (int)std::min<int64_t>(R - r0, kSmRows);
    SampleArgs a = {};
    a.x = (const char*)logits + r0 * row_stride * size; a.x_st = row_stride;
    a.u = uniforms ? uniforms + r0 : nullptr;
    a.t = temperature ? temperature + r0 : nullptr; a.t0 = temperature0;
    a.k = top_k ? top_k + r0 : nullptr; a.k0 = top_k0;
    a.p = top_p ? top_p + r0 : nullptr; a.p0 = top_p0;
    a.m = min_p ? min_p + r0 : nullptr; a.m0 = min_p0;
    a.V = V; a.S = L.S; a.chunk = L.chunk; a.tiles = L.tiles;
    int log = 0;
    while ((1 << log) < V) ++log;
    a.bits = std::min(51, 62 - log);
    a.token = tokens ? tokens + r0 : nullptr;
    a.probs = probs ? (char*)probs + r0 * probs_stride * p_size : nullptr; a.p_st = probs_stride;
    a.best = (uint64_t*)(ws + L.best); a.low = (uint32_t*)(ws + L.low);
    a.cnt = (uint32_t*)(ws + L.cnt); a.mass = (uint64_t*)(ws + L.mass);
    a.state = (SampleState*)(ws + L.state); a.n_list = (int32_t*)(ws + L.n_list);
    a.list = (uint64_t*)(ws + L.list); a.tile = (uint64_t*)(ws + L.tile);
    const bool filter = top_k || top_p || top_k0 > 0 || top_p0 < 1.f;
    if (dtype == 0) sample_launch<float>(a, rows, probs_dtype, filter, st);
    else if (dtype == 1) sample_launch<bf16>(a, rows, probs_dtype, filter, st);
    else sample_launch<__half>(a, rows, probs_dtype, filter, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return kOk;
}
