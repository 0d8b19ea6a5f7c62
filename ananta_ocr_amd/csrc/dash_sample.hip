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
// A short row, or one of many, is one work-group's (sample_row_kernel).  A long one is cut into S chunks of a
// work-group each:
//   sample_max     the best token and the lowest logit of every chunk
//   sample_bins    count and weight of a chunk's tokens in kSmBins bins of equal width in M - x, from M down
//   sample_select  the bins in which the k-th token, the border of p and the one of min_p lie: the bins before
//                  them surely stay, those behind surely do not
//   sample_pick    the tokens between, listed
//   sample_draw    the borders within the list, by the tokens' (logit, id); the chunk, the tile and then the
//                  token that u falls into; the probabilities
// Bound by the latency of dependent launches, and of the passes and barriers within them; the bins' for more than half
// by the vector units.  64 rows of 131,072 bf16 (16.8 MB, which each step over them fetches again: little stays in the
// L2s from launch to launch) 63 us: max 7.0, bins 15.4 (an exponential of 64 bits a token; the LDS atomics 1.5), select
// 6.2, pick 11.3 (a read: only listed tokens are weighed), draw 27.7 (the rows whose top-p leaves thousands).  By the
// instructions counted, four cycles each, the vector units are busy for 3.3, 8.5, 0.2, 3.4 and 0.8 us of these.  48
// rows of 100,003 fp32 with probabilities 68 us: 6.2, 11.8, 6.3, 9.5, 35.9 (busy 2.0, 5.1, 0.2, 2.2, 4.1).  One row of
// 32,000 27 to 30 us where it filters, 6.8 where it is greedy; cut into chunks it took 34 where a work-group took 31.
//
// A list that would be too long (many tokens of one logit) is not made: its work-group reads the row again
// instead, as often as the border needs.
#include <hip/hip_fp16.h>

#include <cfloat>

#include "dash_common.h"

namespace dash {

constexpr int kSmWide = 1024;             // threads of a row's work-group
constexpr int kSmThreads = 256;           // of a chunk's
constexpr int kSmBins = 512;
constexpr int kSmMaxChunks = 16;
constexpr int kSmList = 2048;             // tokens listed of a row
constexpr int kSmFew = 1024;              // so many tokens are all listed (one row 27.9 us; 256: 29.6, 512: 31.3)
constexpr int kSmMaxV = 1 << 20;
constexpr int kSmTiles = 256;             // tiles of a row's work-group, or of a chunk's, at most
constexpr int kSmShort = 32768;           // tokens of a row that one work-group takes
// Rows that take a work-group each, however long: as many as there are CUs.  (255 rows of 131,072 bf16 in chunks, and a
// work-group a row: top-k 50 and top-p 109 us, 94; top-p alone 141, 170.  128 rows: 77, 90; 98, 165.)
constexpr int kSmMany = 256;
constexpr int kSmCut = 256;               // steps a pass of the search for a border

struct SampleState {                      // of a row, once its bins are known
  uint64_t k_mass, k_whole;               // weight of the bins before the k-th token's; of the first k, 0 if unknown
  uint64_t p_mass;                        // weight of the bins before the border of p's
  int32_t k_count, k_bin;                 // tokens of the bins before; -1: no border of k
  int32_t p_lo, p_hi;                     // bins that may hold the border of p; p_lo -1: none
  int32_t sure, end;                      // bins below `sure` stay, bins from `end` on do not
  int32_t listed;                         // tokens to be looked at, -1: too many to list
};

struct SampleArgs {
  const void* x; int64_t x_st;
  const float* u;                         // null: no draw
  const float* t; const int32_t* k; const float* p; const float* m;    // null: the number below
  float t0; int32_t k0; float p0, m0;
  int V, S, chunk;
  int bits;                               // s
  int64_t* token; void* probs; int p_type; int64_t p_st;
  // workspace
  uint64_t* best;                         // [R, S] key and inverted id of a chunk's best token
  float* low;                             // [R, S] lowest logit that is not masked
  uint32_t* cnt; uint64_t* mass;          // [R, S, kSmBins]
  SampleState* state;                     // [R]
  int32_t* n_list;                        // [R]
  uint64_t* list;                         // [R, kSmList]
  uint64_t* sure;                         // [R, S] weight of a chunk's tokens that surely stay
};

__device__ __forceinline__ float sm_in(float x) { return x; }
__device__ __forceinline__ float sm_in(bf16 x) { return (float)x; }
__device__ __forceinline__ float sm_in(__half x) { return __half2float(x); }
__device__ __forceinline__ void sm_out(float x, float& y) { y = x; }
__device__ __forceinline__ void sm_out(float x, bf16& y) { y = (bf16)x; }
__device__ __forceinline__ void sm_out(float x, __half& y) { y = __float2half_rn(x); }

// A vector of kN tokens, 16 bytes at any element's boundary (global loads need no more); masked (-inf) past
// the row's end.
template <typename T>
struct SmVec {
  static constexpr int kN = 16 / sizeof(T);
  typedef uint32_t V __attribute__((ext_vector_type(4), aligned(2)));
  V b;
  __device__ __forceinline__ void load(const T* row, int v, int v1) {
    if (v + kN <= v1) {
      b = *(const V*)(row + v);
    } else {
      T e[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) sm_out(-INFINITY, e[j]);
      if (v < v1) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (v + j < v1) e[j] = row[v + j];
      }
      __builtin_memcpy(&b, e, 16);
    }
  }
  // Logit j: NaN as masked, +inf as the largest number.
  __device__ __forceinline__ float at(int j) const {
    float x;
    if (sizeof(T) == 4) {
      x = __uint_as_float(b[j]);
    } else {
      const uint16_t h = (uint16_t)(b[j / 2] >> (16 * (j & 1)));
      T e;
      __builtin_memcpy(&e, &h, sizeof(T));
      x = sm_in(e);
    }
    return x == x ? fminf(x, FLT_MAX) : -INFINITY;
  }
};

template <typename T, int NT> constexpr int kSmTile = SmVec<T>::kN * NT;     // tokens of NT threads

// Keys order the logits; -0 is 0.
__device__ __forceinline__ uint32_t sm_key(float x) {
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
  float top, t;
  float half_top, bin_scale;              // half of the top; bins of half a logit's distance from it
  double c, scale;                        // log2(e) / T; 2^s
  float min_p;
  int k; float p;
  bool any, greedy, filter;
  int best_id;
};

template <typename A>
__device__ __forceinline__ SampleRow sm_row(const A& a, int64_t r, uint64_t best, float low) {
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
  w.t = t;
  w.c = 1.4426950408889634 / (double)t;
  w.scale = __builtin_bit_cast(double, (uint64_t)(1023 + a.bits) << 52);
  if (w.k >= a.V) w.k = 0;
  w.filter = w.any && !w.greedy && (w.k > 0 || w.p < 1.f || w.min_p > 0.f);
  // past (s + 1) ln 2 T from the top a weight is none
  // (halves: two logits may lie further apart than the largest number)
  w.half_top = 0.5f * w.top;
  const float range = fminf(fmaf(low, -0.5f, w.half_top), (float)(a.bits + 1) * 0.34657359f * t);
  w.bin_scale = range > 5e-31f ? (float)kSmBins / range : 2e-37f;
  return w;
}
// The best token of a row and its lowest logit, from its chunks: a lane each.
template <typename A>
__device__ __forceinline__ SampleRow sm_row_of(const A& a, int64_t r) {
  static_assert(kSmMaxChunks == 16, "four exchanges");
  const int lane = wave_lane();
  uint64_t best = 0;
  float low = INFINITY;
  if (lane < a.S) {
    best = a.best[r * a.S + lane];
    low = a.low[r * a.S + lane];
  }
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) {
    best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, m, kWave));
    low = fminf(low, __shfl_xor(low, m, kWave));
  }
  const uint32_t b0 = __builtin_amdgcn_readfirstlane((uint32_t)best);
  const uint32_t b1 = __builtin_amdgcn_readfirstlane((uint32_t)(best >> 32));
  return sm_row(a, r, (uint64_t)b1 << 32 | b0,
                __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(low))));
}

// exp((x - top) / T) = 2^y = 2^n 2^f with |f| <= 1/2, 2^f by the exponential's series up to the 11th power of
// f ln 2: the next term is below 6.4e-15, less than the half of 2^-46 that whole numbers are rounded by.  Masked: 2^-60.
__device__ __forceinline__ double sm_weight(const SampleRow& w, float x) {
  const double y = fmax(((double)x - (double)w.top) * w.c, -60.0);
  // y rounded to a whole number by adding 3 2^51, in whose last bits that then stands
  const double near = y + 6755399441055744.0;
  const double f = y - (near - 6755399441055744.0);
  constexpr double L = 0.69314718055994530942;
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6,
                   c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
  double s = fma(c11, f, c10);
  s = fma(s, f, c9);
  s = fma(s, f, c8);
  s = fma(s, f, c7);
  s = fma(s, f, c6);
  s = fma(s, f, c5);
  s = fma(s, f, c4);
  s = fma(s, f, c3);
  s = fma(s, f, c2);
  s = fma(s, f, L);
  s = fma(s, f, 1.0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, s);
  const uint32_t top = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, near) << 20);
  return __builtin_bit_cast(double, (uint64_t)top << 32 | (uint32_t)bits);
}
// The weight as a whole number of 2^-s, to the nearest: added to 2^52 it stands in the last bits.
__device__ __forceinline__ uint64_t sm_whole(const SampleRow& w, double e) {
  return __builtin_bit_cast(uint64_t, fma(e, w.scale, 4503599627370496.0)) - 0x4330000000000000ull;
}
// How far a logit lies below the top, in bins.
__device__ __forceinline__ float sm_below(const SampleRow& w, float x) {
  return fmaf(x, -0.5f, w.half_top) * w.bin_scale;
}
__device__ __forceinline__ int sm_bin(const SampleRow& w, float x) {
  return (int)fminf(sm_below(w, x), (float)(kSmBins - 1));
}

// Sum over the earlier ones of the work-group's first NT threads (of the others: nothing in particular);
// total: over all of them.
template <int NT>
__device__ __forceinline__ uint64_t sm_before(uint64_t v, uint64_t* sW, uint64_t& total) {
  const int lane = wave_lane(), wv = threadIdx.x / kWave;
  uint64_t x = v;
  __syncthreads();
  if (wv < NT / kWave) {
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) {
      const uint64_t y = __shfl_up(x, s, kWave);
      if (lane >= s) x += y;
    }
    if (lane == kWave - 1) sW[wv] = x;
  }
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / kWave; ++w) {
    if (w < wv) before += sW[w];
    total += sW[w];
  }
  return before + x - v;
}

// The best token and the lowest logit of a work-group's tokens, on every thread.
template <int NT>
__device__ __forceinline__ void sm_ends(float x, int id, float& low, uint64_t& best, uint64_t* sB, float* sL) {
  best = x > -INFINITY ? sm_place(sm_key(x), id) : 0;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, m, kWave));
    low = fminf(low, __shfl_xor(low, m, kWave));
  }
  if (wave_lane() == 0) { sB[threadIdx.x / kWave] = best; sL[threadIdx.x / kWave] = low; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / kWave; ++w) {
    best = max(best, sB[w]);
    low = fminf(low, sL[w]);
  }
}
__device__ __forceinline__ void sm_see(float x, int v, float& best, int& id, float& low) {
  if (x > best) { best = x; id = v; }
  low = x > -INFINITY ? fminf(low, x) : low;
}
// A token into the bins.
__device__ __forceinline__ void sm_count(const SampleRow& w, float x, uint32_t* sCnt, unsigned long long* sMass) {
  const uint64_t e = sm_whole(w, sm_weight(w, x));
  const int b = sm_bin(w, x);
  if (e == 0) return;
  atomicAdd(&sCnt[b], 1u);
  atomicAdd(&sMass[b], (unsigned long long)e);
}

struct SampleShared {
  uint64_t sW[kSmWide / kWave];
  float sL[kSmWide / kWave];
  uint32_t before[kSmBins + 1];           // tokens of the bins before
  uint64_t k_bin_mass;
  SampleState st;
  int at[2];
  int listed;
  unsigned long long ends[2];
  unsigned long long chunk[kSmMaxChunks];
  unsigned long long tile[kSmTiles];
  uint32_t cnt[kSmBins];
  unsigned long long mass[kSmBins];
  uint64_t list[kSmList];
  uint64_t whole[kSmCut];                 // a token of every step
};

// The row's borders as far as its bins tell, from the counts and weights in s.cnt and s.mass.  A thread adds up
// kSmBins / kSmSelect bins of its own, of the first kSmSelect threads.
constexpr int kSmSelect = 256;
__device__ __forceinline__ void sm_select(const SampleRow& w, SampleShared& s) {
  constexpr int PER = kSmBins / kSmSelect;
  const int tid = threadIdx.x;
  if (tid == 0) s.st = SampleState{0, 0, 0, 0, -1, -1, -1, kSmBins, kSmBins, 0};
  if (w.filter) {
    uint32_t cnt[PER], c = 0;
    uint64_t mass[PER], m = 0, live, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cnt[i] = tid < kSmSelect ? s.cnt[PER * tid + i] : 0;
      mass[i] = tid < kSmSelect ? s.mass[PER * tid + i] : 0;
      c += cnt[i];
      m += mass[i];
    }
    uint64_t cb = sm_before<kSmSelect>(c, s.sW, live), mb = sm_before<kSmSelect>(m, s.sW, all);
    const uint64_t mb0 = mb;
    const bool k_on = w.k > 0 && (uint64_t)w.k < live;
    if (tid == 0 && !k_on) s.st.k_whole = all;
    if (tid == 0) s.before[kSmBins] = (uint32_t)live;
    if (tid < kSmSelect) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        s.before[PER * tid + i] = (uint32_t)cb;
        if (k_on && cb < (uint64_t)w.k && cb + cnt[i] >= (uint64_t)w.k) {
          s.st.k_bin = PER * tid + i;
          s.st.k_count = (int)cb;
          s.st.k_mass = mb;
          s.k_bin_mass = mass[i];
          // (0: the k-th token is not its bin's last)
          s.st.k_whole = cb + cnt[i] == (uint64_t)w.k ? mb + mass[i] : 0;
        }
        cb += cnt[i];
        mb += mass[i];
      }
    }
    __syncthreads();
    const int kb = s.st.k_bin;
    const bool part = s.st.k_whole == 0;
    if (w.p < 1.f && tid < kSmSelect) {
      const double hi = (double)w.p * (double)(part ? s.st.k_mass + s.k_bin_mass : s.st.k_whole);
      const double lo = part ? (double)w.p * (double)s.st.k_mass : hi;
      mb = mb0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int b = PER * tid + i;
        if (mass[i] > 0) {
          // the bin in which the weight reaches p of the first k's, whatever that is between lo and hi
          if ((lo <= 0.0 && b == 0) || ((double)mb < lo && (double)(mb + mass[i]) >= lo)) {
            s.st.p_lo = b;
            s.st.p_mass = mb;
          }
          if ((hi <= 0.0 && b == 0) || ((double)mb < hi && (double)(mb + mass[i]) >= hi)) s.st.p_hi = b;
        }
        mb += mass[i];
      }
    }
    __syncthreads();
    if (tid == 0) {
      SampleState st = s.st;
      if (kb >= 0) {
        st.sure = part ? kb : kb + 1;
        st.end = kb + 1;
      }
      if (st.p_lo >= 0) {
        st.sure = min(st.sure, st.p_lo);
        st.end = min(st.end, st.p_hi + 1);
      }
      if (w.min_p > 0.f) {
        // where exp((x - M) / T) = min_p, and the bins beside it, for what the logarithm may be off by
        const float d = fminf(-logf(w.min_p) * (0.5f * w.t * w.bin_scale), (float)(kSmBins - 1));
        st.sure = min(st.sure, max((int)d - 1, 0));
        st.end = min(st.end, (int)d + 2);
      }
      if (s.before[st.end] <= (uint32_t)kSmFew) st.sure = 0;     // every token that may stay is listed
      int n = s.before[st.end] - s.before[min(st.sure, st.end)];
      if (part && kb >= st.end && st.p_lo >= 0 && st.p_lo < st.end) n += s.before[kb + 1] - s.before[kb];
      st.listed = n <= kSmList ? n : -1;
      s.st = st;
    }
  }
  __syncthreads();
}
// The k-th token lies within a bin; and is to be looked for (for itself or for the border of p).
__device__ __forceinline__ bool sm_seeks_k(const SampleState& st) {
  return st.k_bin >= 0 && st.k_whole == 0 && (st.k_bin < st.end || (st.p_lo >= 0 && st.p_lo < st.end));
}

// The bins' borders as they compare with sm_below: a masked token (inf) lies in none.
struct SampleGate { float sure, end, k0, k1; };
__device__ __forceinline__ SampleGate sm_gate(const SampleState& st) {
  auto edge = [](int b) { return b >= kSmBins ? INFINITY : (float)b; };
  const bool k = sm_seeks_k(st);
  return SampleGate{edge(st.sure), edge(st.end), k ? edge(st.k_bin) : INFINITY, k ? edge(st.k_bin + 1) : 0.f};
}
// A token into the list, if it is to be looked at.
__device__ __forceinline__ void sm_take(const SampleRow& w, const SampleGate& g, float x, int v, uint64_t* list,
                                        int* listed) {
  const float t = sm_below(w, x);
  if (!((t >= g.sure && t < g.end) || (t >= g.k0 && t < g.k1))) return;
  if (sm_whole(w, sm_weight(w, x)) == 0) return;
  const int at = atomicAdd(listed, 1);
  if (at < kSmList) list[at] = sm_place(sm_key(x), v);
}
// Adds `sum` over the wavefront to another.
__device__ __forceinline__ void sm_add(uint64_t sum, unsigned long long* to) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor((unsigned long long)sum, m, kWave);
  if (wave_lane() == 0 && sum > 0) atomicAdd(to, (unsigned long long)sum);
}

// A row, in memory or (HELD) in LDS as well, a vector after the other.
template <typename T, bool HELD>
struct SmSrc {
  const T* row;
  const uint4* held;
  __device__ __forceinline__ SmVec<T> at(int v, int v1) const {
    SmVec<T> x;
    if (HELD) {
      x.b = __builtin_bit_cast(typename SmVec<T>::V, held[v / SmVec<T>::kN]);
    } else {
      x.load(row, v, v1);
    }
    return x;
  }
};
// f(vector, first id) of this thread's vectors of v0 .. v1 - 1, two in flight from memory.
template <int NT, typename T, bool HELD, typename F>
__device__ __forceinline__ void sm_vectors(const SmSrc<T, HELD>& src, int v0, int v1, F f) {
  constexpr int E = SmVec<T>::kN, tile = kSmTile<T, NT>;
  if (HELD) {
#pragma unroll 1
    for (int v = v0 + E * threadIdx.x; v < v1; v += tile) f(src.at(v, v1), v);
    return;
  }
  for (int v = v0 + E * threadIdx.x; v < v1; v += 2 * tile) {
    const SmVec<T> x = src.at(v, v1), y = src.at(v + tile, v1);
    f(x, v);
    if (v + tile < v1) f(y, v + tile);
  }
}
// f(logit, id) of the tokens.
template <int NT, typename T, bool HELD, typename F>
__device__ __forceinline__ void sm_tokens(const SmSrc<T, HELD>& src, int v0, int v1, F f) {
  sm_vectors<NT>(src, v0, v1, [&](const SmVec<T>& x, int v) {
#pragma unroll
    for (int j = 0; j < SmVec<T>::kN; ++j) f(x.at(j), v + j);
  });
}

// f(place, weight) of the row's tokens of bins b0 .. b1 - 1.
template <int NT, typename T, bool HELD, typename F>
__device__ __forceinline__ void sm_of_row(const SampleRow& w, const SmSrc<T, HELD>& row, int V, int b0, int b1, F f) {
  sm_tokens<NT>(row, 0, V, [&](float x, int v) {
    const int b = sm_bin(w, x);
    if (b < b0 || b >= b1) return;
    const uint64_t e = sm_whole(w, sm_weight(w, x));
    if (e > 0) f(sm_place(sm_key(x), v), e);
  });
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ uint64_t sB[kSmThreads / kWave];
  __shared__ float sL[kSmThreads / kWave];
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x, tid = threadIdx.x;
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  const SmSrc<T, false> row = {(const T*)a.x + r * a.x_st, nullptr};
  uint64_t best;
  float top = -INFINITY, low = INFINITY;
  int id = 0;
  sm_tokens<kSmThreads>(row, v0, v1, [&](float x, int v) { sm_see(x, v, top, id, low); });
  sm_ends<kSmThreads>(top, id, low, best, sB, sL);
  if (tid == 0) {
    a.best[r * a.S + c] = best;
    a.low[r * a.S + c] = low;
  }
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_bins_kernel(SampleArgs a) {
  __shared__ uint32_t sCnt[kSmBins];
  __shared__ unsigned long long sMass[kSmBins];
  const int64_t r = blockIdx.y;
  const SampleRow w = sm_row_of(a, r);
  if (!w.any || w.greedy) return;
  const int c = blockIdx.x, tid = threadIdx.x;
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  const SmSrc<T, false> row = {(const T*)a.x + r * a.x_st, nullptr};
  for (int b = tid; b < kSmBins; b += kSmThreads) { sCnt[b] = 0; sMass[b] = 0; }
  __syncthreads();
  uint64_t sum = 0;
  if (w.filter)
    sm_tokens<kSmThreads>(row, v0, v1, [&](float x, int) { sm_count(w, x, sCnt, sMass); });
  else
    sm_tokens<kSmThreads>(row, v0, v1, [&](float x, int) { sum += sm_whole(w, sm_weight(w, x)); });
  if (!w.filter) sm_add(sum, &sMass[0]);
  __syncthreads();
  const int64_t at = (r * a.S + c) * kSmBins;
  for (int b = tid; b < kSmBins; b += kSmThreads) {
    a.cnt[at + b] = sCnt[b];
    a.mass[at + b] = sMass[b];
  }
}

__global__ __launch_bounds__(kSmBins) void sample_select_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const SampleRow w = sm_row_of(a, r);
  if (!w.any || w.greedy) return;
  const uint32_t* cnts = a.cnt + r * a.S * kSmBins + tid;
  const uint64_t* masses = a.mass + r * a.S * kSmBins + tid;
  uint32_t cnt = 0;
  uint64_t mass = 0;
  if (w.filter) {
    uint32_t c[kSmMaxChunks];
    uint64_t m[kSmMaxChunks];
#pragma unroll
    for (int i = 0; i < kSmMaxChunks; ++i) {         // (every load before the first sum)
      c[i] = cnts[min(i, a.S - 1) * kSmBins];
      m[i] = masses[min(i, a.S - 1) * kSmBins];
    }
#pragma unroll
    for (int i = 0; i < kSmMaxChunks; ++i) {
      cnt += i < a.S ? c[i] : 0;
      mass += i < a.S ? m[i] : 0;
    }
  }
  s.cnt[tid] = cnt;
  s.mass[tid] = mass;
  __syncthreads();
  sm_select(w, s);
  if (tid == 0) {
    a.state[r] = s.st;
    a.n_list[r] = 0;
  }
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_pick_kernel(SampleArgs a) {
  __shared__ uint64_t sList[kSmList];
  __shared__ int sN, sAt;
  __shared__ unsigned long long sSum;
  const int64_t r = blockIdx.y;
  const SampleRow w = sm_row_of(a, r);
  if (!w.any || w.greedy) return;
  const SampleState st = a.state[r];
  const int c = blockIdx.x, tid = threadIdx.x;
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  if (tid == 0) { sN = 0; sSum = 0; }
  __syncthreads();
  uint64_t sum = 0;
  for (int b = tid; b < st.sure; b += kSmThreads) sum += a.mass[(r * a.S + c) * kSmBins + b];
  sm_add(sum, &sSum);
  const SampleGate g = sm_gate(st);
  const SmSrc<T, false> row = {(const T*)a.x + r * a.x_st, nullptr};
  if (st.listed > 0)
    sm_tokens<kSmThreads>(row, v0, v1, [&](float x, int v) { sm_take(w, g, x, v, sList, &sN); });
  __syncthreads();
  if (tid == 0) a.sure[r * a.S + c] = sSum;
  const int n = min(sN, kSmList);
  if (n == 0) return;
  if (tid == 0) sAt = atomicAdd(&a.n_list[r], n);
  __syncthreads();
  for (int i = tid; i < n; i += kSmThreads)
    if (sAt + i < kSmList) a.list[r * kSmList + sAt + i] = sList[i];
}

// The last token (by its place) of those in [lo, hi] that the rule keeps: with `need` > 0 the need-th,
// else the last whose predecessors' weight, `mass` of them outside, is below `target` (the first if none
// is).  for_each(f) calls f(place, weight) for the tokens of the source.  mass: with the token found added.
// A pass cuts [lo, hi] into kSmCut steps, which one wavefront adds up; at most eight passes, two for a list of a
// few hundred.
struct SampleCut { uint64_t place, mass; };
template <typename Each>
__device__ SampleCut sm_cut(Each for_each, int need, double target, uint64_t mass, uint64_t lo, uint64_t hi,
                            SampleShared& s) {
  const int tid = threadIdx.x, lane = wave_lane();
  constexpr int PER = kSmCut / kWave;
  uint64_t found = 0;                     // the weight of the token found
  for (;;) {
    // the ends of what there is: logits of 16 bits leave most of a range of places empty
    __syncthreads();
    if (tid == 0) { s.ends[0] = ~0ull; s.ends[1] = 0; }
    if (tid < kSmCut) { s.cnt[tid] = 0; s.mass[tid] = 0; }
    __syncthreads();
    {
      uint64_t mn = ~0ull, mx = 0;
      for_each([&](uint64_t place, uint64_t) {
        if (place < lo || place > hi) return;
        mn = min(mn, place);
        mx = max(mx, place);
      });
      if (__any(mx > 0)) {
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) {
          mn = min(mn, (uint64_t)__shfl_xor((unsigned long long)mn, m, kWave));
          mx = max(mx, (uint64_t)__shfl_xor((unsigned long long)mx, m, kWave));
        }
        if (lane == 0) { atomicMin(&s.ends[0], (unsigned long long)mn); atomicMax(&s.ends[1], (unsigned long long)mx); }
      }
    }
    __syncthreads();
    lo = s.ends[0];
    hi = s.ends[1];
    const uint64_t span = hi - lo;
    const int shift = span ? max(64 - (int)__clzll(span) - 8, 0) : 0;
    for_each([&](uint64_t place, uint64_t e) {
      if (place < lo || place > hi) return;
      const int b = (int)((hi - place) >> shift);
      atomicAdd(&s.cnt[b], 1u);
      atomicAdd(&s.mass[b], (unsigned long long)e);
      s.whole[b] = place;                 // (of a step of one token: that token)
    });
    __syncthreads();
    if (tid < kWave) {
      uint32_t cnt[PER], c = 0;
      uint64_t m[PER], x = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        cnt[i] = s.cnt[PER * lane + i];
        m[i] = s.mass[PER * lane + i];
        c += cnt[i];
        x += m[i];
      }
      uint32_t cb = c;
      uint64_t mb = x;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t yc = __shfl_up(cb, d, kWave);
        const uint64_t ym = __shfl_up((unsigned long long)mb, d, kWave);
        if (lane >= d) { cb += yc; mb += ym; }
      }
      cb -= c;
      mb += mass - x;
      // the last step that has a kept token
      int at = -1;
      uint32_t at_c = 0;
      uint64_t at_m = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (cnt[i] > 0 && (need > 0 ? cb < (uint32_t)need : cb == 0 || (double)mb < target)) {
          at = PER * lane + i;
          at_c = cb;
          at_m = mb;
        }
        cb += cnt[i];
        mb += m[i];
      }
      const uint64_t some = __ballot(at >= 0);
      if (some ? lane == 63 - (int)__clzll(some) : lane == 0) {
        s.at[0] = max(at, 0);
        s.at[1] = (int)at_c;
        s.ends[0] = at_m;
      }
    }
    __syncthreads();
    const int b = s.at[0];
    if (need > 0) need -= s.at[1];
    mass = s.ends[0];
    found = s.mass[b];
    if (shift == 0 || s.cnt[b] <= 1) {    // one token
      hi = s.cnt[b] == 1 ? s.whole[b] : hi - (uint64_t)b;
      break;
    }
    hi -= (uint64_t)b << shift;
    const uint64_t width = (1ull << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
  }
  __syncthreads();
  return SampleCut{hi, mass + found};
}

// The last place that stays (0: every one of the bins before `end`) from the source's tokens.
template <typename Each>
__device__ __forceinline__ uint64_t sm_borders(const SampleRow& w, const SampleState& st, Each tokens,
                                               SampleShared& s) {
  uint64_t last = 0, k_mass = st.k_whole;
  if (sm_seeks_k(st)) {
    const SampleCut z = sm_cut([&](auto f) { tokens(st.k_bin, st.k_bin + 1, f); }, w.k - st.k_count, 0.0, st.k_mass,
                               0, ~0ull, s);
    last = z.place;
    k_mass = z.mass;
  }
  if (st.p_lo >= 0 && st.p_lo < st.end)
    last = max(last, sm_cut([&](auto f) { tokens(st.p_lo, st.end, f); }, 0, (double)w.p * (double)k_mass, st.p_mass,
                            last, ~0ull, s).place);
  return last;
}

// The first (u below 1) or last of `n` weights' sums that exceeds `want`; the sum of those before it.
template <int NT>
__device__ __forceinline__ int sm_find(uint64_t mine, uint64_t ahead, double want, SampleShared& s,
                                       uint64_t& before) {
  const int tid = threadIdx.x;
  uint64_t total;
  ahead += sm_before<NT>(mine, s.sW, total);
  if (tid == 0) { s.at[0] = INT32_MAX; s.at[1] = 0; }
  __syncthreads();
  if (mine > 0) {
    if ((double)(ahead + mine) > want) atomicMin(&s.at[0], tid);
    atomicMax(&s.at[1], tid);
  }
  __syncthreads();
  const int t = s.at[0] == INT32_MAX ? s.at[1] : s.at[0];
  if (tid == t) s.ends[0] = ahead;
  __syncthreads();
  before = s.ends[0];
  return t;
}

// The token of v0 .. v1 - 1 that `want` falls into; `ahead` lies before.  The tile first, then its thread.
template <int NT, typename T, bool HELD, typename Stays>
__device__ __forceinline__ int sm_draw(const SampleRow& w, const SmSrc<T, HELD>& row, double want, uint64_t ahead,
                                       int v0, int v1, SampleShared& s, Stays stays) {
  const int tid = threadIdx.x;
  constexpr int E = SmVec<T>::kN;
  const int nt = (v1 - v0 + kSmTile<T, NT> - 1) / kSmTile<T, NT>;
  int t = 0;
  if (nt > 1) {
    for (int i = tid; i < nt; i += NT) s.tile[i] = 0;
    __syncthreads();
    for (int i = 0; i < nt; i += 2) {
      const int v = v0 + i * kSmTile<T, NT> + E * tid, u = v + kSmTile<T, NT>;
      SmVec<T> x, y;
      if (v < v1) x = row.at(v, v1);
      if (u < v1) y = row.at(u, v1);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < E; ++j) {
        double f;
        if (v < v1 && stays(x.at(j), v + j, f)) sum[0] += sm_whole(w, f);
        if (u < v1 && stays(y.at(j), u + j, f)) sum[1] += sm_whole(w, f);
      }
      if (__any(sum[0] > 0)) sm_add(sum[0], &s.tile[i]);
      if (__any(sum[1] > 0)) sm_add(sum[1], &s.tile[i + 1]);
    }
    __syncthreads();
    uint64_t before;
    t = sm_find<NT>(tid < nt ? s.tile[tid] : 0, ahead, want, s, before);
    ahead = before;
  }
  const int v = v0 + t * kSmTile<T, NT> + E * tid;
  SmVec<T> x;
  if (v < v1) x = row.at(v, v1);
  uint64_t e[E], sum = 0, before;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    double f;
    e[j] = v < v1 && stays(x.at(j), v + j, f) ? sm_whole(w, f) : 0;
    sum += e[j];
  }
  const int th = sm_find<NT>(sum, ahead, want, s, before);
  if (tid == th) {
    uint64_t run = before;
    int first = -1, last = v;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      run += e[j];
      if (e[j] > 0) {
        if (first < 0 && (double)run > want) first = v + j;
        last = v + j;
      }
    }
    s.at[1] = first < 0 ? last : first;
  }
  __syncthreads();
  return s.at[1];
}

__device__ __forceinline__ void sm_put(void* probs, int type, int64_t at, float x) {
  if (type == 0) ((float*)probs)[at] = x;
  else if (type == 1) sm_out(x, ((bf16*)probs)[at]);
  else sm_out(x, ((__half*)probs)[at]);
}
// kN probabilities from v on, in whole vectors at any element's boundary.
template <int N, typename P>
__device__ __forceinline__ void sm_put_all(P* to, const float* x) {
  typedef uint32_t V __attribute__((ext_vector_type(N * sizeof(P) >= 16 ? 4 : 2), aligned(2)));
  constexpr int PER = sizeof(V) / sizeof(P);
#pragma unroll
  for (int j = 0; j < N; j += PER) {
    P e[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) sm_out(x[j + i], e[i]);
    V b;
    __builtin_memcpy(&b, e, sizeof(V));
    *(V*)(to + j) = b;
  }
}
template <typename T>
__device__ __forceinline__ void sm_put_vec(const SampleArgs& a, int64_t r, int v, int v1, const float* x) {
  constexpr int E = SmVec<T>::kN;
  const int64_t at = r * a.p_st + v;
  if (v + E <= v1) {
    if (a.p_type == 0) sm_put_all<E>((float*)a.probs + at, x);
    else if (a.p_type == 1) sm_put_all<E>((bf16*)a.probs + at, x);
    else sm_put_all<E>((__half*)a.probs + at, x);
    return;
  }
#pragma unroll
  for (int j = 0; j < E; ++j)
    if (v + j < v1) sm_put(a.probs, a.p_type, at + j, x[j]);
}

// Whether a token stays, and its weight.
__device__ __forceinline__ bool sm_stays(const SampleRow& w, const SampleGate& g, uint64_t last, float x, int v,
                                         double& e) {
  const float t = sm_below(w, x);
  if (t >= g.end || (t >= g.sure && sm_place(sm_key(x), v) < last)) return false;
  e = sm_weight(w, x);
  return e >= (double)w.min_p;
}
// What a greedy row, or one without any token, gives.
template <int NT>
__device__ __forceinline__ void sm_one(const SampleArgs& a, const SampleRow& w, int64_t r, int c, int v0, int v1) {
  if (c == 0 && threadIdx.x == 0 && a.token) a.token[r] = w.any ? w.best_id : -1;
  if (a.probs)
    for (int v = v0 + threadIdx.x; v < v1; v += NT)
      sm_put(a.probs, a.p_type, r * a.p_st + v, w.any && v == w.best_id ? 1.f : 0.f);
}
// u times the whole.  A number of 1 is exceeded by no running sum: the last token that stays.
__device__ __forceinline__ double sm_want(float u, uint64_t total) {
  u = fmaxf(u, 0.f);
  return u < 1.f ? (double)u * (double)total : (double)INFINITY;
}
// f(place, weight) of the listed tokens of bins b0 .. b1 - 1; their weights in listw, where there is room for them.
template <typename F>
__device__ __forceinline__ void sm_listed(const SampleRow& w, int n, int b0, int b1, const SampleShared& s,
                                          const uint64_t* listw, F f) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t place = s.list[i];
    const float x = sm_logit((uint32_t)(place >> 32));
    const int b = sm_bin(w, x);
    if (b >= b0 && b < b1) f(place, listw ? listw[i] : sm_whole(w, sm_weight(w, x)));
  }
}

// The probabilities of tokens v0 .. v1 - 1.
template <int NT, typename T, bool HELD, typename Stays>
__device__ __forceinline__ void sm_probs(const SampleArgs& a, const SampleRow& w, const SmSrc<T, HELD>& row,
                                         int64_t r, int v0, int v1, uint64_t total, Stays stays) {
  constexpr int E = SmVec<T>::kN;
  const double inv = w.scale / (double)total;
  sm_vectors<NT>(row, v0, v1, [&](const SmVec<T>& x, int v) {
    float p[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      double e;
      p[j] = stays(x.at(j), v + j, e) && sm_whole(w, e) > 0 ? (float)(e * inv) : 0.f;
    }
    sm_put_vec<T>(a, r, v, v1, p);
  });
}

// Every token that may stay is listed: the weight of those that do, and the token that u draws, by their ids as places.
__device__ __forceinline__ uint64_t sm_few(const SampleArgs& a, const SampleRow& w, const SampleState& st,
                                           uint64_t last, int64_t r, bool draw, const uint64_t* listw,
                                           SampleShared& s) {
  auto stay = [&](auto f) {
    sm_listed(w, st.listed, 0, st.end, s, listw, [&](uint64_t place, uint64_t e) {
      if (place >= last && (!(w.min_p > 0.f) || sm_weight(w, sm_logit((uint32_t)(place >> 32))) >= (double)w.min_p))
        f((uint64_t)(uint32_t)place, e);
    });
  };
  __syncthreads();
  if (threadIdx.x == 0) s.chunk[0] = 0;
  __syncthreads();
  stay([&](uint64_t, uint64_t e) { atomicAdd(&s.chunk[0], (unsigned long long)e); });
  __syncthreads();
  const uint64_t total = s.chunk[0];
  if (draw && a.u) {
    // the first whose sum exceeds u times the whole is the last whose predecessors' sum does not
    const double want = sm_want(a.u[r], total);
    const SampleCut z = sm_cut(stay, 0, nextafter(want, (double)INFINITY), 0, 0, ~0ull, s);
    if (threadIdx.x == 0) a.token[r] = (int)~(uint32_t)z.place;
  }
  return total;
}

// NT: kSmWide threads where a row's one work-group draws (64 rows: 27 us, kSmThreads 33), kSmThreads where every chunk's
// has probabilities to write (each finds the borders by itself; 48 rows: 35.8 us, kSmWide 38, a launch of their own for
// them 36.5).
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_draw_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  __shared__ uint64_t sListw[kSmList];
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x, tid = threadIdx.x;
  const SampleRow w = sm_row_of(a, r);
  const int v0 = c * a.chunk, v1 = min(a.V, v0 + a.chunk);
  if (!w.any || w.greedy) {
    sm_one<NT>(a, w, r, c, v0, v1);
    return;
  }
  const SmSrc<T, false> row = {(const T*)a.x + r * a.x_st, nullptr};
  const SampleState st = a.state[r];
  for (int i = tid; i < st.listed; i += NT) {
    s.list[i] = a.list[r * kSmList + i];
    sListw[i] = sm_whole(w, sm_weight(w, sm_logit((uint32_t)(s.list[i] >> 32))));
  }
  if (tid < a.S) s.chunk[tid] = a.sure[r * a.S + tid];
  __syncthreads();
  const SampleGate g = sm_gate(st);
  uint64_t last = 0, total = 0;
  auto stays = [&](float x, int v, double& e) { return sm_stays(w, g, last, x, v, e); };
  auto listed = [&](int b0, int b1, auto f) { sm_listed(w, st.listed, b0, b1, s, sListw, f); };
  if (st.sure == 0 && st.listed > 0) {
    last = sm_borders(w, st, listed, s);
    total = sm_few(a, w, st, last, r, c == 0, sListw, s);
    if (a.probs) sm_probs<NT>(a, w, row, r, v0, v1, total, stays);
    return;
  }
  auto finish = [&](auto tokens) {
    last = sm_borders(w, st, tokens, s);
    tokens(st.sure, st.end, [&](uint64_t place, uint64_t e) {
      if (place >= last && sm_weight(w, sm_logit((uint32_t)(place >> 32))) >= (double)w.min_p)
        atomicAdd(&s.chunk[(int)~(uint32_t)place / a.chunk], (unsigned long long)e);
    });
    __syncthreads();
  };
  if (st.listed > 0)
    finish(listed);
  else if (st.listed < 0)
    finish([&](int b0, int b1, auto f) { sm_of_row<NT>(w, row, a.V, b0, b1, f); });
  for (int i = 0; i < a.S; ++i) total += s.chunk[i];
  if (c == 0 && a.u) {
    const double want = sm_want(a.u[r], total);
    int at = -1, any = 0;
    uint64_t run = 0, ahead = 0, any_ahead = 0;
    for (int i = 0; i < a.S; ++i) {
      const uint64_t e = s.chunk[i];
      if (e > 0) {
        any = i;
        any_ahead = run;
        if (at < 0 && (double)(run + e) > want) {
          at = i;
          ahead = run;
        }
      }
      run += e;
    }
    if (at < 0) {
      at = any;
      ahead = any_ahead;
    }
    const int d0 = at * a.chunk, d1 = min(a.V, d0 + a.chunk);
    const int token = sm_draw<NT>(w, row, want, ahead, d0, d1, s, stays);
    if (tid == 0) a.token[r] = token;
  }
  if (a.probs) sm_probs<NT>(a, w, row, r, v0, v1, total, stays);
}

// The same, a work-group a row.  A short row stays in LDS (HELD): one CU takes 5 us to read 128 KB, from the L2
// too, and four of the five steps read the row.  The room is a row of kSmShort tokens' however short the row is, so that
// a CU takes one at a time: 256 rows of 32,000 fp32 42 us (top-k and top-p), 2,048 of 4,096 160.
template <typename T, bool HELD>
__global__ __launch_bounds__(kSmWide) void sample_row_kernel(SampleArgs a) {
  constexpr int NT = kSmWide, E = SmVec<T>::kN, VECS = HELD ? kSmShort / E : 1;
  __shared__ SampleShared s;
  __shared__ uint4 sRow[VECS];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const SmSrc<T, HELD> row = {(const T*)a.x + r * a.x_st, sRow};
  if constexpr (HELD) {
    SmVec<T> x[VECS / NT];
#pragma unroll
    for (int n = 0; n < VECS / NT; ++n) x[n].load(row.row, E * (n * NT + tid), a.V);
#pragma unroll
    for (int n = 0; n < VECS / NT; ++n) sRow[n * NT + tid] = __builtin_bit_cast(uint4, x[n].b);
  }
  if (tid < kSmBins) { s.cnt[tid] = 0; s.mass[tid] = 0; }
  if (tid == 0) { s.listed = 0; s.chunk[0] = 0; }
  uint64_t best;
  float top = -INFINITY, low = INFINITY;
  int id = 0;
  sm_tokens<NT>(row, 0, a.V, [&](float x, int v) { sm_see(x, v, top, id, low); });
  sm_ends<NT>(top, id, low, best, s.sW, s.sL);
  const SampleRow w = sm_row(a, r, best, low);
  if (!w.any || w.greedy) {
    sm_one<NT>(a, w, r, 0, 0, a.V);
    return;
  }
  uint64_t sum = 0;
  if (w.filter)
    sm_tokens<NT>(row, 0, a.V, [&](float x, int) { sm_count(w, x, s.cnt, s.mass); });
  else
    sm_tokens<NT>(row, 0, a.V, [&](float x, int) { sum += sm_whole(w, sm_weight(w, x)); });
  __syncthreads();
  const uint64_t mass = tid < kSmBins ? s.mass[tid] : 0;
  sm_select(w, s);
  const SampleState st = s.st;
  const SampleGate g = sm_gate(st);
  sm_add(!w.filter ? sum : tid < st.sure ? mass : 0, &s.chunk[0]);
  uint64_t last = 0;
  auto stays = [&](float l, int v, double& e) { return sm_stays(w, g, last, l, v, e); };
  auto finish = [&](auto tokens) {
    last = sm_borders(w, st, tokens, s);
    tokens(st.sure, st.end, [&](uint64_t place, uint64_t e) {
      if (place >= last && sm_weight(w, sm_logit((uint32_t)(place >> 32))) >= (double)w.min_p)
        atomicAdd(&s.chunk[0], (unsigned long long)e);
    });
  };
  if (st.listed > 0) {
    sm_tokens<NT>(row, 0, a.V, [&](float x, int v) { sm_take(w, g, x, v, s.list, &s.listed); });
    __syncthreads();
    auto listed = [&](int b0, int b1, auto f) { sm_listed(w, st.listed, b0, b1, s, nullptr, f); };
    if (st.sure == 0) {
      last = sm_borders(w, st, listed, s);
      const uint64_t whole = sm_few(a, w, st, last, r, true, nullptr, s);
      if (a.probs) sm_probs<NT>(a, w, row, r, 0, a.V, whole, stays);
      return;
    }
    finish(listed);
  } else if (st.listed < 0) {
    finish([&](int b0, int b1, auto f) { sm_of_row<NT>(w, row, a.V, b0, b1, f); });
  }
  __syncthreads();
  const uint64_t total = s.chunk[0];
  if (a.u) {
    const int token = sm_draw<NT>(w, row, sm_want(a.u[r], total), 0, 0, a.V, s, stays);
    if (tid == 0) a.token[r] = token;
  }
  if (a.probs) sm_probs<NT>(a, w, row, r, 0, a.V, total, stays);
}

// Rows of up to kSmShort tokens, and batches of kSmMany rows and more, take a work-group a row.
static bool sample_whole(int64_t R, int V) { return V <= kSmShort || R >= kSmMany; }

// Chunks of a row: work-groups for four a CU in all (two: 78 us where four take 69), a tile each at least.
struct SampleLayout {
  int S, chunk;
  int64_t best, low, cnt, mass, state, n_list, list, sure, total;
};
static SampleLayout sample_layout(int64_t R, int V, int tile) {
  SampleLayout L = {};
  if (R == 0 || sample_whole(R, V)) return L;
  const int64_t want = std::min<int64_t>(kSmMaxChunks, 1024 / R);
  static_assert(kSmMaxV / (1024 / kSmMany) <= kSmTiles * kSmTile<float, kSmThreads> && kSmTiles <= kSmThreads,
                "a chunk's tiles, a thread each");
  L.chunk = (int)(((V + want - 1) / want + tile - 1) / tile * tile);
  L.S = (V + L.chunk - 1) / L.chunk;
  auto align = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t o = 0;
  L.best = o; o = align(o + R * L.S * 8);
  L.low = o; o = align(o + R * L.S * 4);
  L.cnt = o; o = align(o + R * L.S * kSmBins * 4);
  L.mass = o; o = align(o + R * L.S * kSmBins * 8);
  L.state = o; o = align(o + R * (int64_t)sizeof(SampleState));
  L.n_list = o; o = align(o + R * 4);
  L.list = o; o = align(o + R * kSmList * 8);
  L.sure = o; o = align(o + R * L.S * 8);
  L.total = o;
  return L;
}

template <typename T>
static void sample_launch(const SampleArgs& a, int64_t R, hipStream_t st) {
  const dim3 block(kSmThreads);
  if (sample_whole(R, a.V)) {
    const dim3 grid((unsigned)R), wide(kSmWide);
    if (a.V <= kSmShort) hipLaunchKernelGGL((sample_row_kernel<T, true>), grid, wide, 0, st, a);
    else hipLaunchKernelGGL((sample_row_kernel<T, false>), grid, wide, 0, st, a);
    return;
  }
  const dim3 grid(a.S, (unsigned)R);
  hipLaunchKernelGGL(sample_max_kernel<T>, grid, block, 0, st, a);
  hipLaunchKernelGGL(sample_bins_kernel<T>, grid, block, 0, st, a);
  hipLaunchKernelGGL(sample_select_kernel, dim3((unsigned)R), dim3(kSmBins), 0, st, a);
  hipLaunchKernelGGL(sample_pick_kernel<T>, grid, block, 0, st, a);
  if (a.probs) hipLaunchKernelGGL((sample_draw_kernel<T, kSmThreads>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((sample_draw_kernel<T, kSmWide>), dim3(1, (unsigned)R), dim3(kSmWide), 0, st, a);
}

}  // namespace dash

extern "C" int dash_sample_workspace_size(int64_t R, int V, int64_t* bytes) {
  using namespace dash;
  if (!bytes || R < 0 || V <= 0) return kErrInvalid;
  if (V > kSmMaxV) return kErrUnsupported;
  *bytes = std::max(sample_layout(R, V, kSmTile<float, kSmThreads>).total,
                    sample_layout(R, V, kSmTile<bf16, kSmThreads>).total);
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
  if (V > kSmMaxV || !fits_grid(R, kSmWide)) return kErrUnsupported;
  const SampleLayout L = sample_layout(R, V, dtype == 0 ? kSmTile<float, kSmThreads> : kSmTile<bf16, kSmThreads>);
  if (L.total > 0 && (!workspace || workspace_bytes < L.total || (uintptr_t)workspace % 256 != 0))
    return kErrWorkspace;
  char* ws = (char*)workspace;
  hipStream_t st = (hipStream_t)stream;
  SampleArgs a = {};
  a.x = logits; a.x_st = row_stride; a.u = uniforms;
  a.t = temperature; a.t0 = temperature0; a.k = top_k; a.k0 = top_k0;
  a.p = top_p; a.p0 = top_p0; a.m = min_p; a.m0 = min_p0;
  a.V = V; a.S = L.S; a.chunk = L.chunk;
  int log = 0;
  while ((1 << log) < V) ++log;
  a.bits = std::min(51, 62 - log);
  a.token = tokens; a.probs = probs; a.p_type = probs_dtype; a.p_st = probs_stride;
  a.best = (uint64_t*)(ws + L.best); a.low = (float*)(ws + L.low);
  a.cnt = (uint32_t*)(ws + L.cnt); a.mass = (uint64_t*)(ws + L.mass);
  a.state = (SampleState*)(ws + L.state); a.n_list = (int32_t*)(ws + L.n_list);
  a.list = (uint64_t*)(ws + L.list); a.sure = (uint64_t*)(ws + L.sure);
  if (dtype == 0) sample_launch<float>(a, R, st);
  else if (dtype == 1) sample_launch<bf16>(a, R, st);
  else sample_launch<__half>(a, R, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
