// Rotary positions on gfx950: a part [start, start + 2 m) of every head row is turned by angles
// pos * inv_freq[j], alone (queries, keys, their gradients) or as the keys and values are written to a
// paged cache.
//
// Pair j of a row is (x_j, x_{j + m}) of the part (halves) or (x_2j, x_{2j+1}) (interleaved), and
//   (x, y) -> (x c - y s, y c + x s),   c = f cos(pos * inv_freq[j]), s = f sin(pos * inv_freq[j]).
// The map's transpose is the turn by -pos with the same factor f, which is the gradient's.
//
// The angle is a product in 64 bits: a position of 10^5 has 10^5 radians, whose 32-bit rounding alone is 4e-3.  Its
// sine and cosine are series in 64 bits, good to 1.2e-10 (33 bits, beside the 24 that they are rounded to), once a
// (token, pair), in LDS, for all heads; the turn is two products and an addition in 32 bits, rounded once to the row's
// type.
//
// A work-group takes a token, or a few of few heads, and all its heads.  Its units are two 16-byte chunks: the two
// that a pair of the halves' layout needs, or two neighbours (single elements where an address, a stride or the
// part does not fit 16 bytes).  Their loads start before the sines are there.
//
// Bound by HBM: 8,190 tokens of 10 + 10 + 10 heads of 128 bf16 in 38 us (126 MB read and written, 3.3 TB/s), 20 heads
// turned as interleaved pairs 30.6 us (84 MB, 2.7 TB/s); replayed over the same rows, which the last cache then holds, 31
// and 21.2.  With two or four units a thread in flight, or loads and stores past the caches, 40 to 46 and (replayed) 25 to
// 33.  Six wavefronts a SIMD: 38 us, five 44, eight (registers to memory) 46; replayed, seven 31.2, six 32.7.
// A few tokens 4 us, of latency.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "dash_common.h"

namespace dash {

constexpr int kRpThreads = 256;
constexpr int kRpTokens = 4;        // of a work-group, at most
constexpr int kRpMaxPairs = 256;

struct RopeRows {                   // rows [B, S, heads, D] in elements; slots: y is a cache of pages
  const void* x; int64_t x_sb, x_st, x_sh;
  void* y; int64_t y_sb, y_st, y_sh;       // slots: y_sb the page's stride
  int heads;
  int turn;                         // 0: copied
  int slots;                        // written at the token's slot
};
struct RopeArgs {
  RopeRows r[3];
  int n, heads;                     // row sets and their heads
  const void* pos; int pos64; int64_t pos_sb, pos_st;
  const double* inv_freq;
  double sign, factor;
  const int64_t* slots; int page; int64_t num_slots;
  int B, S, D, m, start;
  int units;                        // of a head row
  int per;                          // tokens of a work-group
};

template <typename T, int E> struct RopeChunk {
  typedef uint32_t V __attribute__((ext_vector_type(E * sizeof(T) / 4)));
  union { V v; T e[E]; };
};
template <typename T> struct RopeChunk<T, 1> {
  typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type V;
  union { V v; T e[1]; };
};
__device__ __forceinline__ float rp_in(float x) { return x; }
__device__ __forceinline__ float rp_in(bf16 x) { return (float)x; }
__device__ __forceinline__ float rp_in(__half x) { return __half2float(x); }
__device__ __forceinline__ void rp_out(float x, float& y) { y = x; }
__device__ __forceinline__ void rp_out(float x, bf16& y) { y = (bf16)x; }
__device__ __forceinline__ void rp_out(float x, __half& y) { y = __float2half_rn(x); }

// factor (cos, sin) of pos * f.  In turns: pos f / (2 pi) = pos (g + h) with g + h = f / (2 pi) to twice the digits.
// Its whole part goes within one fused step, before anything is rounded (the product and its rounding apart, as two
// terms of a sum, were fused by the compiler, which counted the rounding twice: a position of 2^31 was off by 2e-7, one
// of 2^47 by 5e-3).  Then the nearest quarter turn, and the series of sine and cosine on [-pi / 4, pi / 4], whose next
// terms are below 1.2e-10.
__device__ __forceinline__ float2 rp_turn(double pos, double f, double factor) {
  constexpr double c0 = 0.15915494309189535, c1 = -9.839338337591243e-18;   // 1 / (2 pi)
  const double g = f * c0, h = fma(f, c0, -g) + f * c1;
  const double r = fma(pos, h, fma(pos, g, -__builtin_rint(pos * g)));
  const double q = __builtin_rint(4.0 * r);
  const double x = fma(q, -0.25, r) * 6.283185307179586, y = x * x;
  double k3 = -1.0 / 6.0, k5 = 1.0 / 120.0, k7 = -1.0 / 5040.0, k9 = 1.0 / 362880.0;
  asm("" : "+s"(k3), "+s"(k5), "+s"(k7), "+s"(k9));      // (in vector registers they would be spilled)
  double s = fma(y, -1.0 / 39916800.0, k9);
  s = fma(s, y, k7);
  s = fma(s, y, k5);
  s = fma(s, y, k3);
  s = fma(s * y, x, x);
  double c = fma(y, -1.0 / 3628800.0, 1.0 / 40320.0);
  c = fma(c, y, -1.0 / 720.0);
  c = fma(c, y, 1.0 / 24.0);
  c = fma(c, y, -0.5);
  c = fma(c, y, 1.0);
  const int k = (int)q & 3;
  const double u = k & 1 ? s : c, v = k & 1 ? c : s;
  return make_float2((float)((k == 1 || k == 2 ? -u : u) * factor), (float)((k & 2 ? -v : v) * factor));
}

template <typename T, int E, bool PAIRS>
__global__ __launch_bounds__(kRpThreads, 7) void rope_kernel(RopeArgs a) {
  typedef typename std::remove_reference<decltype(RopeChunk<T, E>::v)>::type V;
  __shared__ float2 sCs[kRpTokens * kRpMaxPairs];
  __shared__ int64_t sSlot[kRpTokens];
  const int tid = threadIdx.x;
  const int64_t tokens = (int64_t)a.B * a.S, t0 = (int64_t)blockIdx.x * a.per;
  const int nt = (int)min((int64_t)a.per, tokens - t0);
  const int per_token = a.heads * a.units, total = nt * per_token;
  const int nturn = a.m / E;                 // units of a turned row that hold pairs

  struct Unit { int token, set, u; int64_t x, y; bool live; };
  auto unit_of = [&](int i) {
    Unit w;
    w.live = i < total;
    i = min(i, total - 1);
    w.token = i / per_token;
    i -= w.token * per_token;
    int h = i / a.units;
    w.u = i - h * a.units;
    w.set = 0;
    while (h >= a.r[w.set].heads) h -= a.r[w.set++].heads;
    const RopeRows& r = a.r[w.set];
    const int64_t t = t0 + w.token;
    const int b = a.B == 1 ? 0 : (int)(t / a.S);
    const int64_t s = t - (int64_t)b * a.S;
    w.x = b * r.x_sb + s * r.x_st + h * r.x_sh;
    w.y = h * r.y_sh + (r.slots ? 0 : b * r.y_sb + s * r.y_st);
    return w;
  };
  // first elements of a unit's two chunks
  auto chunks = [&](const Unit& w, int& e0, int& e1) {
    if (a.r[w.set].turn && w.u < nturn) {
      e0 = a.start + (PAIRS ? 2 * w.u * E : w.u * E);
      e1 = e0 + (PAIRS ? E : a.m);
      return;
    }
    int c = 2 * (w.u - (a.r[w.set].turn ? nturn : 0)), d = c + 1;
    if (a.r[w.set].turn) {                   // chunks outside of the part
      const int s = a.start / E;
      c += c >= s ? 2 * nturn : 0;
      d += d >= s ? 2 * nturn : 0;
    }
    e0 = c * E;
    e1 = d * E;
  };
  for (int i0 = 0; i0 < total; i0 += kRpThreads) {
    const Unit w = unit_of(i0 + tid);
    const RopeRows& r = a.r[w.set];
    int e0, e1;
    chunks(w, e0, e1);
    RopeChunk<T, E> p, q;
    p.v = *(const V*)((const T*)r.x + w.x + e0);
    q.v = *(const V*)((const T*)r.x + w.x + e1);
    if (i0 == 0) {
      for (int i = tid; i < nt * a.m; i += kRpThreads) {
        const int t = i / a.m, j = i - t * a.m;
        const int b = a.B == 1 ? 0 : (int)((t0 + t) / a.S);
        const int64_t at = b * a.pos_sb + (t0 + t - (int64_t)b * a.S) * a.pos_st;
        const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
        sCs[t * kRpMaxPairs + j] = rp_turn(a.sign * pos, a.inv_freq[j], a.factor);
      }
      if (a.slots && tid < nt) sSlot[tid] = a.slots[t0 + tid];
      __syncthreads();
    }
    if (!w.live) continue;
    if (r.turn && w.u < nturn) {
      const float2* cs = sCs + w.token * kRpMaxPairs + w.u * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        // pair e of the unit: element e of each chunk, or elements 2e, 2e + 1 of both in a row
        T& xe = PAIRS ? (2 * e < E ? p.e[(2 * e) % E] : q.e[(2 * e) % E]) : p.e[e];
        T& ye = PAIRS ? (2 * e + 1 < E ? p.e[(2 * e + 1) % E] : q.e[(2 * e + 1) % E]) : q.e[e];
        const float2 z = cs[e];
        const float x = rp_in(xe), y = rp_in(ye);
        rp_out(fmaf(x, z.x, -(y * z.y)), xe);
        rp_out(fmaf(y, z.x, x * z.y), ye);
      }
    }
    int64_t y = w.y;
    if (r.slots) {
      const int64_t s = sSlot[w.token];
      if (s < 0 || s >= a.num_slots) continue;
      const int64_t pg = s / a.page;
      y += pg * r.y_sb + (s - pg * a.page) * r.y_st;
    }
    T* out = (T*)r.y + y;
    *(V*)(out + e0) = p.v;
    *(V*)(out + e1) = q.v;
  }
}

// Whether every row of the sets starts at a multiple of `bytes`.
static bool rope_fits(const RopeArgs& a, int size, int bytes) {
  const int e = bytes / size;
  if (a.m % e || a.start % e || a.D % (2 * e)) return false;
  for (int i = 0; i < a.n; ++i) {
    const RopeRows& r = a.r[i];
    const int64_t strides[] = {r.x_sb, r.x_st, r.x_sh, r.y_sb, r.y_st, r.y_sh};
    for (int64_t s : strides)
      if (s % e) return false;
    if ((uintptr_t)r.x % bytes || (uintptr_t)r.y % bytes) return false;
  }
  return true;
}

template <typename T>
static int rope_launch(RopeArgs& a, bool pairs, hipStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const bool wide = rope_fits(a, sizeof(T), 16);
  a.units = a.D / 2 / (wide ? E : 1);
  const int64_t tokens = (int64_t)a.B * a.S;
  if ((int64_t)a.heads * a.units * kRpTokens > INT32_MAX / 2) return kErrUnsupported;
  // four tokens (8,190 of 20 heads 21.6 us, one at a time 23.3), one where rows go to a cache (37.8 us, four 45.8)
  // unless that leaves threads without a unit, or the CUs without a work-group
  a.per = a.slots ? std::max(1, std::min(kRpTokens, kRpThreads / (a.heads * a.units))) : kRpTokens;
  if (tokens < 1024) a.per = 1;      // (1,023 of 20 heads 16.2 us replayed, four at a time 16.9; 1,536: 16.9, 16.7)
  const int64_t groups = (tokens + a.per - 1) / a.per;
  if (!fits_grid(groups, kRpThreads)) return kErrUnsupported;
  const dim3 grid((unsigned)groups), block(kRpThreads);
  if (wide && pairs) hipLaunchKernelGGL((rope_kernel<T, E, true>), grid, block, 0, st, a);
  else if (wide) hipLaunchKernelGGL((rope_kernel<T, E, false>), grid, block, 0, st, a);
  else if (pairs) hipLaunchKernelGGL((rope_kernel<T, 1, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rope_kernel<T, 1, false>), grid, block, 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}

static int rope_run(RopeArgs& a, int dtype, int interleaved, void* stream) {
  if (a.B < 0 || a.S < 0 || a.D <= 0 || a.m < 0 || a.start < 0 || dtype < 0 || dtype > 2) return kErrInvalid;
  if ((int64_t)a.B * a.S == 0) return kOk;
  if (a.D % 2 || a.m > kRpMaxPairs || (int64_t)a.start + 2 * a.m > a.D) return kErrUnsupported;
  if (!a.pos || (a.m > 0 && !a.inv_freq)) return kErrInvalid;
  // sets without heads are left out
  int n = 0;
  a.heads = 0;
  for (int i = 0; i < a.n; ++i) {
    if (a.r[i].heads < 0) return kErrInvalid;
    if (a.r[i].heads == 0) continue;
    if (!a.r[i].x || !a.r[i].y) return kErrInvalid;
    if (a.r[i].heads > INT32_MAX / 8) return kErrUnsupported;
    a.heads += a.r[i].heads;
    a.r[n++] = a.r[i];
  }
  a.n = n;
  if (n == 0) return kOk;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return rope_launch<float>(a, interleaved != 0, st);
  if (dtype == 1) return rope_launch<bf16>(a, interleaved != 0, st);
  return rope_launch<__half>(a, interleaved != 0, st);
}

}  // namespace dash

extern "C" int dash_rope(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int H, void* q_out,
                         int64_t qo_sb, int64_t qo_st, int64_t qo_sh, const void* k, int64_t k_sb,
                         int64_t k_st, int64_t k_sh, int Hkv, void* k_out, int64_t ko_sb, int64_t ko_st,
                         int64_t ko_sh, int dtype, const void* positions, int positions_int64,
                         int64_t pos_sb, int64_t pos_st, const double* inv_freq, int pairs, int start,
                         int interleaved, int back, double factor, int B, int S, int D, void* stream) {
  using namespace dash;
  RopeArgs a = {};
  a.r[0] = RopeRows{q, q_sb, q_st, q_sh, q_out, qo_sb, qo_st, qo_sh, H, 1, 0};
  a.r[1] = RopeRows{k, k_sb, k_st, k_sh, k_out, ko_sb, ko_st, ko_sh, Hkv, 1, 0};
  a.n = 2;
  a.pos = positions; a.pos64 = positions_int64; a.pos_sb = pos_sb; a.pos_st = pos_st;
  a.inv_freq = inv_freq; a.sign = back ? -1.0 : 1.0; a.factor = factor;
  a.B = B; a.S = S; a.D = D; a.m = pairs; a.start = start;
  return rope_run(a, dtype, interleaved, stream);
}

extern "C" int dash_rope_append(const void* q, int64_t q_st, int64_t q_sh, int H, void* q_out, int64_t qo_st,
                                int64_t qo_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                                int64_t v_st, int64_t v_sh, int Hkv, int dtype, const void* positions,
                                int positions_int64, const int64_t* slots, void* k_cache, int64_t kc_sp,
                                int64_t kc_st, int64_t kc_sh, void* v_cache, int64_t vc_sp, int64_t vc_st,
                                int64_t vc_sh, int page_size, int num_pages, const double* inv_freq,
                                int pairs, int start, int interleaved, double factor, int T, int D,
                                void* stream) {
  using namespace dash;
  if (page_size <= 0 || num_pages < 0 || (T > 0 && !slots)) return kErrInvalid;
  RopeArgs a = {};
  a.r[0] = RopeRows{q, 0, q_st, q_sh, q_out, 0, qo_st, qo_sh, H, 1, 0};
  a.r[1] = RopeRows{k, 0, k_st, k_sh, k_cache, kc_sp, kc_st, kc_sh, Hkv, 1, 1};
  a.r[2] = RopeRows{v, 0, v_st, v_sh, v_cache, vc_sp, vc_st, vc_sh, Hkv, 0, 1};
  a.n = num_pages > 0 ? 3 : 1;
  a.pos = positions; a.pos64 = positions_int64; a.pos_st = 1;
  a.inv_freq = inv_freq; a.sign = 1.0; a.factor = factor;
  a.slots = slots; a.page = page_size; a.num_slots = (int64_t)num_pages * page_size;
  a.B = 1; a.S = T; a.D = D; a.m = pairs; a.start = start;
  return rope_run(a, dtype, interleaved, stream);
}
