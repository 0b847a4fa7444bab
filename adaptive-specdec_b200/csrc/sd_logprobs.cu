// Log-probabilities of given tokens with their rank, the entropy of the
// distribution and its largest entries (sm_100a).
//
// For a row of logits x, temperature T and a token t, with y = x / T:
//   logprob = y_t - log sum_j exp(y_j)
//   entropy = -sum_j p_j log p_j = log z - (sum_j (y_j - m) exp(y_j - m)) / z,
//             z = sum_j exp(y_j - m), m = max y: both terms are >= 0, nothing
//             cancels
//   rank    = 1 + #{j : x_j > x_t} + #{j < t : x_j = x_t}
//   top n   = the n first entries by (x falling, id rising)
// A NaN counts as the largest value, -0 equals +0.  The sampling kernels of
// the verify round give a token and its probability after top-k / top-p; a
// caller that ranks samples needs the untruncated log-probabilities.
//
// One pass over the logits.  A row is cut into parts; a part's CTA streams its
// 16-byte units, LP_UNITS per thread and step with the next step's loads in
// flight, each thread keeping its maximum, sums in base 2 against a reference
// that moves only when a step's maximum passes it by LP_HEADROOM, and the count
// of elements ahead of the token (packed compares and adds).
// logp_part_kernel leaves per part the sums at the part's maximum, the count,
// and the part's top n as sorted 64-bit keys (value key, complement of the id);
// logp_rows_kernel (a programmatic dependent launch) joins a row's parts in part
// order.  No atomics reach a result: the list below is filled in any order and
// then ranked by unique keys.
//
// Top n of a part without comparing every element: with M_w the thread maxima
// of warp w, T = max(max_w (n-th largest of M_w), min_w (ceil(n/8)-th largest
// of M_w)) has at least n elements at or above it, and few more; only threads
// whose maximum reaches T look through their units again (from L2).
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <cfloat>

#include "sd_common.cuh"

namespace sd {

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNITS = 4;                     // 16-byte units per thread and step
constexpr int LP_CTAS = 3;                      // per SM
constexpr int LP_STEP = LP_THREADS * LP_UNITS;  // units per step of a CTA
constexpr float LP_HEADROOM = 8.f;              // base 2
constexpr int LP_LIST = 2048;                   // a part's flagged elements; a row's parts * n
constexpr int LP_MAX_PARTS = 64;
static_assert(LP_MAX_PARTS * SD_TOPN_MAX <= LP_LIST, "a row's lists fit the join's list");
static_assert(SD_TOPN_MAX <= 32, "the n-th largest thread maximum of one warp");
constexpr int LP_ROW_THREADS = 128;

struct LpPart {
  float m, s, e;                                // max (logit units), sum 2^d, sum d 2^d
  int ahead;                                    // elements at or ahead of the token
};

struct LpParams {
  const void* x;
  int64_t bs, ps;
  const int64_t* ids;
  int64_t ids_bs;
  int B, L, V, top, parts, dtype;
  float temperature, c;                         // c = log2(e) / temperature
  float* logprob;
  int64_t* rank;
  float* entropy;
  int64_t* top_ids;
  float* top_lp;
  LpPart* part;
  unsigned long long* keys;                     // [rows][parts][top]
};

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 32-bit order key: NaN (either sign) largest, -0 = +0; 0 is no value's key.
__device__ __forceinline__ uint32_t lp_key(float f) {
  return f != f ? 0xFFFFFFFFu : fkey(f);
}
// An exponent held at or above -256, where 2^x is 0: an element far below the
// maximum (-inf, or a mask of the type's lowest value) then adds 0 * -256 to
// the entropy sum, not 0 * -inf.  A NaN stays.
__device__ __forceinline__ float lp_hold(float x) { return x < -256.f ? -256.f : x; }
__device__ __forceinline__ float lp_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// What the kernel does on a 32-bit word of the logits' type (two 16-bit
// elements or one float): maximum with NaN winning, elements, and counting the
// elements that are not below a threshold (a NaN is not) with packed compares
// and adds: 4 * LP_UNITS per half and step, which bf16 holds exactly (up to 256).
template <typename T> struct Word;
template <> struct Word<__nv_bfloat16> {
  static constexpr int N = 2;
  static constexpr uint32_t NEG_INF = 0xFF80FF80u;
  __device__ static __nv_bfloat162 v(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  __device__ static uint32_t w(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
  __device__ static uint32_t vmax(uint32_t a, uint32_t b) { return w(__hmax2_nan(v(a), v(b))); }
  __device__ static float get(uint32_t x, int e) {
    return __uint_as_float(e ? (x & 0xFFFF0000u) : (x << 16));
  }
  __device__ static uint32_t count(uint32_t c, uint32_t x, uint32_t thr) {
    return w(__hadd2(v(c), __hgeu2(v(x), v(thr))));
  }
  __device__ static float total(uint32_t c) { return get(c, 0) + get(c, 1); }
  __device__ static bool any(uint32_t x, uint32_t thr) { return w(__hgeu2(v(x), v(thr))) != 0u; }
  // both halves the element's bits; the next larger value of a finite one
  __device__ static uint32_t splat(float f) { return (__float_as_uint(f) >> 16) * 0x10001u; }
  __device__ static uint32_t above(float f) {
    const uint32_t b = __float_as_uint(f) >> 16;
    return (f == 0.f ? 1u : (b & 0x8000u) ? b - 1u : b + 1u) * 0x10001u;
  }
};
template <> struct Word<__half> {
  static constexpr int N = 2;
  static constexpr uint32_t NEG_INF = 0xFC00FC00u;
  __device__ static __half2 v(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
  __device__ static uint32_t w(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
  __device__ static uint32_t vmax(uint32_t a, uint32_t b) { return w(__hmax2_nan(v(a), v(b))); }
  __device__ static float get(uint32_t x, int e) {
    return e ? __high2float(v(x)) : __low2float(v(x));
  }
  __device__ static uint32_t count(uint32_t c, uint32_t x, uint32_t thr) {
    return w(__hadd2(v(c), __hgeu2(v(x), v(thr))));
  }
  __device__ static float total(uint32_t c) { return get(c, 0) + get(c, 1); }
  __device__ static bool any(uint32_t x, uint32_t thr) { return w(__hgeu2(v(x), v(thr))) != 0u; }
  __device__ static uint32_t bits(float f) { return __half_as_ushort(__float2half_rn(f)); }
  __device__ static uint32_t splat(float f) { return bits(f) * 0x10001u; }
  __device__ static uint32_t above(float f) {
    const uint32_t b = bits(f);
    return (f == 0.f ? 1u : (b & 0x8000u) ? b - 1u : b + 1u) * 0x10001u;
  }
};
template <> struct Word<float> {
  static constexpr int N = 1;
  static constexpr uint32_t NEG_INF = 0xFF800000u;
  __device__ static uint32_t vmax(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static float get(uint32_t x, int) { return __uint_as_float(x); }
  __device__ static uint32_t count(uint32_t c, uint32_t x, uint32_t thr) {
    return c + !(__uint_as_float(x) < __uint_as_float(thr));
  }
  __device__ static float total(uint32_t c) { return (float)(int)c; }
  __device__ static bool any(uint32_t x, uint32_t thr) {
    return !(__uint_as_float(x) < __uint_as_float(thr));
  }
  __device__ static uint32_t splat(float f) { return __float_as_uint(f); }
  __device__ static uint32_t above(float f) {
    const uint32_t b = __float_as_uint(f);
    return f == 0.f ? 1u : (b & 0x80000000u) ? b - 1u : b + 1u;
  }
};

// Two floats in one 64-bit register for the packed FP32 instructions.
__device__ __forceinline__ unsigned long long pair2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(unsigned long long p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b,
                                                   unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The n largest of the cnt unique keys in `list` (shared memory), in falling
// order, to out[0..n): all threads of the block call it.  cnt <= LP_LIST;
// slots past cnt keys are 0.  A long list is first cut to its n largest by
// finding the n-th key bit by bit.
template <int THREADS>
__device__ void sort_top(unsigned long long* list, int cnt, int n, unsigned long long* out,
                         int* counter) {
  const int t = threadIdx.x;
  if (cnt > 2 * THREADS) {
    unsigned long long nth = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long cand = nth | (1ULL << bit);
      int c = 0;
      for (int i0 = 0; i0 < cnt; i0 += THREADS)
        c += __syncthreads_count(i0 + t < cnt && list[i0 + t] >= cand);
      if (c >= n) nth = cand;
    }
    // the n keys >= nth move to the front, a block of THREADS at a time
    int kept = 0;
    for (int i0 = 0; i0 < cnt; i0 += THREADS) {
      const unsigned long long k = i0 + t < cnt ? list[i0 + t] : 0ULL;
      __syncthreads();                               // everybody has read its key
      if (t == 0) *counter = kept;
      __syncthreads();
      if (k >= nth && k != 0ULL) list[atomicAdd(counter, 1)] = k;   // at most i0 + THREADS so far
      __syncthreads();
      kept = *counter;
    }
    cnt = kept;
    __syncthreads();
  }
  for (int i = t; i < cnt; i += THREADS) {
    const unsigned long long k = list[i];
    int r = 0;
    for (int j = 0; j < cnt; ++j) r += list[j] > k;
    if (r < n) out[r] = k;
  }
  for (int i = cnt + t; i < n; i += THREADS) out[i] = 0ULL;
}

// A thread's running state over its units.
template <typename T>
struct LpRun {
  using Wd = Word<T>;
  uint32_t wm;                                       // maximum, a NaN wins
  float ref, nref, ahead;                            // reference of the sums and its negative
  unsigned long long s2, e2;                         // sum 2^d, sum d 2^d, d = (x - ref) c
  __device__ void init() {
    wm = Wd::NEG_INF;
    ref = nref = 0.f;
    ahead = 0.f;
    s2 = e2 = 0ULL;
  }
  // One step: units u, u + LP_THREADS, ...; `first`: the reference is set, not moved.
  __device__ __forceinline__ void step(const uint4 (&d)[LP_UNITS], int u, bool first, float c,
                                       unsigned long long c2, int tu, uint32_t thr_at,
                                       uint32_t thr_up) {
    uint32_t g = Wd::vmax(Wd::vmax(d[0].x, d[0].y), Wd::vmax(d[0].z, d[0].w));
#pragma unroll
    for (int i = 1; i < LP_UNITS; ++i)
      g = Wd::vmax(g, Wd::vmax(Wd::vmax(d[i].x, d[i].y), Wd::vmax(d[i].z, d[i].w)));
    wm = Wd::vmax(wm, g);
    const float gm = fmaxf(Wd::get(g, 0), Wd::get(g, Wd::N - 1));
    const float up = (gm - ref) * c;
    if (first ? gm > -CUDART_INF_F && gm < CUDART_INF_F : up > LP_HEADROOM && gm < CUDART_INF_F) {
      // the sums so far move to the new reference (2^-256 is 0)
      const float dm = fmaxf(-up, -256.f), f = lp_ex2(dm);
      const unsigned long long f2 = pair2(f, f);
      if (!first) {
        e2 = mul2(f2, fma2(pair2(dm, dm), s2, e2));
        s2 = mul2(f2, s2);
      }
      ref = gm;
      nref = -gm;
    }
    const unsigned long long nr2 = pair2(nref, nref);
    uint32_t cnt = 0u;
#pragma unroll
    for (int i = 0; i < LP_UNITS; ++i) {
      const uint32_t thr = u + i * LP_THREADS <= tu ? thr_at : thr_up;
      const uint32_t w[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) cnt = Wd::count(cnt, w[q], thr);
#pragma unroll
      for (int q = 0; q < 4; q += 3 - Wd::N) {
        const unsigned long long x2 = Wd::N == 2 ? pair2(Wd::get(w[q], 0), Wd::get(w[q], 1))
                                                 : pair2(Wd::get(w[q], 0), Wd::get(w[q | 1], 0));
        float a, b;
        unpair(mul2(add2(x2, nr2), c2), a, b);
        // -inf elements add 0 * -256, not 0 * -inf
        a = fmaxf(a, -256.f);
        b = fmaxf(b, -256.f);
        const unsigned long long p2 = pair2(lp_ex2(a), lp_ex2(b));
        s2 = add2(s2, p2);
        e2 = fma2(pair2(a, b), p2, e2);
      }
    }
    ahead += Wd::total(cnt);
  }
};

// A step's units from p on (p: this thread's first); those past `left` units
// of the part are -inf.
__device__ __forceinline__ void lp_load(uint4 (&d)[LP_UNITS], const uint4* p) {
#pragma unroll
  for (int i = 0; i < LP_UNITS; ++i) d[i] = __ldcs(p + i * LP_THREADS);
}
template <typename T>
__device__ __forceinline__ void lp_load_rest(uint4 (&d)[LP_UNITS], const uint4* p, int left) {
#pragma unroll
  for (int i = 0; i < LP_UNITS; ++i) {
    constexpr uint32_t ni = Word<T>::NEG_INF;
    d[i] = i * LP_THREADS < left ? __ldcs(p + i * LP_THREADS) : make_uint4(ni, ni, ni, ni);
  }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) logp_part_kernel(const LpParams P) {
  using Wd = Word<T>;
  constexpr int E = 4 * Wd::N;                       // elements per 16-byte unit
  extern __shared__ __align__(16) unsigned char lp_smem[];
  unsigned long long* list = reinterpret_cast<unsigned long long*>(lp_smem);   // TOP only
  __shared__ float red_m[LP_WARPS], red_s[LP_WARPS], red_e[LP_WARPS];
  __shared__ int red_c[LP_WARPS];
  __shared__ uint32_t kth[LP_WARPS], jth[LP_WARPS];
  __shared__ unsigned long long red_k[LP_WARPS];
  __shared__ int n_list, counter;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int64_t item = blockIdx.x;
  const int64_t r = item / P.parts;
  const int part = (int)(item - r * P.parts);
  const int64_t rb = r / P.L, rl = r - rb * P.L;
  const int64_t row0 = rb * P.bs + rl * P.ps;
  const T* row = reinterpret_cast<const T*>(P.x) + row0;
  const int V = P.V;
  // whole 16-byte units between the row's first and last aligned address; the
  // < 2 E elements outside them go one each to threads of part 0
  const int h0 = min((int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)), V);
  const int units = (V - h0) / E, tail = V - h0 - units * E;
  const int per = (units + P.parts - 1) / P.parts;
  const int u0 = min(part * per, units), u1 = min(u0 + per, units);
  const uint4* body = reinterpret_cast<const uint4*>(row + h0);
  uint4 cur[LP_UNITS], nxt[LP_UNITS];
  // whole steps two by two, the loads of one in flight while the other is
  // worked on; then what is left (k whole steps, `left` units past this thread)
  const uint4* p = body + u0 + t;
  int k = (u1 - u0) / LP_STEP;
  const int left = u1 - u0 - k * LP_STEP - t;
  if (k > 0) lp_load(cur, p); else lp_load_rest<T>(cur, p, left);
  if (t == 0) n_list = 0;
  const bool lone = part == 0 && t < h0 + tail;      // this thread's extra element
  const int xi = t < h0 ? t : V - tail + (t - h0);
  const float xe = lone ? load_logit(P.x, P.dtype, row0 + xi) : -CUDART_INF_F;
  const int64_t tok = P.ids[rb * P.ids_bs + rl];
  const bool have = tok >= 0 && tok < V;
  const float xt = have ? load_logit(P.x, P.dtype, row0 + tok) : CUDART_INF_F;
  // elements at ids up to the token's count when not below it, later ones when
  // above it: units up to the token's compare with x_t, later ones with the
  // next larger value
  const bool plain = have && xt > -CUDART_INF_F && xt < CUDART_INF_F;
  const int tu = tok < h0 ? -1 : (int)((tok - h0) / E);
  const uint32_t thr_at = Wd::splat(xt), thr_up = Wd::above(xt);
  const unsigned long long c2 = pair2(P.c, P.c);
  LpRun<T> run;
  run.init();
  int u = u0 + t;
  bool first = true;
  auto step = [&](const uint4 (&d)[LP_UNITS]) {
    run.step(d, u, first, P.c, c2, tu, thr_at, thr_up);
    // the reference is set by the first step that has a finite element
    first = first && run.s2 == 0ULL;
    u += LP_STEP;
  };
#pragma unroll 1
  for (; k >= 2; k -= 2) {
    p += LP_STEP;
    lp_load(nxt, p);
    step(cur);
    p += LP_STEP;
    if (k > 2) lp_load(cur, p); else lp_load_rest<T>(cur, p, left);
    step(nxt);
  }
  if (k == 1) {
    lp_load_rest<T>(nxt, p + LP_STEP, left);
    step(cur);
    step(nxt);
  } else {
    step(cur);
  }
  float m = __uint_as_float(Word<float>::vmax(
      Word<float>::vmax(__float_as_uint(Wd::get(run.wm, 0)),
                        __float_as_uint(Wd::get(run.wm, Wd::N - 1))),
      __float_as_uint(xe)));
  const bool nan = m != m;
  // the thread's sums at its own maximum, with its extra element
  const float m0 = m == -CUDART_INF_F || m == CUDART_INF_F || nan ? 0.f : m;
  float s, es;
  {
    float a, b;
    unpair(run.s2, s, b);
    unpair(run.e2, es, a);
    s += b;
    es += a;
    const float dm = s > 0.f ? fmaxf((run.ref - m0) * P.c, -256.f) : 0.f, f = lp_ex2(dm);
    es = f * fmaf(dm, s, es);
    s *= f;
    const float dd = fmaxf((xe - m0) * P.c, -256.f), p = lp_ex2(dd);
    s += p;
    es = fmaf(dd, p, es);
  }
  const uint32_t kt = lp_key(xt);
  int ahead = 0;
  if (plain) {
    ahead = (int)run.ahead;
    if (tu >= u0 && tu < u1 && (tu - u0) % LP_THREADS == t) {
      // the token's own unit: entries behind it that equal it were counted
      for (int e = (int)((tok - h0) % E) + 1; e < E; ++e)
        ahead -= load_logit(P.x, P.dtype, row0 + h0 + tu * E + e) == xt;
    }
  } else if (have) {
    // an infinite or NaN token: by keys
#pragma unroll 1
    for (int u = u0 + t; u < u1; u += LP_THREADS)
      for (int e = 0; e < E; ++e) {
        const int idx = h0 + u * E + e;
        const uint32_t k = lp_key(load_logit(P.x, P.dtype, row0 + idx));
        ahead += k > kt || (k == kt && idx <= tok);
      }
  }
  if (lone && have) {
    const uint32_t k = lp_key(xe);
    ahead += k > kt || (k == kt && xi <= tok);
  }
  // join over the block: the maxima first, then the sums at the block's maximum
  float bm = warp_max(nan ? -CUDART_INF_F : m);
  if (lane == 0) red_m[w] = bm;
  const bool any = u0 + t < u1 || lone;              // this thread holds an element
  if (TOP) {
    // this warp's sorted thread maxima (bitonic over lanes, falling)
    uint32_t k = any ? lp_key(m) : 0u;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
      for (int st = size >> 1; st > 0; st >>= 1) {
        const uint32_t o = __shfl_xor_sync(0xffffffffu, k, st);
        const bool up = ((lane & size) == 0) == ((lane & st) == 0);
        k = up ? max(k, o) : min(k, o);
      }
    const int j = (P.top + LP_WARPS - 1) / LP_WARPS;
    if (lane == P.top - 1) kth[w] = k;
    if (lane == j - 1) jth[w] = k;
  }
  __syncthreads();
  bm = red_m[0];
#pragma unroll
  for (int q = 1; q < LP_WARPS; ++q) bm = fmaxf(bm, red_m[q]);
  const float dm = lp_hold((m - bm) * P.c), f = lp_ex2(dm);
  float sj = f * s, ej = f * fmaf(dm, s, es);
  if (m == -CUDART_INF_F) sj = ej = 0.f;             // nothing above -inf
  if (nan || m == CUDART_INF_F) sj = CUDART_NAN_F;   // as the formula: inf - inf
  sj = warp_sum(sj);
  ej = warp_sum(ej);
  ahead = warp_sum(ahead);
  if (lane == 0) {
    red_s[w] = sj;
    red_e[w] = ej;
    red_c[w] = ahead;
  }
  if (TOP) {
    uint32_t T1 = 0, T2 = 0xFFFFFFFFu;
#pragma unroll
    for (int q = 0; q < LP_WARPS; ++q) {
      T1 = max(T1, kth[q]);
      T2 = min(T2, jth[q]);
    }
    const uint32_t thr = max(max(T1, T2), 1u);
    auto put = [&](uint32_t k, int idx) {
      const int at = atomicAdd(&n_list, 1);
      if (at < LP_LIST) list[at] = ((unsigned long long)k << 32) | (uint32_t)~(uint32_t)idx;
    };
    // the warp looks through its flagged threads' units, four threads at a time
    const uint32_t tw = Wd::splat(lp_value(thr));
    if (lone && lp_key(xe) >= thr) put(lp_key(xe), xi);
    uint32_t flagged = __ballot_sync(0xffffffffu, any && lp_key(m) >= thr);
    while (flagged) {
      int at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at[i] = flagged ? u0 + 32 * w + __ffs(flagged) - 1 : u1;
        flagged &= flagged - 1;
      }
#pragma unroll 1
      for (int o = lane * LP_THREADS; u0 + 32 * w + o < u1; o += 32 * LP_THREADS) {
        uint4 d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          constexpr uint32_t ni = Wd::NEG_INF;
          d[i] = at[i] + o < u1 ? __ldg(body + at[i] + o) : make_uint4(ni, ni, ni, ni);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (at[i] + o >= u1) continue;
          const uint32_t x[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (!Wd::any(x[q], tw)) continue;
#pragma unroll
            for (int e = 0; e < Wd::N; ++e) {
              const uint32_t key = lp_key(Wd::get(x[q], e));
              if (key >= thr) put(key, h0 + (at[i] + o) * E + q * Wd::N + e);
            }
          }
        }
      }
    }
    __syncthreads();
    int found = n_list;
    if (found > LP_LIST) {
      // More elements than the list holds reach the threshold (flat logits):
      // the n largest keys one after the other, a pass over the part for each.
      unsigned long long last = ~0ULL;
      for (int n = 0; n < P.top; ++n) {
        unsigned long long best = 0ULL;
        auto see = [&](float x, int idx) {
          const unsigned long long k =
              ((unsigned long long)lp_key(x) << 32) | (uint32_t)~(uint32_t)idx;
          if (k < last && k > best) best = k;
        };
#pragma unroll 1
        for (int v = u0 + t; v < u1; v += LP_THREADS) {
          const uint4 d = __ldg(body + v);
          const uint32_t x[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < Wd::N; ++e) see(Wd::get(x[q], e), h0 + v * E + q * Wd::N + e);
        }
        if (lone) see(xe, xi);
        best = warp_max(best);
        __syncthreads();                             // red_k of the last round has been read
        if (lane == 0) red_k[w] = best;
        __syncthreads();
        best = red_k[0];
#pragma unroll
        for (int q = 1; q < LP_WARPS; ++q) best = red_k[q] > best ? red_k[q] : best;
        if (t == 0) list[n] = best;
        last = best;
      }
      found = P.top;
      __syncthreads();
    }
    sort_top<LP_THREADS>(list, found, P.top, P.keys + item * P.top, &counter);
  } else {
    __syncthreads();
  }
  if (t == 0) {
    LpPart o;
    o.m = bm;
    o.s = 0.f;
    o.e = 0.f;
    o.ahead = 0;
#pragma unroll
    for (int q = 0; q < LP_WARPS; ++q) {
      o.s += red_s[q];
      o.e += red_e[q];
      o.ahead += red_c[q];
    }
    P.part[item] = o;
  }
}

// One CTA per row: the parts' sums at the row's maximum, the token, the
// entropy, and the row's top n from the parts' lists.
__global__ void __launch_bounds__(LP_ROW_THREADS) logp_rows_kernel(const LpParams P) {
  extern __shared__ __align__(16) unsigned char lp_smem[];
  unsigned long long* list = reinterpret_cast<unsigned long long*>(lp_smem);   // [parts * top]
  __shared__ float sh_m, sh_lz;
  __shared__ int counter, n_list;
  __shared__ unsigned long long sh_t, best[SD_TOPN_MAX];
  const int t = threadIdx.x;
  const int64_t r = blockIdx.x, rb = r / P.L, rl = r % P.L;
  const int64_t tok = P.ids[rb * P.ids_bs + rl];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const LpPart* part = P.part + r * P.parts;
  if (t < 32) {
    float m = -CUDART_INF_F;
    for (int i = t; i < P.parts; i += 32) m = fmaxf(m, part[i].m);
    m = warp_max(m);
    float s = 0.f, e = 0.f;
    int ahead = 0;
    for (int i = t; i < P.parts; i += 32) {
      const LpPart q = part[i];
      ahead += q.ahead;
      if (q.m == -CUDART_INF_F && q.s == q.s) continue;          // nothing finite, no NaN
      const float dm = lp_hold((q.m - m) * P.c), f = lp_ex2(dm);
      s = fmaf(f, q.s, s);
      e = fmaf(f, fmaf(dm, q.s, q.e), e);
    }
    s = warp_sum(s);
    e = warp_sum(e);
    ahead = warp_sum(ahead);
    if (t == 0) {
      const float lz = logf(s);
      sh_m = m;
      sh_lz = lz;
      const bool none = !(m > -CUDART_INF_F);                    // every entry is -inf
      const bool have = tok >= 0 && tok < P.V;
      P.entropy[r] = none || m == CUDART_INF_F ? CUDART_NAN_F
                                               : lz - 0.69314718055994531f * (e / s);
      P.rank[r] = have ? (int64_t)ahead : 0;
      float lp = CUDART_NAN_F;
      if (have && !none)
        lp = __fdiv_rn(load_logit(P.x, P.dtype, rb * P.bs + rl * P.ps + tok) - m, P.temperature) - lz;
      P.logprob[r] = lp;
    }
  }
  __syncthreads();
  if (P.top == 0) return;
  // Each part's keys are sorted: the best part's n-th key, and the least of the
  // parts' ceil(n / parts)-th keys, have n keys at or above them.
  const unsigned long long* keys = P.keys + r * P.parts * P.top;
  const int all = P.parts * P.top, j = (P.top + P.parts - 1) / P.parts;
  if (t < 32) {
    unsigned long long T1 = 0ULL, T2 = ~0ULL;
    for (int i = t; i < P.parts; i += 32) {
      const unsigned long long a = keys[i * P.top + P.top - 1], b = keys[i * P.top + j - 1];
      T1 = a > T1 ? a : T1;
      T2 = b < T2 ? b : T2;
    }
    T1 = warp_max(T1);
    T2 = warp_min(T2);
    if (t == 0) {
      sh_t = T1 > T2 ? T1 : T2;
      n_list = 0;
    }
  }
  __syncthreads();
  const unsigned long long thr = sh_t > 1ULL ? sh_t : 1ULL;    // absent keys are 0
  for (int i = t; i < all; i += LP_ROW_THREADS) {
    const unsigned long long k = keys[i];
    if (k >= thr) list[atomicAdd(&n_list, 1)] = k;
  }
  __syncthreads();
  const int found = n_list;
  __syncthreads();
  sort_top<LP_ROW_THREADS>(list, found, P.top, best, &counter);
  __syncthreads();
  if (t < P.top) {
    const unsigned long long k = best[t];
    const float v = lp_value((uint32_t)(k >> 32));
    P.top_ids[r * P.top + t] = (int64_t)(uint32_t)~(uint32_t)k;
    P.top_lp[r * P.top + t] = __fdiv_rn(v - sh_m, P.temperature) - sh_lz;
  }
}

// Parts per row: the CTAs run in rounds of LP_CTAS per SM, a round takes a
// part's units plus about LP_FIXED units' time for its start and its join, and
// the fewest of round * length wins.
constexpr int LP_FIXED = 2048;
static int lp_parts(int64_t rows, int V, int dtype) {
  const int E = dtype == SD_DTYPE_F32 ? 4 : 8;
  const int64_t units = ((int64_t)V + E - 1) / E, slots = LP_CTAS * 148;
  const int64_t most = std::min<int64_t>(std::max<int64_t>(units / LP_THREADS, 1), LP_MAX_PARTS);
  int best = 1;
  int64_t least = -1;
  for (int p = 1; p <= most; ++p) {
    const int64_t rounds = (rows * p + slots - 1) / slots;
    const int64_t cost = rounds * ((units + p - 1) / p + LP_FIXED);
    if (least < 0 || cost < least) {
      least = cost;
      best = p;
    }
  }
  return best;
}

template <typename T>
static int launch_logprobs(const LpParams& P, cudaStream_t st) {
  const int64_t rows = (int64_t)P.B * P.L;
  const dim3 grid((unsigned)(rows * P.parts));
  if (P.top > 0)
    logp_part_kernel<T, true><<<grid, LP_THREADS, LP_LIST * sizeof(unsigned long long), st>>>(P);
  else
    logp_part_kernel<T, false><<<grid, LP_THREADS, 0, st>>>(P);
  if (cudaGetLastError() != cudaSuccess) return SD_ELAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows);
  cfg.blockDim = dim3(LP_ROW_THREADS);
  cfg.dynamicSmemBytes = (size_t)P.parts * P.top * sizeof(unsigned long long);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, logp_rows_kernel, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // namespace sd

using namespace sd;

extern "C" {

size_t sd_token_logprobs_workspace_bytes(int B, int L, int V, int dtype, int top_n) {
  if (B <= 0 || L <= 0 || V <= 0 || V > SD_LOGPROBS_MAX_V || top_n < 0 || top_n > SD_TOPN_MAX)
    return 0;
  const int64_t rows = (int64_t)B * L;
  const size_t items = (size_t)rows * lp_parts(rows, V, dtype);
  return items * (sizeof(LpPart) + (size_t)top_n * sizeof(unsigned long long));
}

int sd_token_logprobs(const void* logits, int64_t bs, int64_t ps, int dtype, const int64_t* ids,
                      int64_t ids_bs, int B, int L, int V, float temperature, int top_n,
                      float* logprob, int64_t* rank, float* entropy, int64_t* top_ids,
                      float* top_logprobs, void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (B < 0 || L < 0) return SD_EINVAL;
  if (B == 0 || L == 0) return SD_OK;
  if (!logits || !ids || !logprob || !rank || !entropy || V <= 0) return SD_EINVAL;
  if (dtype != SD_DTYPE_F32 && dtype != SD_DTYPE_F16 && dtype != SD_DTYPE_BF16) return SD_EINVAL;
  if (!(temperature > 0.f) || temperature > FLT_MAX) return SD_EINVAL;
  if (top_n < 0 || top_n > V || (top_n > 0 && (!top_ids || !top_logprobs))) return SD_EINVAL;
  const int64_t rows = (int64_t)B * L;
  if (V > SD_LOGPROBS_MAX_V || top_n > SD_TOPN_MAX) return SD_ENOTSUP;
  const int parts = lp_parts(rows, V, dtype);
  if (rows * parts > 0x7FFFFFFF) return SD_ENOTSUP;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == SD_DTYPE_F32 ? 4 : 2)) return SD_EINVAL;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
      workspace_bytes < sd_token_logprobs_workspace_bytes(B, L, V, dtype, top_n))
    return SD_ENOSPC;
  LpParams P;
  P.x = logits; P.bs = bs; P.ps = ps; P.dtype = dtype;
  P.ids = ids; P.ids_bs = ids_bs;
  P.B = B; P.L = L; P.V = V; P.top = top_n; P.parts = parts;
  P.temperature = temperature;
  P.c = (float)(1.4426950408889634 / (double)temperature);
  P.logprob = logprob; P.rank = rank; P.entropy = entropy;
  P.top_ids = top_ids; P.top_lp = top_logprobs;
  // keys first: both arrays then sit on their own alignment
  P.keys = reinterpret_cast<unsigned long long*>(workspace);
  P.part = reinterpret_cast<LpPart*>(P.keys + (size_t)rows * parts * top_n);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == SD_DTYPE_BF16) return launch_logprobs<__nv_bfloat16>(P, st);
  if (dtype == SD_DTYPE_F16) return launch_logprobs<__half>(P, st);
  return launch_logprobs<float>(P, st);
}

}  // extern "C"
