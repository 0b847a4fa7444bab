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
// One pass over the logits, one launch.  (Small vocabularies: a warp per row, see
// logp_warp_kernel.)  Clusters of 1, 2, 4 or 8 CTAs take
// either a whole row per CTA or one row together, a part each: whole rows while
// there is one for every SM, then parts, so that the SMs end together.  A CTA
// streams its part's 16-byte
// units, LP_UNITS per thread and step with the next step's loads in flight,
// each thread keeping its maximum, sums in base 2 against a reference that
// moves only when a step's maximum passes it by LP_HEADROOM (rows whose largest
// logit is beyond LP_TAME in base-2 units take a second pass), and the count of
// elements ahead of the token (packed compares and adds).  Each CTA leaves its
// sums at the part's maximum, its count and its top n as sorted 64-bit keys
// (value key, complement of the id) in the shared memory of the cluster's first
// CTA, which joins them in part order.  No atomics reach a result: the list
// below is filled in any order and then ranked by unique keys.
//
// Top n of a part without comparing every element: of 32 to 64 maxima of up to 8
// threads each, the n-th largest has at least n elements at or above it, and
// few more; only threads whose maximum reaches it look through their units
// again (from L2), a warp together.
//
// The list holds 2048 elements; where more reach the threshold (flat logits; fewer
// than n of the groups with anything above -inf, as under a mask that leaves a few
// neighbouring ids), the part is read once per alternative: 320 rows with 15 live
// entries take 408 us with five alternatives, 1127 with twenty.
//
// Bound by HBM with many rows: 2048 rows of 151936 bf16 in 117 us, 5.3 TB/s (the
// copy rate here is 6.57); by latency with few: one row in 6 us, 320 rows with five
// alternatives in 29 (3.4 TB/s: 2.2 rows per SM, whose tails show).
#include <cuda_runtime.h>
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>

#include "sd_common.cuh"

namespace sd {

namespace cg = cooperative_groups;

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNITS = 4;                     // 16-byte units per thread and step
constexpr int LP_CTAS = 4;                      // per SM
constexpr int LP_SMS = 148;
constexpr int LP_STEP = LP_THREADS * LP_UNITS;  // units per step of a CTA
constexpr float LP_HEADROOM = 8.f;              // base 2
// The largest reference, in base-2 units.  A reference is the float next to m c;
// from 2^31 on it may be more than 128 away from it, so that the maximum's own
// exponent d = fma(m, c, -R) is no longer near 0 and 2^d leaves the float range.
// Up to 2^20 they are within 1/32.
constexpr float LP_TAME = 1048576.f;
constexpr int LP_LIST = 2048;                   // a part's flagged elements
constexpr int LP_GROUPS = 64;                   // groups of threads behind the top n's threshold
constexpr int LP_MAX_PARTS = 8;                 // CTAs of a cluster
constexpr int LP_WARP_V = 1024;                 // largest vocabulary of a warp per row
constexpr int LP_WLIST = 256;                   // its flagged elements
static_assert(LP_MAX_PARTS * SD_TOPN_MAX <= LP_THREADS, "a thread per key of the join");
static_assert(SD_TOPN_MAX <= LP_GROUPS / 2 && LP_THREADS / 8 >= LP_GROUPS / 2,
              "the n-th largest of the group maxima");

struct LpPart {
  double ref;                                   // reference of the sums (base-2 units)
  float s, e;                                   // sum 2^d, sum d 2^d
  int ahead;                                    // elements at or ahead of the token
};

struct LpParams {
  const void* x;
  int64_t bs, ps;
  const int64_t* ids;
  int64_t ids_bs;
  int B, L, V, top, dtype;
  int csize, whole;                             // CTAs per cluster; clusters of whole rows
  float c;                                      // log2(e) / temperature
  float* logprob;
  int64_t* rank;
  float* entropy;
  int64_t* top_ids;
  float* top_lp;
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
// ln2 (x c - ref - lz): a log-probability from a logit, the reference and the base-2
// log of the sum.  In 64 bits, where x c is exact and the difference loses
// nothing; the rounding of the sum alone may not make a probability above 1.
__device__ __forceinline__ float lp_final(float x, float c, double ref, float lz) {
  const double v = 0.69314718055994530942 * ((double)x * (double)c - ref - (double)lz);
  return v > 0.0 ? 0.f : (float)v;
}
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

// A thread's running state over its units.  Exponents are d = fma(x, c, -R) with
// the reference R a float in base-2 units, |R| <= LP_TAME: one rounding of d, as
// long as everything is measured against the same R.  A thread whose maximum is
// below that range has sums of 0, which is what they are worth beside a maximum
// within it; one above it has no valid sums (the block notices).
template <typename T>
struct LpRun {
  using Wd = Word<T>;
  uint32_t wm;                                       // maximum, a NaN wins
  float R, ahead;
  unsigned long long s2, e2;                         // sums of 2^d and d 2^d
  __device__ void init() {
    wm = Wd::NEG_INF;
    R = ahead = 0.f;
    s2 = e2 = 0ULL;
  }
  // One step: units u, u + LP_THREADS, ...
  __device__ __forceinline__ void step(const uint4 (&d)[LP_UNITS], int u, float c, int tu,
                                       uint32_t thr_at, uint32_t thr_up) {
    uint32_t g = Wd::vmax(Wd::vmax(d[0].x, d[0].y), Wd::vmax(d[0].z, d[0].w));
#pragma unroll
    for (int i = 1; i < LP_UNITS; ++i)
      g = Wd::vmax(g, Wd::vmax(Wd::vmax(d[i].x, d[i].y), Wd::vmax(d[i].z, d[i].w)));
    wm = Wd::vmax(wm, g);
    const float gs = fmaxf(Wd::get(g, 0), Wd::get(g, Wd::N - 1)) * c;
    // nothing summed yet: any maximum is the reference
    const bool first = s2 == 0ULL;
    if (fabsf(gs) <= LP_TAME && (first || gs - R > LP_HEADROOM)) {
      // the sums so far move to the new reference (2^-256 is 0)
      const float dm = fmaxf(R - gs, -256.f), f = lp_ex2(dm);
      const unsigned long long f2 = pair2(f, f);
      e2 = mul2(f2, fma2(pair2(dm, dm), s2, e2));
      s2 = mul2(f2, s2);
      if (first) s2 = e2 = 0ULL;
      R = gs;
    }
    const unsigned long long c2 = pair2(c, c), nR2 = pair2(-R, -R);
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
        unpair(fma2(x2, c2, nR2), a, b);
        // elements far below (-inf, masks) add 0 * -256, not 0 * -inf
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
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) logp_kernel(const LpParams P) {
  using Wd = Word<T>;
  constexpr int E = 4 * Wd::N;                       // elements per 16-byte unit
  extern __shared__ __align__(16) unsigned char lp_smem[];
  unsigned long long* list = reinterpret_cast<unsigned long long*>(lp_smem);   // TOP only
  __shared__ float red_m[LP_WARPS], red_s[LP_WARPS], red_e[LP_WARPS];
  __shared__ int red_c[LP_WARPS];
  __shared__ uint32_t group_k[LP_GROUPS];
  __shared__ unsigned long long red_k[LP_WARPS];
  __shared__ int n_list, counter;
  // of the cluster's first CTA: what every part found
  __shared__ LpPart parts[LP_MAX_PARTS];
  __shared__ unsigned long long part_keys[LP_MAX_PARTS * SD_TOPN_MAX];
  // log2 of the sum of all exponentials: the reference and the rest
  __shared__ double sh_ref;
  __shared__ float sh_lz;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const cg::cluster_group cluster = cg::this_cluster();
  const int cid = (int)(blockIdx.x / P.csize), crank = (int)(blockIdx.x % P.csize);
  const bool split = cid >= P.whole && P.csize > 1;
  const int64_t r = split ? (int64_t)P.whole * P.csize + (cid - P.whole)
                          : (int64_t)cid * P.csize + crank;
  const int part = split ? crank : 0, nparts = split ? P.csize : 1;
  // the first CTA's shared memory may be written once its CTA has started
  if (split) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t rb = r / P.L, rl = r - rb * P.L;
  const int64_t row0 = rb * P.bs + rl * P.ps;
  const T* row = reinterpret_cast<const T*>(P.x) + row0;
  const int V = P.V;
  // whole 16-byte units between the row's first and last aligned address; the
  // < 2 E elements outside them go one each to threads of part 0
  const int h0 = min((int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)), V);
  const int units = (V - h0) / E, tail = V - h0 - units * E;
  const int per = (units + nparts - 1) / nparts;
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
  LpRun<T> run;
  run.init();
  int u = u0 + t;
  auto step = [&](const uint4 (&d)[LP_UNITS]) {
    run.step(d, u, P.c, tu, thr_at, thr_up);
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
  // the thread's sums at its own maximum (base-2 units), with its extra element
  const float ms = m * P.c;
  const float m0 = fabsf(ms) <= LP_TAME ? ms : 0.f;
  float s, es;
  {
    float a, b;
    unpair(run.s2, s, b);
    unpair(run.e2, es, a);
    s += b;
    es += a;
    const float dm = s > 0.f ? fmaxf(run.R - m0, -256.f) : 0.f, f = lp_ex2(dm);
    es = f * fmaf(dm, s, es);
    s *= f;
    const float dd = fmaxf(fmaf(xe, P.c, -m0), -256.f), p = lp_ex2(dd);
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
  if (split) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  // join over the block: the maxima first, then the sums at the block's maximum
  float bx = warp_max(nan ? -CUDART_INF_F : m);
  if (lane == 0) red_m[w] = bx;
  const bool any = u0 + t < u1 || lone;              // this thread holds an element
  int size = 8;
  if (TOP) {
    // the maximum of 8 threads each, of fewer when few hold a unit: at least 32
    // groups that hold something, at most 64
    while (size > 1 && u1 - u0 < 32 * size) size /= 2;
    uint32_t k = any ? lp_key(m) : 0u;
    if (size == 8) {
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
    } else {
#pragma unroll 1
      for (int o = size / 2; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
    }
    if (t % size == 0 && t / size < LP_GROUPS) group_k[t / size] = k;
  }
  __syncthreads();
  bx = red_m[0];
#pragma unroll
  for (int q = 1; q < LP_WARPS; ++q) bx = fmaxf(bx, red_m[q]);
  const float bm = bx * P.c;
  const bool wild = !(fabsf(bm) <= LP_TAME) && fabsf(bx) < CUDART_INF_F;
  float sj, ej;
  if (wild) {
    // No float is near enough to the maximum's x c: once more over the part (from
    // L2, or HBM), with d = (x - bx) c, which is 0 at the maximum.
    sj = ej = 0.f;
    auto add = [&](float x) {
      const float d = fmaxf((x - bx) * P.c, -256.f), p = lp_ex2(d);
      sj += p;
      ej = fmaf(d, p, ej);
    };
#pragma unroll 1
    for (int v = u0 + t; v < u1; v += LP_THREADS) {
      const uint4 d = __ldg(body + v);
      const uint32_t x[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < Wd::N; ++e) add(Wd::get(x[q], e));
    }
    if (lone) add(xe);
  } else {
    const float dm = lp_hold(ms - bm), f = lp_ex2(dm);
    sj = f * s;
    ej = f * fmaf(dm, s, es);
    if (ms == -CUDART_INF_F) sj = ej = 0.f;          // nothing above -inf
  }
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
    // the largest group maximum with n group maxima at or above it
    const uint32_t mine = group_k[lane];
    uint32_t at_or_above = 0u;                       // a group maximum with n at or above it
    if (size == 8) {
      int above = 0;
#pragma unroll
      for (int q = 0; q < LP_THREADS / 8; ++q) above += group_k[q] >= mine;
      if (above >= P.top) at_or_above = mine;
    } else {
      const uint32_t mine2 = group_k[lane + 32];
      int above = 0, above2 = 0;
#pragma unroll 1
      for (int q = 0; q < LP_GROUPS; ++q) {
        above += group_k[q] >= mine;
        above2 += group_k[q] >= mine2;
      }
      at_or_above = max(above >= P.top ? mine : 0u, above2 >= P.top ? mine2 : 0u);
    }
    const uint32_t thr = max(__reduce_max_sync(0xffffffffu, at_or_above), 1u);
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
    sort_top<LP_THREADS>(list, found, P.top,
                         (split ? cluster.map_shared_rank(part_keys, 0) : part_keys) + part * P.top,
                         &counter);
  } else {
    __syncthreads();
  }
  if (t == 0) {
    LpPart o;
    o.ref = wild ? (double)bx * (double)P.c : (double)bm;
    o.s = 0.f;
    o.e = 0.f;
    o.ahead = 0;
#pragma unroll
    for (int q = 0; q < LP_WARPS; ++q) {
      o.s += red_s[q];
      o.e += red_e[q];
      o.ahead += red_c[q];
    }
    (split ? cluster.map_shared_rank(parts, 0) : parts)[part] = o;
  }
  // the cluster's first CTA joins; the others leave once all have delivered
  if (split) cluster.sync(); else __syncthreads();
  if (part != 0) return;
  if (t == 0) {
    double rm = -CUDART_INF;
    float rs = 0.f, re = 0.f;
    int ra = 0;
    for (int i = 0; i < nparts; ++i) rm = fmax(rm, parts[i].ref);
    for (int i = 0; i < nparts; ++i) {
      const LpPart q = parts[i];
      ra += q.ahead;
      if (q.ref == -CUDART_INF && q.s == q.s) continue;          // nothing above -inf, no NaN
      const float dj = (float)fmax(q.ref - rm, -256.0), fj = lp_ex2(dj);
      rs = fmaf(fj, q.s, rs);
      re = fmaf(fj, fmaf(dj, q.s, q.e), re);
    }
    // every entry is -inf, or one +inf: NaN, as the formula
    const bool none = !(fabs(rm) < CUDART_INF);
    const float lz = none ? CUDART_NAN_F : log2f(rs);
    sh_ref = rm;
    sh_lz = lz;
    const float h = 0.69314718055994531f * (lz - re / rs);
    P.entropy[r] = h < 0.f ? 0.f : h;
    P.rank[r] = have ? (int64_t)ra : 0;
    P.logprob[r] = have ? lp_final(xt, P.c, rm, lz) : CUDART_NAN_F;
  }
  if (!TOP) return;
  __syncthreads();
  if (t < nparts * P.top) {
    const unsigned long long key = part_keys[t];
    int rank = 0;
    if (nparts == 1) {
      rank = t;                                      // sorted already
    } else {
      for (int q = 0; q < nparts * P.top; ++q) rank += part_keys[q] > key;
    }
    if (rank < P.top) {                              // absent keys (0) rank behind the V >= n real ones
      P.top_ids[r * P.top + rank] = (int64_t)(uint32_t)~(uint32_t)key;
      P.top_lp[r * P.top + rank] =
          lp_final(lp_value((uint32_t)(key >> 32)), P.c, sh_ref, sh_lz);
    }
  }
}

__device__ __forceinline__ float lp_f(float x) { return x; }
__device__ __forceinline__ float lp_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float lp_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ unsigned long long lp_entry(float x, int idx) {
  return ((unsigned long long)lp_key(x) << 32) | (uint32_t)~(uint32_t)idx;
}

// Small vocabularies, up to 32 NE entries: a warp per row, the row in its
// registers (entry 32 i + lane in x[i]).  Of 64 maxima, of the lanes' even and odd
// entries, the n-th largest has at least n entries at or above it (some 45 for n =
// 32): those go to the warp's list and are ranked there; when it is too short (flat
// logits), the n largest one after the other.
// Bound by the loads' latency and the list.
template <typename T, int NE>
__global__ void __launch_bounds__(LP_THREADS) logp_warp_kernel(const LpParams P, int64_t rows) {
  __shared__ unsigned long long lists[LP_WARPS][LP_WLIST];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, V = P.V;
  const int64_t r = (int64_t)blockIdx.x * LP_WARPS + w;
  if (r >= rows) return;
  const int64_t rb = r / P.L, rl = r - rb * P.L;
  const T* row = reinterpret_cast<const T*>(P.x) + rb * P.bs + rl * P.ps;
  const int64_t tok = P.ids[rb * P.ids_bs + rl];
  float x[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int idx = 32 * i + lane;
    x[i] = idx < V ? lp_f(row[idx]) : -CUDART_INF_F;
  }
  const bool have = tok >= 0 && tok < V;
  const float xt = have ? lp_f(row[tok]) : CUDART_INF_F;
  const uint32_t kt = lp_key(xt);
  uint32_t mk[2] = {0u, 0u};                         // the largest keys of the even and odd i
  int ahead = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int idx = 32 * i + lane;
    if (idx >= V) break;
    const uint32_t k = lp_key(x[i]);
    mk[i & 1] = max(mk[i & 1], k);
    ahead += k > kt || (k == kt && idx <= tok);
  }
  ahead = warp_sum(ahead);
  const uint32_t wk = __reduce_max_sync(0xffffffffu, max(mk[0], mk[1]));
  const float m = lp_value(wk);                      // (a NaN's key: NaN)
  const bool finite = fabsf(m) < CUDART_INF_F;
  const float m0 = finite ? m : 0.f;
  float s0 = 0.f, s1 = 0.f, e0 = 0.f, e1 = 0.f;
#pragma unroll
  for (int i = 0; i < NE; i += 2) {
    const float a = fmaxf((x[i] - m0) * P.c, -256.f), b = fmaxf((x[i + 1] - m0) * P.c, -256.f);
    const float pa = lp_ex2(a), pb = lp_ex2(b);
    s0 += pa;
    s1 += pb;
    e0 = fmaf(a, pa, e0);
    e1 = fmaf(b, pb, e1);
  }
  const float rs = warp_sum(s0 + s1), re = warp_sum(e0 + e1);
  // all -inf, +inf or NaN among them: as the formula, NaN
  const float lz = finite ? log2f(rs) : CUDART_NAN_F;
  const double ref = (double)m * (double)P.c;
  if (lane == 0) {
    const float h = 0.69314718055994531f * (lz - re / rs);
    P.entropy[r] = h < 0.f ? 0.f : h;
    P.rank[r] = have ? (int64_t)ahead : 0;
    P.logprob[r] = have ? lp_final(xt, P.c, ref, lz) : CUDART_NAN_F;
  }
  const int n = P.top;
  if (n == 0) return;
  unsigned long long* list = lists[w];
  int above[2] = {0, 0};
#pragma unroll 4
  for (int q = 0; q < 32; ++q) {
    const uint32_t a = __shfl_sync(0xffffffffu, mk[0], q), b = __shfl_sync(0xffffffffu, mk[1], q);
    above[0] += (a >= mk[0]) + (b >= mk[0]);
    above[1] += (a >= mk[1]) + (b >= mk[1]);
  }
  // (a group without an entry has the key 0; n <= V groups or 32 hold one)
  const uint32_t thr = max(__reduce_max_sync(0xffffffffu, max(above[0] >= n ? mk[0] : 0u,
                                                             above[1] >= n ? mk[1] : 0u)), 1u);
  int cnt = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    if (32 * i >= V) break;
    const bool hit = 32 * i + lane < V && lp_key(x[i]) >= thr;
    const uint32_t hits = __ballot_sync(0xffffffffu, hit);
    const int at = cnt + __popc(hits & ((1u << lane) - 1u));
    if (hit && at < LP_WLIST) list[at] = lp_entry(x[i], 32 * i + lane);
    cnt += __popc(hits);
  }
  auto put = [&](int rank, unsigned long long key) {
    P.top_ids[r * n + rank] = (int64_t)(uint32_t)~(uint32_t)key;
    P.top_lp[r * n + rank] = lp_final(lp_value((uint32_t)(key >> 32)), P.c, ref, lz);
  };
  __syncwarp();
  if (cnt <= LP_WLIST) {
    for (int i = lane; i < cnt; i += 32) {
      const unsigned long long key = list[i];
      int rank = 0;
      for (int j = 0; j < cnt; ++j) rank += list[j] > key;
      if (rank < n) put(rank, key);
    }
    return;
  }
  unsigned long long last = ~0ULL;
  for (int k = 0; k < n; ++k) {
    unsigned long long best = 0ULL;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      if (32 * i + lane >= V) break;
      const unsigned long long key = lp_entry(x[i], 32 * i + lane);
      if (key < last && key > best) best = key;
    }
    last = warp_max(best);
    if (lane == 0) put(k, last);
  }
}

// How the rows are cut.  Up to one row per SM, every row is split, over as many
// CTAs as fit the machine at once; beyond, whole rows while there is one for
// every SM and the rest in halves, so that the SMs end together.  Clusters of four
// do not fill all of the machine's 592 places (four CTAs per SM): 142 of them run
// at once, so four parts end at 15/16 of the places, 138 rows.  Measured (bf16, V =
// 151936, five alternatives; us): 8 rows in 8 parts 8.5, in 4 8.8, in 2 11.4, in 1
// 15.5; 18 rows in 8 9.5, in 4 9.7; 30 rows in 4 10.9, in 2 13.7; 100 rows in 4
// 14.5, in 2 17.0, in 1 21.0; 138 rows in 4 17.3, in 2 17.8; 142 in 4 17.4, 143 in 4
// 21.5, in 2 18.1; 148 rows in 4 22.2, in 2 18.1, in 1 21.9; 320 rows, 296 of
// them whole and 24 in halves 29.2, all whole 33.5, all in halves 37.1 (700 rows:
// 51, 55.5, 60.7).  Shorter rows gain less: 111 rows of 32003 fp32 take 12.7 in 4
// parts and 12.1 in 2, 37 rows 9.6 and 9.9.  A part has at least a unit per thread.
struct LpPlan { int csize, whole; int64_t ctas; };
static LpPlan lp_plan(int64_t rows, int V, int dtype) {
  const int units = V / (dtype == SD_DTYPE_F32 ? 4 : 8);
  LpPlan p = {2, 0, 0};
  if (rows * 8 <= LP_SMS)
    p.csize = 8;
  else if (rows * 4 <= LP_SMS * LP_CTAS * 15 / 16)
    p.csize = 4;
  while (p.csize > 1 && units / p.csize < LP_THREADS) p.csize /= 2;
  const int64_t full = p.csize == 1 ? rows : rows <= LP_SMS ? 0 : rows / LP_SMS * LP_SMS;
  p.whole = (int)(full / p.csize);
  p.ctas = full + (rows - full) * p.csize;
  return p;
}

// Up to LP_WARP_V entries a warp takes a row: 4000 rows of 300 bf16 in 5.1 us (a CTA
// each: 27.8), 4000 x 1000 9.3 (28.0), with five alternatives 18.9 (70.6), 1000 x 1000
// with five 8.6 (20.7), one row of 1000 with five 7.3 (8.1), without 3.7 (3.5).  Beyond,
// 64 entries in a thread's registers leave one CTA per SM: 4000 x 2000 bf16 in 25 us
// against 28, with five alternatives 52 against 70, but fp32 25 and 52 against 25 and
// 43.
template <typename T>
static int launch_warps(const LpParams& P, cudaStream_t st) {
  const int64_t rows = (int64_t)P.B * P.L, ctas = (rows + LP_WARPS - 1) / LP_WARPS;
  if (ctas > 0x7FFFFFFF) return SD_ENOTSUP;
  if (P.V <= 512)
    logp_warp_kernel<T, 16><<<(unsigned)ctas, LP_THREADS, 0, st>>>(P, rows);
  else
    logp_warp_kernel<T, 32><<<(unsigned)ctas, LP_THREADS, 0, st>>>(P, rows);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

template <typename T>
static int launch_logprobs(const LpParams& P, int64_t ctas, cudaStream_t st) {
  if (P.V <= LP_WARP_V) return launch_warps<T>(P, st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(LP_THREADS);
  cfg.dynamicSmemBytes = P.top > 0 ? LP_LIST * sizeof(unsigned long long) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)P.csize;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t rc = P.top > 0 ? cudaLaunchKernelEx(&cfg, logp_kernel<T, true>, P)
                                   : cudaLaunchKernelEx(&cfg, logp_kernel<T, false>, P);
  if (rc != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // namespace sd

using namespace sd;

extern "C" {

int sd_token_logprobs(const void* logits, int64_t bs, int64_t ps, int dtype, const int64_t* ids,
                      int64_t ids_bs, int B, int L, int V, float temperature, int top_n,
                      float* logprob, int64_t* rank, float* entropy, int64_t* top_ids,
                      float* top_logprobs, void* stream) {
  if (B < 0 || L < 0) return SD_EINVAL;
  if (B == 0 || L == 0) return SD_OK;
  if (!logits || !ids || !logprob || !rank || !entropy || V <= 0) return SD_EINVAL;
  if (dtype != SD_DTYPE_F32 && dtype != SD_DTYPE_F16 && dtype != SD_DTYPE_BF16) return SD_EINVAL;
  if (!(temperature >= 1e-6f && temperature <= 1e6f)) return SD_EINVAL;
  if (top_n < 0 || top_n > V || (top_n > 0 && (!top_ids || !top_logprobs))) return SD_EINVAL;
  const int64_t rows = (int64_t)B * L;
  if (V > SD_LOGPROBS_MAX_V || top_n > SD_TOPN_MAX) return SD_ENOTSUP;
  const LpPlan plan = lp_plan(rows, V, dtype);
  if (plan.ctas > 0x7FFFFFFF) return SD_ENOTSUP;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == SD_DTYPE_F32 ? 4 : 2)) return SD_EINVAL;
  LpParams P;
  P.x = logits; P.bs = bs; P.ps = ps; P.dtype = dtype;
  P.ids = ids; P.ids_bs = ids_bs;
  P.B = B; P.L = L; P.V = V; P.top = top_n;
  P.csize = plan.csize; P.whole = plan.whole;
  P.c = (float)(1.4426950408889634 / (double)temperature);
  P.logprob = logprob; P.rank = rank; P.entropy = entropy;
  P.top_ids = top_ids; P.top_lp = top_logprobs;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == SD_DTYPE_BF16) return launch_logprobs<__nv_bfloat16>(P, plan.ctas, st);
  if (dtype == SD_DTYPE_F16) return launch_logprobs<__half>(P, plan.ctas, st);
  return launch_logprobs<float>(P, plan.ctas, st);
}

}  // extern "C"
