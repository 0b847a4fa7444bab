// Constraints on logits (sm_100a): penalties for repeated tokens, biases and
// grammar masks at every position of a verify or draft forward, and the token
// history behind the penalties.
//
//   x = logit;  seen (in the prompt, written, or on the node's path):
//   x = x > 0 ? x / r : x r;  x -= f c;  x -= p [c > 0];  x += bias;  x = -inf where not allowed
//
// What it has to move is a logit in and out (and, per row, 16 bits of history per
// token; per position, one bit of mask), so HBM bounds it while paths and biases touch few
// entries.  A CTA takes a chunk of a row's vocabulary for up to LG_POS positions and passes
// over it once: 16-byte units of the input, wherever they start in the row (rows of an odd
// vocabulary are aligned differently), with -inf for what the mask bans; a unit that it bans
// whole is written without being read.  Tokens that have a history (some thousand of 151936)
// get their penalties on the way: the CTA takes the chunk's history to shared memory once for
// all its positions, with a bit per token, and a thread loops over the bits of its unit.  The
// tokens of the position's path and the biases are written over what the pass left; where
// out is the logits themselves, they have been computed before the pass.
// 320 positions of 151936 bf16 logits, 64 rows of history, masks, 16 biases (220 MB): 46.9 us
// (fp16 47.2, fp32 68.0), 832 positions (531 MB): 101 us; without history and biases 32 and
// 79, a copy's rate.  What is left is the penalties' arithmetic (3 and 5 us), the history's way
// to shared memory ahead of the pass, and the sparse entries behind it.  In place a CTA takes
// one position, and so the history to shared memory for each: 73.8 and 162 us.
// A touched entry costs a walk over its row's N tokens and M biases, so a position's cost
// grows by (N + M)^2: 320 positions with 300 biases take 261 us, with 1024 2.5 ms, 832 positions
// 703 us and 6.2 ms; 256 rows of 64 nodes over a vocabulary of 1000 (65 MB) 107 us without
// biases, 909 us with 300.
// Measured and left: the tokens with a history listed and written over the pass's output
// (47.3 and 111; 33 instead of 23 for fp32 rows of 32003), units asked for a position ahead
// (51, 108: fewer CTAs fit), one run of positions per resident CTA (60, 121), the history
// looked up in global memory for every unit (60, 127) or for the units whose bits are set
// (53, 110).
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>

#include "sd_common.cuh"
#include "sd_tree.cuh"

namespace sd {

constexpr int LG_THREADS = 256;
constexpr int LG_UNITS = 4;                  // most 16-byte units per thread and position
constexpr int LG_AHEAD = 4;                  // units whose loads are on their way at once
constexpr int LG_POS = 8;                    // most positions of a CTA
constexpr int LG_CTAS = 4 * 148;             // enough CTAs: four per SM
constexpr int LG_CHUNK = LG_UNITS * LG_THREADS * 8;          // most tokens of a chunk

struct LogitsParams {
  const void* logits; int64_t bs, ps;
  int B, L, V;
  const int64_t* tokens; int64_t tokens_bs;
  const int32_t* masks; int64_t mask_bs;
  int N, W, first;
  const int16_t* history; int64_t history_bs;
  const float* repetition; const float* presence; const float* frequency;
  const int64_t* bias_ids; const float* bias_values; int64_t bias_bs; int M;
  const int32_t* allowed; int64_t allowed_bs, allowed_ps;
  void* out; int64_t out_bs, out_ps;
  int chunk, chunks;                         // elements of a CTA's chunk, chunks of a position
  int lg, groups;                            // positions of a CTA, CTAs along the positions
};

template <int DT> struct LgType;
template <> struct LgType<SD_DTYPE_F32> { using T = float; };
template <> struct LgType<SD_DTYPE_F16> { using T = __half; };
template <> struct LgType<SD_DTYPE_BF16> { using T = __nv_bfloat16; };
__device__ __forceinline__ float lg_in(float x) { return x; }
__device__ __forceinline__ float lg_in(__half x) { return __half2float(x); }
__device__ __forceinline__ float lg_in(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void lg_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void lg_out(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void lg_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// A unit with -inf for the elements whose bit of `on` is 0: 16-bit ones by a byte permutation of
// a word and a pair of -inf, whose selector is 0x3210 where both stay and 0x7654 where none does.
template <int DT>
__device__ __forceinline__ uint4 lg_ban(uint4 v, uint32_t on) {
  if constexpr (DT == SD_DTYPE_F32) {
    const uint32_t none = 0xFF800000u;
    return make_uint4(on & 1u ? v.x : none, on & 2u ? v.y : none, on & 4u ? v.z : none, on & 8u ? v.w : none);
  } else {
    const uint32_t none = DT == SD_DTYPE_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
    auto pick = [&](uint32_t word, uint32_t two) {
      return __byte_perm(word, none, 0x7654u - 0x44u * ((two | two << 7) & 0x101u));
    };
    return make_uint4(pick(v.x, on & 3u), pick(v.y, (on >> 2) & 3u), pick(v.z, (on >> 4) & 3u),
                      pick(v.w, (on >> 6) & 3u));
  }
}

struct LgPenalty {
  float r, p, f;
  __device__ __forceinline__ float operator()(float x, int h, int path) const {
    const int c = (h & 0x7FFF) + path;
    if (c > 0 || h < 0) {
      x = x > 0.f ? __fdiv_rn(x, r) : x * r;
      x -= f * (float)c;
      if (c > 0) x -= p;
    }
    return x;
  }
};

// Eight bits from bit `at` on of a bit string whose last word is `last`.
__device__ __forceinline__ uint32_t lg_bits(const uint32_t* p, int at, int last) {
  const int w = at >> 5;
  return __funnelshift_r(p[w], p[min(w + 1, last)], at & 31);
}

// What a CTA knows of a position: its node's path and how its tokens become logits.
struct LgPosition {
  const int32_t* mask;                               // the node's ancestor bits; null: a chain
  int node;
};
__device__ __forceinline__ bool lg_on_path(const LogitsParams& P, const LgPosition& q, int i) {
  return q.mask ? (tree_word(q.mask, P.W, P.N, i >> 5) >> (i & 31)) & 1u : i <= q.node;
}
// Entry id of a position, in full: its history, its path, its biases, its mask.
template <typename T>
__device__ __forceinline__ float lg_entry(const LogitsParams& P, const LgPosition& q, const LgPenalty& pen,
                                       const T* x, const int16_t* hist, const uint32_t* allow, int b,
                                       int id) {
  float z = lg_in(x[id]);
  if (hist) {
    int c = 0;
    for (int i = 0; i < P.N; ++i)
      c += P.tokens[b * P.tokens_bs + i] == id && lg_on_path(P, q, i);
    z = pen(z, hist[id], c);
  }
  float bias = 0.f;                                  // (in the list's order: the same sum every time)
  for (int k = 0; k < P.M; ++k)
    if (P.bias_ids[b * P.bias_bs + k] == id) bias += P.bias_values[b * P.bias_bs + k];
  z += bias;
  return !allow || ((allow[id >> 5] >> (id & 31)) & 1u) ? z : -CUDART_INF_F;
}

// Element j of a unit with its penalties.
template <int DT>
__device__ __forceinline__ void lg_penalize(uint4& v, int j, const LgPenalty& pen, int h) {
  if constexpr (DT == SD_DTYPE_F32) {
    const uint32_t z = __float_as_uint(pen(__uint_as_float(j & 2 ? (j & 1 ? v.w : v.z) : (j & 1 ? v.y : v.x)), h, 0));
    if (j == 0) v.x = z;
    if (j == 1) v.y = z;
    if (j == 2) v.z = z;
    if (j == 3) v.w = z;
  } else {
    using T = typename LgType<DT>::T;
    const uint32_t word = j & 4 ? (j & 2 ? v.w : v.z) : (j & 2 ? v.y : v.x);
    const unsigned short in = (unsigned short)(word >> (16 * (j & 1)));
    T out;
    lg_out(&out, pen(lg_in(*reinterpret_cast<const T*>(&in)), h, 0));
    const uint32_t z =
        __byte_perm(word, *reinterpret_cast<const unsigned short*>(&out), j & 1 ? 0x5410 : 0x3254);
    const int w = j >> 1;
    if (w == 0) v.x = z;
    if (w == 1) v.y = z;
    if (w == 2) v.z = z;
    if (w == 3) v.w = z;
  }
}

// INPLACE: out is the logits (one position per CTA; what is sparse is computed before the pass)
template <int DT, bool INPLACE>
__global__ void __launch_bounds__(LG_THREADS, INPLACE ? 5 : 6) process_logits_kernel(const __grid_constant__ LogitsParams P) {
  using T = typename LgType<DT>::T;
  constexpr int E = 16 / sizeof(T);                  // elements of a unit
  constexpr uint32_t ALL = (1u << E) - 1u;
  constexpr int SPARSE = INPLACE ? SD_TREE_MAX + SD_BIAS_MAX : 1;
  // the chunk's history, and which of its tokens have one
  __shared__ __align__(16) int16_t past[LG_CHUNK];
  __shared__ uint32_t some[LG_CHUNK / 32 + 1];
  __shared__ int at[SPARSE];
  __shared__ float val[SPARSE];
  __shared__ int n_at;
  const int t = threadIdx.x;
  const int chunk = (int)(blockIdx.x % P.chunks), bg = (int)(blockIdx.x / P.chunks);
  const int b = bg / P.groups, l0 = (bg - b * P.groups) * P.lg, nl = min(P.lg, P.L - l0);
  const int c0 = chunk * P.chunk, c1 = min(P.V, c0 + P.chunk);
  const int16_t* hist = P.history ? P.history + b * P.history_bs : nullptr;
  LgPenalty pen = {1.f, 0.f, 0.f};
  if (hist) {
    if (P.repetition) pen.r = P.repetition[b];
    if (P.presence) pen.p = P.presence[b];
    if (P.frequency) pen.f = P.frequency[b];
  }
  auto logits = [&](int l) { return reinterpret_cast<const T*>(P.logits) + b * P.bs + (int64_t)l * P.ps; };
  auto output = [&](int l) { return reinterpret_cast<T*>(P.out) + b * P.out_bs + (int64_t)l * P.out_ps; };
  auto mask = [&](int l) {
    return P.allowed ? reinterpret_cast<const uint32_t*>(P.allowed) + b * P.allowed_bs +
                           (int64_t)l * P.allowed_ps : nullptr;
  };
  auto position = [&](int l) {
    const int node = P.first + l;
    return LgPosition{P.masks ? P.masks + b * P.mask_bs + (int64_t)node * P.W : nullptr, node};
  };
  if (hist) {
    // eight tokens a thread; behind the chunk's end 0
    const bool vec = (reinterpret_cast<uintptr_t>(hist) & 15) == 0;
    unsigned char* bits = reinterpret_cast<unsigned char*>(some);
#pragma unroll 1
    for (int i = t; i < P.chunk / 8 + 4; i += LG_THREADS) {
      const int e = c0 + 8 * i, n = min(8, c1 - e);
      uint32_t h[4] = {0u, 0u, 0u, 0u};
      if (vec && n == 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(hist + e));
        h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) h[k >> 1] |= (uint32_t)(unsigned short)hist[e + k] << (16 * (k & 1));
      }
      uint32_t on = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) on |= (uint32_t)(((h[k >> 1] >> (16 * (k & 1))) & 0xFFFFu) != 0u) << k;
      bits[i] = (unsigned char)on;
      if (8 * i < P.chunk) *reinterpret_cast<uint4*>(&past[8 * i]) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
  if (INPLACE && t == 0) n_at = 0;
  __syncthreads();
  // the entries that a position's path or the biases touch
  const int np = hist ? P.N : 0;
  auto sparse_id = [&](const LgPosition& q, int i) -> int {
    int64_t id = -1;
    if (i < np) {
      if (lg_on_path(P, q, i)) id = P.tokens[b * P.tokens_bs + i];
    } else {
      id = P.bias_ids[b * P.bias_bs + i - np];
    }
    return id >= c0 && id < c1 ? (int)id : -1;
  };
  if (INPLACE) {
    const LgPosition q = position(l0);
    for (int i = t; i < np + P.M; i += LG_THREADS) {
      const int id = sparse_id(q, i);
      if (id < 0) continue;
      const int k = atomicAdd(&n_at, 1);
      at[k] = id;
      val[k] = lg_entry(P, q, pen, logits(l0), hist, mask(l0), b, id);   // (twice: the same value)
    }
    __syncthreads();
  }
  // ---- the pass, position by position: 16-byte units of the input, wherever they start in the row
  const int words = (P.V + 31) / 32 - 1;
#pragma unroll 1
  for (int l = l0; l < l0 + nl; ++l) {
    const T* x = logits(l) + c0;
    T* y = output(l) + c0;
    const int head = (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15)) & 15u) / (int)sizeof(T);
    const int nu = c0 + head <= c1 ? (c1 - c0 - head) / E : 0;
    const uint32_t* allow = mask(l);
    x += head;
    y += head;
    const bool wide = (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll 1
    for (int u0 = t; u0 < nu; u0 += LG_THREADS * LG_AHEAD) {
      uint4 v[LG_AHEAD];
      uint32_t on[LG_AHEAD];
#pragma unroll
      for (int k = 0; k < LG_AHEAD; ++k) {
        const int u = u0 + k * LG_THREADS;
        on[k] = u < nu ? ALL : 0u;
        if (allow && u < nu) on[k] = lg_bits(allow, c0 + head + u * E, words) & ALL;
      }
#pragma unroll
      for (int k = 0; k < LG_AHEAD; ++k) {
        v[k] = make_uint4(0u, 0u, 0u, 0u);
        if (on[k]) v[k] = (reinterpret_cast<const uint4*>(x))[u0 + k * LG_THREADS];
      }
#pragma unroll
      for (int k = 0; k < LG_AHEAD; ++k) {
        const int u = u0 + k * LG_THREADS;
        if (u >= nu) continue;
        if (hist) {
          const int e = head + u * E;
          for (uint32_t which = lg_bits(some, e, LG_CHUNK / 32) & on[k]; which; which &= which - 1) {
            const int j = __ffs((int)which) - 1;
            lg_penalize<DT>(v[k], j, pen, past[e + j]);
          }
        }
        if (on[k] != ALL) v[k] = lg_ban<DT>(v[k], on[k]);
        if (wide) {
          reinterpret_cast<uint4*>(y)[u] = v[k];
        } else {
          const uint32_t word[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int j = 0; j < E; ++j) {
            if constexpr (E == 4) reinterpret_cast<uint32_t*>(y)[u * E + j] = word[j];
            else reinterpret_cast<unsigned short*>(y)[u * E + j] = (unsigned short)(word[j / 2] >> (16 * (j & 1)));
          }
        }
      }
    }
  }
  // the elements before the first and behind the last unit, at most 2 E - 2 of a position
  for (int i = t; i < nl * 2 * E; i += LG_THREADS) {
    const int l = l0 + i / (2 * E), k = i % (2 * E);
    const T* x = logits(l);
    const int head = (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(x + c0) & 15)) & 15u) / (int)sizeof(T);
    const int body = c0 + head <= c1 ? (c1 - c0 - head) / E * E : 0;
    int e;
    if (k < E) e = k < head ? c0 + k : -1;
    else e = c0 + head + body + k - E;
    if (e < 0 || e >= c1) continue;
    const uint32_t* allow = mask(l);
    T* y = output(l) + e;
    if (allow && !((allow[e >> 5] >> (e & 31)) & 1u)) lg_out(y, -CUDART_INF_F);
    else if (hist) lg_out(y, pen(lg_in(x[e]), past[e - c0], 0));
    else *y = x[e];
  }
  if (np + P.M == 0) return;
  __syncthreads();
  if (INPLACE) {
    for (int k = t; k < n_at; k += LG_THREADS) lg_out(&output(l0)[at[k]], val[k]);
  } else {
    for (int i = t; i < nl * (np + P.M); i += LG_THREADS) {
      const int l = l0 + i / (np + P.M);
      const LgPosition q = position(l);
      const int id = sparse_id(q, i % (np + P.M));
      if (id >= 0) lg_out(&output(l)[id], lg_entry(P, q, pen, logits(l), hist, mask(l), b, id));
    }
  }
}

// A thread per token.  Counts stop at 32767; order does not matter.
__global__ void __launch_bounds__(256)
history_add_kernel(int16_t* history, int64_t history_bs, int V, const int64_t* ids, int64_t ids_bs,
                   int n_ids, const int32_t* path, int64_t path_bs, const int64_t* counts, int n,
                   int prompt) {
  const int b = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n || (counts && i >= counts[b])) return;
  int k = i;
  if (path) {
    k = path[b * path_bs + i];
    if ((unsigned)k >= (unsigned)n_ids) return;
  }
  const int64_t id = ids[b * ids_bs + k];
  if (id < 0 || id >= V) return;
  unsigned short* p = reinterpret_cast<unsigned short*>(history + b * history_bs + id);
  unsigned short old = *reinterpret_cast<volatile unsigned short*>(p);
  while (true) {
    const unsigned short add = prompt ? (unsigned short)(old | 0x8000u)
                                      : (unsigned short)((old & 0x7FFFu) == 0x7FFFu ? old : old + 1);
    if (add == old) return;
    const unsigned short was = atomicCAS(p, old, add);
    if (was == old) return;                          // (else another thread got through)
    old = was;
  }
}

}  // namespace sd

using namespace sd;

extern "C" {

int sd_process_logits(const void* logits, int64_t bs, int64_t ps, int dtype, int B, int L, int V,
                      const int64_t* tokens, int64_t tokens_bs, const int32_t* masks,
                      int64_t mask_bs, int N, int first, const int16_t* history,
                      int64_t history_bs, const float* repetition, const float* presence,
                      const float* frequency, const int64_t* bias_ids, const float* bias_values,
                      int64_t bias_bs, int M, const int32_t* allowed, int64_t allowed_bs,
                      int64_t allowed_ps, void* out, int64_t out_bs, int64_t out_ps,
                      void* stream) {
  if (B < 0 || L < 0 || V < 1 || N < 0 || M < 0 || first < 0) return SD_EINVAL;
  if (B == 0 || L == 0) return SD_OK;
  if (!logits || !out) return SD_EINVAL;
  if (dtype != SD_DTYPE_F32 && dtype != SD_DTYPE_F16 && dtype != SD_DTYPE_BF16) return SD_EINVAL;
  if (N > 0 && (!tokens || first + L > N)) return SD_EINVAL;
  if (M > 0 && (!bias_ids || !bias_values)) return SD_EINVAL;
  if (N > SD_TREE_MAX || M > SD_BIAS_MAX || V > 1 << 30) return SD_ENOTSUP;
  LogitsParams P = {};
  P.logits = logits; P.bs = bs; P.ps = ps; P.B = B; P.L = L; P.V = V;
  P.tokens = tokens; P.tokens_bs = tokens_bs; P.masks = masks; P.mask_bs = mask_bs;
  P.N = N; P.W = (N + 31) / 32; P.first = first;
  P.history = history; P.history_bs = history_bs;
  P.repetition = repetition; P.presence = presence; P.frequency = frequency;
  P.bias_ids = bias_ids; P.bias_values = bias_values; P.bias_bs = bias_bs; P.M = M;
  P.allowed = allowed; P.allowed_bs = allowed_bs; P.allowed_ps = allowed_ps;
  P.out = out; P.out_bs = out_bs; P.out_ps = out_ps;
  const int E = dtype == SD_DTYPE_F32 ? 4 : 8, size = 16 / E;
  // the memory of one may overlap the other's: a CTA has to read its sparse entries first
  auto span = [&](const void* p, int64_t s0, int64_t s1, uintptr_t* lo, uintptr_t* hi) {
    const int64_t d0 = (B - 1) * s0 * size, d1 = (L - 1) * s1 * size, base = (int64_t)(uintptr_t)p;
    *lo = (uintptr_t)(base + std::min<int64_t>(d0, 0) + std::min<int64_t>(d1, 0));
    *hi = (uintptr_t)(base + std::max<int64_t>(d0, 0) + std::max<int64_t>(d1, 0) + (int64_t)V * size);
  };
  uintptr_t a0, a1, b0, b1;
  span(logits, bs, ps, &a0, &a1);
  span(out, out_bs, out_ps, &b0, &b1);
  const bool inplace = a0 < b1 && b0 < a1;
  // the same elements, or memory that a position may be read from after it was written
  if (inplace && (logits != out || (B > 1 && bs != out_bs) || (L > 1 && ps != out_ps))) return SD_EINVAL;
  // one CTA per entry of the output
  if (!rows_apart<2>(V, {B, L}, {out_bs, out_ps})) return SD_EINVAL;
  if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & (size - 1)) return SD_EINVAL;
  // a chunk is up to 4 units per thread, and a CTA takes up to 8 positions, less where that would
  // leave SMs without a CTA: first the positions, then the chunk
  int units = LG_UNITS;
  P.lg = inplace ? 1 : std::min(L, LG_POS);
  auto ctas = [&]() {
    P.chunk = units * LG_THREADS * E;
    P.chunks = (V + P.chunk - 1) / P.chunk;
    P.groups = (L + P.lg - 1) / P.lg;
    return (int64_t)B * P.groups * P.chunks;
  };
  while (P.lg > 1 && ctas() < 2 * LG_CTAS) P.lg = (P.lg + 1) / 2;
  while (units > 1 && ctas() < LG_CTAS) units /= 2;
  const int64_t grid = ctas();
  if ((double)B * P.groups * P.chunks > 0x7FFFFFFF) return SD_ENOTSUP;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) { kernel<<<(unsigned)grid, LG_THREADS, 0, st>>>(P); };
  if (dtype == SD_DTYPE_F32)
    inplace ? go(process_logits_kernel<SD_DTYPE_F32, true>) : go(process_logits_kernel<SD_DTYPE_F32, false>);
  else if (dtype == SD_DTYPE_F16)
    inplace ? go(process_logits_kernel<SD_DTYPE_F16, true>) : go(process_logits_kernel<SD_DTYPE_F16, false>);
  else
    inplace ? go(process_logits_kernel<SD_DTYPE_BF16, true>) : go(process_logits_kernel<SD_DTYPE_BF16, false>);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

int sd_history_add(int16_t* history, int64_t history_bs, int V, const int64_t* ids,
                   int64_t ids_bs, int n_ids, const int32_t* path, int64_t path_bs,
                   const int64_t* counts, int n, int B, int prompt, void* stream) {
  if (B < 0 || n < 0 || V < 1 || n_ids < 0) return SD_EINVAL;
  if (B == 0 || n == 0) return SD_OK;
  if (!history || !ids) return SD_EINVAL;
  if (!path && n > n_ids) return SD_EINVAL;
  if (B > 65535) return SD_ENOTSUP;
  history_add_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)B), 256, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(
      history, history_bs, V, ids, ids_bs, n_ids, path, path_bs, counts, n, prompt);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // extern "C"
