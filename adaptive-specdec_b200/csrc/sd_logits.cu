// Constraints on logits (sm_100a): penalties for repeated tokens, biases and
// grammar masks at every position of a verify or draft forward, and the token
// history behind the penalties.
//
//   x = logit;  seen (in the prompt, written, or on the node's path):
//   x = x > 0 ? x / r : x r;  x -= f c;  x -= p [c > 0];  x += bias;  x = -inf where not allowed
//
// One pass: what it has to move is a logit in and out (and, per row, 16 bits of
// history per token; per position, one bit of mask), so HBM bounds it.  A CTA
// takes a chunk of one position's vocabulary.  Nearly every 16-byte unit of the
// history is zero (a row has written some thousand of 151936 tokens), so a unit is
// tested whole.  A unit that the mask bans whole is written without being read.
// What is sparse (the tokens of the path, the biases) is not looked up element by
// element: the CTA computes those of its chunk first, from the logits as they
// came, and writes them over what the pass left, so out may be the logits.
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>

#include "sd_common.cuh"
#include "sd_tree.cuh"

namespace sd {

constexpr int LG_THREADS = 256;
constexpr int LG_UNITS = 8;                  // most 16-byte units per thread
constexpr int LG_AHEAD = 4;                  // units whose loads are on their way at once

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

template <int DT>
__global__ void __launch_bounds__(LG_THREADS) process_logits_kernel(const __grid_constant__ LogitsParams P) {
  using T = typename LgType<DT>::T;
  constexpr int E = 16 / sizeof(T);                  // elements of a unit
  // the path's tokens, the biases, and the entries of this chunk that they touch
  __shared__ int path_tok[SD_TREE_MAX], bias_id[SD_BIAS_MAX];
  __shared__ float bias_val[SD_BIAS_MAX];
  __shared__ int at[SD_TREE_MAX + SD_BIAS_MAX];
  __shared__ float val[SD_TREE_MAX + SD_BIAS_MAX];
  __shared__ int n_path, n_at;
  const int t = threadIdx.x;
  const int chunk = (int)(blockIdx.x % P.chunks);
  const int64_t pos = blockIdx.x / P.chunks;
  const int b = (int)(pos / P.L), l = (int)(pos - (int64_t)b * P.L);
  const int c0 = chunk * P.chunk, c1 = min(P.V, c0 + P.chunk);
  const T* x = reinterpret_cast<const T*>(P.logits) + b * P.bs + l * P.ps;
  T* y = reinterpret_cast<T*>(P.out) + b * P.out_bs + l * P.out_ps;
  const int16_t* hist = P.history ? P.history + b * P.history_bs : nullptr;
  const uint32_t* allow = P.allowed ? reinterpret_cast<const uint32_t*>(P.allowed) +
                                          b * P.allowed_bs + l * P.allowed_ps : nullptr;
  LgPenalty pen = {1.f, 0.f, 0.f};
  if (hist) {
    if (P.repetition) pen.r = P.repetition[b];
    if (P.presence) pen.p = P.presence[b];
    if (P.frequency) pen.f = P.frequency[b];
  }
  const bool sparse = (hist && P.N > 0) || P.M > 0;
  if (sparse) {
    if (t == 0) n_path = n_at = 0;
    __syncthreads();
    const int node = P.first + l;
    if (hist) {
      const int32_t* m = P.masks ? P.masks + b * P.mask_bs + (int64_t)node * P.W : nullptr;
      for (int i = t; i < P.N; i += LG_THREADS) {
        const bool on = m ? (tree_word(m, P.W, P.N, i >> 5) >> (i & 31)) & 1u : i <= node;
        if (!on) continue;
        const int64_t id = P.tokens[b * P.tokens_bs + i];
        if (id >= 0 && id < P.V) path_tok[atomicAdd(&n_path, 1)] = (int)id;
      }
    }
    for (int i = t; i < P.M; i += LG_THREADS) {
      const int64_t id = P.bias_ids[b * P.bias_bs + i];
      bias_id[i] = id >= 0 && id < P.V ? (int)id : -1;
      bias_val[i] = P.bias_values[b * P.bias_bs + i];
    }
    __syncthreads();
    const int np = n_path;
    for (int i = t; i < np + P.M; i += LG_THREADS) {
      const int id = i < np ? path_tok[i] : bias_id[i - np];
      if (id < c0 || id >= c1) continue;
      int c = 0;
      for (int k = 0; k < np; ++k) c += path_tok[k] == id;
      float z = lg_in(x[id]);
      if (hist) z = pen(z, hist[id], c);
      float bias = 0.f;
      for (int k = 0; k < P.M; ++k)
        if (bias_id[k] == id) bias += bias_val[k];   // (in the list's order: the same sum every time)
      z += bias;
      if (allow && !((allow[id >> 5] >> (id & 31)) & 1u)) z = -CUDART_INF_F;
      const int k = atomicAdd(&n_at, 1);
      at[k] = id;
      val[k] = z;                                    // (an id that is there twice: the same value)
    }
    __syncthreads();
  }
  // units of 16 bytes where everything is aligned to them, else element by element
  const bool wide = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0 &&
                    (!hist || (reinterpret_cast<uintptr_t>(hist) & (2 * E - 1)) == 0);
  int e0 = c0;                                       // what the units leave
  if (wide) {
    const int nu = (c1 - c0) / E;
    for (int u0 = t; u0 < nu; u0 += LG_THREADS * LG_AHEAD) {
      uint32_t on[LG_AHEAD];
      uint4 v[LG_AHEAD];
      uint4 h[LG_AHEAD];
#pragma unroll
      for (int k = 0; k < LG_AHEAD; ++k) {
        const int u = u0 + k * LG_THREADS, e = c0 + u * E;
        on[k] = u < nu ? (1u << E) - 1u : 0u;
        if (allow && u < nu) on[k] &= __ldg(allow + (e >> 5)) >> (e & 31);
      }
#pragma unroll
      for (int k = 0; k < LG_AHEAD; ++k) {
        const int64_t e = c0 + (int64_t)(u0 + k * LG_THREADS) * E;
        v[k] = h[k] = make_uint4(0u, 0u, 0u, 0u);
        if (on[k]) {
          v[k] = __ldcs(reinterpret_cast<const uint4*>(x + e));
          if (hist) {
            if constexpr (E == 8) {
              h[k] = __ldg(reinterpret_cast<const uint4*>(hist + e));
            } else {
              const uint2 z = __ldg(reinterpret_cast<const uint2*>(hist + e));
              h[k].x = z.x;
              h[k].y = z.y;
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < LG_AHEAD; ++k) {
        const int u = u0 + k * LG_THREADS;
        if (u >= nu) continue;
        T* xe = reinterpret_cast<T*>(&v[k]);
        if ((h[k].x | h[k].y | h[k].z | h[k].w) != 0u) {
          const int16_t* he = reinterpret_cast<const int16_t*>(&h[k]);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (he[e] != 0) lg_out(&xe[e], pen(lg_in(xe[e]), he[e], 0));
        }
        if (on[k] != (1u << E) - 1u) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (!((on[k] >> e) & 1u)) lg_out(&xe[e], -CUDART_INF_F);
        }
        __stcs(reinterpret_cast<uint4*>(y + c0 + (int64_t)u * E), v[k]);
      }
    }
    e0 = c0 + nu * E;
  }
  for (int i0 = e0 + t; i0 < c1; i0 += LG_THREADS * LG_UNITS) {
    T v[LG_UNITS];
    int h[LG_UNITS];
    uint32_t on[LG_UNITS];
#pragma unroll
    for (int k = 0; k < LG_UNITS; ++k) {
      const int i = i0 + k * LG_THREADS;
      on[k] = 0u;
      h[k] = 0;
      if (i < c1) {
        v[k] = x[i];
        if (hist) h[k] = hist[i];
        on[k] = allow ? (__ldg(allow + (i >> 5)) >> (i & 31)) & 1u : 1u;
      }
    }
#pragma unroll
    for (int k = 0; k < LG_UNITS; ++k) {
      const int i = i0 + k * LG_THREADS;
      if (i >= c1) continue;
      if (!on[k]) lg_out(&y[i], -CUDART_INF_F);
      else if (h[k] != 0) lg_out(&y[i], pen(lg_in(v[k]), h[k], 0));
      else y[i] = v[k];
    }
  }
  if (sparse) {
    __syncthreads();
    for (int k = t; k < n_at; k += LG_THREADS) lg_out(&y[at[k]], val[k]);
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
  const int E = dtype == SD_DTYPE_F32 ? 4 : 8;
  // a chunk is 8 units per thread, less where that would leave SMs without a CTA
  int units = LG_UNITS;
  while (units > 1 && (int64_t)B * L * ((V + units * LG_THREADS * E - 1) / (units * LG_THREADS * E)) <
                          4 * 148)
    units /= 2;
  P.chunk = units * LG_THREADS * E;
  P.chunks = (V + P.chunk - 1) / P.chunk;
  const int64_t grid = (int64_t)B * L * P.chunks;
  if (grid > 0x7FFFFFFF) return SD_ENOTSUP;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == SD_DTYPE_F32)
    process_logits_kernel<SD_DTYPE_F32><<<(unsigned)grid, LG_THREADS, 0, st>>>(P);
  else if (dtype == SD_DTYPE_F16)
    process_logits_kernel<SD_DTYPE_F16><<<(unsigned)grid, LG_THREADS, 0, st>>>(P);
  else
    process_logits_kernel<SD_DTYPE_BF16><<<(unsigned)grid, LG_THREADS, 0, st>>>(P);
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
