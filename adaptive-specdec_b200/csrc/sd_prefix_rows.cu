// Attention over a paged cache, row by row on the CUDA cores (sm_100a): the
// shapes of prefix attention that the tensor-core path does not take (fp32, head
// sizes other than 128, very wide head groups).
//
// A cluster of S CTAs holds 8 query rows of one (row, kv head); their keys go out
// in groups of 32 to the cluster's 8 S warps in turn.  Per group a lane has one key:
//   s_r = scale log2(e) q_r . k        q_r from shared memory, k by the lane itself
//   p_r = 2^(s_r - m_r)                m_r the warp's running maximum
// and then, key by key, a lane has every 32nd column of V: acc_r += p_r v.  Each
// warp's (m, l, acc) are merged over the CTA in shared memory and over the cluster
// in distributed shared memory, in warp order: one launch, no workspace, and the
// same sums whatever runs beside it.
// What bounds a verify step is latency (one 32-key group after another in a warp),
// so S is as large as the machine has room for; with many rows the products (each
// K and V element meets only 8 rows).  8 rows of 3 queries, 8 / 2 heads of 64 over
// 460 fp32 keys: 14 us (the verify kernels, which split a row every 1024 keys, 134);
// 64 rows of 5 queries, 32 / 8 heads of 128 over 4096 keys: 2.3 ms, 9.3 TFLOP/s
// (4.9 ms).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>

#include "sd_attn.cuh"
#include "sd_common.cuh"

namespace sd {

constexpr int PR_ROWS = 8;                     // query rows of a cluster
constexpr int PR_WARPS = 8;
constexpr int PR_KEYS = 32;                    // keys of a group: one per lane
constexpr int PR_AHEAD = 8;                    // V rows on their way at once
constexpr int PR_CTAS = 2 * 148;               // enough CTAs: two per SM

__device__ __forceinline__ float pr_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pr_f(float x) { return x; }
__device__ __forceinline__ float pr_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float4 pr_load4(const float* p) {
  return __ldg(reinterpret_cast<const float4*>(p));
}
__device__ __forceinline__ float4 pr_load4(const __nv_bfloat16* p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void pr_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float pr_remote(const float* p, int rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}

// The merge of (m, l) pairs keeps a NaN sum whatever its maximum.
__device__ __forceinline__ float pr_weight(float m, float gm) {
  return m == -CUDART_INF_F ? 0.f : pr_ex2(m - gm);
}
__device__ __forceinline__ float pr_part(float f, float l) { return l != l ? l : f * l; }

// VEC: 16 (fp32) or 8 (bf16) byte loads of K, D a multiple of 4
template <typename T, int DV, bool VEC>
__global__ void __launch_bounds__(PR_WARPS * 32)
prefix_rows_kernel(const __grid_constant__ AttnParams P, int blocks, int S) {
  __shared__ __align__(16) float qs[PR_ROWS][32 * DV];
  __shared__ float accs[PR_WARPS][PR_ROWS][32 * DV];
  __shared__ float ms[PR_WARPS][PR_ROWS], ls[PR_WARPS][PR_ROWS];
  __shared__ float acc1[PR_ROWS][32 * DV], m1[PR_ROWS], l1[PR_ROWS];     // of the CTA
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, D = P.D;
  const int rank = (int)(blockIdx.x % S), unit = (int)(blockIdx.x / S);
  const int rb = unit % blocks, bh = unit / blocks, b = bh / P.Hkv, h = bh - b * P.Hkv;
  const int r0 = rb * PR_ROWS, R = min(PR_ROWS, P.R - r0);
  const float sl2 = P.scale * 1.4426950408889634f;
  for (int i = t; i < PR_ROWS * 32 * DV; i += PR_WARPS * 32) {
    const int r = i / (32 * DV), d = i % (32 * DV);
    float x = 0.f;
    if (r < R && d < D) {
      const int j = (r0 + r) / P.group, hq = h * P.group + (r0 + r) % P.group;
      x = pr_f(reinterpret_cast<const T*>(P.q)[b * P.qbs + hq * P.qhs + j * P.qqs + d]) * sl2;
    }
    qs[r][d] = x;
  }
  int lim[PR_ROWS];                                  // rows r0 + r see the keys below lim[r]
#pragma unroll
  for (int r = 0; r < PR_ROWS; ++r) lim[r] = row_limit(P, b, (r0 + min(r, R - 1)) / P.group);
  const int kmax = lim[PR_ROWS - 1];                 // limits rise with the query
  float m[PR_ROWS], l[PR_ROWS], acc[PR_ROWS][DV];
#pragma unroll
  for (int r = 0; r < PR_ROWS; ++r) {
    m[r] = -CUDART_INF_F;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[r][i] = 0.f;
  }
  __syncthreads();
#pragma unroll 1
  for (int s0 = (rank * PR_WARPS + w) * PR_KEYS; s0 < kmax; s0 += S * PR_WARPS * PR_KEYS) {
    const int nk = min(PR_KEYS, kmax - s0), key = s0 + lane;
    const int64_t at = kv_row(P, b, h, s0) * D;      // a group lies in one page
    const T* k = reinterpret_cast<const T*>(P.k) + at + (int64_t)min(lane, nk - 1) * D;
    const T* v = reinterpret_cast<const T*>(P.v) + at;
    float s[PR_ROWS];
#pragma unroll
    for (int r = 0; r < PR_ROWS; ++r) s[r] = 0.f;
    if (VEC) {
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        const float4 x = pr_load4(k + d);
#pragma unroll
        for (int r = 0; r < PR_ROWS; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(&qs[r][d]);
          s[r] = fmaf(q.x, x.x, fmaf(q.y, x.y, fmaf(q.z, x.z, fmaf(q.w, x.w, s[r]))));
        }
      }
    } else {
#pragma unroll 4
      for (int d = 0; d < D; ++d) {
        const float x = pr_f(k[d]);
#pragma unroll
        for (int r = 0; r < PR_ROWS; ++r) s[r] = fmaf(qs[r][d], x, s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < PR_ROWS; ++r) {
      if (key >= lim[r]) s[r] = -CUDART_INF_F;
      const float mn = fmaxf(m[r], warp_max(s[r]));
      const float alpha = pr_weight(m[r], mn);
      s[r] = s[r] == -CUDART_INF_F ? 0.f : pr_ex2(s[r] - mn);
      m[r] = mn;
      l[r] = fmaf(l[r], alpha, s[r]);
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[r][i] *= alpha;
    }
#pragma unroll 1
    for (int k0 = 0; k0 < nk; k0 += PR_AHEAD) {
      float x[PR_AHEAD][DV];
#pragma unroll
      for (int e = 0; e < PR_AHEAD; ++e)
#pragma unroll
        for (int i = 0; i < DV; ++i) {
          const int d = lane + 32 * i;
          x[e][i] = k0 + e < nk && d < D ? pr_f(v[(int64_t)(k0 + e) * D + d]) : 0.f;
        }
#pragma unroll
      for (int e = 0; e < PR_AHEAD; ++e)
#pragma unroll
        for (int r = 0; r < PR_ROWS; ++r) {
          const float p = __shfl_sync(0xffffffffu, s[r], k0 + e);
          if (p == 0.f) continue;                    // a key that the row does not see: V may be NaN
#pragma unroll
          for (int i = 0; i < DV; ++i) acc[r][i] = fmaf(p, x[e][i], acc[r][i]);
        }
    }
  }
  // the warps' parts, in order
#pragma unroll
  for (int r = 0; r < PR_ROWS; ++r) {
    l[r] = warp_sum(l[r]);
    if (lane == 0) {
      ms[w][r] = m[r];
      ls[w][r] = l[r];
    }
#pragma unroll
    for (int i = 0; i < DV; ++i) accs[w][r][lane + 32 * i] = acc[r][i];
  }
  __syncthreads();
  for (int i = t; i < PR_ROWS * 32 * DV; i += PR_WARPS * 32) {
    const int r = i / (32 * DV), d = i % (32 * DV);
    float gm = -CUDART_INF_F, L = 0.f, a = 0.f;
#pragma unroll
    for (int x = 0; x < PR_WARPS; ++x) gm = fmaxf(gm, ms[x][r]);
#pragma unroll
    for (int x = 0; x < PR_WARPS; ++x) {
      const float f = pr_weight(ms[x][r], gm);
      L += pr_part(f, ls[x][r]);
      if (f != 0.f) a = fmaf(f, accs[x][r][d], a);
    }
    acc1[r][d] = a;
    if (d == 0) {
      m1[r] = gm;
      l1[r] = L;
    }
  }
  // the CTAs' parts, in order: row r by the CTA of rank r % S
  if (S > 1) pr_cluster_sync(); else __syncthreads();
  for (int i = t; i < PR_ROWS * 32 * DV; i += PR_WARPS * 32) {
    const int r = i / (32 * DV), d = i % (32 * DV);
    if (r % S != rank || r >= R || d >= D) continue;
    float gm = m1[r], L = l1[r], a = acc1[r][d];
    if (S > 1) {
      gm = -CUDART_INF_F;
      L = a = 0.f;
      for (int x = 0; x < S; ++x) gm = fmaxf(gm, pr_remote(&m1[r], x));
      for (int x = 0; x < S; ++x) {
        const float f = pr_weight(pr_remote(&m1[r], x), gm);
        L += pr_part(f, pr_remote(&l1[r], x));
        if (f != 0.f) a = fmaf(f, pr_remote(&acc1[r][d], x), a);
      }
    }
    const int j = (r0 + r) / P.group, hq = h * P.group + (r0 + r) % P.group;
    const float y = L == 0.f ? 0.f : a / L;          // (a NaN sum: NaN)
    T* out = reinterpret_cast<T*>(P.out) + b * P.obs + j * P.oqs + hq * P.ohs + d;
    if constexpr (sizeof(T) == 4) *out = y; else *out = __float2bfloat16(y);
  }
  if (S > 1) pr_cluster_sync();                      // nobody leaves while its parts are read
}

template <typename T, int DV, bool VEC>
static int launch_rows(const AttnParams& P, int blocks, int S, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)P.B * P.Hkv * blocks * S));
  cfg.blockDim = dim3(PR_WARPS * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, prefix_rows_kernel<T, DV, VEC>, P, blocks, S) != cudaSuccess)
    return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}
template <typename T>
static int rows_of(const AttnParams& P, int blocks, int S, cudaStream_t st) {
  const uintptr_t mask = 4 * sizeof(T) - 1;
  const bool vec = P.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(P.k) & mask) == 0);
  if (P.D <= 32) return vec ? launch_rows<T, 1, true>(P, blocks, S, st)
                            : launch_rows<T, 1, false>(P, blocks, S, st);
  if (P.D <= 64) return vec ? launch_rows<T, 2, true>(P, blocks, S, st)
                            : launch_rows<T, 2, false>(P, blocks, S, st);
  return vec ? launch_rows<T, 4, true>(P, blocks, S, st) : launch_rows<T, 4, false>(P, blocks, S, st);
}

int prefix_rows(const AttnParams& P, int dtype, cudaStream_t st) {
  if (P.D > 128) return SD_ENOTSUP;
  const int64_t blocks = ((int64_t)P.R + PR_ROWS - 1) / PR_ROWS, units = blocks * P.B * P.Hkv;
  // CTAs up to two per SM, and no more than the table has groups of keys for
  int S = 1;
  while (S < 8 && units * S < PR_CTAS && S * PR_WARPS * PR_KEYS < P.C) S *= 2;
  if (units * S > 0x7FFFFFFF) return SD_ENOTSUP;
  return dtype == SD_DTYPE_BF16 ? rows_of<__nv_bfloat16>(P, (int)blocks, S, st)
                                : rows_of<float>(P, (int)blocks, S, st);
}

}  // namespace sd
