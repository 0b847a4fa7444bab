// Tree attention on the CUDA cores (sm_100a): the shapes that the tensor-core
// kernel does not take (fp32, head sizes other than 64 and 128, very wide head groups).
//
// A cluster of S CTAs holds TR_ROWS query rows (node, head) of one (row, kv head).
// The keys go out in groups of 32 to the cluster's 8 S warps in turn.  Per group
// a lane has one key,
//   s_r = scale log2(e) q_r . k_lane    (q_r from shared memory)
//   p_r = 2^(s_r - m_r)                 m_r the warp's running maximum, and 0 for
//                                       a key that node r does not see
// and then every 32nd column of V:  acc_r += p_r v.  The warps' (m, l, acc) are
// merged over the CTA in shared memory and over the cluster in distributed shared
// memory, in warp order: one launch, no workspace, the same sums on every run.
// A key that a node does not see adds nothing to it whatever K and V hold there.
// Bound by latency for few rows (so S grows while the machine has room), else by
// the products: each K and V element meets TR_ROWS query rows.  8 rows of 9 nodes over up
// to 460 fp32 keys of 64: 12.4 to 14.1 us, about eight dependent trips to memory; 32 rows of 26
// nodes over 2048 keys: 1.01 ms with fp32 heads of 64, 1.84 with 128, 1.17 with bf16 in heads of
// 64 or a little less, 1.90, 2.04 and 2.15 with 80, 96 and 112 (9 to 15 TFLOP/s of the 74 that
// the FMA pipes have).  P V is what holds it there: a (key, row) costs a shuffle and a test of its
// weight for D / 32 multiply-adds of a lane, and in Q K a 16-byte load of q feeds four.  Two CTAs
// per SM, at 128 registers a thread, beat one with more of K and V on the way (1.03, 2.36,
// 1.33 ms) and three (1.10, 2.02, 1.46).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>

#include "sd_common.cuh"
#include "sd_tree.cuh"

namespace sd {

constexpr int TR_ROWS = 8;
constexpr int TR_WARPS = 8;
constexpr int TR_AHEAD = 8;                    // V rows on their way at once
constexpr int TR_CTAS = 2 * 148;               // enough CTAs: two per SM

__device__ __forceinline__ float tr_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float tr_f(float x) { return x; }
__device__ __forceinline__ float tr_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float4 tr_load4(const float* p) {
  return __ldg(reinterpret_cast<const float4*>(p));
}
__device__ __forceinline__ float4 tr_load4(const __nv_bfloat16* p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void tr_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float tr_remote(const float* p, int rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}
// Weight of a part with maximum m under the joint maximum gm; its sum keeps a NaN.
__device__ __forceinline__ float tr_weight(float m, float gm) {
  return m == -CUDART_INF_F ? 0.f : tr_ex2(m - gm);
}
__device__ __forceinline__ float tr_part(float f, float l) { return l != l ? l : f * l; }

// VEC: 16 (fp32) or 8 (bf16) byte loads of K, D a multiple of 4
template <typename T, int DV, bool VEC>
__global__ void __launch_bounds__(TR_WARPS * 32, TR_CTAS / 148)
tree_rows_kernel(const __grid_constant__ TreeParams P, int blocks, int S) {
  __shared__ __align__(16) float qs[TR_ROWS][32 * DV];
  __shared__ float accs[TR_WARPS][TR_ROWS][32 * DV];
  __shared__ float ms[TR_WARPS][TR_ROWS], ls[TR_WARPS][TR_ROWS];
  __shared__ float acc1[TR_ROWS][32 * DV], m1[TR_ROWS], l1[TR_ROWS];     // of the CTA
  const AttnParams& A = P.A;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, D = A.D;
  const int rank = (int)(blockIdx.x % S), unit = (int)(blockIdx.x / S);
  const int rb = unit % blocks, bh = unit / blocks, b = bh / A.Hkv, h = bh - b * A.Hkv;
  const int r0 = rb * TR_ROWS, R = min(TR_ROWS, A.R - r0);
  const float sl2 = A.scale * 1.4426950408889634f;
  const int base = tree_base(P, b), kmax = tree_end(P, base);
  // lane r: the bits of row r's node
  const int32_t* mask = P.masks + (int64_t)b * P.mask_bs +
                        (int64_t)(P.first + (r0 + min(lane, R - 1)) / A.group) * P.W;
  const uint32_t there =                             // rows whose node is present
      __ballot_sync(0xffffffffu, lane < R && tree_present(mask, P.W, P.N));
  for (int i = t; i < TR_ROWS * 32 * DV; i += TR_WARPS * 32) {
    const int r = i / (32 * DV), d = i % (32 * DV);
    float x = 0.f;
    if (r < R && d < D) {
      const int j = (r0 + r) / A.group, hq = h * A.group + (r0 + r) % A.group;
      x = tr_f(reinterpret_cast<const T*>(A.q)[b * A.qbs + hq * A.qhs + j * A.qqs + d]) * sl2;
    }
    qs[r][d] = x;
  }
  float m[TR_ROWS], l[TR_ROWS], acc[TR_ROWS][DV];
#pragma unroll
  for (int r = 0; r < TR_ROWS; ++r) {
    m[r] = -CUDART_INF_F;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[r][i] = 0.f;
  }
  __syncthreads();
#pragma unroll 1
  for (int s0 = (rank * TR_WARPS + w) * 32; s0 < kmax && there; s0 += S * TR_WARPS * 32) {
    const int nk = min(32, kmax - s0);
    const int64_t at = kv_row(A, b, h, s0) * D;      // a group lies in one page
    const T* k = reinterpret_cast<const T*>(A.k) + at + (int64_t)min(lane, nk - 1) * D;
    const T* v = reinterpret_cast<const T*>(A.v) + at;
    float s[TR_ROWS];
#pragma unroll
    for (int r = 0; r < TR_ROWS; ++r) s[r] = 0.f;
    if (VEC) {
#pragma unroll 2
      for (int d = 0; d < D; d += 4) {
        const float4 x = tr_load4(k + d);
#pragma unroll
        for (int r = 0; r < TR_ROWS; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(&qs[r][d]);
          s[r] = fmaf(q.x, x.x, fmaf(q.y, x.y, fmaf(q.z, x.z, fmaf(q.w, x.w, s[r]))));
        }
      }
    } else {
#pragma unroll 4
      for (int d = 0; d < D; ++d) {
        const float x = tr_f(k[d]);
#pragma unroll
        for (int r = 0; r < TR_ROWS; ++r) s[r] = fmaf(qs[r][d], x, s[r]);
      }
    }
    uint32_t hidden = 0;
    if (s0 + 32 > base) {                            // some keys of the group are the tree's
      const uint32_t sees = tree_sees(mask, P.W, P.N, base, s0);
#pragma unroll
      for (int r = 0; r < TR_ROWS; ++r)
        hidden |= (~(__shfl_sync(0xffffffffu, sees, r) >> lane) & 1u) << r;
    }
    const uint32_t hid = (lane < nk ? hidden : 0xFFu) | ~there;    // rows that do not see this lane's key
#pragma unroll
    for (int r = 0; r < TR_ROWS; ++r) {
      const bool out = (hid >> r) & 1u;
      if (out) s[r] = -CUDART_INF_F;
      const float mn = fmaxf(m[r], warp_max(s[r]));
      const float alpha = tr_weight(m[r], mn);
      s[r] = out || s[r] == -CUDART_INF_F ? 0.f : tr_ex2(s[r] - mn);
      m[r] = mn;
      l[r] = fmaf(l[r], alpha, s[r]);
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[r][i] *= alpha;
    }
#pragma unroll 1
    for (int k0 = 0; k0 < nk; k0 += TR_AHEAD) {
      float x[TR_AHEAD][DV];
#pragma unroll
      for (int e = 0; e < TR_AHEAD; ++e)
#pragma unroll
        for (int i = 0; i < DV; ++i) {
          const int d = lane + 32 * i;
          x[e][i] = k0 + e < nk && d < D ? tr_f(v[(int64_t)(k0 + e) * D + d]) : 0.f;
        }
#pragma unroll
      for (int e = 0; e < TR_AHEAD; ++e)
#pragma unroll
        for (int r = 0; r < TR_ROWS; ++r) {
          const float p = __shfl_sync(0xffffffffu, s[r], k0 + e);
          if (p == 0.f) continue;                    // a key that the row does not see: V may be NaN
#pragma unroll
          for (int i = 0; i < DV; ++i) acc[r][i] = fmaf(p, x[e][i], acc[r][i]);
        }
    }
  }
  // the warps' parts, in order
#pragma unroll
  for (int r = 0; r < TR_ROWS; ++r) {
    l[r] = warp_sum(l[r]);
    if (lane == 0) {
      ms[w][r] = m[r];
      ls[w][r] = l[r];
    }
#pragma unroll
    for (int i = 0; i < DV; ++i) accs[w][r][lane + 32 * i] = acc[r][i];
  }
  __syncthreads();
  for (int i = t; i < TR_ROWS * 32 * DV; i += TR_WARPS * 32) {
    const int r = i / (32 * DV), d = i % (32 * DV);
    float gm = -CUDART_INF_F, L = 0.f, a = 0.f;
#pragma unroll
    for (int x = 0; x < TR_WARPS; ++x) gm = fmaxf(gm, ms[x][r]);
#pragma unroll
    for (int x = 0; x < TR_WARPS; ++x) {
      const float f = tr_weight(ms[x][r], gm);
      L += tr_part(f, ls[x][r]);
      if (f != 0.f) a = fmaf(f, accs[x][r][d], a);
    }
    acc1[r][d] = a;
    if (d == 0) {
      m1[r] = gm;
      l1[r] = L;
    }
  }
  // the CTAs' parts, in order: row r by the CTA of rank r % S
  if (S > 1) tr_cluster_sync(); else __syncthreads();
  for (int i = t; i < TR_ROWS * 32 * DV; i += TR_WARPS * 32) {
    const int r = i / (32 * DV), d = i % (32 * DV);
    if (r % S != rank || r >= R || d >= D) continue;
    float gm = m1[r], L = l1[r], a = acc1[r][d];
    if (S > 1) {
      gm = -CUDART_INF_F;
      L = a = 0.f;
      for (int x = 0; x < S; ++x) gm = fmaxf(gm, tr_remote(&m1[r], x));
      for (int x = 0; x < S; ++x) {
        const float f = tr_weight(tr_remote(&m1[r], x), gm);
        L += tr_part(f, tr_remote(&l1[r], x));
        if (f != 0.f) a = fmaf(f, tr_remote(&acc1[r][d], x), a);
      }
    }
    const int j = (r0 + r) / A.group, hq = h * A.group + (r0 + r) % A.group;
    const float y = L == 0.f ? 0.f : a / L;          // (a NaN sum: NaN)
    T* out = reinterpret_cast<T*>(A.out) + b * A.obs + j * A.oqs + hq * A.ohs + d;
    if constexpr (sizeof(T) == 4) *out = y; else *out = __float2bfloat16(y);
  }
  if (S > 1) tr_cluster_sync();                      // nobody leaves while its parts are read
}

template <typename T, int DV, bool VEC>
static int launch_tree_rows(const TreeParams& P, int blocks, int S, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)P.A.B * P.A.Hkv * blocks * S));
  cfg.blockDim = dim3(TR_WARPS * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, tree_rows_kernel<T, DV, VEC>, P, blocks, S) != cudaSuccess)
    return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}
template <typename T>
static int tree_rows_of(const TreeParams& P, int blocks, int S, cudaStream_t st) {
  const uintptr_t mask = 4 * sizeof(T) - 1;
  const bool vec = P.A.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(P.A.k) & mask) == 0);
  if (P.A.D <= 32) return vec ? launch_tree_rows<T, 1, true>(P, blocks, S, st)
                              : launch_tree_rows<T, 1, false>(P, blocks, S, st);
  if (P.A.D <= 64) return vec ? launch_tree_rows<T, 2, true>(P, blocks, S, st)
                              : launch_tree_rows<T, 2, false>(P, blocks, S, st);
  return vec ? launch_tree_rows<T, 4, true>(P, blocks, S, st)
             : launch_tree_rows<T, 4, false>(P, blocks, S, st);
}

int tree_rows(const TreeParams& P, int dtype, cudaStream_t st) {
  const int64_t blocks = ((int64_t)P.A.R + TR_ROWS - 1) / TR_ROWS, units = blocks * P.A.B * P.A.Hkv;
  // CTAs up to two per SM, and no more than the cache has groups of keys for
  int S = 1;
  while (S < 8 && units * S < TR_CTAS && S * TR_WARPS * 32 < P.A.C) S *= 2;
  if (units * S > 0x7FFFFFFF) return SD_ENOTSUP;
  return dtype == SD_DTYPE_BF16 ? tree_rows_of<__nv_bfloat16>(P, (int)blocks, S, st)
                                : tree_rows_of<float>(P, (int)blocks, S, st);
}

}  // namespace sd
