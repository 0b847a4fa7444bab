// Attention of a tree's nodes over the cache (sm_100a): host entry, and the tensor-core
// kernels for bf16 heads of 128.
//
// The query rows of a (row, kv head) are its nodes times the heads of the group:
// 64 nodes under 32 / 8 heads are 256 rows that read the same keys.  An item is one
// (row, kv head) and up to 256 of them, on two tiles of 128; it goes over the row's
// keys in tiles of 128 ("pages", whether the cache is paged or not):
//   S = Q K^T,  p = 2^(s - m) under a lazy running maximum m,  O += P V
// Every page but the last few is seen whole by every node; in those that hold
// the tree a row keeps the scores whose bit its node's mask has.
// tree_tc_kernel    persistent, stream-K: the pages of all items lie end to end
//                   and a CTA takes one contiguous run; an item that lies within a
//                   run is written out, a cut one leaves (m, l, O) per piece
// tree_join_kernel  merges the pieces of cut items, in order (programmatic dependent)
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "sd_common.cuh"
#include "sd_softmax.cuh"
#include "sd_tcgen05.cuh"
#include "sd_tree.cuh"

namespace sd {

constexpr int TT_D = 128;
constexpr int TT_TILE = 128;                 // query rows of a tile
constexpr int TT_THREADS = 352;              // warps 0-7: softmax; 8: TMA of K, V; 9: MMA; 10: TMA of Q
constexpr int TT_CTAS = 148;                 // one CTA per SM
constexpr int TT_OVH = 3;                    // schedule cost of an item beyond its pages, in pages
constexpr int TT_MIN_SHARE = TT_OVH + 1;     // fewest schedule units per CTA: a one-page item
constexpr int TT_BASES = 512;                // rows whose bases a CTA keeps
constexpr int TT_WORDS = SD_TREE_MAX / 32;
constexpr int TJ_THREADS = 256;
constexpr int TJ_ROWS = 32;                  // query rows of a join CTA

struct TreeTcParams {
  TreeParams T;
  int np, ni, nt;                            // items of a (row, kv head); nodes of an item, of a tile
  int rs;                                    // rows of a piece: ni * group, rounded up to 32
  int out_vec;                               // 16-byte stores of the output are aligned
  // workspace
  int* rowpre;                               // [B + 1] exclusive prefix of a row's units per item
  int* status;                               // [TT_CTAS] a bounded wait gave up
  float4* pacc;                              // [2 TT_CTAS][32 column groups][rs] pieces
  float2* pml;                               // [2 TT_CTAS][rs]
};

__device__ __forceinline__ int tt_units(int end) { return (end + SD_KV_PAGE - 1) / SD_KV_PAGE + TT_OVH; }
__device__ __forceinline__ int tt_share(int total) {
  return max(TT_MIN_SHARE, (total + TT_CTAS - 1) / TT_CTAS);
}

// NT: tiles of query rows of an item
template <int NT>
struct TtSmem {
  static constexpr int SLOTS = NT == 2 ? 4 : 5;      // 32 KB K / V tiles in flight
  alignas(1024) unsigned char q[NT][2][128 * 128];           // [tile][64-col box][128 rows x 128 B]
  alignas(1024) unsigned char kv[SLOTS][2][128 * 128];       // [slot][64-col box][128 keys x 128 B]
  alignas(16) unsigned char out[8][32 * 64];         // a warp's 32 rows x 32 outputs
  // sfull, pfull by step parity; oready by tile and page parity; xch by lane quarter
  alignas(8) unsigned long long full[SLOTS], empty[SLOTS], sfull[2], pfull[2], oready[NT][2], qfull[NT],
      qempty[NT], fin;
  uint32_t mask[NT][128][TT_WORDS];          // the query rows: their nodes' bits
  // what the threads of a row tell one another: [exchange parity][warpgroup][row], (value, number)
  unsigned long long peer[2][2][128];
  int base[TT_BASES];
  int red[33];
  int first[2];                              // the CTA's first row and the units before it
  int abort_;
  uint32_t tmem;
};
static_assert(sizeof(TtSmem<2>) + 1024 <= 227 * 1024, "shared memory, with room to align");
static_assert(sizeof(TtSmem<1>) + 1024 <= 227 * 1024, "shared memory, with room to align");

// A CTA's run of schedule units as segments of items, walked identically by
// every role: row-major, kv head and then the item inner; TT_OVH virtual units in
// front of each item's pages.
struct TtSeg {
  int b, h, p, base, tb, off, tt, t1, ncost, j0, j1;         // pages [j0, j1) of the segment
};
template <int NT>
__device__ __forceinline__ int tt_base(const TtSmem<NT>& S, const TreeParams& T, int b) {
  return b < TT_BASES ? S.base[b] : tree_base(T, b);
}
__device__ __forceinline__ void tt_bounds(TtSeg& s) {
  s.ncost = min(s.tb - s.off, s.t1 - s.tt);
  s.j0 = max(s.off, TT_OVH) - TT_OVH;
  s.j1 = max(s.off + s.ncost - TT_OVH, s.j0);
}
template <int NT>
__device__ __forceinline__ bool tt_next(TtSeg& s, const TtSmem<NT>& S, const TreeTcParams& P) {
  s.tt += s.ncost;
  if (s.tt >= s.t1) return false;
  s.off = 0;
  if (++s.p == P.np) {
    s.p = 0;
    if (++s.h == P.T.A.Hkv) {
      s.h = 0;
      ++s.b;                                         // units remain, and every row has some
      s.base = tt_base(S, P.T, s.b);
      s.tb = tt_units(tree_end(P.T, s.base));
    }
  }
  tt_bounds(s);
  return true;
}
// On to the current or next segment with pages; false when none is left.
template <int NT>
__device__ __forceinline__ bool tt_real(TtSeg& s, const TtSmem<NT>& S, const TreeTcParams& P) {
  while (s.j1 == s.j0)
    if (!tt_next(s, S, P)) return false;
  return true;
}

// The schedule: every CTA sums the rows' units and finds its own first row.  The
// units per CTA and, in S.first, where the run of this one starts.
template <int NT>
__device__ __forceinline__ void tt_plan(TtSmem<NT>& S, const TreeTcParams& P, int* total, int* share) {
  const TreeParams& T = P.T;
  const int t = threadIdx.x, cta = (int)blockIdx.x, B = T.A.B, per = T.A.Hkv * P.np;
  int mine = 0, ex = 0, all = 0;
  if (B <= TT_THREADS) {                             // one pass does both
    if (t < B) {
      const int base = tree_base(T, t);
      S.base[t] = base;
      mine = tt_units(tree_end(T, base));
    }
    ex = block_excl_scan<int>(mine, S.red, &all);
  } else {
    for (int b = t; b < B; b += TT_THREADS) {
      const int base = tree_base(T, b);
      if (b < TT_BASES) S.base[b] = base;
      mine += tt_units(tree_end(T, base));
    }
    all = block_sum<int>(mine, S.red);
  }
  *total = all * per;
  *share = tt_share(*total);
  const int64_t t0 = (int64_t)cta * *share;
  int carry = 0;
  for (int b0 = 0; b0 < B; b0 += TT_THREADS) {
    const int b = b0 + t;
    if (B > TT_THREADS) {
      __syncthreads();
      mine = b < B ? tt_units(tree_end(T, tt_base(S, T, b))) : 0;
      int sum;
      ex = carry + block_excl_scan<int>(mine, S.red, &sum);
      carry += sum;
    }
    if (b < B) {
      if (cta == 0) P.rowpre[b] = ex;
      if ((int64_t)ex * per <= t0 && t0 < (int64_t)(ex + mine) * per) {
        S.first[0] = b;
        S.first[1] = ex * per;
      }
    }
  }
  if (cta == 0 && t == 0) P.rowpre[B] = all;
}

// A whole warp's arrival, as one.
__device__ __forceinline__ void tt_arrive(unsigned long long* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) tc_arrive(bar);
}
__device__ __forceinline__ void tt_tma_4d(void* dst, const void* tmap, int x, int y, int z, int u,
                                          unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%2, %3, %4, %5}], [%6];"
               :: "r"(smem_addr(dst)), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_addr(bar))
               : "memory");
}

// Scores of `n` columns from scol on, keys k0 on: to -inf where the row's node does not
// see the key, in TMEM, 32 columns at a time (a short loop: cold whenever it runs).
__device__ __forceinline__ void tt_hide(const uint32_t* m, const TreeParams& T, int base, int end,
                                        int k0, int n, uint32_t scol) {
#pragma unroll 1
  for (int c = 0; c < n; c += 32) {
    const int d = base - (k0 + c);
    uint32_t sees = 0xFFFFFFFFu;
    if (d < 32) {
      if (d > 0) {
        sees = ((1u << d) - 1u) | ((m[0] & tree_valid(T.N, 0)) << d);
      } else {
        const int a = -d, w = a >> 5;
        sees = __funnelshift_r(w < T.W ? m[w] & tree_valid(T.N, w) : 0u,
                               w + 1 < T.W ? m[w + 1] & tree_valid(T.N, w + 1) : 0u, a & 31);
      }
      const int left = end - (k0 + c);               // (the capacity may cut the tree)
      if (left < 32) sees &= left > 0 ? (1u << left) - 1u : 0u;
    }
    if (__all_sync(0xffffffffu, sees == 0xFFFFFFFFu)) continue;
    uint32_t s[32];
    TC_LD32(s, scol + (uint32_t)c);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 32; ++e) s[e] = (sees >> e) & 1u ? s[e] : 0xFF800000u;
    TC_ST32(scol + (uint32_t)c, s);
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// V of the keys [kg, kg + 32) that no query of the row sees to zero (they may hold NaN), in
// the boxes [box0, box1) of a slot; uni: lane w holds word w of what any query sees.
__device__ __forceinline__ bool tt_blank(unsigned char (*v)[128 * 128], const TreeParams& T, uint32_t uni,
                                         int base, int end, int kg, int row, int box0, int box1,
                                         unsigned long long* full, uint32_t par, int* abort_) {
  const int lane = threadIdx.x & 31, d = base - kg;
  uint32_t any = 0xFFFFFFFFu;
  const int a = d > 0 ? 0 : -d, w = a >> 5;
  const uint32_t lo = __shfl_sync(0xffffffffu, uni, min(w, 31));
  const uint32_t hi = __shfl_sync(0xffffffffu, uni, min(w + 1, 31));
  if (d < 32) {
    any = d > 0 ? ((1u << d) - 1u) | (lo << d) : __funnelshift_r(lo, hi, a & 31);
    const int left = end - kg;
    if (left < 32) any &= left > 0 ? (1u << left) - 1u : 0u;
  }
  if (any == 0xFFFFFFFFu) return true;
  if (!__all_sync(0xffffffffu, tc_wait(full, par, abort_))) return false;
#pragma unroll 1
  for (int k4 = 0; k4 < 32; k4 += 4) {               // four keys of a 128-byte box at a time
    const int kr = k4 + (lane >> 3);
    if ((any >> kr) & 1u) continue;
    for (int x = box0; x < box1; ++x)
      *reinterpret_cast<uint4*>(v[x] + (row + kr) * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  return true;
}

// 32 columns of O, as outputs of the warp's 32 rows: over a swizzled 2 KB buffer, so that
// four lanes write 64 bytes of a row.  dst: the row's output from the first column on.
__device__ __forceinline__ void tt_write(unsigned char* stage, const float (&o)[32], __nv_bfloat16* dst,
                                         bool live, bool vec) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint4 u;
    u.x = pack_bf16(o[8 * e], o[8 * e + 1]);
    u.y = pack_bf16(o[8 * e + 2], o[8 * e + 3]);
    u.z = pack_bf16(o[8 * e + 4], o[8 * e + 5]);
    u.w = pack_bf16(o[8 * e + 6], o[8 * e + 7]);
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) = u;
  }
  __syncwarp();
  const unsigned long long mine = live ? reinterpret_cast<unsigned long long>(dst) : 0ULL;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2), e = lane & 3;
    const uint4 u = *reinterpret_cast<const uint4*>(stage + row * 64 + ((e ^ ((row >> 1) & 3)) << 4));
    __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(__shfl_sync(0xffffffffu, mine, row));
    if (to != nullptr) {
      to += 8 * e;
      if (vec) {
        *reinterpret_cast<uint4*>(to) = u;
      } else {
        const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(&u);
#pragma unroll
        for (int k = 0; k < 8; ++k) to[k] = x[k];
      }
    }
  }
  __syncwarp();
}

#ifndef TTV
#define TTV 0
#endif
__device__ __forceinline__ void tt_weights(const uint32_t (&s)[32], uint32_t* p,
                                           unsigned long long (&sum)[2], unsigned long long sl22,
                                           unsigned long long nm2) {
#if TTV == 0
  px_weights(s, p, sum, sl22, nm2);
#elif TTV == 1
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float a, b;
    const unsigned long long s2 = pair2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
    unpair(fma2(s2, sl22, nm2), a, b);
    const unsigned long long p2 = pair2(ex2f(a), ex2f(b));
    sum[e & 1] = add2(sum[e & 1], p2);
    unpair(p2, a, b);
    p[e] = pack_bf16(a, b);
  }
#elif TTV == 2
  float sl, nm, d, t0, t1, t2, t3;
  unpair(sl22, sl, d); unpair(nm2, nm, d); unpair(sum[0], t0, t1); unpair(sum[1], t2, t3);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float a = ex2f(fmaf(__uint_as_float(s[2 * e]), sl, nm)), b = ex2f(fmaf(__uint_as_float(s[2 * e + 1]), sl, nm));
    if (e & 1) { t0 += a; t1 += b; } else { t2 += a; t3 += b; }
    p[e] = pack_bf16(a, b);
  }
  sum[0] = pair2(t0, t1); sum[1] = pair2(t2, t3);
#elif TTV == 3
  float sl, nm, d, t0, t1, t2, t3;
  unpair(sl22, sl, d); unpair(nm2, nm, d); unpair(sum[0], t0, t1); unpair(sum[1], t2, t3);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float a, b;
    if (e % 8 == 1) unpair(px_exp2(fmaf(__uint_as_float(s[2 * e]), sl, nm), fmaf(__uint_as_float(s[2 * e + 1]), sl, nm)), a, b);
    else { a = ex2f(fmaf(__uint_as_float(s[2 * e]), sl, nm)); b = ex2f(fmaf(__uint_as_float(s[2 * e + 1]), sl, nm)); }
    if (e & 1) { t0 += a; t1 += b; } else { t2 += a; t3 += b; }
    p[e] = pack_bf16(a, b);
  }
  sum[0] = pair2(t0, t1); sum[1] = pair2(t2, t3);
#endif
}

template <int NT>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_tc_kernel(const __grid_constant__ TreeTcParams P, const __grid_constant__ CUtensorMap tmk,
               const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmq) {
  extern __shared__ __align__(1024) unsigned char tt_raw[];
  const uint32_t pad = (1024u - (smem_addr(tt_raw) & 1023u)) & 1023u;   // swizzle atoms: 1024 B
  TtSmem<NT>& S = *reinterpret_cast<TtSmem<NT>*>(tt_raw + pad);
  constexpr int SLOTS = TtSmem<NT>::SLOTS;
  const TreeParams& T = P.T;
  const AttnParams& A = T.A;
  const int t = threadIdx.x, w = t >> 5, lane = t & 31, cta = (int)blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (w == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_addr(&S.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (t == 256) {
    for (int i = 0; i < SLOTS; ++i) {
      tc_bar_init(&S.full[i], 1);
      tc_bar_init(&S.empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      tc_bar_init(&S.sfull[x], 1);
      tc_bar_init(&S.pfull[x], 8);
    }
    for (int x = 0; x < NT; ++x) {
      tc_bar_init(&S.qfull[x], 1);
      tc_bar_init(&S.qempty[x], 1);
      tc_bar_init(&S.oready[x][0], 1);
      tc_bar_init(&S.oready[x][1], 1);
    }
    tc_bar_init(&S.fin, 1);
    S.abort_ = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = t; i < 2 * 2 * 128; i += TT_THREADS) S.peer[0][0][i] = 0ULL;     // (numbers start at 1)
  // the rows of a tile that no query fills stay 0
  for (int i = P.nt * A.group * 8 + t; i < NT * 2 * 128 * 8; i += TT_THREADS)
    if (i % 1024 >= P.nt * A.group * 8)
      reinterpret_cast<uint4*>(S.q[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  int total, share;
  tt_plan(S, P, &total, &share);
  const bool work = (int64_t)cta * share < total;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = S.tmem;
  if (work) {
    const int t0 = cta * share, t1 = t0 + min(total - t0, share);
    TtSeg seg;
    seg.b = S.first[0];
    seg.base = tt_base(S, T, seg.b);
    seg.tb = tt_units(tree_end(T, seg.base));
    const int u = t0 - S.first[1], it = u / seg.tb;
    seg.off = u % seg.tb;
    seg.h = it / P.np;
    seg.p = it % P.np;
    seg.tt = t0;
    seg.t1 = t1;
    tt_bounds(seg);
    bool more = tt_real(seg, S, P);

    // Q of a tile of a segment's item: its nodes x heads
    auto ask_q = [&](const TtSeg& g, int ti) {
      const int j = g.p * P.ni + P.nt * ti;
      tc_expect_tx(&S.qfull[ti], 2u * 128u * (uint32_t)(P.nt * A.group));
      tt_tma_4d(S.q[ti][0], &tmq, 0, g.h * A.group, j, g.b, &S.qfull[ti]);
      tt_tma_4d(S.q[ti][1], &tmq, 64, g.h * A.group, j, g.b, &S.qfull[ti]);
    };
    if (w == 8) {
      if (lane == 0) {
        // ---------------- TMA producer: K then V of each page, SLOTS tiles ahead; the first
        // segment's Q in front, before all SMs' K and V are on their way
        for (int ti = 0; ti < NT && more; ++ti) ask_q(seg, ti);
        uint32_t idx = 0;
        bool ok = true;
        while (more && ok) {
          for (int j = seg.j0; j < seg.j1 && ok; ++j) {
            const int y = (int)kv_row(A, seg.b, seg.h, j * SD_KV_PAGE);
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv, ++idx) {
              const int sl = (int)(idx % SLOTS);
              if (idx >= (uint32_t)SLOTS)
                ok = tc_wait(&S.empty[sl], ((idx / SLOTS) - 1) & 1u, &S.abort_);
              if (!ok) break;
              tc_expect_tx(&S.full[sl], 2u * 128u * 128u);
              const void* map = kv ? (const void*)&tmv : (const void*)&tmk;
              tc_tma_2d(S.kv[sl][0], map, 0, y, &S.full[sl]);
              tc_tma_2d(S.kv[sl][1], map, 64, y, &S.full[sl]);
            }
          }
          if (ok) more = tt_next(seg, S, P) && tt_real(seg, S, P);
        }
        if (!ok) {
          // let the copies already issued land before the CTA leaves
          for (uint32_t q = idx > (uint32_t)SLOTS ? idx - SLOTS : 0u; q < idx; ++q) {
            int dummy = 0;
            tc_wait(&S.full[q % SLOTS], (q / SLOTS) & 1u, &dummy);
          }
        }
      }
    } else if (w == 9) {
      // ---------------- MMA issuer (the whole warp): S(0) S(1) P.V(0) S(2) P.V(1) ... in steps
      // of (page, tile), tile inner; S of a step lies in buffer step & 1, P over it
      constexpr uint32_t ID1 = tc_idesc(128, 128, 0, 0);     // S = Q . K^T
      constexpr uint32_t ID2 = tc_idesc(128, 128, 0, 1);     // O += P . V (V [key][d]: N-major)
      const uint32_t kv0 = smem_addr(S.kv[0][0]), q0 = smem_addr(S.q[0][0]);
      TtSeg back = seg;
      int ahead = seg.j1 - seg.j0, behind = ahead;   // pages left of the segments of S and of P . V
      uint32_t ga = 0, gc = 0, xa = 0, xc = 0;       // pages and tiles of the next S, the next P . V
      uint32_t a = 0, c = 0, qn = 0;                 // steps issued; segments begun by S
      bool ok = true, acc = false;
      long long idle = 0;
      while (ok) {
        const uint32_t ki = 2u * ga, vi = 2u * gc + 1u;
        unsigned long long* kfull = &S.full[ki % SLOTS];
        // S comes first, up to two ahead; where its tiles are late, P . V does not wait for it
        bool s_go = false, p_go = false;
        if (more && a < c + 2u)
          s_go = __all_sync(0xffffffffu, tc_test(kfull, (ki / SLOTS) & 1u) && tc_test(&S.qfull[xa], qn & 1u));
        if (!s_go && c < a) {
          unsigned long long* vfull = &S.full[vi % SLOTS];
          if (more && a < c + 2u)
            p_go = __all_sync(0xffffffffu, tc_test(vfull, (vi / SLOTS) & 1u) &&
                                               tc_test(&S.pfull[c & 1u], (c >> 1) & 1u));
          else
            p_go = ok = tc_wait2_warp(vfull, (vi / SLOTS) & 1u, &S.pfull[c & 1u], (c >> 1) & 1u, &S.abort_);
          if (!ok) break;
        }
        if (!s_go && !p_go) {
          if (c == a && !more) break;
          const long long now = clock64();
          if (idle == 0) idle = now;
          if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&S.abort_) || now - idle > TC_WAIT)) {
            *reinterpret_cast<volatile int*>(&S.abort_) = 1;
            break;
          }
          continue;
        }
        idle = 0;
        tc_fence_after();
        if (s_go) {
          const uint32_t sl = ki % SLOTS, d = tm + 128u * (a & 1u);
          const uint64_t dq = tc_desc(q0 + xa * 32768u, 16, 1024, 2);
          const uint64_t dk = tc_desc(kv0 + sl * 32768u, 16, 1024, 2);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {           // 16 of 128 d: 32 B, the second box 16 KB on
            const uint64_t o = (uint64_t)((ks & 3) * 2 + (ks >> 2) * 1024);
            tc_mma_warp(d, dq + o, dk + o, ID1, ks > 0 ? 1 : 0);
          }
          tc_commit_warp(&S.sfull[a & 1u]);
          if (ahead == 1) tc_commit_warp(&S.qempty[xa]);     // the segment's last S of the tile
          ++a;
          if (++xa == (uint32_t)NT) {
            xa = 0;
            tc_commit_warp(&S.empty[sl]);
            ++ga;
            if (--ahead == 0) {
              more = tt_next(seg, S, P) && tt_real(seg, S, P);
              ahead = seg.j1 - seg.j0;
              ++qn;
            }
          }
          continue;
        }
        const uint32_t sl = vi % SLOTS, pa = tm + 128u * (c & 1u);
        const uint64_t dv = tc_desc(kv0 + sl * 32768u, 16384, 1024, 2);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)               // 16 keys: 2 KB; P of 64 keys every 64 columns
          tc_mma_ts_warp(tm + 256u + 128u * xc, pa + 64u * (ks >> 2) + 8u * (ks & 3),
                         dv + (uint64_t)(ks * 128), ID2, ks || acc ? 1 : 0);
        tc_commit_warp(&S.oready[xc][gc & 1u]);
        ++c;
        if (++xc == (uint32_t)NT) {
          xc = 0;
          tc_commit_warp(&S.empty[sl]);
          ++gc;
          acc = true;
          if (--behind == 0) {
            if (!(tt_next(back, S, P) && tt_real(back, S, P))) break;
            behind = back.j1 - back.j0;
            acc = false;
          }
        }
      }
      // every MMA this warp issued has finished before the CTA leaves
      tc_commit_warp(&S.fin);
      int dummy = 0;
      tc_wait(&S.fin, 0u, &dummy);
    } else if (w == 10) {
      if (lane == 0) {
        // ---------------- TMA producer of the later segments' Q, once a tile's last S is done
        uint32_t sent = more ? NT : 0u;              // tiles asked for, tile inner
        bool ok = true;
        while (ok && more && tt_next(seg, S, P) && tt_real(seg, S, P)) {
          for (int ti = 0; ti < NT; ++ti, ++sent) {
            ok = tc_wait(&S.qempty[ti], (sent / NT - 1) & 1u, &S.abort_);
            if (!ok) break;
            ask_q(seg, ti);
          }
        }
        if (!ok) {
          // let the copies already issued land before the CTA leaves
          for (uint32_t q = sent > (uint32_t)NT ? sent - NT : 0u; q < sent; ++q) {
            int dummy = 0;
            tc_wait(&S.qfull[q % NT], (q / NT) & 1u, &dummy);
          }
        }
      }
    } else {
      // ---------------- softmax warps: the threads of warpgroups 0 and 1 with the same lane own
      // the same query row of every tile; warpgroup x takes the keys [64 x, 64 x + 64) of a page
      const int x = w >> 2, wq = w & 3, r = t & 127;
      const uint32_t lcol = tm + ((uint32_t)(32 * wq) << 16);
      const float sl2 = A.scale * 1.4426950408889634f;
      unsigned char* stage = S.out[w];
      // rows of tile ti of a segment's item
      auto rows_of = [&](const TtSeg& g, int ti) {
        return A.group * min(min(P.nt, P.ni - P.nt * ti), A.qlen - g.p * P.ni - P.nt * ti);
      };
      uint32_t k = 0, n = 0, xn = 0;                 // steps and pages done; exchanges with the peer
      bool ok = true;
      // A value to the thread with the row's other keys, and that thread's (a word of shared memory
      // holds the value and the exchange's number; two of them by parity, as the peer may be one
      // exchange ahead).  `ok` is false when a bounded wait gives up.
      auto tell = [&](float v) {
        ++xn;
        *reinterpret_cast<volatile unsigned long long*>(&S.peer[xn & 1u][x][r]) =
            ((unsigned long long)xn << 32) | __float_as_uint(v);
      };
      auto told = [&]() {
        const volatile unsigned long long* from = &S.peer[xn & 1u][x ^ 1][r];
        unsigned long long v = *from;
        long long since = 0;
        while ((uint32_t)(v >> 32) != xn) {
          const long long now = clock64();
          if (since == 0) since = now;
          if (*reinterpret_cast<volatile int*>(&S.abort_) || now - since > TC_WAIT) {
            *reinterpret_cast<volatile int*>(&S.abort_) = 1;
            ok = false;
            break;
          }
          v = *from;
        }
        ok = __all_sync(0xffffffffu, ok);
        return __uint_as_float((uint32_t)v);
      };
      // P . V of page n - 1 is in O (that of page n - 2 may be under way, too: two barriers)
      auto o_ready = [&](int ti) {
        return tc_wait(&S.oready[ti][(n - 1) & 1u], ((n - 1) >> 1) & 1u, &S.abort_);
      };
      int seen_b = -1, seen_p = -1;                  // the segment that these are of:
      uint32_t uni = 0;
      bool settled = false;
      uint32_t there = 0, dead = 0;                  // bit ti: the row's node is present; no row in the warp
      while (more) {
        const TtSeg cur = seg;
        more = tt_next(seg, S, P) && tt_real(seg, S, P);
        const int pages = cur.j1 - cur.j0, end = tree_end(T, cur.base);
        const int32_t* mask0 = T.masks + (int64_t)cur.b * T.mask_bs + (int64_t)T.first * T.W;
        // the rows' bits to shared memory (both warpgroups write the same), unless they are there:
        // asked for now, used in the tree's pages
        if (seen_p != cur.p || (seen_b != cur.b && (T.mask_bs != 0 || seen_b < 0))) {
          if (!settled) asm volatile("cp.async.wait_all;" ::: "memory");   // an older copy first
          dead = 0;
#pragma unroll
          for (int ti = 0; ti < NT; ++ti) {
            const bool live = r < rows_of(cur, ti);
            dead |= __all_sync(0xffffffffu, !live) ? 1u << ti : 0u;
            const int32_t* m = mask0 + (int64_t)(cur.p * P.ni + P.nt * ti + r / A.group) * T.W;
            for (int i = 0; i < T.W; ++i) {
              if (live)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                             :: "r"(smem_addr(&S.mask[ti][r][i])), "l"(m + i) : "memory");
              else
                S.mask[ti][r][i] = 0u;
            }
          }
          settled = false;
          seen_b = cur.b;
          seen_p = cur.p;
        }
        auto settle = [&]() {
          asm volatile("cp.async.wait_all;" ::: "memory");
          there = 0;
#pragma unroll
          for (int ti = 0; ti < NT; ++ti) {
            uint32_t some = 0;
            for (int i = 0; i < T.W; ++i) some |= S.mask[ti][r][i] & tree_valid(T.N, i);
            there |= some != 0u ? 1u << ti : 0u;
          }
          // lane i: word i of what any query of the row sees
          uni = 0u;
          for (int i = 0; i < T.W; ++i) {
            uint32_t word = 0;
#pragma unroll 4
            for (int q = lane; q < A.qlen; q += 32) word |= tree_word(mask0 + (int64_t)q * T.W, T.W, T.N, i);
            word = __reduce_or_sync(0xffffffffu, word);
            if (lane == i) uni = word;
          }
          settled = true;
        };
        // of the tile in turn, and of the other one
        float m = -CUDART_INF_F, l = 0.f, m2 = -CUDART_INF_F, l2 = 0.f;
        bool wild = false, wild2 = false;
#pragma unroll 1
        for (int i = 0; i < pages && ok; ++i, ++n) {
#pragma unroll 1
          for (int ti = 0; ti < NT; ++ti, ++k) {
            ok = __all_sync(0xffffffffu, tc_wait(&S.sfull[k & 1u], (k >> 1) & 1u, &S.abort_));
            if (!ok) break;
            tc_fence_after();
            const uint32_t scol = lcol + 128u * (k & 1u) + 64u * x;
            const int key0 = (cur.j0 + i) * SD_KV_PAGE;
            const bool idle = (dead >> ti) & 1u;
            if (key0 + SD_KV_PAGE > cur.base) {
              // the tree's pages, and what lies behind it
              if (!settled) settle();
              if (!idle) tt_hide(S.mask[ti][r], T, cur.base, end, key0 + 64 * x, 64, scol);
              if (ti == 0) {
                // each warpgroup its half of the keys, two warps 32 of them
                const uint32_t vi = 2u * n + 1u;
                const int grp = 2 * x + (wq & 1);
                ok = tt_blank(S.kv[vi % SLOTS], T, uni, cur.base, end, key0 + 32 * grp, 32 * grp,
                              wq >> 1, (wq >> 1) + 1, &S.full[vi % SLOTS], (vi / SLOTS) & 1u,
                              &S.abort_);
                if (!ok) break;
              }
            }
            if (!idle) {
              uint32_t s0[32], s1[32], pk[32];
              unsigned long long ls[2];
              auto largest = [&]() {
                float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  px_max3(mx[e & 2], s0[e], s0[e + 1]);
                  px_max3(mx[(e & 2) + 1], s1[e], s1[e + 1]);
                }
                return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
              };
              if (i == 0) {                            // a reference for the segment
                TC_LD32(s0, scol);
                TC_LD32(s1, scol + 32u);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                const float mine = largest();
                tell(mine);
                m = fmaxf(mine, told());
                if (!ok) break;
                wild = px_wild(m);
              }
              // weights under the reference as it is, and the largest score beside them: where
              // that is too far above it (rare), the reference moves and the weights are made again
              while (true) {
                TC_LD32(s0, scol);
                TC_LD32(s1, scol + 32u);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                const float mine = largest();
                if (wild) {
                  px_scale(s0, sl2);
                  px_scale(s1, sl2);
                }
                const float mc = m == -CUDART_INF_F ? 0.f : m, sf = wild ? 1.f : sl2;
                const unsigned long long sl22 = pair2(sf, sf), nm2 = pair2(-mc, -mc);
                ls[0] = ls[1] = 0ULL;                  // (0.f, 0.f)
                tell(mine);
                tt_weights(s0, pk, ls, sl22, nm2);
                tt_weights(s1, pk + 16, ls, sl22, nm2);
                const float mt = fmaxf(mine, told());
                if (!ok) break;
                const bool move = mt > m + PX_HEADROOM;
                if (!__any_sync(0xffffffffu, move)) break;
                const float mn = move ? mt : m;
                const float alpha = move ? (m == -CUDART_INF_F ? 0.f : ex2f(m - mn)) : 1.f;
                m = mn;
                l *= alpha;
                wild = px_wild(m);
                if (i > 0) {
                  // O holds this segment's earlier pages: the last P . V into it first; each
                  // warpgroup half of the columns
                  ok = __all_sync(0xffffffffu, o_ready(ti));
                  if (!ok) break;
                  tc_fence_after();
#pragma unroll 1
                  for (int q = 0; q < 4; ++q) {
                    const uint32_t oc = lcol + 256u + 128u * ti + 64u * x + 16u * q;
                    uint32_t o[16];
                    TC_LD16(o, oc);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    TC_ST16(oc, o);
                  }
                }
              }
              if (!ok) break;
              TC_ST32(scol, pk);                       // over columns that have been read
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              float la, lb;
              unpair(add2(ls[0], ls[1]), la, lb);
              l += la + lb;
            }
            tc_fence_before();
            tt_arrive(&S.pfull[k & 1u]);
            if constexpr (NT == 2) {                   // the other tile's turn
              const float tm0 = m, tl0 = l;
              const bool tw0 = wild;
              m = m2; l = l2; wild = wild2;
              m2 = tm0; l2 = tl0; wild2 = tw0;
            }
          }
        }
        if (!ok) break;
        // ---- the segment's end: O divided by the row's sum and written out, or as a piece; each
        // warpgroup half of the columns
        const bool whole = cur.j0 == 0 && cur.j1 + TT_OVH == cur.tb;
        const int slot = 2 * cta + (cur.j0 == 0);
#pragma unroll 1
        for (int ti = 0; ti < NT; ++ti) {
          if (!((dead >> ti) & 1u)) {
            tell(l);
            const float lp = told();
            ok = ok && __all_sync(0xffffffffu, o_ready(ti));
            if (!ok) break;
            tc_fence_after();
            l = x ? lp + l : l + lp;                 // (the first warpgroup's half first, in both)
            const int pr = P.nt * A.group * ti + r;
            const bool live = r < rows_of(cur, ti);
            const float il = !whole ? 1.f : l == 0.f || !((there >> ti) & 1u) ? 0.f : 1.f / l;
            const int jt = r / A.group, j = cur.p * P.ni + P.nt * ti + jt;
            const int hq = cur.h * A.group + r - jt * A.group;
            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(A.out) + cur.b * A.obs + j * A.oqs +
                                 hq * A.ohs;
            float4* part = P.pacc + (int64_t)slot * (TT_D / 4) * P.rs + pr;
#pragma unroll 1
            for (int q = 2 * x; q < 2 * x + 2; ++q) {
              uint32_t u[32];
              TC_LD32(u, lcol + 256u + 128u * ti + 32u * q);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
              float o[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = il == 0.f ? 0.f : il * __uint_as_float(u[e]);
              if (whole) {
                tt_write(stage, o, out + 32 * q, live, P.out_vec != 0);
              } else if (live) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  part[(int64_t)(8 * q + e) * P.rs] =
                      make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
              }
              __syncwarp();
            }
            if (!whole && live && x == 0) P.pml[(int64_t)slot * P.rs + pr] = make_float2(m, l);
          }
          m = m2;
          l = l2;
        }
        if (!ok) break;
        tc_fence_before();
      }
    }
  }
  tc_fence_before();
  __syncthreads();                                   // every role is done
  if (t == 0) P.status[cta] = S.abort_;
  if (w == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 :: "r"(tm), "r"(512u) : "memory");
  }
}

// CTA (boundary c, rows): where CTA c's run ends inside an item that it is the first to
// work on, the item's pieces are merged, in order; a lane takes a query row, a warp
// 16 columns.
__global__ void __launch_bounds__(TJ_THREADS) tree_join_kernel(const __grid_constant__ TreeTcParams P) {
  const TreeParams& T = P.T;
  const AttnParams& A = T.A;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int c = (int)blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int stop = t < TT_CTAS ? P.status[t] : 0;
  const int per = A.Hkv * P.np, total = P.rowpre[A.B] * per, share = tt_share(total);
  if (__syncthreads_or(stop)) {
    // a wait gave up somewhere: say so in the output
    const int64_t n = (int64_t)A.B * A.qlen * A.Hq * TT_D, nt = (int64_t)gridDim.x * gridDim.y * TJ_THREADS;
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + c) * TJ_THREADS + t; i < n; i += nt) {
      const int64_t v = i / TT_D, bj = v / A.Hq;
      reinterpret_cast<__nv_bfloat16*>(A.out)[(bj / A.qlen) * A.obs + (bj % A.qlen) * A.oqs +
                                              (v % A.Hq) * A.ohs + i % TT_D] =
          __float2bfloat16(CUDART_NAN_F);
    }
    return;
  }
  const int64_t U = (int64_t)(c + 1) * share;
  if (U >= total) return;
  int lo = 0, hi = A.B;                              // the last row that starts at or before U
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)P.rowpre[mid] * per <= U) lo = mid + 1; else hi = mid;
  }
  const int b = lo - 1, u0 = P.rowpre[b] * per, tb = P.rowpre[b + 1] - P.rowpre[b];
  const int it = ((int)U - u0) / tb, h = it / P.np, p = it % P.np;
  const int start = u0 + it * tb + TT_OVH;           // the unit of the item's first page
  const int c0 = start / share, c1 = (u0 + it * tb + tb - 1) / share;
  if (c0 != c || c1 == c) return;
  const int rows = A.group * min(P.ni, A.qlen - p * P.ni), np = c1 - c0 + 1;
  const int r = (int)blockIdx.y * TJ_ROWS + lane;
  if (r >= rows) return;
  // piece i: the item's start in its first CTA, then a CTA's start each
  auto slot_of = [&](int i) { return (int64_t)(2 * (c + i) + (i == 0)); };
  float gm = -CUDART_INF_F;
#pragma unroll 4
  for (int i = 0; i < np; ++i) gm = fmaxf(gm, __ldcg(&P.pml[slot_of(i) * P.rs + r]).x);
  float L = 0.f;
  float4 a[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int i = 0; i < np; ++i) {
    const float2 ml = __ldcg(&P.pml[slot_of(i) * P.rs + r]);
    const float4* src = P.pacc + (slot_of(i) * (TT_D / 4) + 4 * w) * P.rs + r;
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __ldcg(src + (int64_t)k * P.rs);
    const float fw = ml.x == -CUDART_INF_F ? 0.f : ex2f(ml.x - gm);
    L += ml.y != ml.y ? ml.y : fw * ml.y;
    if (fw != 0.f) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k].x = fmaf(fw, v[k].x, a[k].x); a[k].y = fmaf(fw, v[k].y, a[k].y);
        a[k].z = fmaf(fw, v[k].z, a[k].z); a[k].w = fmaf(fw, v[k].w, a[k].w);
      }
    }
  }
  const int ji = r / A.group, j = p * P.ni + ji, hq = h * A.group + r - ji * A.group;
  const int32_t* mask = T.masks + (int64_t)b * T.mask_bs + (int64_t)(T.first + j) * T.W;
  const bool none = L == 0.f || !tree_present(mask, T.W, T.N);
  const float il = none ? 0.f : 1.f / L;
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(A.out) + b * A.obs + j * A.oqs + hq * A.ohs + 16 * w;
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (!none) {
      u.x = pack_bf16(a[k].x * il, a[k].y * il);
      u.y = pack_bf16(a[k].z * il, a[k].w * il);
      u.z = pack_bf16(a[k + 1].x * il, a[k + 1].y * il);
      u.w = pack_bf16(a[k + 1].z * il, a[k + 1].w * il);
    }
    if (P.out_vec) {
      *reinterpret_cast<uint4*>(dst + 4 * k) = u;
    } else {
      const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&u);
#pragma unroll
      for (int q = 0; q < 8; ++q) dst[4 * k + q] = e[q];
    }
  }
}

// The shapes of the tensor-core path.
static bool tt_fast(int dtype, int D, int group) {
  return dtype == SD_DTYPE_BF16 && D == TT_D && group <= 128;
}

struct TtLayout {
  size_t status, acc, ml, bytes;
  int np, ni, nt, rs;
};
static TtLayout tt_layout(int qlen, int group, int B) {
  TtLayout L;
  // items of up to two tiles of whole nodes, of about the same size, and so their tiles
  const int most = TT_TILE / group;
  L.np = (qlen + 2 * most - 1) / (2 * most);
  L.ni = (qlen + L.np - 1) / L.np;
  L.nt = qlen <= most ? qlen : (L.ni + 1) / 2;
  L.rs = (L.ni * group + 31) / 32 * 32;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t o = up(((size_t)B + 1) * sizeof(int));
  L.status = o; o = up(o + TT_CTAS * sizeof(int));
  L.acc = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * TT_D * sizeof(float));
  L.ml = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * 2 * sizeof(float));
  L.bytes = o;
  return L;
}

template <int NT>
static int launch_tc(const TreeTcParams& P, const CUtensorMap& mk, const CUtensorMap& mv,
                     const CUtensorMap& mq, cudaStream_t st) {
  const int sm = (int)sizeof(TtSmem<NT>) + 1024;   // room to align
  static std::atomic<uint64_t> ready{0};             // devices whose kernel may use that much
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SD_ELAUNCH;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load() & bit) || !bit) {
    if (cudaFuncSetAttribute(tree_tc_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) !=
        cudaSuccess)
      return SD_ELAUNCH;
    ready.fetch_or(bit);
  }
  tree_tc_kernel<NT><<<TT_CTAS, TT_THREADS, sm, st>>>(P, mk, mv, mq);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

static int tree_tc(TreeTcParams& P, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  AttnParams& A = P.T.A;
  // TMA boxes of the queries and the caches
  if ((reinterpret_cast<uintptr_t>(A.q) & 15) || A.qbs % 8 || A.qhs % 8 || A.qqs % 8 ||
      (reinterpret_cast<uintptr_t>(A.k) & 15) || (reinterpret_cast<uintptr_t>(A.v) & 15))
    return SD_EINVAL;
  if ((A.B > 1 && A.qbs <= 0) || (A.Hq > 1 && A.qhs <= 0) || (A.qlen > 1 && A.qqs <= 0)) return SD_EINVAL;
  const int64_t rows = A.bt ? (int64_t)A.npages * A.Hkv * SD_KV_PAGE : (int64_t)A.B * A.Hkv * A.C;
  if (rows >= (int64_t)1 << 31) return SD_ENOTSUP;   // a TMA coordinate
  const TtLayout L = tt_layout(A.qlen, A.group, A.B);
  // the schedule counts units in 32 bits
  const int64_t tiles = ((int64_t)A.C + SD_KV_PAGE - 1) / SD_KV_PAGE + TT_OVH;
  if (tiles * A.B > 0x7FFFFFFF / ((int64_t)A.Hkv * L.np)) return SD_ENOTSUP;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < L.bytes)
    return SD_ENOSPC;
  char* ws = reinterpret_cast<char*>(workspace);
  P.np = L.np; P.ni = L.ni; P.nt = L.nt; P.rs = L.rs;
  P.rowpre = reinterpret_cast<int*>(ws);
  P.status = reinterpret_cast<int*>(ws + L.status);
  P.pacc = reinterpret_cast<float4*>(ws + L.acc);
  P.pml = reinterpret_cast<float2*>(ws + L.ml);
  P.out_vec = (reinterpret_cast<uintptr_t>(A.out) & 15) == 0 && A.obs % 8 == 0 && A.oqs % 8 == 0 &&
              A.ohs % 8 == 0;
  CUtensorMap mk, mv, mq;
  if (!cache_map(&mk, A.k, rows) || !cache_map(&mv, A.v, rows)) return SD_ENOTSUP;
  // the queries of a tile: 64 columns of `group` heads of L.nt nodes of a row
  const int64_t sizes[4] = {TT_D, A.Hq, A.qlen, A.B}, strides[3] = {A.qhs, A.qqs, A.qbs};
  const int box[4] = {64, A.group, L.nt, 1};
  if (!tile_map(&mq, A.q, sizes, strides, box)) return SD_ENOTSUP;
  if (int rc = L.nt < L.ni ? launch_tc<2>(P, mk, mv, mq, st) : launch_tc<1>(P, mk, mv, mq, st)) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3(TT_CTAS - 1, (unsigned)((L.rs + TJ_ROWS - 1) / TJ_ROWS));
  cfg.blockDim = dim3(TJ_THREADS);
  if (cudaLaunchKernelEx(&cfg, tree_join_kernel, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // namespace sd

using namespace sd;

extern "C" {

size_t sd_tree_attn_workspace_bytes(int B, int Hq, int Hkv, int D, int C, int qlen, int dtype) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || C <= 0 || qlen <= 0) return 0;
  if (!tt_fast(dtype, D, Hq / Hkv) || (int64_t)qlen * (Hq / Hkv) > 0x7FFFFFFF) return 0;
  return tt_layout(qlen, Hq / Hkv, B).bytes;
}

int sd_tree_attn(const void* q, int64_t qbs, int64_t qhs, int64_t qqs, const void* kcache,
                 const void* vcache, const int32_t* block_table, int bt_stride, int npages,
                 const int64_t* lengths, const int32_t* masks, int64_t mask_bs, int N, int first,
                 int B, int Hq, int Hkv, int D, int C, int qlen, float scale, void* out,
                 int64_t obs, int64_t oqs, int64_t ohs, int dtype, void* workspace,
                 size_t workspace_bytes, void* stream) {
  if (B < 0 || qlen < 0 || N < 0 || first < 0) return SD_EINVAL;
  if (B == 0 || qlen == 0) return SD_OK;
  if (!q || !kcache || !vcache || !lengths || !masks || !out) return SD_EINVAL;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || first + qlen > N) return SD_EINVAL;
  if (!(scale > 0.f) || scale > 3e38f) return SD_EINVAL;
  if (dtype != SD_DTYPE_BF16 && dtype != SD_DTYPE_F32) return SD_ENOTSUP;
  if (N > SD_TREE_MAX) return SD_ENOTSUP;
  if (block_table) {
    if (bt_stride <= 0 || npages <= 0) return SD_EINVAL;
    if ((int64_t)bt_stride * SD_KV_PAGE > 0x7FFFFFFF) return SD_ENOTSUP;
    C = bt_stride * SD_KV_PAGE;
  }
  if (C <= 0) return SD_EINVAL;
  // the end of the last key's tile is a 32-bit number
  if (C > 0x7FFFFFFF - 2 * SD_KV_PAGE - SD_TREE_MAX) return SD_ENOTSUP;
  const int group = Hq / Hkv;
  const int64_t R = (int64_t)qlen * group;
  if (R > 0x7FFFFFFF) return SD_ENOTSUP;
  TreeTcParams P = {};
  AttnParams& A = P.T.A;
  A.q = q; A.qbs = qbs; A.qhs = qhs; A.qqs = qqs;
  A.k = kcache; A.v = vcache; A.lengths = lengths;
  A.B = B; A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.C = C; A.qlen = qlen;
  A.group = group; A.R = (int)R; A.scale = scale;
  A.out = out; A.obs = obs; A.oqs = oqs; A.ohs = ohs;
  A.bt = block_table; A.bt_stride = bt_stride; A.npages = npages;
  P.T.masks = masks; P.T.mask_bs = mask_bs; P.T.N = N; P.T.W = (N + 31) / 32; P.T.first = first;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return tt_fast(dtype, D, group) ? tree_tc(P, workspace, workspace_bytes, st)
                                  : tree_rows(P.T, dtype, st);
}

}  // extern "C"
