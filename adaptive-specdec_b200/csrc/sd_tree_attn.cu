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
constexpr int TT_ROWS = 256;                 // query rows of an item: two tiles of 128
constexpr int TT_SLOTS = 4;                  // 32 KB K / V tiles in flight (two pages)
constexpr int TT_THREADS = 320;              // warps 0-3, 4-7: softmax of tile 0, 1; 8 TMA; 9 MMA
constexpr int TT_CTAS = 148;                 // one CTA per SM
constexpr int TT_OVH = 2;                    // schedule cost of an item beyond its pages, in pages
constexpr int TT_MIN_SHARE = TT_OVH + 1;     // fewest schedule units per CTA: a one-page item
constexpr int TT_BASES = 1024;               // rows whose bases a CTA keeps
constexpr int TJ_THREADS = 256;
constexpr int TJ_ROWS = 32;                  // query rows of a join CTA

struct TreeTcParams {
  TreeParams T;
  int np, rs;                                // items of a (row, kv head); rows of a piece
  int out_vec;                               // 16-byte stores of the output are aligned
  // workspace
  int* rowpre;                               // [B + 1] exclusive prefix of a row's units per item
  int* status;                               // [TT_CTAS] a bounded wait gave up
  float* pacc;                               // [2 TT_CTAS][rs][128] pieces
  float* pml;                                // [2 TT_CTAS][rs][2]
};

__device__ __forceinline__ int tt_units(int end) { return (end + SD_KV_PAGE - 1) / SD_KV_PAGE + TT_OVH; }
__device__ __forceinline__ int tt_share(int total) {
  return max(TT_MIN_SHARE, (total + TT_CTAS - 1) / TT_CTAS);
}

struct TtSmem {
  alignas(1024) unsigned char q[2][2][128 * 128];            // [tile][64-col box][128 rows x 128 B]
  alignas(1024) unsigned char kv[TT_SLOTS][2][128 * 128];    // [slot][64-col box][128 keys x 128 B]
  alignas(8) unsigned long long full[TT_SLOTS], empty[TT_SLOTS];
  alignas(8) unsigned long long sfull[2], pfull[2], oready[2], qfull[2], fin;
  alignas(8) unsigned long long mlfull, ofree;       // where both tiles work on the same rows
  float ml[2][128][2];                       // the tiles' (m, l) where both work on the same rows
  int base[TT_BASES];
  int red[33];
  int first[2];                              // the CTA's first row and the units before it
  int abort_;
  uint32_t tmem;
};
static_assert(sizeof(TtSmem) + 1024 <= 227 * 1024, "shared memory, with room to align");

// A CTA's run of schedule units as segments of items, walked identically by
// every role: row-major, kv head and then the 256 query rows inner; TT_OVH virtual
// units in front of each item's pages.
struct TtSeg {
  int b, h, p, base, tb, off, tt, t1, ncost, j0, j1;         // pages [j0, j1) of the segment
  bool dup;                                          // one tile of rows: both tiles work on it
};
__device__ __forceinline__ int tt_base(const TtSmem& S, const TreeParams& T, int b) {
  return b < TT_BASES ? S.base[b] : tree_base(T, b);
}
__device__ __forceinline__ void tt_bounds(TtSeg& s, const TreeTcParams& P) {
  s.dup = P.T.A.R - s.p * TT_ROWS <= TT_ROWS / 2;
  s.ncost = min(s.tb - s.off, s.t1 - s.tt);
  s.j0 = max(s.off, TT_OVH) - TT_OVH;
  s.j1 = max(s.off + s.ncost - TT_OVH, s.j0);
}
__device__ __forceinline__ bool tt_next(TtSeg& s, const TtSmem& S, const TreeTcParams& P) {
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
  tt_bounds(s, P);
  return true;
}
// On to the current or next segment with pages; false when none is left.
__device__ __forceinline__ bool tt_real(TtSeg& s, const TtSmem& S, const TreeTcParams& P) {
  while (s.j1 == s.j0)
    if (!tt_next(s, S, P)) return false;
  return true;
}

// Eight outputs of a query row.
__device__ __forceinline__ void tt_store8(__nv_bfloat16* dst, const float* o, bool vec) {
  uint4 u;
  u.x = pack_bf16(o[0], o[1]);
  u.y = pack_bf16(o[2], o[3]);
  u.z = pack_bf16(o[4], o[5]);
  u.w = pack_bf16(o[6], o[7]);
  if (vec) {
    *reinterpret_cast<uint4*>(dst) = u;
  } else {
    const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = e[i];
  }
}

__global__ void __launch_bounds__(TT_THREADS, 1)
tree_tc_kernel(const __grid_constant__ TreeTcParams P, const __grid_constant__ CUtensorMap tmk,
               const __grid_constant__ CUtensorMap tmv) {
  extern __shared__ __align__(1024) unsigned char tt_raw[];
  const uint32_t pad = (1024u - (smem_addr(tt_raw) & 1023u)) & 1023u;   // swizzle atoms: 1024 B
  TtSmem& S = *reinterpret_cast<TtSmem*>(tt_raw + pad);
  const TreeParams& T = P.T;
  const AttnParams& A = T.A;
  const int t = threadIdx.x, w = t >> 5, lane = t & 31, cta = (int)blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (w == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_addr(&S.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (t == 0) {
    for (int i = 0; i < TT_SLOTS; ++i) {
      tc_bar_init(&S.full[i], 1);
      tc_bar_init(&S.empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      tc_bar_init(&S.qfull[x], 128);
      tc_bar_init(&S.sfull[x], 1);
      tc_bar_init(&S.pfull[x], 128);
      tc_bar_init(&S.oready[x], 1);
    }
    tc_bar_init(&S.fin, 1);
    tc_bar_init(&S.mlfull, 256);
    tc_bar_init(&S.ofree, 256);
    S.abort_ = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // ---- the schedule: every CTA sums the rows' units, then looks for its own first row
  const int per = A.Hkv * P.np;                      // items of a row
  int sum = 0;
  for (int b0 = 0; b0 < A.B; b0 += TT_THREADS) {
    const int b = b0 + t;
    if (b < A.B) {
      const int base = tree_base(T, b);
      if (b < TT_BASES) S.base[b] = base;
      sum += tt_units(tree_end(T, base));
    }
  }
  const int rows_units = block_sum<int>(sum, S.red);
  const int total = rows_units * per, share = tt_share(total);
  const bool work = (int64_t)cta * share < total;
  const int t0 = work ? cta * share : 0, t1 = t0 + min(total - t0, share);
  int carry = 0;
  for (int b0 = 0; b0 < A.B; b0 += TT_THREADS) {
    const int b = b0 + t;
    const int u = b < A.B ? tt_units(tree_end(T, tt_base(S, T, b))) : 0;
    int all;
    const int ex = carry + block_excl_scan<int>(u, S.red, &all);
    if (b < A.B) {
      if (cta == 0) P.rowpre[b] = ex;
      if (ex * per <= t0 && t0 < (ex + u) * per) {
        S.first[0] = b;
        S.first[1] = ex * per;
      }
    }
    carry += all;
    __syncthreads();                                 // red is written again next
  }
  if (cta == 0 && t == 0) P.rowpre[A.B] = carry;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = S.tmem;
  if (work) {
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
    tt_bounds(seg, P);
    bool more = tt_real(seg, S, P);

    if (w == 8) {
      if (lane == 0) {
        // ---------------- TMA producer: K then V of each page, TT_SLOTS tiles ahead
        uint32_t idx = 0;
        bool ok = true;
        while (more && ok) {
          for (int j = seg.j0; j < seg.j1 && ok; ++j) {
            const int y = (int)kv_row(A, seg.b, seg.h, j * SD_KV_PAGE);
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv, ++idx) {
              const int sl = (int)(idx % TT_SLOTS);
              if (idx >= (uint32_t)TT_SLOTS)
                ok = tc_wait(&S.empty[sl], ((idx / TT_SLOTS) - 1) & 1u, &S.abort_);
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
          for (uint32_t q = idx > (uint32_t)TT_SLOTS ? idx - TT_SLOTS : 0u; q < idx; ++q) {
            int dummy = 0;
            tc_wait(&S.full[q % TT_SLOTS], (q / TT_SLOTS) & 1u, &dummy);
          }
        }
      }
    } else if (w == 9) {
      // ---------------- MMA issuer (the whole warp): S0(0) S1(0) | PV0(i) S0(i + 1)
      // PV1(i) S1(i + 1) | ...
      constexpr uint32_t ID1 = tc_idesc(128, 128, 0, 0);     // S = Q . K^T
      constexpr uint32_t ID1H = tc_idesc(128, 64, 0, 0);     // of half a page
      constexpr uint32_t ID2 = tc_idesc(128, 128, 0, 1);     // O += P . V (V [key][d]: N-major)
      const uint32_t kv0 = smem_addr(S.kv[0][0]), q0 = smem_addr(S.q[0][0]);
      uint32_t qn = 0, g = 0;                        // segments, pages done
      bool ok = true, dup = false;
      // K of ring page g is in slot 2 (g & 1), its V in slot 2 (g & 1) + 1
      auto issue_s = [&](uint32_t x, uint32_t ring) {
        const uint32_t sl = 2u * (ring & 1u), d = tm + 128u * x, id = dup ? ID1H : ID1;
        const uint64_t dq = tc_desc(q0 + x * 32768u, 16, 1024, 2);
        const uint64_t dk = tc_desc(kv0 + sl * 32768u + (dup ? x * 8192u : 0u), 16, 1024, 2);
        ok = tc_wait2_warp(&S.full[sl], (ring >> 1) & 1u, &S.qfull[x], qn & 1u, &S.abort_);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {             // 16 of 128 d: 32 B, the second box 16 KB on
          const uint64_t o = (uint64_t)((ks & 3) * 2 + (ks >> 2) * 1024);
          tc_mma_warp(d, dq + o, dk + o, id, ks > 0 ? 1 : 0);
        }
        tc_commit_warp(&S.sfull[x]);
        if (x == 1u) tc_commit_warp(&S.empty[sl]);
      };
      auto issue_pv = [&](uint32_t x, bool first) {
        const uint32_t sl = 2u * (g & 1u) + 1u, a = tm + 128u * x;
        const uint64_t dv = tc_desc(kv0 + sl * 32768u + (dup ? x * 8192u : 0u), 16384, 1024, 2);
        ok = tc_wait2_warp(&S.full[sl], (g >> 1) & 1u, &S.pfull[x], g & 1u, &S.abort_);
        if (!ok) return;
        tc_fence_after();
        for (int k4 = 0; k4 < 8; k4 += 4) {          // 16 keys: 2 KB
          if (k4 > 0 && dup) break;
#pragma unroll
          for (int ks = k4; ks < k4 + 4; ++ks)
            tc_mma_ts_warp(a + 256u, a + 8u * ks, dv + (uint64_t)(ks * 128), ID2,
                           ks || !first ? 1 : 0);
        }
        tc_commit_warp(&S.oready[x]);
        if (x == 1u) tc_commit_warp(&S.empty[sl]);
      };
      while (more && ok) {
        const int pages = seg.j1 - seg.j0;
        dup = seg.dup;
        // page i: P . V of a tile, then its S of page i + 1; i = -1: the first S
#pragma unroll 1
        for (int i = -1; i < pages && ok; ++i) {
#pragma unroll 1
          for (uint32_t x = 0; x < 2u && ok; ++x) {
            if (i >= 0) issue_pv(x, i == 0);
            if (ok && i + 1 < pages) issue_s(x, i < 0 ? g : g + 1u);
          }
          if (i >= 0) ++g;
        }
        ++qn;
        if (ok) more = tt_next(seg, S, P) && tt_real(seg, S, P);
      }
      // every MMA this warp issued has finished before the CTA leaves
      tc_commit_warp(&S.fin);
      int dummy = 0;
      tc_wait(&S.fin, 0u, &dummy);
    } else {
      // ---------------- softmax warps of tile x: thread r owns query row r
      const int x = w >> 2, wq = w & 3, r = t & 127;
      const uint32_t lrow = (uint32_t)(32 * wq) << 16;
      const uint32_t scol = tm + lrow + 128u * x, ocol = scol + 256u;
      const float sl2 = A.scale * 1.4426950408889634f;
      // the tile's 128 query rows, 16 lanes a row (rows past the item's: zeros)
      auto load_q = [&](const TtSeg& g) {
        const int r0 = g.p * TT_ROWS + (g.dup ? 0 : 128 * x);
        const __nv_bfloat16* Q = reinterpret_cast<const __nv_bfloat16*>(A.q) + g.b * A.qbs;
        const int c = lane & 15;
        unsigned char* dst = S.q[x][c >> 3];
#pragma unroll 1
        for (int i0 = 0; i0 < 16; i0 += 8) {
          uint4 v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = 32 * wq + 2 * (i0 + i) + (lane >> 4), f = r0 + row;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (f < A.R) {
              const int j = f / A.group, hq = g.h * A.group + f - j * A.group;
              v[i] = __ldg(reinterpret_cast<const uint4*>(Q + hq * A.qhs + j * A.qqs) + c);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = 32 * wq + 2 * (i0 + i) + (lane >> 4);
            *reinterpret_cast<uint4*>(dst + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[i];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_arrive(&S.qfull[x]);
      };
      uint32_t n = 0, dn = 0;                        // pages done; segments that both tiles did
      bool ok = true;
      if (more) load_q(seg);
      while (more) {
        const TtSeg cur = seg;
        more = tt_next(seg, S, P) && tt_real(seg, S, P);
        const int pages = cur.j1 - cur.j0, halves = cur.dup ? 1 : 2;
        const int f = cur.p * TT_ROWS + (cur.dup ? 0 : 128 * x) + r;     // row of the (row, kv head)
        const bool live = f < A.R;
        const bool dead = __all_sync(0xffffffffu, !live);    // a warp without rows
        const int32_t* mask0 = T.masks + (int64_t)cur.b * T.mask_bs + (int64_t)T.first * T.W;
        const int32_t* mask = mask0 + (int64_t)(live ? f / A.group : 0) * T.W;
        const int end = tree_end(T, cur.base);
        float m = -CUDART_INF_F, l = 0.f;
        bool wild = false;
#pragma unroll 1
        for (int i = 0; i < pages; ++i) {
          ok = __all_sync(0xffffffffu, tc_wait(&S.sfull[x], n & 1u, &S.abort_));
          if (!ok) break;
          tc_fence_after();
          // the segment's S are all done with Q: the next segment's may come
          if (i == pages - 1 && more) load_q(seg);
          const int key0 = (cur.j0 + i) * SD_KV_PAGE;
          if (key0 + SD_KV_PAGE > cur.base) {
            // The tree's pages, and what lies behind it.  Scores that the row's node does
            // not see to -inf, in TMEM, 32 columns at a time (a short loop: this code is
            // cold whenever it runs).
            const int k0 = key0 + (cur.dup ? 64 * x : 0);
            if (!dead) {
#pragma unroll 1
              for (int c = 0; c < 2 * halves; ++c) {
                uint32_t sees = tree_sees(mask, T.W, T.N, cur.base, k0 + 32 * c);
                const int left = end - (k0 + 32 * c);        // (the capacity may cut the tree)
                if (left < 32) sees &= left > 0 ? (1u << left) - 1u : 0u;
                if (__all_sync(0xffffffffu, sees == 0xFFFFFFFFu)) continue;
                uint32_t s[32];
                TC_LD32(s, scol + 32u * c);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int e = 0; e < 32; ++e) s[e] = (sees >> e) & 1u ? s[e] : 0xFF800000u;
                TC_ST32(scol + 32u * c, s);
              }
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            // Slots that no node sees may hold NaN: their V to zero.  The warps of tile 0
            // (of both, each its half, where both work on the same rows) take 32 keys each.
            if (x == 0 || cur.dup) {
              const int grp = cur.dup ? 2 * x + (wq & 1) : wq;
              const int kg = key0 + 32 * grp;
              uint32_t any = 0;
              for (int q = lane; q < A.qlen; q += 32) {
                const int32_t* mq = mask0 + (int64_t)q * T.W;
                if (tree_present(mq, T.W, T.N)) any |= tree_sees(mq, T.W, T.N, cur.base, kg);
              }
              any = __reduce_or_sync(0xffffffffu, any);
              const int left = end - kg;
              if (left < 32) any &= left > 0 ? (1u << left) - 1u : 0u;
              if (any != 0xFFFFFFFFu) {
                const uint32_t sl = 2u * (n & 1u) + 1u;
                ok = __all_sync(0xffffffffu, tc_wait(&S.full[sl], (n >> 1) & 1u, &S.abort_));
                if (!ok) break;
                // four keys of a 128-byte box at a time
                for (int k4 = 0; k4 < 32; k4 += 4) {
                  const int kr = k4 + (lane >> 3);
                  if ((any >> kr) & 1u) continue;
                  const int at = (32 * grp + kr) * 128 + (lane & 7) * 16;
                  if (!cur.dup || wq < 2)
                    *reinterpret_cast<uint4*>(S.kv[sl][0] + at) = make_uint4(0u, 0u, 0u, 0u);
                  if (!cur.dup || wq >= 2)
                    *reinterpret_cast<uint4*>(S.kv[sl][1] + at) = make_uint4(0u, 0u, 0u, 0u);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              }
            }
          }
          if (!dead) {
            // the scores twice from TMEM, 64 columns at a time: for the maximum, then
            // for the exponentials
            uint32_t sa[32], sb[32];
            float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll 1
            for (int c = 0; c < halves; ++c) {
              TC_LD32(sa, scol + 64u * c);
              TC_LD32(sb, scol + 64u * c + 32u);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                px_max3(mx[e & 2], sa[e], sa[e + 1]);
                px_max3(mx[(e & 2) + 1], sb[e], sb[e + 1]);
              }
            }
            const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
            const bool move = mt > m + PX_HEADROOM;
            if (__any_sync(0xffffffffu, move)) {
              const float mn = move ? mt : m;
              const float alpha = move ? (m == -CUDART_INF_F ? 0.f : ex2f(m - mn)) : 1.f;
              m = mn;
              l *= alpha;
              wild = px_wild(m);
              if (i > 0) {
                // O holds this segment's earlier pages: the last P . V into it first
                ok = __all_sync(0xffffffffu, tc_wait(&S.oready[x], (n - 1) & 1u, &S.abort_));
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                  uint32_t o[32];
                  TC_LD32(o, ocol + 32u * q);
                  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                  TC_ST32(ocol + 32u * q, o);
                }
              }
            }
            const float mc = m == -CUDART_INF_F ? 0.f : m, sf = wild ? 1.f : sl2;
            const unsigned long long sl22 = pair2(sf, sf), nm2 = pair2(-mc, -mc);
            unsigned long long ls[2] = {0ULL, 0ULL};   // (0.f, 0.f)
            uint32_t pk[32];
#pragma unroll 1
            for (int c = 0; c < halves; ++c) {
              TC_LD32(sa, scol + 64u * c);
              TC_LD32(sb, scol + 64u * c + 32u);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
              if (wild) {
                px_scale(sa, sl2);
                px_scale(sb, sl2);
              }
              px_weights(sa, pk, ls, sl22, nm2);
              px_weights(sb, pk + 16, ls, sl22, nm2);
              TC_ST32(scol + 32u * c, pk);             // over columns that have been read
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            float la, lb;
            unpair(add2(ls[0], ls[1]), la, lb);
            l += la + lb;
          }
          tc_fence_before();
          tc_arrive(&S.pfull[x]);
          ++n;
        }
        if (!ok) break;
        // ---- the segment's end: the row's sum and O, divided and written out, or as a piece
        ok = __all_sync(0xffffffffu, tc_wait(&S.oready[x], (n - 1) & 1u, &S.abort_));
        if (cur.dup) {
          // both tiles hold a part of the same rows: each writes half of the columns
          S.ml[x][r][0] = m;
          S.ml[x][r][1] = l;
          tc_arrive(&S.mlfull);
          ok = ok && __all_sync(0xffffffffu, tc_wait(&S.mlfull, dn & 1u, &S.abort_) &&
                                                 tc_wait(&S.oready[x ^ 1], (n - 1) & 1u, &S.abort_));
        }
        if (!ok) break;
        {
          tc_fence_after();
          float w0 = 1.f, w1 = 0.f;
          if (cur.dup) {
            const float m0 = S.ml[0][r][0], m1 = S.ml[1][r][0], l0 = S.ml[0][r][1], l1 = S.ml[1][r][1];
            m = fmaxf(m0, m1);
            w0 = m0 == -CUDART_INF_F ? 0.f : ex2f(m0 - m);
            w1 = m1 == -CUDART_INF_F ? 0.f : ex2f(m1 - m);
            l = (l0 != l0 ? l0 : w0 * l0) + (l1 != l1 ? l1 : w1 * l1);
          }
          const bool whole = cur.j0 == 0 && cur.j1 + TT_OVH == cur.tb;
          const bool there = live && tree_present(mask, T.W, T.N);
          const float il = l == 0.f ? 0.f : 1.f / l;             // (a NaN sum: NaN)
          const int j = f / A.group, hq = cur.h * A.group + f - j * A.group;
          __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(A.out) + cur.b * A.obs +
                               j * A.oqs + hq * A.ohs;
          const int slot = 2 * cta + (cur.j0 == 0), pr = f - cur.p * TT_ROWS;
          float* acc = P.pacc + ((int64_t)slot * P.rs + pr) * TT_D;
          const uint32_t o0 = tm + lrow + 256u + (cur.dup ? 0u : 128u * x);
#pragma unroll 1
          for (int q = cur.dup ? 2 * x : 0; q < (cur.dup ? 2 * x + 2 : 4) && !dead; ++q) {
            uint32_t a[32], c[32];
            TC_LD32(a, o0 + 32u * q);
            if (cur.dup) TC_LD32(c, o0 + 128u + 32u * q);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            float o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              o[e] = __uint_as_float(a[e]);
              if (cur.dup)
                o[e] = (w0 == 0.f ? 0.f : w0 * o[e]) + (w1 == 0.f ? 0.f : w1 * __uint_as_float(c[e]));
            }
            if (live && whole) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = there ? o[e] * il : 0.f;
#pragma unroll
              for (int e = 0; e < 32; e += 8) tt_store8(out + 32 * q + e, o + e, P.out_vec != 0);
            } else if (live) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(acc + 32 * q + e) =
                    make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
            __syncwarp();
          }
          if (!whole && live && (!cur.dup || x == 0)) {
            float* pm = P.pml + ((int64_t)slot * P.rs + pr) * 2;
            pm[0] = m;
            pm[1] = l;
          }
          tc_fence_before();
        }
        if (cur.dup) {
          // both have read O and (m, l): the next P . V may come
          tc_arrive(&S.ofree);
          ok = __all_sync(0xffffffffu, tc_wait(&S.ofree, dn & 1u, &S.abort_));
          ++dn;
          if (!ok) break;
        }
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
// work on, the item's pieces are merged, in order; a warp takes a query row, a lane
// four columns.
__global__ void __launch_bounds__(TJ_THREADS) tree_join_kernel(const __grid_constant__ TreeTcParams P) {
  const TreeParams& T = P.T;
  const AttnParams& A = T.A;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int c = (int)blockIdx.x, r0 = (int)blockIdx.y * TJ_ROWS;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int stop = t < TT_CTAS ? P.status[t] : 0;
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
  const int per = A.Hkv * P.np, total = P.rowpre[A.B] * per, share = tt_share(total);
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
  const int rows = min(TT_ROWS, A.R - p * TT_ROWS), np = c1 - c0 + 1;
  for (int r = r0 + w; r < min(r0 + TJ_ROWS, rows); r += TJ_THREADS / 32) {
    const int f = p * TT_ROWS + r, j = f / A.group, hq = h * A.group + f - j * A.group;
    // piece i: the item's start in its first CTA, then a CTA's start each
    auto row_of = [&](int i) { return (int64_t)(2 * (c + i) + (i == 0)) * P.rs + r; };
    float gm = -CUDART_INF_F;
    for (int i = lane; i < np; i += 32) gm = fmaxf(gm, __ldcg(&P.pml[row_of(i) * 2]));
    gm = warp_max(gm);
    float L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < np; i0 += 4) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ml[k] = make_float2(-CUDART_INF_F, 0.f);
        v[k] = a;
        if (i0 + k < np) {
          ml[k] = __ldcg(reinterpret_cast<const float2*>(P.pml + row_of(i0 + k) * 2));
          v[k] = __ldcg(reinterpret_cast<const float4*>(P.pacc + row_of(i0 + k) * TT_D) + lane);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float fw = ml[k].x == -CUDART_INF_F ? 0.f : ex2f(ml[k].x - gm);
        L += ml[k].y != ml[k].y ? ml[k].y : fw * ml[k].y;
        if (fw == 0.f) continue;
        a.x = fmaf(fw, v[k].x, a.x); a.y = fmaf(fw, v[k].y, a.y);
        a.z = fmaf(fw, v[k].z, a.z); a.w = fmaf(fw, v[k].w, a.w);
      }
    }
    const int32_t* mask = T.masks + (int64_t)b * T.mask_bs + (int64_t)(T.first + j) * T.W;
    const float il = !tree_present(mask, T.W, T.N) || L == 0.f ? 0.f : 1.f / L;
    if (il == 0.f) a = make_float4(0.f, 0.f, 0.f, 0.f);
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(A.out) + b * A.obs + j * A.oqs +
                         hq * A.ohs + 4 * lane;
    const uint2 pk = make_uint2(pack_bf16(a.x * il, a.y * il), pack_bf16(a.z * il, a.w * il));
    if (P.out_vec) {
      *reinterpret_cast<uint2*>(dst) = pk;
    } else {
      const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&pk);
#pragma unroll
      for (int k = 0; k < 4; ++k) dst[k] = e[k];
    }
  }
}

// The shapes of the tensor-core path.
static bool tt_fast(int dtype, int D, int group) {
  return dtype == SD_DTYPE_BF16 && D == TT_D && group <= 128;
}

struct TtLayout {
  size_t status, acc, ml, bytes;
  int np, rs;
};
static TtLayout tt_layout(int B, int R) {
  TtLayout L;
  L.np = (R + TT_ROWS - 1) / TT_ROWS;
  L.rs = std::min(TT_ROWS, (R + 31) / 32 * 32);
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t o = up(((size_t)B + 1) * sizeof(int));
  L.status = o; o = up(o + TT_CTAS * sizeof(int));
  L.acc = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * TT_D * sizeof(float));
  L.ml = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * 2 * sizeof(float));
  L.bytes = o;
  return L;
}

static int tree_tc(TreeTcParams& P, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  AttnParams& A = P.T.A;
  // 16-byte loads of q rows and TMA boxes of the caches
  if ((reinterpret_cast<uintptr_t>(A.q) & 15) || A.qbs % 8 || A.qhs % 8 || A.qqs % 8 ||
      (reinterpret_cast<uintptr_t>(A.k) & 15) || (reinterpret_cast<uintptr_t>(A.v) & 15))
    return SD_EINVAL;
  const int64_t rows = A.bt ? (int64_t)A.npages * A.Hkv * SD_KV_PAGE : (int64_t)A.B * A.Hkv * A.C;
  if (rows >= (int64_t)1 << 31) return SD_ENOTSUP;   // a TMA coordinate
  const TtLayout L = tt_layout(A.B, A.R);
  // the schedule counts units in 32 bits
  const int64_t tiles = ((int64_t)A.C + SD_KV_PAGE - 1) / SD_KV_PAGE + TT_OVH;
  if (tiles * A.B > 0x7FFFFFFF / ((int64_t)A.Hkv * L.np)) return SD_ENOTSUP;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < L.bytes)
    return SD_ENOSPC;
  char* ws = reinterpret_cast<char*>(workspace);
  P.np = L.np; P.rs = L.rs;
  P.rowpre = reinterpret_cast<int*>(ws);
  P.status = reinterpret_cast<int*>(ws + L.status);
  P.pacc = reinterpret_cast<float*>(ws + L.acc);
  P.pml = reinterpret_cast<float*>(ws + L.ml);
  P.out_vec = (reinterpret_cast<uintptr_t>(A.out) & 15) == 0 && A.obs % 8 == 0 && A.oqs % 8 == 0 &&
              A.ohs % 8 == 0;
  CUtensorMap mk, mv;
  if (!cache_map(&mk, A.k, rows) || !cache_map(&mv, A.v, rows)) return SD_ENOTSUP;
  const int sm = (int)sizeof(TtSmem) + 1024;         // room to align
  static std::atomic<uint64_t> ready{0};             // devices whose kernel may use that much
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SD_ELAUNCH;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load() & bit) || !bit) {
    if (cudaFuncSetAttribute(tree_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) !=
        cudaSuccess)
      return SD_ELAUNCH;
    ready.fetch_or(bit);
  }
  tree_tc_kernel<<<TT_CTAS, TT_THREADS, sm, st>>>(P, mk, mv);
  if (cudaGetLastError() != cudaSuccess) return SD_ELAUNCH;
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
  return tt_layout(B, qlen * (Hq / Hkv)).bytes;
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
