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
constexpr int TT_THREADS = 384;              // warps 0-3, 4-7: softmax; 8: TMA; 9: MMA; two idle
// Registers after the start, when the softmax warps take what the others give: 8 x 200 + 4 x 104
// a warp's lane, as many as 12 x 168.
constexpr int TT_REGS_SOFTMAX = 200, TT_REGS_OTHER = 104;
static_assert(8 * TT_REGS_SOFTMAX + 4 * TT_REGS_OTHER <= 12 * 168, "of what the launch has");
constexpr int TT_CTAS = 148;                 // one CTA per SM
constexpr int TT_OVH = 2;                    // schedule cost of an item beyond its pages, in pages
constexpr int TT_MIN_SHARE = TT_OVH + 1;     // fewest schedule units per CTA: a one-page item
constexpr int TT_BASES = 512;                // rows whose bases a CTA keeps
constexpr int TT_WORDS = SD_TREE_MAX / 32;
constexpr int TJ_THREADS = 256;
constexpr int TJ_ROWS = 32;                  // query rows of a join CTA

struct TreeTcParams {
  TreeParams T;
  int np, ri, tr;                            // items of a (row, kv head), their query rows, a tile's
  int rs;                                    // rows of a piece: ri, rounded up to 32
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

// PAIR: two tiles of query rows; else one, whose keys the softmax warps share.
template <bool PAIR>
struct TtSmem {
  static constexpr int SLOTS = PAIR ? 4 : 5;         // 32 KB K / V tiles in flight
  static constexpr int TILES = PAIR ? 2 : 1;
  alignas(1024) unsigned char q[TILES][2][128 * 128];        // [tile][64-col box][128 rows x 128 B]
  alignas(1024) unsigned char kv[SLOTS][2][128 * 128];       // [slot][64-col box][128 keys x 128 B]
  alignas(16) unsigned char out[8][32 * 64];         // a warp's 32 rows x 32 outputs
  alignas(8) unsigned long long full[SLOTS], empty[SLOTS];
  // PAIR: by tile; else S by page parity, P by warpgroup and page parity
  alignas(8) unsigned long long sfull[2], pfull[2][2], oready[2], qfull[2], fin, mlfull, ofree;
  uint32_t mask[256][TT_WORDS];              // each softmax thread's row: its node's bits
  float ml[2][128][2];                       // !PAIR: the warpgroups' (m, l)
  int base[TT_BASES];
  int red[33];
  int first[2];                              // the CTA's first row and the units before it
  int abort_;
  uint32_t tmem;
};
static_assert(sizeof(TtSmem<true>) + 1024 <= 227 * 1024, "shared memory, with room to align");
static_assert(sizeof(TtSmem<false>) + 1024 <= 227 * 1024, "shared memory, with room to align");

// A CTA's run of schedule units as segments of items, walked identically by
// every role: row-major, kv head and then the item inner; TT_OVH virtual units in
// front of each item's pages.
struct TtSeg {
  int b, h, p, base, tb, off, tt, t1, ncost, j0, j1;         // pages [j0, j1) of the segment
};
template <bool PAIR>
__device__ __forceinline__ int tt_base(const TtSmem<PAIR>& S, const TreeParams& T, int b) {
  return b < TT_BASES ? S.base[b] : tree_base(T, b);
}
__device__ __forceinline__ void tt_bounds(TtSeg& s) {
  s.ncost = min(s.tb - s.off, s.t1 - s.tt);
  s.j0 = max(s.off, TT_OVH) - TT_OVH;
  s.j1 = max(s.off + s.ncost - TT_OVH, s.j0);
}
template <bool PAIR>
__device__ __forceinline__ bool tt_next(TtSeg& s, const TtSmem<PAIR>& S, const TreeTcParams& P) {
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
template <bool PAIR>
__device__ __forceinline__ bool tt_real(TtSeg& s, const TtSmem<PAIR>& S, const TreeTcParams& P) {
  while (s.j1 == s.j0)
    if (!tt_next(s, S, P)) return false;
  return true;
}

// The schedule: every CTA sums the rows' units and finds its own first row.  The
// units per CTA and, in S.first, where the run of this one starts.
template <bool PAIR>
__device__ __forceinline__ void tt_plan(TtSmem<PAIR>& S, const TreeTcParams& P, int* total, int* share) {
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

// What a softmax thread knows of its segment.
struct TtRow {
  int f;                                             // its query row of the (row, kv head)
  bool live, dead, there;                            // there is one; none in the warp; its node is present
};

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
        sees = ((1u << d) - 1u) | (m[0] << d);
      } else {
        const int a = -d, w = a >> 5;
        sees = __funnelshift_r(w < T.W ? m[w] : 0u, w + 1 < T.W ? m[w + 1] : 0u, a & 31);
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

template <bool PAIR>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_tc_kernel(const __grid_constant__ TreeTcParams P, const __grid_constant__ CUtensorMap tmk,
               const __grid_constant__ CUtensorMap tmv) {
  extern __shared__ __align__(1024) unsigned char tt_raw[];
  const uint32_t pad = (1024u - (smem_addr(tt_raw) & 1023u)) & 1023u;   // swizzle atoms: 1024 B
  TtSmem<PAIR>& S = *reinterpret_cast<TtSmem<PAIR>*>(tt_raw + pad);
  constexpr int SLOTS = TtSmem<PAIR>::SLOTS;
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
      tc_bar_init(&S.qfull[x], PAIR ? 128 : 256);
      tc_bar_init(&S.sfull[x], 1);
      tc_bar_init(&S.pfull[x][0], 128);
      tc_bar_init(&S.pfull[x][1], 128);
      tc_bar_init(&S.oready[x], 1);
    }
    tc_bar_init(&S.fin, 1);
    tc_bar_init(&S.mlfull, 256);
    tc_bar_init(&S.ofree, 256);
    S.abort_ = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
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

    if (w >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(TT_REGS_OTHER));
      if (w == 8 && lane == 0) {
        // ---------------- TMA producer: K then V of each page, SLOTS tiles ahead
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
      } else if (w == 9) {
        // ---------------- MMA issuer (the whole warp)
        constexpr uint32_t ID1 = tc_idesc(128, 128, 0, 0);     // S = Q . K^T
        constexpr uint32_t ID2 = tc_idesc(128, 128, 0, 1);     // O += P . V (V [key][d]: N-major)
        const uint32_t kv0 = smem_addr(S.kv[0][0]), q0 = smem_addr(S.q[0][0]);
        auto k_desc = [&](uint32_t g) { return tc_desc(kv0 + (2u * g % SLOTS) * 32768u, 16, 1024, 2); };
        auto v_desc = [&](uint32_t g) {
          return tc_desc(kv0 + ((2u * g + 1u) % SLOTS) * 32768u, 16384, 1024, 2);
        };
        auto full = [&](uint32_t idx, unsigned long long* other, uint32_t par) {
          return tc_wait2_warp(&S.full[idx % SLOTS], (idx / SLOTS) & 1u, other, par, &S.abort_);
        };
        // S of 128 query rows (tile x) and the 128 keys of page g
        auto issue_s = [&](uint32_t x, uint32_t d, uint32_t g) {
          const uint64_t dq = tc_desc(q0 + x * 32768u, 16, 1024, 2), dk = k_desc(g);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {             // 16 of 128 d: 32 B, the second box 16 KB on
            const uint64_t o = (uint64_t)((ks & 3) * 2 + (ks >> 2) * 1024);
            tc_mma_warp(d, dq + o, dk + o, ID1, ks > 0 ? 1 : 0);
          }
        };
        // O += P . V of 64 keys (half of page g)
        auto issue_pv = [&](uint32_t o, uint32_t pa, uint32_t g, int half, bool acc) {
          const uint64_t dv = v_desc(g) + (uint64_t)(half * 512);      // 16 keys: 2 KB
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            tc_mma_ts_warp(o, pa + 8u * ks, dv + (uint64_t)(ks * 128), ID2, ks || acc ? 1 : 0);
        };
        uint32_t g = 0, qn = 0;                        // pages whose S is issued, segments
        bool ok = true;
        if constexpr (PAIR) {
          // S0(0) S1(0) | PV0(i) S0(i + 1) PV1(i) S1(i + 1) | ...: a tile's P lies over its S,
          // so S of its next page comes behind P . V; the tiles take turns, so that one's
          // softmax runs under the other's products.  P . V starts with the first half of P.
          for (uint32_t x = 0; x < 2u && ok; ++x) {
            ok = full(0, &S.qfull[x], 0u);
            if (!ok) break;
            tc_fence_after();
            issue_s(x, tm + 128u * x, 0);
            tc_commit_warp(&S.sfull[x]);
          }
          if (ok) tc_commit_warp(&S.empty[0]);
          ++g;
          bool acc = false;
          int left = seg.j1 - seg.j0;                  // pages of the segment of page g - 1
          while (ok) {
            const uint32_t c = g - 1u;                 // the page whose P . V comes
            bool last = false, turn = false;
            if (--left == 0) {
              turn = true;
              more = tt_next(seg, S, P) && tt_real(seg, S, P);
              last = !more;
              if (more) {
                left = seg.j1 - seg.j0;
                ++qn;
              }
            }
#pragma unroll 1
            for (uint32_t x = 0; x < 2u && ok; ++x) {
              const uint32_t s = tm + 128u * x, o = s + 256u;
              ok = full(2u * c + 1u, &S.pfull[x][0], c & 1u);
              if (!ok) break;
              tc_fence_after();
              issue_pv(o, s, c, 0, acc);
              // the rest of P, K of the next page and, at a segment's start, its Q
              ok = last ? tc_wait2_warp(&S.pfull[x][1], c & 1u, &S.pfull[x][1], c & 1u, &S.abort_)
                        : full(2u * g, &S.pfull[x][1], c & 1u) &&
                              (!turn || tc_wait2_warp(&S.qfull[x], qn & 1u, &S.qfull[x], qn & 1u,
                                                      &S.abort_));
              if (!ok) break;
              tc_fence_after();
              issue_pv(o, s + 32u, c, 1, true);
              tc_commit_warp(&S.oready[x]);
              if (x == 1u) tc_commit_warp(&S.empty[(2u * c + 1u) % SLOTS]);
              if (last) continue;
              issue_s(x, s, g);
              tc_commit_warp(&S.sfull[x]);
              if (x == 1u) tc_commit_warp(&S.empty[2u * g % SLOTS]);
            }
            if (last) break;
            acc = !turn;
            ++g;
          }
        } else {
          // S(0) | S(1) PV(0) | S(2) PV(1) | ...: S twice, by page parity; a warpgroup's half of
          // the keys has an O of its own
          TtSeg back = seg;
          // pages left of the segments of S and of P . V
          int ahead = seg.j1 - seg.j0, behind = ahead;
          bool acc = false;
          uint32_t c = 0;                              // pages whose P . V is issued
          while (ok) {
            if (more) {
              ok = full(2u * g, &S.qfull[0], qn & 1u);
              if (!ok) break;
              tc_fence_after();
              issue_s(0, tm + 128u * (g & 1u), g);
              tc_commit_warp(&S.sfull[g & 1u]);
              tc_commit_warp(&S.empty[2u * g % SLOTS]);
              ++g;
              if (--ahead == 0) {
                more = tt_next(seg, S, P) && tt_real(seg, S, P);
                ahead = more ? seg.j1 - seg.j0 : 0;
                ++qn;
              }
              if (g < 2u && more) continue;            // two S before the first P . V
            }
            if (c == g) break;
#pragma unroll 1
            for (uint32_t x = 0; x < 2u && ok; ++x) {
              ok = full(2u * c + 1u, &S.pfull[x][c & 1u], (c >> 1) & 1u);
              if (!ok) break;
              tc_fence_after();
              issue_pv(tm + 256u + 128u * x, tm + 128u * (c & 1u) + 64u * x, c, (int)x, acc);
              tc_commit_warp(&S.oready[x]);
            }
            if (!ok) break;
            tc_commit_warp(&S.empty[(2u * c + 1u) % SLOTS]);
            ++c;
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
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(TT_REGS_SOFTMAX));
      // ---------------- softmax warps.  PAIR: tile x, thread r owns its query row r; else
      // both warpgroups own the same rows, x takes the keys [64 x, 64 x + 64) of a page
      const int x = w >> 2, wq = w & 3, r = t & 127;
      const uint32_t lrow = (uint32_t)(32 * wq) << 16;
      const float sl2 = A.scale * 1.4426950408889634f;
      unsigned char* stage = S.out[w];
      // the tile's query rows, 16-byte chunks (rows past the item's: zeros)
      auto load_q = [&](const TtSeg& g) {
        const int r0 = g.p * P.ri + (PAIR ? P.tr * x : 0);
        const int rows = min(min(P.tr, P.ri - (PAIR ? P.tr * x : 0)), A.R - r0);
        const __nv_bfloat16* Q = reinterpret_cast<const __nv_bfloat16*>(A.q) + g.b * A.qbs;
        // PAIR: 16 lanes a row; else 8 lanes half a row (the warpgroup's box)
        constexpr int LANES = PAIR ? 16 : 8, RPI = 32 / LANES, STEPS = 32 / RPI;
        const int c = (PAIR ? 0 : 8 * x) + lane % LANES;
        unsigned char* dst = S.q[PAIR ? x : 0][c >> 3];
#pragma unroll 1
        for (int i0 = 0; i0 < STEPS; i0 += 8) {
          uint4 v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = 32 * wq + RPI * (i0 + i) + lane / LANES, f = r0 + row;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row < rows) {
              const int j = f / A.group, hq = g.h * A.group + f - j * A.group;
              v[i] = __ldg(reinterpret_cast<const uint4*>(Q + hq * A.qhs + j * A.qqs) + c);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = 32 * wq + RPI * (i0 + i) + lane / LANES;
            *reinterpret_cast<uint4*>(dst + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[i];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_arrive(&S.qfull[PAIR ? x : 0]);
      };
      uint32_t n = 0, dn = 0;                        // pages and segments done
      int uni_b = -1;
      uint32_t uni = 0;                              // lane w: word w of what any query of row uni_b sees
      bool ok = true;
      if (more) load_q(seg);
      while (more) {
        const TtSeg cur = seg;
        more = tt_next(seg, S, P) && tt_real(seg, S, P);
        const int pages = cur.j1 - cur.j0, end = tree_end(T, cur.base);
        const int pr = (PAIR ? P.tr * x : 0) + r, f = cur.p * P.ri + pr;     // row of the item, of all
        const bool live = r < P.tr && pr < P.ri && f < A.R;
        const bool dead = __all_sync(0xffffffffu, !live);    // a warp without rows
        const int32_t* mask0 = T.masks + (int64_t)cur.b * T.mask_bs + (int64_t)T.first * T.W;
        // the row's bits, and what any query sees
        uint32_t* mine = S.mask[t];
        uint32_t some = 0;
        for (int k = 0; k < T.W; ++k) {
          mine[k] = live ? tree_word(mask0 + (int64_t)(f / A.group) * T.W, T.W, T.N, k) : 0u;
          some |= mine[k];
        }
        const bool there = some != 0u;
        if (uni_b < 0 || (uni_b != cur.b && T.mask_bs != 0)) {
          uni = 0u;
          for (int q0 = 0; q0 < A.qlen; q0 += 32)
            for (int k = 0; k < T.W; ++k) {
              const int q = q0 + lane;
              const uint32_t word = q < A.qlen ? tree_word(mask0 + (int64_t)q * T.W, T.W, T.N, k) : 0u;
              const uint32_t all = __reduce_or_sync(0xffffffffu, word);
              if (lane == k) uni |= all;
            }
        }
        uni_b = cur.b;
        float m = -CUDART_INF_F, l = 0.f;
        bool wild = false;
#pragma unroll 1
        for (int i = 0; i < pages; ++i) {
          const uint32_t sb = PAIR ? (uint32_t)x : n & 1u;               // buffer of S
          ok = __all_sync(0xffffffffu, tc_wait(&S.sfull[sb], (PAIR ? n : n >> 1) & 1u, &S.abort_));
          if (!ok) break;
          tc_fence_after();
          // the segment's S are all done with Q: the next segment's may come
          if (i == pages - 1 && more) load_q(seg);
          const uint32_t scol = tm + lrow + 128u * sb + (PAIR ? 0u : 64u * x);
          const int key0 = (cur.j0 + i) * SD_KV_PAGE;
          if (key0 + SD_KV_PAGE > cur.base) {
            // the tree's pages, and what lies behind it
            if (!dead) tt_hide(mine, T, cur.base, end, key0 + (PAIR ? 0 : 64 * x), PAIR ? 128 : 64, scol);
            // PAIR: tile 0 blanks V for both (the issuer asks for its P first); else each
            // warpgroup its half, two warps 32 keys
            if (!PAIR || x == 0) {
              const uint32_t vi = 2u * n + 1u;
              const int grp = PAIR ? wq : 2 * x + (wq & 1);
              ok = tt_blank(S.kv[vi % SLOTS], T, uni, cur.base, end, key0 + 32 * grp, 32 * grp,
                            PAIR ? 0 : wq >> 1, PAIR ? 2 : (wq >> 1) + 1, &S.full[vi % SLOTS],
                            (vi / SLOTS) & 1u, &S.abort_);
              if (!ok) break;
            }
          }
          unsigned long long* half0 = PAIR ? &S.pfull[x][0] : &S.pfull[x][n & 1u];
          if (!dead) {
            constexpr int NC = PAIR ? 4 : 2;         // 32-column chunks of a thread
            uint32_t s[NC][32];
#pragma unroll
            for (int c = 0; c < NC; ++c) TC_LD32(s[c], scol + 32u * c);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 2) px_max3(mx[(e >> 1) & 3], s[c][e], s[c][e + 1]);
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
                for (int q = 0; q < 8; ++q) {
                  uint32_t o[16];
                  TC_LD16(o, tm + lrow + 256u + 128u * x + 16u * q);
                  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                  TC_ST16(tm + lrow + 256u + 128u * x + 16u * q, o);
                }
              }
            }
            if (wild)
#pragma unroll
              for (int c = 0; c < NC; ++c) px_scale(s[c], sl2);
            const float mc = m == -CUDART_INF_F ? 0.f : m, sf = wild ? 1.f : sl2;
            const unsigned long long sl22 = pair2(sf, sf), nm2 = pair2(-mc, -mc);
            unsigned long long ls[2] = {0ULL, 0ULL};   // (0.f, 0.f)
#pragma unroll
            for (int c = 0; c < NC; c += 2) {
              uint32_t pk[32];
              px_weights(s[c], pk, ls, sl22, nm2);
              px_weights(s[c + 1], pk + 16, ls, sl22, nm2);
              TC_ST32(scol + 16u * c, pk);             // over columns that have been read
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              if (PAIR && c == 0) {
                tc_fence_before();
                tc_arrive(half0);
              }
            }
            float la, lb;
            unpair(add2(ls[0], ls[1]), la, lb);
            l += la + lb;
          } else if (PAIR) {
            tc_arrive(half0);
          }
          tc_fence_before();
          tc_arrive(PAIR ? &S.pfull[x][1] : half0);
          ++n;
        }
        if (!ok) break;
        // ---- the segment's end: O divided by the row's sum and written out, or as a piece
        ok = __all_sync(0xffffffffu, tc_wait(&S.oready[x], (n - 1) & 1u, &S.abort_));
        if (!PAIR) {
          // each warpgroup writes half of the columns, of both O
          S.ml[x][r][0] = m;
          S.ml[x][r][1] = l;
          tc_arrive(&S.mlfull);
          ok = ok && __all_sync(0xffffffffu, tc_wait(&S.mlfull, dn & 1u, &S.abort_) &&
                                                 tc_wait(&S.oready[x ^ 1], (n - 1) & 1u, &S.abort_));
        }
        if (!ok) break;
        tc_fence_after();
        float w0 = 1.f, w1 = 0.f;
        if (!PAIR) {
          const float m0 = S.ml[0][r][0], m1 = S.ml[1][r][0], l0 = S.ml[0][r][1], l1 = S.ml[1][r][1];
          m = fmaxf(m0, m1);
          w0 = m0 == -CUDART_INF_F ? 0.f : ex2f(m0 - m);
          w1 = m1 == -CUDART_INF_F ? 0.f : ex2f(m1 - m);
          l = (l0 != l0 ? l0 : w0 * l0) + (l1 != l1 ? l1 : w1 * l1);
        }
        if (!dead) {
          const bool whole = cur.j0 == 0 && cur.j1 + TT_OVH == cur.tb;
          if (whole) {
            const float il = l == 0.f || !there ? 0.f : 1.f / l;   // (a NaN sum: NaN)
            w0 *= il;
            w1 *= il;
          }
          const int j = f / A.group, hq = cur.h * A.group + f - j * A.group;
          __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(A.out) + cur.b * A.obs +
                               j * A.oqs + hq * A.ohs;
          const int slot = 2 * cta + (cur.j0 == 0);
          float4* acc = P.pacc + (int64_t)slot * (TT_D / 4) * P.rs + pr;
          const uint32_t o0 = tm + lrow + 256u + (PAIR ? 128u * x : 0u);
#pragma unroll 1
          for (int q = PAIR ? 0 : 2 * x; q < (PAIR ? 4 : 2 * x + 2); ++q) {
            uint32_t a[32], c[32];
            TC_LD32(a, o0 + 32u * q);
            if constexpr (!PAIR) TC_LD32(c, o0 + 128u + 32u * q);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            float o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              o[e] = w0 == 0.f ? 0.f : w0 * __uint_as_float(a[e]);
              if constexpr (!PAIR) o[e] += w1 == 0.f ? 0.f : w1 * __uint_as_float(c[e]);
            }
            if (whole) {
              tt_write(stage, o, out + 32 * q, live, P.out_vec != 0);
            } else if (live) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                acc[(int64_t)(8 * q + e) * P.rs] =
                    make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            __syncwarp();
          }
          if (!whole && live && (PAIR || x == 0)) P.pml[(int64_t)slot * P.rs + pr] = make_float2(m, l);
        }
        tc_fence_before();
        if (!PAIR) {
          // both have read O and (m, l): the next P . V may come
          tc_arrive(&S.ofree);
          ok = __all_sync(0xffffffffu, tc_wait(&S.ofree, dn & 1u, &S.abort_));
          if (!ok) break;
        }
        ++dn;
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
  const int rows = min(P.ri, A.R - p * P.ri), np = c1 - c0 + 1;
  const int r = (int)blockIdx.y * TJ_ROWS + lane, f = p * P.ri + r;
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
  const int j = f / A.group, hq = h * A.group + f - j * A.group;
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
  int np, ri, tr, rs;
};
static TtLayout tt_layout(int B, int R) {
  TtLayout L;
  // items of up to two tiles of query rows, of about the same size, and so their tiles
  L.np = (R + 2 * TT_TILE - 1) / (2 * TT_TILE);
  L.ri = (R + L.np - 1) / L.np;
  L.tr = R <= TT_TILE ? R : std::min(TT_TILE, ((L.ri + 1) / 2 + 31) / 32 * 32);
  L.rs = (L.ri + 31) / 32 * 32;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t o = up(((size_t)B + 1) * sizeof(int));
  L.status = o; o = up(o + TT_CTAS * sizeof(int));
  L.acc = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * TT_D * sizeof(float));
  L.ml = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * 2 * sizeof(float));
  L.bytes = o;
  return L;
}

template <bool PAIR>
static int launch_tc(const TreeTcParams& P, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  const int sm = (int)sizeof(TtSmem<PAIR>) + 1024;   // room to align
  static std::atomic<uint64_t> ready{0};             // devices whose kernel may use that much
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SD_ELAUNCH;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load() & bit) || !bit) {
    if (cudaFuncSetAttribute(tree_tc_kernel<PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) !=
        cudaSuccess)
      return SD_ELAUNCH;
    ready.fetch_or(bit);
  }
  tree_tc_kernel<PAIR><<<TT_CTAS, TT_THREADS, sm, st>>>(P, mk, mv);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
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
  P.np = L.np; P.ri = L.ri; P.tr = L.tr; P.rs = L.rs;
  P.rowpre = reinterpret_cast<int*>(ws);
  P.status = reinterpret_cast<int*>(ws + L.status);
  P.pacc = reinterpret_cast<float4*>(ws + L.acc);
  P.pml = reinterpret_cast<float2*>(ws + L.ml);
  P.out_vec = (reinterpret_cast<uintptr_t>(A.out) & 15) == 0 && A.obs % 8 == 0 && A.oqs % 8 == 0 &&
              A.ohs % 8 == 0;
  CUtensorMap mk, mv;
  if (!cache_map(&mk, A.k, rows) || !cache_map(&mv, A.v, rows)) return SD_ENOTSUP;
  if (int rc = A.R > TT_TILE ? launch_tc<true>(P, mk, mv, st) : launch_tc<false>(P, mk, mv, st)) return rc;
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
