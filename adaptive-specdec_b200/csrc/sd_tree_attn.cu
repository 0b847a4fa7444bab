// Attention of a tree's nodes over the cache (sm_100a): host entry, and the tensor-core
// kernels for bf16 heads of 64 and 128.
//
// The query rows of a (row, kv head) are its nodes times the heads of the group:
// 64 nodes under 32 / 8 heads are 256 rows that read the same keys.  An item is one
// (row, kv head) and up to 256 of them, on two tiles of 128; it goes over the row's
// keys in tiles of 128 ("pages", whether the cache is paged or not):
//   S = Q K^T,  p = 2^(s - m) under a lazy running maximum m,  O += P V
// Every page but the last few is seen whole by every node; in those that hold
// the tree a row keeps the scores whose bit its node's mask has.  The weights are
// rounded to bf16 for P V (both operands of an MMA have one type, V's), each off by up to
// 2^-8 of itself like the output: over 40 keys the error against 64 bits is 1.75e-3
// (rms, relative) where 32-bit weights leave 1.65e-3, over 500 keys and more 1 % above
// theirs or less.  Scores, maxima, sums, O and the pieces are 32 bits.
// tree_tc_kernel    persistent, stream-K: the pages of all items lie end to end
//                   and a CTA takes one contiguous run; an item that lies within a
//                   run is written out, a cut one leaves (m, l, O) per piece
// tree_join_kernel  merges the pieces of cut items, in order (programmatic dependent)
//
// What bounds it.  K and V are read once for all nodes and heads, so up to 128 query
// rows it is HBM: 32 rows of 26 nodes over 128 to 4096 keys (294 MB) take 64 us in a graph,
// 5.0 TB/s in the main kernel, and a start (plan, first loads) and join of 3 and 6 us;
// 2 rows of 33 nodes over 30011 keys (246 MB) 53 to 58 us.  With two tiles it is the chain of S,
// softmax and P V of a tile: 64 rows of 64 nodes over 512 to 8192 keys take 337 us, the
// tensor pipe is busy 47 % of the time.  (The CUDA-core kernel: 20.2 ms.)  These are bursts at
// 1965 MHz.  Back to back for 0.4 s the power cap lowers the clock: 64 rows of 64 nodes then take
// 404 us near 1500 MHz, 32 rows of 26 nodes 71 us at 1635 MHz.
// One tile: S of the next page stands ready in TMEM's second buffer, and its 128 columns go
// to two warpgroups, so that a page's softmax takes half as long.  Two tiles: S and O of both
// fill TMEM, so S comes in halves of 64 keys (tt_issue_pair); whole pages of S took 422 us.
// Heads of 64 halve the tiles and so put twice as many on their way: 32 rows of 26 nodes over
// 2048 keys take 52 us (CUDA cores: 1.17 ms).
// Queries come by TMA (the softmax threads' own loads waited 8000 cycles behind K and V),
// the nodes' bits late and by asynchronous copies, as only the tree's pages look at them.
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

constexpr int TT_TILE = 128;                 // query rows of a tile
constexpr int TT_THREADS = 352;              // warps 0-7: softmax; 8: TMA of K, V; 9: MMA; 10: TMA of Q
constexpr int TT_CTAS = 148;                 // one CTA per SM
constexpr int TT_OVH = 3;                    // schedule cost of an item beyond its pages, in pages
constexpr int TT_MIN_SHARE = TT_OVH + 1;     // fewest schedule units per CTA: a one-page item
constexpr int TT_BASES = 512;                // rows whose bases a CTA keeps
constexpr int TT_WORDS = SD_TREE_MAX / 32;
constexpr int TJ_THREADS = 256;
constexpr int TJ_ROWS = 32;                  // query rows and columns of a join CTA
constexpr int TJ_COLS = 32;
static_assert(TJ_THREADS == TJ_COLS / 4 * 32 && TJ_THREADS == TJ_ROWS * (TJ_COLS / 4));

struct TreeTcParams {
  TreeParams T;
  int np, ni, nt;                            // items of a (row, kv head); nodes of an item, of a tile
  int rs;                                    // rows of a piece: ni * group, rounded up to 32
  int out_vec;                               // 16-byte stores of the output are aligned
  // workspace
  int4* cut;                                 // [TT_CTAS] the item that is cut at a CTA's end, if it is the
                                             // first to work on it: row, kv head, item, pieces (0: none)
  int* status;                               // [TT_CTAS] a bounded wait gave up
  float4* pacc;                              // [2 TT_CTAS][32 column groups][rs] pieces
  float2* pml;                               // [2 TT_CTAS][rs]
};

__device__ __forceinline__ int tt_units(int end) { return (end + SD_KV_PAGE - 1) / SD_KV_PAGE + TT_OVH; }
__device__ __forceinline__ int tt_share(int total) {
  return max(TT_MIN_SHARE, (total + TT_CTAS - 1) / TT_CTAS);
}

// NT: tiles of query rows of an item; D: head size, 64 or 128
template <int NT, int D>
struct TtSmem {
  static constexpr int BOXES = D / 64;               // of 64 columns
  static constexpr uint32_t TILE = BOXES * 16384u;   // bytes of a tile of 128 rows
  static constexpr int SLOTS = (NT == 2 ? 4 : 5) * 2 / BOXES;          // K / V tiles in flight
  alignas(1024) unsigned char q[NT][BOXES][128 * 128];       // [tile][64-col box][128 rows x 128 B]
  alignas(1024) unsigned char kv[SLOTS][BOXES][128 * 128];   // [slot][64-col box][128 keys x 128 B]
  alignas(16) unsigned char out[8][32 * 64];         // a warp's 32 rows x 32 outputs
  // one tile: sfull, pfull and oready by page parity; two: by tile, of the two halves of S (slo,
  // shi), of S's second half in registers (sread)
  alignas(8) unsigned long long full[SLOTS], empty[SLOTS], sfull[2], pfull[2], oready[2], qfull[NT],
      qempty[NT], slo[2], shi[2], sread[2], fin;
  uint32_t mask[NT][128][TT_WORDS];          // the query rows: their nodes' bits
  // what the threads of a row tell one another: [exchange parity][warpgroup][row], (value, number)
  unsigned long long peer[2][2][128];
  int base[TT_BASES];
  int red[33];
  int first[2];                              // the CTA's first row and the units before it
  int abort_;
  uint32_t tmem;
};
static_assert(sizeof(TtSmem<2, 128>) + 1024 <= 227 * 1024, "shared memory, with room to align");
static_assert(sizeof(TtSmem<1, 128>) + 1024 <= 227 * 1024, "shared memory, with room to align");
static_assert(sizeof(TtSmem<2, 64>) + 1024 <= 227 * 1024, "shared memory, with room to align");
static_assert(sizeof(TtSmem<1, 64>) + 1024 <= 227 * 1024, "shared memory, with room to align");

// A CTA's run of schedule units as segments of items, walked identically by
// every role: row-major, kv head and then the item inner; TT_OVH virtual units in
// front of each item's pages.
struct TtSeg {
  int b, h, p, base, tb, off, tt, t1, ncost, j0, j1;         // pages [j0, j1) of the segment
};
template <int NT, int D>
__device__ __forceinline__ int tt_base(const TtSmem<NT, D>& S, const TreeParams& T, int b) {
  return b < TT_BASES ? S.base[b] : tree_base(T, b);
}
__device__ __forceinline__ void tt_bounds(TtSeg& s) {
  s.ncost = min(s.tb - s.off, s.t1 - s.tt);
  s.j0 = max(s.off, TT_OVH) - TT_OVH;
  s.j1 = max(s.off + s.ncost - TT_OVH, s.j0);
}
template <int NT, int D>
__device__ __forceinline__ bool tt_next(TtSeg& s, const TtSmem<NT, D>& S, const TreeTcParams& P) {
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
template <int NT, int D>
__device__ __forceinline__ bool tt_real(TtSeg& s, const TtSmem<NT, D>& S, const TreeTcParams& P) {
  while (s.j1 == s.j0)
    if (!tt_next(s, S, P)) return false;
  return true;
}

// The schedule: every CTA sums the rows' units and finds its own first row.  The
// units per CTA and, in S.first, where the run of this one starts.
template <int NT, int D>
__device__ __forceinline__ void tt_plan(TtSmem<NT, D>& S, const TreeTcParams& P, int* total, int* share) {
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
      if ((int64_t)ex * per <= t0 && t0 < (int64_t)(ex + mine) * per) {
        S.first[0] = b;
        S.first[1] = ex * per;
      }
    }
  }
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

// ---- the roles of a CTA's warps ---------------------------------------------------------------
// Q of a tile of a segment's item: its nodes x heads.
template <int NT, int D>
__device__ __forceinline__ void tt_ask_q(TtSmem<NT, D>& S, const TreeTcParams& P, const CUtensorMap& tmq,
                                         const TtSeg& g, int ti) {
  const int group = P.T.A.group, j = g.p * P.ni + P.nt * ti;
  tc_expect_tx(&S.qfull[ti], 2u * D * (uint32_t)(P.nt * group));
#pragma unroll
  for (int x = 0; x < D / 64; ++x) tt_tma_4d(S.q[ti][x], &tmq, 64 * x, g.h * group, j, g.b, &S.qfull[ti]);
}

// TMA producer (one thread): K then V of each page, SLOTS tiles ahead; the first segment's Q
// in front, before all SMs' K and V are on their way.
template <int NT, int D>
__device__ __forceinline__ void tt_load_kv(TtSmem<NT, D>& S, const TreeTcParams& P, const CUtensorMap& tmk,
                                           const CUtensorMap& tmv, const CUtensorMap& tmq, TtSeg seg,
                                           bool more, int share) {
  constexpr int SLOTS = TtSmem<NT, D>::SLOTS;
  int4 cut = make_int4(0, 0, 0, 0);
  for (int ti = 0; ti < NT && more; ++ti) tt_ask_q(S, P, tmq, seg, ti);
  uint32_t idx = 0;
  bool ok = true;
  while (more && ok) {
    for (int j = seg.j0; j < seg.j1 && ok; ++j) {
      const int y = (int)kv_row(P.T.A, seg.b, seg.h, j * SD_KV_PAGE);
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv, ++idx) {
        const int sl = (int)(idx % SLOTS);
        if (idx >= (uint32_t)SLOTS) ok = tc_wait(&S.empty[sl], ((idx / SLOTS) - 1) & 1u, &S.abort_);
        if (!ok) break;
        tc_expect_tx(&S.full[sl], TtSmem<NT, D>::TILE);
        const void* map = kv ? (const void*)&tmv : (const void*)&tmk;
#pragma unroll
        for (int x = 0; x < D / 64; ++x) tc_tma_2d(S.kv[sl][x], map, 64 * x, y, &S.full[sl]);
      }
    }
    if (seg.j0 == 0 && seg.j1 + TT_OVH < seg.tb)     // (the last segment)
      cut = make_int4(seg.b, seg.h, seg.p, (seg.tt - seg.off + seg.tb - 1) / share - (int)blockIdx.x + 1);
    if (ok) more = tt_next(seg, S, P) && tt_real(seg, S, P);
  }
  P.cut[blockIdx.x] = cut;
  if (!ok) {
    // let the copies already issued land before the CTA leaves
    for (uint32_t q = idx > (uint32_t)SLOTS ? idx - SLOTS : 0u; q < idx; ++q) {
      int dummy = 0;
      tc_wait(&S.full[q % SLOTS], (q / SLOTS) & 1u, &dummy);
    }
  }
}

// TMA producer (one thread) of the later segments' Q, once a tile's last S is done.
template <int NT, int D>
__device__ __forceinline__ void tt_load_q(TtSmem<NT, D>& S, const TreeTcParams& P, const CUtensorMap& tmq,
                                          TtSeg seg, bool more) {
  uint32_t sent = more ? NT : 0u;                    // tiles asked for, tile inner
  bool ok = true;
  while (ok && more && tt_next(seg, S, P) && tt_real(seg, S, P)) {
    for (int ti = 0; ti < NT; ++ti, ++sent) {
      ok = tc_wait(&S.qempty[ti], (sent / NT - 1) & 1u, &S.abort_);
      if (!ok) break;
      tt_ask_q(S, P, tmq, seg, ti);
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

constexpr uint32_t TT_ID_S = tc_idesc(128, 128, 0, 0);       // S = Q . K^T of 128 keys
constexpr uint32_t TT_ID_H = tc_idesc(128, 64, 0, 0);        // of 64 keys
template <int D> constexpr uint32_t TT_ID_O = tc_idesc(128, D, 0, 1);           // O += P . V (V [key][d]: N-major)

// S = Q . K^T by a warp: 16 of D columns an MMA: 32 B, the second box 16 KB on.
template <int D>
__device__ __forceinline__ void tt_mma_s(uint32_t d, uint32_t q, uint32_t k, uint32_t id) {
  const uint64_t dq = tc_desc(q, 16, 1024, 2), dk = tc_desc(k, 16, 1024, 2);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const uint64_t o = (uint64_t)((ks & 3) * 2 + (ks >> 2) * 1024);
    tc_mma_warp(d, dq + o, dk + o, id, ks > 0 ? 1 : 0);
  }
}
// O (+)= P . V by a warp: 16 keys an MMA: 2 KB of V, 8 columns of P, whose second 64 keys start
// at column `half`.
template <int D>
__device__ __forceinline__ void tt_mma_o(uint32_t o, uint32_t p, uint32_t half, uint32_t v, bool acc) {
  const uint64_t dv = tc_desc(v, 16384, 1024, 2);
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
    tc_mma_ts_warp(o, p + half * (ks >> 2) + 8u * (ks & 3), dv + (uint64_t)(ks * 128), TT_ID_O<D>,
                   ks || acc ? 1 : 0);
}
// An issuer that has found nothing to do since `idle` (0: it has just begun): whether it goes on.
__device__ __forceinline__ bool tt_idle(long long& idle, int* abort_) {
  const long long now = clock64();
  if (idle == 0) idle = now;
  if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(abort_) || now - idle > TC_WAIT)) {
    *reinterpret_cast<volatile int*>(abort_) = 1;
    return false;
  }
  return true;
}
// Every MMA that this warp issued has finished before the CTA leaves.
__device__ __forceinline__ void tt_finish(unsigned long long* bar) {
  tc_commit_warp(bar);
  int dummy = 0;
  tc_wait(bar, 0u, &dummy);
}

// MMA issuer of one tile: S(0) S(1) P.V(0) S(2) P.V(1) ...; S of page i in buffer i & 1 (128
// columns each), P over it; where S's tiles are late, P . V does not wait for it.
template <int D>
__device__ __forceinline__ void tt_issue_one(TtSmem<1, D>& S, const TreeTcParams& P, TtSeg seg, bool more) {
  constexpr int SLOTS = TtSmem<1, D>::SLOTS;
  const uint32_t kv0 = smem_addr(S.kv[0][0]), q0 = smem_addr(S.q[0][0]), tm = S.tmem;
  TtSeg back = seg;
  int ahead = seg.j1 - seg.j0, behind = ahead;       // pages left of the segments of S and of P . V
  uint32_t a = 0, c = 0, qn = 0;                     // pages issued; segments begun by S
  bool ok = true, acc = false;
  long long idle = 0;
  while (ok) {
    const uint32_t ki = 2u * a, vi = 2u * c + 1u;
    unsigned long long* vfull = &S.full[vi % SLOTS];
    bool s_go = false, p_go = false;
    if (more && a < c + 2u)
      s_go = __all_sync(0xffffffffu, tc_test(&S.full[ki % SLOTS], (ki / SLOTS) & 1u) &&
                                         tc_test(&S.qfull[0], qn & 1u));
    if (!s_go && c < a) {
      if (more && a < c + 2u)
        p_go = __all_sync(0xffffffffu, tc_test(vfull, (vi / SLOTS) & 1u) &&
                                           tc_test(&S.pfull[c & 1u], (c >> 1) & 1u));
      else
        p_go = ok = tc_wait2_warp(vfull, (vi / SLOTS) & 1u, &S.pfull[c & 1u], (c >> 1) & 1u, &S.abort_);
    }
    if (!s_go && !p_go) {
      if (!ok || (c == a && !more) || !tt_idle(idle, &S.abort_)) break;
      continue;
    }
    idle = 0;
    tc_fence_after();
    if (s_go) {
      tt_mma_s<D>(tm + 128u * (a & 1u), q0, kv0 + (ki % SLOTS) * TtSmem<1, D>::TILE, TT_ID_S);
      tc_commit_warp(&S.sfull[a & 1u]);
      tc_commit_warp(&S.empty[ki % SLOTS]);
      ++a;
      if (--ahead == 0) {                            // the segment's last S: Q may be replaced
        tc_commit_warp(&S.qempty[0]);
        more = tt_next(seg, S, P) && tt_real(seg, S, P);
        ahead = seg.j1 - seg.j0;
        ++qn;
      }
      continue;
    }
    tt_mma_o<D>(tm + 256u, tm + 128u * (c & 1u), 64u, kv0 + (vi % SLOTS) * TtSmem<1, D>::TILE, acc);
    tc_commit_warp(&S.oready[c & 1u]);
    tc_commit_warp(&S.empty[vi % SLOTS]);
    ++c;
    acc = true;
    if (--behind == 0) {
      if (!(tt_next(back, S, P) && tt_real(back, S, P))) break;
      behind = back.j1 - back.j0;
      acc = false;
    }
  }
  tt_finish(&S.fin);
}

// MMA issuer of two tiles.  S comes in halves of 64 keys: with H0, H1 the two 64-column halves
// of a tile's S, page i has its first half in H(i & 1) and its second in the other one; P of the
// whole page lies over the first, so the second is free as soon as it is in registers, and the
// next page's first half goes there before this page's P is made.  The tiles take turns in a fixed
// order, half a page apart: left to themselves they fall into step, and softmax and tensor cores
// wait for one another (8 rows of 64 nodes over 16384 keys: 171 us instead of 167).
template <int D>
__device__ __forceinline__ void tt_issue_pair(TtSmem<2, D>& S, const TreeTcParams& P, TtSeg seg, bool more) {
  constexpr int SLOTS = TtSmem<2, D>::SLOTS;
  const uint32_t kv0 = smem_addr(S.kv[0][0]), q0 = smem_addr(S.q[0][0]), tm = S.tmem;
  uint32_t g = 0, qn = 0;                            // page of the next P . V; segments done
  bool ok = true;
  // the first or second half of S of page i of tile x
  auto issue_s = [&](uint32_t x, uint32_t i, uint32_t half) {
    tt_mma_s<D>(tm + 128u * x + 64u * ((i + half) & 1u), q0 + x * TtSmem<1, D>::TILE,
             kv0 + (2u * i % SLOTS) * TtSmem<1, D>::TILE + half * 8192u, TT_ID_H);
    tc_commit_warp(half ? &S.shi[x] : &S.slo[x]);
    if (half && x == 1u) tc_commit_warp(&S.empty[2u * i % SLOTS]);
  };
  while (more && ok) {
    int pages = seg.j1 - seg.j0;
    // the segment's first S, of both tiles
#pragma unroll 1
    for (uint32_t x = 0; x < 2u && ok; ++x) {
      ok = tc_wait2_warp(&S.full[2u * g % SLOTS], (2u * g / SLOTS) & 1u, &S.qfull[x], qn & 1u, &S.abort_);
      if (!ok) break;
      tc_fence_after();
      issue_s(x, g, 0u);
      issue_s(x, g, 1u);
      if (pages == 1) tc_commit_warp(&S.qempty[x]);
    }
#pragma unroll 1
    for (; pages > 0 && ok; --pages, ++g) {
      const uint32_t ki = 2u * (g + 1u), vi = 2u * g + 1u;
#pragma unroll 1
      for (uint32_t x = 0; x < 2u; ++x) {
        if (pages > 1) {
          ok = tc_wait2_warp(&S.full[ki % SLOTS], (ki / SLOTS) & 1u, &S.sread[x], g & 1u, &S.abort_);
          if (!ok) break;
          tc_fence_after();
          issue_s(x, g + 1u, 0u);
        }
        ok = tc_wait2_warp(&S.full[vi % SLOTS], (vi / SLOTS) & 1u, &S.pfull[x], g & 1u, &S.abort_);
        if (!ok) break;
        tc_fence_after();
        tt_mma_o<D>(tm + 256u + 128u * x, tm + 128u * x + 64u * (g & 1u), 32u, kv0 + (vi % SLOTS) * TtSmem<1, D>::TILE,
                 pages < seg.j1 - seg.j0);
        tc_commit_warp(&S.oready[x]);
        if (x == 1u) tc_commit_warp(&S.empty[vi % SLOTS]);
        if (pages > 1) issue_s(x, g + 1u, 1u);
        if (pages == 2) tc_commit_warp(&S.qempty[x]);        // the segment's last S: Q may be replaced
      }
    }
    ++qn;
    if (ok) more = tt_next(seg, S, P) && tt_real(seg, S, P);
  }
  tt_finish(&S.fin);
}

// What the softmax warps know of a segment's nodes.
struct TtNodes {
  int b = -1, p = -1;                                // the row and item that these are of
  uint32_t uni = 0;                                  // lane i: word i of what any query of the row sees
  bool settled = false, there = false;               // the bits are in; the thread's node is present
};
// A thread's row r of tile ti: its node's bits to shared memory (asked for now, used in the
// tree's pages), unless they are there.
template <int NT, int D>
__device__ __forceinline__ void tt_ask_nodes(TtNodes& N, TtSmem<NT, D>& S, const TreeTcParams& P,
                                             const TtSeg& g, int ti, int r, bool live) {
  const TreeParams& T = P.T;
  if (N.p == g.p && (N.b == g.b || (N.b >= 0 && T.mask_bs == 0))) return;
  if (!N.settled) asm volatile("cp.async.wait_all;" ::: "memory");       // an older copy first
  const int32_t* m = T.masks + (int64_t)g.b * T.mask_bs +
                     (int64_t)(T.first + g.p * P.ni + P.nt * ti + r / T.A.group) * T.W;
  for (int i = 0; i < T.W; ++i) {
    if (live)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                   :: "r"(smem_addr(&S.mask[ti][r][i])), "l"(m + i) : "memory");
    else
      S.mask[ti][r][i] = 0u;
  }
  N.settled = false;
  N.b = g.b;
  N.p = g.p;
}
template <int NT, int D>
__device__ __forceinline__ void tt_settle(TtNodes& N, const TtSmem<NT, D>& S, const TreeTcParams& P,
                                          const TtSeg& g, int ti, int r) {
  const TreeParams& T = P.T;
  const int lane = threadIdx.x & 31;
  const int32_t* m = T.masks + (int64_t)g.b * T.mask_bs + (int64_t)T.first * T.W;
  asm volatile("cp.async.wait_all;" ::: "memory");
  uint32_t some = 0, uni = 0;
  for (int i = 0; i < T.W; ++i) {
    some |= S.mask[ti][r][i] & tree_valid(T.N, i);
    uint32_t word = 0;
#pragma unroll 4
    for (int q = lane; q < T.A.qlen; q += 32) word |= tree_word(m + (int64_t)q * T.W, T.W, T.N, i);
    word = __reduce_or_sync(0xffffffffu, word);
    if (lane == i) uni = word;
  }
  N.uni = uni;
  N.there = some != 0u;
  N.settled = true;
}

// The largest of 64 scores.
__device__ __forceinline__ float tt_largest(const uint32_t (&s0)[32], const uint32_t (&s1)[32]) {
  float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    px_max3(mx[e & 2], s0[e], s0[e + 1]);
    px_max3(mx[(e & 2) + 1], s1[e], s1[e + 1]);
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// The weights of 64 scores as bf16 pairs under the reference m, and their sum.
__device__ __forceinline__ float tt_weights(uint32_t (&s0)[32], uint32_t (&s1)[32], uint32_t (&pk)[32],
                                            float m, float sl2, bool wild) {
  if (wild) {
    px_scale(s0, sl2);
    px_scale(s1, sl2);
  }
  const float mc = m == -CUDART_INF_F ? 0.f : m, sf = wild ? 1.f : sl2;
  const unsigned long long sl22 = pair2(sf, sf), nm2 = pair2(-mc, -mc);
  unsigned long long ls[2] = {0ULL, 0ULL};           // (0.f, 0.f)
  px_weights(s0, pk, ls, sl22, nm2);
  px_weights(s1, pk + 16, ls, sl22, nm2);
  float a, b;
  unpair(add2(ls[0], ls[1]), a, b);
  return a + b;
}
// Columns [col, col + n) of O times alpha.
__device__ __forceinline__ void tt_rescale(uint32_t col, int n, float alpha) {
#pragma unroll 1
  for (int q = 0; q < n; q += 16) {
    uint32_t o[16];
    TC_LD16(o, col + (uint32_t)q);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
    TC_ST16(col + (uint32_t)q, o);
  }
}
// Columns [32 q0, 32 q1) of a thread's row of O: divided by the row's sum and written out, or as
// a piece.  oc: TMEM column of O (with the warp's lanes).
template <int NT, int D>
__device__ __forceinline__ void tt_emit(TtSmem<NT, D>& S, const TreeTcParams& P, const TtSeg& g, int ti, int r,
                                        bool live, bool there, float m, float l, uint32_t oc, int q0, int q1) {
  const AttnParams& A = P.T.A;
  const bool whole = g.j0 == 0 && g.j1 + TT_OVH == g.tb;
  const float il = !whole ? 1.f : l == 0.f || !there ? 0.f : 1.f / l;    // (a NaN sum: NaN)
  const int jt = r / A.group, j = g.p * P.ni + P.nt * ti + jt, hq = g.h * A.group + r - jt * A.group;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(A.out) + g.b * A.obs + j * A.oqs + hq * A.ohs;
  const int slot = 2 * (int)blockIdx.x + (g.j0 == 0), pr = P.nt * A.group * ti + r;
  float4* part = P.pacc + (int64_t)slot * (D / 4) * P.rs + pr;
#pragma unroll 1
  for (int q = q0; q < q1; ++q) {
    uint32_t u[32];
    TC_LD32(u, oc + 32u * q);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    float o[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = il == 0.f ? 0.f : il * __uint_as_float(u[e]);
    if (whole) {
      tt_write(S.out[threadIdx.x >> 5], o, out + 32 * q, live, P.out_vec != 0);
    } else if (live) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        part[(int64_t)(8 * q + e) * P.rs] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
    }
    __syncwarp();
  }
  if (!whole && live && q0 == 0) P.pml[(int64_t)slot * P.rs + pr] = make_float2(m, l);
}
// Query rows of tile ti of a segment's item.
__device__ __forceinline__ int tt_rows(const TreeTcParams& P, const TtSeg& g, int ti) {
  const AttnParams& A = P.T.A;
  return A.group * min(min(P.nt, P.ni - P.nt * ti), A.qlen - g.p * P.ni - P.nt * ti);
}
// What moves from reference m to mn: 2^(m - mn) of the sums and of O.
__device__ __forceinline__ float tt_alpha(float m, float mn) {
  return m == -CUDART_INF_F ? 0.f : ex2f(m - mn);
}

// Softmax of one tile: the threads of warpgroups 0 and 1 with the same lane own the same query
// row, x takes the keys [64 x, 64 x + 64) of a page and half of the columns of O.
template <int D>
__device__ __forceinline__ void tt_softmax_one(TtSmem<1, D>& S, const TreeTcParams& P, TtSeg seg, bool more) {
  constexpr int SLOTS = TtSmem<1, D>::SLOTS;
  const TreeParams& T = P.T;
  const int t = threadIdx.x, w = t >> 5, x = w >> 2, wq = w & 3, r = t & 127;
  const uint32_t lcol = S.tmem + ((uint32_t)(32 * wq) << 16), ocol = lcol + 256u;
  const float sl2 = T.A.scale * 1.4426950408889634f;
  uint32_t n = 0, xn = 0;                            // pages done; exchanges with the peer
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
  auto o_ready = [&]() {
    return __all_sync(0xffffffffu,
                      tc_wait(&S.oready[(n - 1) & 1u], ((n - 1) >> 1) & 1u, &S.abort_));
  };
  TtNodes nodes;
  while (more) {
    const TtSeg cur = seg;
    more = tt_next(seg, S, P) && tt_real(seg, S, P);
    const int pages = cur.j1 - cur.j0, end = tree_end(T, cur.base);
    const bool live = r < tt_rows(P, cur, 0), dead = __all_sync(0xffffffffu, !live);
    tt_ask_nodes(nodes, S, P, cur, 0, r, live);
    float m = -CUDART_INF_F, l = 0.f;
    bool wild = false;
#pragma unroll 1
    for (int i = 0; i < pages; ++i, ++n) {
      ok = __all_sync(0xffffffffu, tc_wait(&S.sfull[n & 1u], (n >> 1) & 1u, &S.abort_));
      if (!ok) break;
      tc_fence_after();
      const uint32_t scol = lcol + 128u * (n & 1u) + 64u * x;
      const int key0 = (cur.j0 + i) * SD_KV_PAGE;
      if (key0 + SD_KV_PAGE > cur.base) {
        // the tree's pages, and what lies behind it
        if (!nodes.settled) tt_settle(nodes, S, P, cur, 0, r);
        if (!dead) tt_hide(S.mask[0][r], T, cur.base, end, key0 + 64 * x, 64, scol);
        // V: each warpgroup its half of the keys, two warps 32 of them
        const uint32_t vi = 2u * n + 1u;
        const int grp = 2 * x + (wq & 1);
        ok = tt_blank(S.kv[vi % SLOTS], T, nodes.uni, cur.base, end, key0 + 32 * grp, 32 * grp, wq >> 1,
                      D == 128 ? (wq >> 1) + 1 : 1, &S.full[vi % SLOTS], (vi / SLOTS) & 1u, &S.abort_);
        if (!ok) break;
      }
      if (!dead) {
        uint32_t s0[32], s1[32], pk[32];
        if (i == 0) {                                // a reference for the segment, for both halves
          TC_LD32(s0, scol);
          TC_LD32(s1, scol + 32u);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          const float mine = tt_largest(s0, s1) * sl2;
          tell(mine);
          m = fmaxf(mine, told());
          if (!ok) break;
          wild = px_wild(m);
        }
        // weights under the reference as it is, and the largest score beside them: where that is
        // too far above it (rare), the reference moves and the weights are made again
        float sum;
        while (true) {
          TC_LD32(s0, scol);
          TC_LD32(s1, scol + 32u);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          const float mine = tt_largest(s0, s1) * sl2;
          tell(mine);
          sum = tt_weights(s0, s1, pk, m, sl2, wild);
          const float mt = fmaxf(mine, told());
          if (!ok) break;
          const bool move = mt > m + PX_HEADROOM;
          if (!__any_sync(0xffffffffu, move)) break;
          const float mn = move ? mt : m, alpha = move ? tt_alpha(m, mn) : 1.f;
          m = mn;
          l *= alpha;
          wild = px_wild(m);
          if (i > 0) {
            // O holds this segment's earlier pages: the last P . V into it first
            ok = o_ready();
            if (!ok) break;
            tc_fence_after();
            tt_rescale(ocol + (D / 2) * x, D / 2, alpha);
          }
        }
        if (!ok) break;
        l += sum;
        TC_ST32(scol, pk);                           // over columns that have been read
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      tc_fence_before();
      tt_arrive(&S.pfull[n & 1u]);
    }
    if (!ok) break;
    if (!dead) {
      tell(l);
      const float lp = told();
      ok = ok && o_ready();
      if (!ok) break;
      tc_fence_after();
      l = x ? lp + l : l + lp;                       // (the first warpgroup's half first, in both)
      tt_emit(S, P, cur, 0, r, live, nodes.there, m, l, ocol, D / 64 * x, D / 64 * (x + 1));
    }
    tc_fence_before();
  }
}

// Softmax of two tiles: a thread owns its query row of tile x, warpgroup x.
template <int D>
__device__ __forceinline__ void tt_softmax_pair(TtSmem<2, D>& S, const TreeTcParams& P, TtSeg seg, bool more) {
  constexpr int SLOTS = TtSmem<2, D>::SLOTS;
  const TreeParams& T = P.T;
  const int t = threadIdx.x, w = t >> 5, x = w >> 2, wq = w & 3, r = t & 127;
  const uint32_t lcol = S.tmem + ((uint32_t)(32 * wq) << 16) + 128u * x, ocol = lcol + 256u;
  const float sl2 = T.A.scale * 1.4426950408889634f;
  uint32_t n = 0;                                    // pages done
  bool ok = true;
  // P . V of page n - 1 is in O
  auto o_ready = [&]() {
    return __all_sync(0xffffffffu, tc_wait(&S.oready[x], (n - 1) & 1u, &S.abort_));
  };
  TtNodes nodes;
  while (more) {
    const TtSeg cur = seg;
    more = tt_next(seg, S, P) && tt_real(seg, S, P);
    const int pages = cur.j1 - cur.j0, end = tree_end(T, cur.base);
    const bool live = r < tt_rows(P, cur, x), dead = __all_sync(0xffffffffu, !live);
    tt_ask_nodes(nodes, S, P, cur, x, r, live);
    float m = -CUDART_INF_F, l = 0.f;
    bool wild = false;
#pragma unroll 1
    for (int i = 0; i < pages; ++i, ++n) {
      const uint32_t pcol = lcol + 64u * (n & 1u);   // P, over the page's first half of S
      const int key0 = (cur.j0 + i) * SD_KV_PAGE;
      const bool tree = key0 + SD_KV_PAGE > cur.base;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        ok = __all_sync(0xffffffffu, tc_wait(half ? &S.shi[x] : &S.slo[x], n & 1u, &S.abort_));
        if (!ok) break;
        tc_fence_after();
        const uint32_t scol = lcol + 64u * ((n + (uint32_t)half) & 1u);
        if (tree) {
          // the tree's pages, and what lies behind it (V: both tiles the same)
          if (!nodes.settled) tt_settle(nodes, S, P, cur, x, r);
          if (!dead) tt_hide(S.mask[x][r], T, cur.base, end, key0 + 64 * half, 64, scol);
          if (half) {
            const uint32_t vi = 2u * n + 1u;
            ok = tt_blank(S.kv[vi % SLOTS], T, nodes.uni, cur.base, end, key0 + 32 * wq, 32 * wq, 0, D / 64,
                          &S.full[vi % SLOTS], (vi / SLOTS) & 1u, &S.abort_);
            if (!ok) break;
          }
        }
        if (dead) {
          if (half) tt_arrive(&S.sread[x]);
          continue;
        }
        uint32_t s0[32], s1[32], pk[32];
        TC_LD32(s0, scol);
        TC_LD32(s1, scol + 32u);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (half) {
          tc_fence_before();
          tt_arrive(&S.sread[x]);
        }
        const float mt = tt_largest(s0, s1) * sl2;
        const bool move = mt > m + PX_HEADROOM;
        if (__any_sync(0xffffffffu, move)) {
          // (between the halves by a whole number, or next to one: the weights already made are
          // scaled by a power of two, which rounds nothing)
          const float up = half && m != -CUDART_INF_F ? m + ceilf(mt - m) : mt;
          const float mn = move ? up : m, alpha = move ? tt_alpha(m, mn) : 1.f;
          m = mn;
          l *= alpha;
          wild = px_wild(m);
          if (half) {
            // the page's first weights, already made
            TC_LD32(pk, pcol);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const __nv_bfloat162 a2 = __float2bfloat162_rn(alpha);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&pk[e]), a2);
              pk[e] = *reinterpret_cast<uint32_t*>(&v);
            }
            TC_ST32(pcol, pk);
          }
          if (i > 0) {
            // O holds this segment's earlier pages: the last P . V into it first
            ok = o_ready();
            if (!ok) break;
            tc_fence_after();
            tt_rescale(ocol, D, alpha);
          }
        }
        l += tt_weights(s0, s1, pk, m, sl2, wild);
        TC_ST32(pcol + 32u * half, pk);              // over columns that have been read
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      if (!ok) break;
      tc_fence_before();
      tt_arrive(&S.pfull[x]);
    }
    if (!ok) break;
    if (!dead) {
      ok = o_ready();
      if (!ok) break;
      tc_fence_after();
      tt_emit(S, P, cur, x, r, live, nodes.there, m, l, ocol, 0, D / 32);
    }
    tc_fence_before();
  }
}

template <int NT, int D>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_tc_kernel(const __grid_constant__ TreeTcParams P, const __grid_constant__ CUtensorMap tmk,
               const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmq) {
  extern __shared__ __align__(1024) unsigned char tt_raw[];
  const uint32_t pad = (1024u - (smem_addr(tt_raw) & 1023u)) & 1023u;   // swizzle atoms: 1024 B
  TtSmem<NT, D>& S = *reinterpret_cast<TtSmem<NT, D>*>(tt_raw + pad);
  const TreeParams& T = P.T;
  const int t = threadIdx.x, w = t >> 5, lane = t & 31, cta = (int)blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (w == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_addr(&S.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (t == 256) {
    for (int i = 0; i < TtSmem<NT, D>::SLOTS; ++i) {
      tc_bar_init(&S.full[i], 1);
      tc_bar_init(&S.empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      tc_bar_init(&S.sfull[x], 1);
      tc_bar_init(&S.slo[x], 1);
      tc_bar_init(&S.shi[x], 1);
      tc_bar_init(&S.sread[x], 4);
      tc_bar_init(&S.pfull[x], NT == 2 ? 4 : 8);     // warps
      tc_bar_init(&S.oready[x], 1);
    }
    tc_bar_init(&S.fin, 1);
    for (int x = 0; x < NT; ++x) {
      tc_bar_init(&S.qfull[x], 1);
      tc_bar_init(&S.qempty[x], 1);
    }
    S.abort_ = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = t; i < 2 * 2 * 128; i += TT_THREADS) S.peer[0][0][i] = 0ULL;     // (numbers start at 1)
  // the rows of a tile that no query fills stay 0
  const int filled = P.nt * T.A.group * 8;
  for (int i = t; i < NT * (D / 64) * 128 * 8; i += TT_THREADS)
    if (i % 1024 >= filled) reinterpret_cast<uint4*>(S.q[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");         // what the kernel before this one wrote
  int total, share;
  tt_plan(S, P, &total, &share);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if ((int64_t)cta * share < total) {
    const int t0 = cta * share;
    TtSeg seg;
    seg.b = S.first[0];
    seg.base = tt_base(S, T, seg.b);
    seg.tb = tt_units(tree_end(T, seg.base));
    const int u = t0 - S.first[1], it = u / seg.tb;
    seg.off = u % seg.tb;
    seg.h = it / P.np;
    seg.p = it % P.np;
    seg.tt = t0;
    seg.t1 = t0 + min(total - t0, share);
    tt_bounds(seg);
    const bool more = tt_real(seg, S, P);
    if (w == 8) {
      if (lane == 0) tt_load_kv(S, P, tmk, tmv, tmq, seg, more, share);
    } else if (w == 10) {
      if (lane == 0) tt_load_q(S, P, tmq, seg, more);
    } else if constexpr (NT == 2) {
      if (w == 9) tt_issue_pair(S, P, seg, more);
      else if (w < 8) tt_softmax_pair(S, P, seg, more);
    } else {
      if (w == 9) tt_issue_one(S, P, seg, more);
      else if (w < 8) tt_softmax_one(S, P, seg, more);
    }
  }
  if ((int64_t)cta * share >= total && t == 0) P.cut[cta] = make_int4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();                                   // every role is done
  if (t == 0) P.status[cta] = S.abort_;
  if (w == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 :: "r"(S.tmem), "r"(512u) : "memory");
  }
}

// CTA (c, rows, columns): the item that the run of CTA c of the main kernel cuts, if any: its
// pieces are merged, in order; a lane takes a query row, a warp four columns of each of NC
// column blocks.  One block and eight pieces at once where that makes few CTAs (16 items of
// 33 rows in ten pieces each: 60 us the call, 70 with four blocks and two pieces), else all
// four and two (148 cut items of 104 rows: 64.5 us the call, 70 with one).
template <int NC>
__global__ void __launch_bounds__(TJ_THREADS) tree_join_kernel(const __grid_constant__ TreeTcParams P) {
  constexpr int AT_ONCE = 8 / NC;
  __shared__ __align__(16) uint2 tile[TJ_ROWS][NC][TJ_COLS / 4 + 1];
  const TreeParams& T = P.T;
  const AttnParams& A = T.A;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int c = (int)blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int stop = t < TT_CTAS ? P.status[t] : 0;
  const int4 cut = P.cut[c];
  if (__syncthreads_or(stop)) {
    // a wait gave up somewhere: say so in the output
    const int64_t n = (int64_t)A.B * A.qlen * A.Hq * A.D;
    const int64_t nt = (int64_t)gridDim.x * gridDim.y * gridDim.z * TJ_THREADS;
    const int64_t cta = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + c;
    for (int64_t i = cta * TJ_THREADS + t; i < n; i += nt) {
      const int64_t v = i / A.D, bj = v / A.Hq;
      reinterpret_cast<__nv_bfloat16*>(A.out)[(bj / A.qlen) * A.obs + (bj % A.qlen) * A.oqs +
                                              (v % A.Hq) * A.ohs + i % A.D] =
          __float2bfloat16(CUDART_NAN_F);
    }
    return;
  }
  const int b = cut.x, h = cut.y, p = cut.z, np = cut.w;
  if (np == 0) return;
  const int rows = A.group * min(P.ni, A.qlen - p * P.ni), r0 = (int)blockIdx.y * TJ_ROWS;
  if (r0 >= rows) return;
  auto node_of = [&](int r) { return p * P.ni + r / A.group; };
  const int r = min(r0 + lane, rows - 1), col = (int)blockIdx.z * NC * (TJ_COLS / 4) + w;
  const bool there =
      tree_present(T.masks + (int64_t)b * T.mask_bs + (int64_t)(T.first + node_of(r)) * T.W, T.W, T.N);
  float gm = -CUDART_INF_F, L = 0.f;
  float4 a[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = 0; i0 < np; i0 += AT_ONCE) {
    float2 ml[AT_ONCE];
    float4 v[AT_ONCE][NC];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      // piece i: the item's start in its first CTA, then a CTA's start each
      const int64_t slot = 2 * (c + i0 + i) + (i0 + i == 0);
      const bool is = i0 + i < np;
      ml[i] = is ? __ldcg(&P.pml[slot * P.rs + r]) : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
      for (int k = 0; k < NC; ++k)
        v[i][k] = is ? __ldcg(P.pacc + (slot * (A.D / 4) + col + k * (TJ_COLS / 4)) * P.rs + r)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mx = gm;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) mx = fmaxf(mx, ml[i].x);
    const float old = gm == -CUDART_INF_F ? 0.f : ex2f(gm - mx);
    gm = mx;
    L = L != L ? L : old * L;                        // (a NaN sum stays)
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (old == 0.f) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      else a[k] = make_float4(a[k].x * old, a[k].y * old, a[k].z * old, a[k].w * old);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const float fw = ml[i].x == -CUDART_INF_F ? 0.f : ex2f(ml[i].x - gm);
      L += ml[i].y != ml[i].y ? ml[i].y : fw * ml[i].y;
      if (fw != 0.f) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          a[k].x = fmaf(fw, v[i][k].x, a[k].x); a[k].y = fmaf(fw, v[i][k].y, a[k].y);
          a[k].z = fmaf(fw, v[i][k].z, a[k].z); a[k].w = fmaf(fw, v[i][k].w, a[k].w);
        }
      }
    }
  }
  const bool none = L == 0.f || !there;
  const float il = none ? 0.f : 1.f / L;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    uint2 u = make_uint2(0u, 0u);
    if (!none) {
      u.x = pack_bf16(a[k].x * il, a[k].y * il);
      u.y = pack_bf16(a[k].z * il, a[k].w * il);
    }
    tile[lane][k][w] = u;
  }
  __syncthreads();
  // eight threads a row
  const int ro = r0 + (t >> 3);
  if (ro >= rows) return;
  const int j = node_of(ro), hq = h * A.group + ro % A.group;
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(A.out) + b * A.obs + j * A.oqs + hq * A.ohs +
                       (int)blockIdx.z * NC * TJ_COLS + 4 * (t & 7);
#pragma unroll
  for (int k = 0; k < NC; ++k, dst += TJ_COLS) {
    const uint2 u = tile[t >> 3][k][t & 7];
    if (P.out_vec) {
      *reinterpret_cast<uint2*>(dst) = u;
    } else {
      const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&u);
#pragma unroll
      for (int q = 0; q < 4; ++q) dst[q] = e[q];
    }
  }
}

// The shapes of the tensor-core path.
static bool tt_fast(int dtype, int D, int group) {
  return dtype == SD_DTYPE_BF16 && (D == 64 || D == 128) && group <= 128;
}

struct TtLayout {
  size_t status, acc, ml, bytes;
  int np, ni, nt, rs;
};
static TtLayout tt_layout(int qlen, int group, int D) {
  TtLayout L;
  // items of up to two tiles of whole nodes, of about the same size, and so their tiles
  const int most = TT_TILE / group;
  L.np = (qlen + 2 * most - 1) / (2 * most);
  L.ni = (qlen + L.np - 1) / L.np;
  L.nt = qlen <= most ? qlen : (L.ni + 1) / 2;
  L.rs = (L.ni * group + 31) / 32 * 32;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  size_t o = up(TT_CTAS * sizeof(int4));
  L.status = o; o = up(o + TT_CTAS * sizeof(int));
  L.acc = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * D * sizeof(float));
  L.ml = o; o = up(o + (size_t)2 * TT_CTAS * L.rs * 2 * sizeof(float));
  L.bytes = o;
  return L;
}

template <int NT, int D>
static int launch_tc(const TreeTcParams& P, const CUtensorMap& mk, const CUtensorMap& mv,
                     const CUtensorMap& mq, cudaStream_t st) {
  const int sm = (int)sizeof(TtSmem<NT, D>) + 1024;   // room to align
  static std::atomic<uint64_t> ready{0};             // devices whose kernel may use that much
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SD_ELAUNCH;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load() & bit) || !bit) {
    if (cudaFuncSetAttribute(tree_tc_kernel<NT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) !=
        cudaSuccess)
      return SD_ELAUNCH;
    ready.fetch_or(bit);
  }
  // (its start, up to the first read of memory, beside the end of the kernel before it)
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3(TT_CTAS);
  cfg.blockDim = dim3(TT_THREADS);
  cfg.dynamicSmemBytes = sm;
  if (cudaLaunchKernelEx(&cfg, tree_tc_kernel<NT, D>, P, mk, mv, mq) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

static int tree_tc(TreeTcParams& P, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  AttnParams& A = P.T.A;
  // TMA boxes of the queries (the stride of a dimension of one is any) and the caches
  auto odd = [](int n, int64_t stride) { return n > 1 && (stride <= 0 || stride % 8); };
  if ((reinterpret_cast<uintptr_t>(A.q) & 15) || odd(A.B, A.qbs) || odd(A.Hq, A.qhs) || odd(A.qlen, A.qqs) ||
      (reinterpret_cast<uintptr_t>(A.k) & 15) || (reinterpret_cast<uintptr_t>(A.v) & 15))
    return SD_EINVAL;
  const int64_t rows = A.bt ? (int64_t)A.npages * A.Hkv * SD_KV_PAGE : (int64_t)A.B * A.Hkv * A.C;
  if (rows >= (int64_t)1 << 31) return SD_ENOTSUP;   // a TMA coordinate
  const TtLayout L = tt_layout(A.qlen, A.group, A.D);
  // the schedule counts units in 32 bits
  const int64_t tiles = ((int64_t)A.C + SD_KV_PAGE - 1) / SD_KV_PAGE + TT_OVH;
  if (tiles * A.B > (0x7FFFFFFF - TT_CTAS) / ((int64_t)A.Hkv * L.np)) return SD_ENOTSUP;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < L.bytes)
    return SD_ENOSPC;
  char* ws = reinterpret_cast<char*>(workspace);
  P.np = L.np; P.ni = L.ni; P.nt = L.nt; P.rs = L.rs;
  P.cut = reinterpret_cast<int4*>(ws);
  P.status = reinterpret_cast<int*>(ws + L.status);
  P.pacc = reinterpret_cast<float4*>(ws + L.acc);
  P.pml = reinterpret_cast<float2*>(ws + L.ml);
  P.out_vec = (reinterpret_cast<uintptr_t>(A.out) & 15) == 0 && A.obs % 8 == 0 && A.oqs % 8 == 0 &&
              A.ohs % 8 == 0;
  CUtensorMap mk, mv, mq;
  if (!cache_map(&mk, A.k, rows, SD_KV_PAGE, A.D) || !cache_map(&mv, A.v, rows, SD_KV_PAGE, A.D)) return SD_ENOTSUP;
  // the queries of a tile: 64 columns of `group` heads of L.nt nodes of a row
  const int64_t sizes[4] = {A.D, A.Hq, A.qlen, A.B}, strides[3] = {A.qhs, A.qqs, A.qbs};
  const int box[4] = {64, A.group, L.nt, 1};
  if (!tile_map(&mq, A.q, sizes, strides, box)) return SD_ENOTSUP;
  const int rc = A.D == 64 ? L.nt < L.ni ? launch_tc<2, 64>(P, mk, mv, mq, st)
                                         : launch_tc<1, 64>(P, mk, mv, mq, st)
                           : L.nt < L.ni ? launch_tc<2, 128>(P, mk, mv, mq, st)
                                         : launch_tc<1, 128>(P, mk, mv, mq, st);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.blockDim = dim3(TJ_THREADS);
  // (at most as many items are cut as there are)
  const int blocks = A.D / TJ_COLS;
  const int64_t cut = std::min<int64_t>(TT_CTAS, (int64_t)A.B * A.Hkv * L.np) * (L.rs / TJ_ROWS) * blocks;
  const bool few = cut <= TT_CTAS * 4;
  cfg.gridDim = dim3(TT_CTAS, (unsigned)(L.rs / TJ_ROWS), few ? blocks : 1);
  const auto join = few ? tree_join_kernel<1> : blocks == 2 ? tree_join_kernel<2> : tree_join_kernel<4>;
  if (cudaLaunchKernelEx(&cfg, join, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // namespace sd

using namespace sd;

extern "C" {

size_t sd_tree_attn_workspace_bytes(int B, int Hq, int Hkv, int D, int C, int qlen, int dtype) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || C <= 0 || qlen <= 0) return 0;
  if (!tt_fast(dtype, D, Hq / Hkv) || (int64_t)qlen * (Hq / Hkv) > 0x7FFFFFFF) return 0;
  return tt_layout(qlen, Hq / Hkv, D).bytes;
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
  if (N > SD_TREE_MAX || D > 128) return SD_ENOTSUP;
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
  // one CTA per entry of the output
  if (!rows_apart<3>(D, {B, qlen, Hq}, {obs, oqs, ohs})) return SD_EINVAL;
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
