// Attention over a paged cache whose rows share a prefix (sm_100a).
//
// The rows of a group (samples of one prompt, requests under one system
// prompt) hold the same pages in front: block_table[b, 0..pages_g) is equal
// for every row b of group g.  With the softmax split over two key ranges,
//   out = (2^(m1 - m) O1 + 2^(m2 - m) O2) / (2^(m1 - m) l1 + 2^(m2 - m) l2),
//   m = max(m1, m2), (m_i, l_i, O_i) the running maximum (base 2), sum and
//   unnormalised output over range i,
// the shared range is computed for all query rows of a group at once and each
// row's own range by itself:
//   prefix_plan_kernel  lays out the work of both from the device lengths, and
//                       copies the queries kv head by kv head, so that TMA
//                       brings any run of a group's query rows;
//   prefix_tc_kernel    some CTAs: the shared pages, query rows of the whole group
//                       on the M side of tcgen05.mma: K and V are read once per
//                       256 query rows instead of once per row; the others: the
//                       rows' own pages, four rows at a time;
//   prefix_join_kernel  merges the partials, in piece order, into the output.
// Each is launched as a programmatic dependent of the one before and reads what
// that one wrote (and what it had waited for) behind its own wait.  64 rows of 5
// queries, 32 / 8 heads, 64 shared pages and up to 1 K own keys: 96 us for the
// call; kernel by kernel, with cold caches, 7 + 82 + 14.
// A row whose first query does not see the whole shared range (an empty or a
// padding row, a short cap) takes no part in it: its own range starts at 0, so
// the shared range needs no mask and no row meets another row's masked keys.
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "sd_attn.cuh"
#include "sd_common.cuh"
#include "sd_softmax.cuh"
#include "sd_tcgen05.cuh"

namespace sd {

constexpr int PX_D = 128;
constexpr int PX_ROWS = 256;                 // query rows per item: two tiles of 128
constexpr int PX_SLOTS = 4;                  // 32 KB K / V tiles in flight (two pages)
constexpr int PX_THREADS = 320;              // warps 0-3, 4-7: softmax of tile 0, 1; 8 TMA; 9 MMA
constexpr int PX_PLAN_THREADS = 1024;
constexpr int PX_CTAS = 148;                 // one CTA per SM
constexpr int PX_OVH = 2;                    // schedule cost of an item beyond its pages, in pages
constexpr int PX_MIN_SHARE = PX_OVH + 1;     // fewest schedule units per CTA: a one-page item
constexpr int PX_JOIN_THREADS = 256;
constexpr int PX_JOIN_CTAS = 4;              // per SM
constexpr int PX_JOIN_LOADS = 4;             // pieces of a row on their way at once
constexpr int OW_STAGES = 3;                 // K + V tiles in flight (own ranges: of the
                                             // PX_THREADS warps 0-3 softmax, 4 TMA, 5 MMA)
constexpr int OW_OVH = 2;                    // schedule cost of a (row, kv head) beyond its pages
constexpr int OW_MIN_SHARE = OW_OVH + 1;

struct PrefixParams {
  AttnParams A;
  const int32_t* starts;                     // [G + 1] first row of each group
  const int32_t* pages;                      // [G] shared pages of each group
  int G, max_items;
  // workspace
  int* g_unit;                               // [G + 1] exclusive prefix of schedule units
  int* g_item;                               // [G + 1] exclusive prefix of items
  int* g_row0;                               // [G]
  int* g_rows;                               // [G]
  int* g_pages;                              // [G] 0: the group shares nothing
  int4* rowjoin;                             // [B][2] what the join needs of the row, see PxRow
  int4* totals;                              // own and shared ranges: schedule units, units per CTA
  int* rowstart;                             // [B] first key of the row's own range, a page bound
  int qc, nq, chunks;                        // queries per chunk; lane quarters of a chunk's rows
  int slots;                                 // partial slots of a chunk of the own ranges
  uint4* qp;                                 // queries [Hkv][B][qlen][group][D]
  float* pacc;                               // [slot][2 tiles][4 chunks][128 rows][32]
  float* pml;                                // [slot][PX_ROWS][2]
};

// What the join needs of a row, in one load: its units of the own ranges and the
// ones before them; its group's units and items before, rows (0: it takes no
// part) and pages, and the row's place in it.
struct __align__(16) PxRow {
  int pre, tb, unit, item, rows, pages, place, unused;
};
static_assert(sizeof(PxRow) == 2 * sizeof(int4), "two loads");

// The items of a group: (kv head, 256 query rows), kv head outer.
__device__ __forceinline__ int px_pairs(const PrefixParams& P, int rows) {
  return (rows * P.A.R + PX_ROWS - 1) / PX_ROWS;
}
__device__ __forceinline__ int px_share(int total) {
  return max(PX_MIN_SHARE, (total + PX_CTAS - 1) / PX_CTAS);
}

// Units per CTA of the own ranges.  Where the shared ranges leave SMs idle, only
// the CTAs that come up on those get work, if it then ends before the ones that
// have to wait for a busy SM would (a shared page takes about 1.5 own ones).  32 / 8
// heads, 1 query: 8 rows, 16 shared pages, up to 1000 own keys 23.1 us for the call
// (27.2 with the work over all SMs); 64 rows, 8 pages, up to 300 keys 35.0 (39.7); 16
// rows the same 21.3 (21.0), 4 rows, 4 pages, up to 100 keys 20.4 (19.8).
__device__ __forceinline__ int ow_share(const PrefixParams& P, int total, int units, int ps) {
  int share = max(OW_MIN_SHARE, (total + PX_CTAS - 1) / PX_CTAS);
  if (units > 0 && P.qc >= P.A.qlen) {
    const int idle = PX_CTAS - (units + ps - 1) / ps;
    if (idle > 0) {
      const int apart = max(share, (total + idle - 1) / idle);
      if (apart - share < ps + ps / 2) share = apart;
    }
  }
  return share;
}

// CTA 0 plans, the others pack: 16 threads copy a query row.
__global__ void __launch_bounds__(PX_PLAN_THREADS) prefix_plan_kernel(const PrefixParams P) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x > 0) {
    const AttnParams& A = P.A;
    const int64_t i = ((int64_t)(blockIdx.x - 1) * PX_PLAN_THREADS + threadIdx.x) >> 4;
    if (i >= (int64_t)A.B * A.Hq * A.qlen) return;
    const int c = threadIdx.x & 15;
    const int hb = (int)(i / A.R), f = (int)(i - (int64_t)hb * A.R), h = hb / A.B, b = hb - h * A.B;
    const int j = f / A.group, hq = h * A.group + f - j * A.group;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(A.q);
    P.qp[i * 16 + c] =
        __ldg(reinterpret_cast<const uint4*>(q + b * A.qbs + hq * A.qhs + j * A.qqs) + c);
    return;
  }
  __shared__ long long red[33];
  __shared__ int redi[33];
  const AttnParams& A = P.A;
  const int t = threadIdx.x;
  if (t == 0) *A.status = 0;
  const int W = A.bt_stride;
  long long items0 = 0, units0 = 0;
  for (int g0 = 0; g0 < P.G; g0 += 1024) {
    const int g = g0 + t;
    long long items = 0, units = 0;
    if (g < P.G) {
      const int s0 = min(max(P.starts[g], 0), A.B), s1 = min(max(P.starts[g + 1], s0), A.B);
      const int rows = s1 - s0;
      const int pg = rows < 2 ? 0 : min(max(P.pages[g], 0), W);   // one row shares with nobody
      if (pg > 0) {
        items = (long long)A.Hkv * (((long long)rows * A.R + PX_ROWS - 1) / PX_ROWS);
        units = items * (pg + PX_OVH);
      }
      P.g_row0[g] = s0;
      P.g_rows[g] = rows;
      P.g_pages[g] = pg;
    }
    long long si, su;
    const long long xi = block_excl_scan<long long>(items, red, &si);
    __syncthreads();
    const long long xu = block_excl_scan<long long>(units, red, &su);
    if (g < P.G) {
      P.g_item[g] = (int)(items0 + xi);
      P.g_unit[g] = (int)(units0 + xu);
    }
    items0 += si;
    units0 += su;
    __syncthreads();
  }
  // groups that overlap could ask for more items than the workspace holds:
  // then nothing is shared
  const bool share = items0 <= P.max_items && units0 <= 0x7FFFFFFF;
  if (t == 0) {
    P.g_item[P.G] = share ? (int)items0 : 0;
    P.g_unit[P.G] = share ? (int)units0 : 0;
  }
  __syncthreads();
  int carry = 0;
  for (int b0 = 0; b0 < A.B; b0 += 1024) {
    const int b = b0 + t;
    int tiles = 0;
    PxRow row = {};
    if (b < A.B) {
      int lo = 0, hi = P.G;                          // the last group that starts at or before b
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (P.starts[mid] <= b) lo = mid + 1; else hi = mid;
      }
      const int g = lo - 1;
      int start = 0;
      if (share && g >= 0 && b < P.g_row0[g] + P.g_rows[g] && b >= P.g_row0[g]) {
        const int keys = P.g_pages[g] * SD_KV_PAGE;
        if (row_limit(A, b, 0) >= keys) start = keys;
      }
      if (start > 0) {
        row.unit = P.g_unit[g];
        row.item = P.g_item[g];
        row.rows = P.g_rows[g];
        row.pages = P.g_pages[g];
        row.place = b - P.g_row0[g];
      }
      const int km = row_limit(A, b, A.qlen - 1);
      P.rowstart[b] = start;
      A.rowkmax[b] = km;
      tiles = (max(km - start, 0) + SD_KV_PAGE - 1) / SD_KV_PAGE;
      if (tiles > 0) tiles += OW_OVH;
    }
    int sum;
    const int ex = block_excl_scan<int>(tiles, redi, &sum);
    if (b < A.B) {
      A.rowpre[b] = row.pre = carry + ex;
      row.tb = tiles;
      P.rowjoin[2 * b] = make_int4(row.pre, row.tb, row.unit, row.item);
      P.rowjoin[2 * b + 1] = make_int4(row.rows, row.pages, row.place, 0);
    }
    carry += sum;
    __syncthreads();
  }
  if (t == 0) {
    A.rowpre[A.B] = carry;
    const int own = carry * A.Hkv, shared = share ? (int)units0 : 0, ps = px_share(shared);
    *P.totals = make_int4(own, shared, ow_share(P, own, shared, ps), ps);
  }
}

// A CTA's run of schedule units as segments of items, walked identically by
// every role.
struct PxSeg {
  int g, rows, h, p, np, tb, off, tt, t1, ncost, j0, j1;     // pages [j0, j1) of the segment
  bool dup;                                          // one tile of rows: both tiles work on it
};
__device__ __forceinline__ void px_item(PxSeg& s, const PrefixParams& P) {
  s.dup = s.rows * P.A.R - s.p * PX_ROWS <= PX_ROWS / 2;
}
__device__ __forceinline__ void px_bounds(PxSeg& s) {
  s.ncost = min(s.tb - s.off, s.t1 - s.tt);
  s.j0 = max(s.off, PX_OVH) - PX_OVH;
  s.j1 = max(s.off + s.ncost - PX_OVH, s.j0);
}
// first: the group's index, its first unit, its rows and pages
__device__ __forceinline__ void px_init(PxSeg& s, const PrefixParams& P, const int (&first)[4],
                                        int t0, int t1) {
  s.g = first[0];
  s.rows = first[2];
  s.np = px_pairs(P, s.rows);
  s.tb = first[3] + PX_OVH;
  const int u = t0 - first[1], it = u / s.tb;
  s.off = u % s.tb;
  s.h = it / s.np;
  s.p = it % s.np;
  s.tt = t0;
  s.t1 = t1;
  px_item(s, P);
  px_bounds(s);
}
__device__ __forceinline__ bool px_next(PxSeg& s, const PrefixParams& P) {
  s.tt += s.ncost;
  if (s.tt >= s.t1) return false;
  s.off = 0;
  if (++s.p == s.np) {
    s.p = 0;
    if (++s.h == P.A.Hkv) {
      s.h = 0;
      do { ++s.g; } while (P.g_pages[s.g] == 0);     // units remain, so a sharing group follows
      s.rows = P.g_rows[s.g];
      s.np = px_pairs(P, s.rows);
      s.tb = P.g_pages[s.g] + PX_OVH;
    }
  }
  px_item(s, P);
  px_bounds(s);
  return true;
}
struct PxSmem {
  alignas(1024) unsigned char q[2][2][128 * 128];            // [tile][64-col box][128 rows x 128 B]
  alignas(1024) unsigned char kv[PX_SLOTS][2][128 * 128];    // [slot][64-col box][128 keys x 128 B]
  alignas(8) unsigned long long full[PX_SLOTS], empty[PX_SLOTS];
  alignas(128) unsigned char out[8][32 * 128];               // a warp's 32 rows x 32 floats of O
  alignas(8) unsigned long long sfull[2], pfull[2], oready[2], qfull[2], fin;
  int first[4];                                      // the CTA's first group: g, unit, rows, pages
  int abort_;
};
static_assert(sizeof(PxSmem) + 2048 <= 227 * 1024, "shared memory, with room to align");

// A group's first unit, the next one's, rows and pages
__device__ __forceinline__ int4 px_group(const PrefixParams& P, int g) {
  return make_int4(P.g_unit[g], P.g_unit[g + 1], P.g_rows[g], P.g_pages[g]);
}

// Persistent, stream-K: the (item, page) units lie end to end and each CTA
// takes one contiguous run.  Per page of 128 keys and tile of 128 query rows:
//   S[128 rows, 128 keys] = Q . K^T      (tcgen05.mma, operands in shared memory)
//   thread t of the tile's four softmax warps owns row t (TMEM lane t): its
//   128 scores in registers, a lazy reference maximum (moved when a score
//   passes it by PX_HEADROOM), p = 2^(s - m) as bf16 back into the first 64
//   columns of S
//   O[128 rows, 128 d] += P . V          (tcgen05.mma, A in TMEM)
// TMEM holds S and O of both tiles, all 512 columns, so P has to lie over S, and
// S of a tile's next page is issued behind P . V of this one (MMAs run in issue
// order).  One issuer takes the tiles in turns, so that one tile's softmax runs
// under the other's tensor work.  Measured on the way, cycles per page with both
// tiles (2072 of them MMAs): one issuer on a single thread 4950 (an issue gap of
// 500 cycles at every wait); two such issuers, one per tile, 5400 (the tiles fall
// into step: softmax, then tensor cores); half pages with S of N = 64, 4170 (an
// MMA of N = 64 takes as long as one of N = 128); this form 3550.  A tile's own
// chain is what bounds it: 1900 cycles of softmax, then P . V and the next S with
// their latencies.  Two warps per 32 rows, each with half of the keys, left the
// softmax as long (1850: the pipes of the SM quarter are shared); weights and
// maximum in one pass over S, 3600.  128 rows of 5 queries over 128 pages, 32 / 8
// heads: 150 us as a launch of its own, 1.15 PFLOP/s.
// An item with rows for one tile only is worked on by both: tile 0 takes the
// first, tile 1 the second half of every page's keys.
__device__ __forceinline__ void shared_ranges(const PrefixParams& P, const CUtensorMap& tmk,
                                              const CUtensorMap& tmv, const CUtensorMap& tmq,
                                              int4 totals, int4 group, const uint32_t* tmem) {
  extern __shared__ __align__(1024) unsigned char px_raw[];
  const uint32_t pad = (1024u - (smem_addr(px_raw) & 1023u)) & 1023u;   // swizzle atoms: 1024 B
  PxSmem& S = *reinterpret_cast<PxSmem*>(px_raw + pad);
  const AttnParams& A = P.A;
  const int t = threadIdx.x, w = t >> 5, lane = t & 31;
  if (t == 0) {
    for (int i = 0; i < PX_SLOTS; ++i) {
      tc_bar_init(&S.full[i], 1);
      tc_bar_init(&S.empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      tc_bar_init(&S.qfull[x], 1);
      tc_bar_init(&S.sfull[x], 1);
      tc_bar_init(&S.pfull[x], 128);
      tc_bar_init(&S.oready[x], 1);
    }
    tc_bar_init(&S.fin, 1);
    S.abort_ = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int t0 = (int)blockIdx.x * totals.w, t1 = min(totals.y, t0 + totals.w);
  for (int g = t; g < P.G; g += PX_THREADS) {
    if (g != t) group = px_group(P, g);
    if (group.x <= t0 && t0 < group.y) {
      S.first[0] = g;
      S.first[1] = group.x;
      S.first[2] = group.z;
      S.first[3] = group.w;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = *tmem;
  PxSeg seg;
  px_init(seg, P, S.first, t0, t1);

  if (w >= 8) {
    if (w == 8 && lane == 0) {
      // ---------------- TMA producer: K then V of each page, PX_SLOTS tiles ahead
      uint32_t idx = 0;
      bool ok = true;
      do {
        const int32_t* bt = A.bt + (int64_t)P.g_row0[seg.g] * A.bt_stride;
        for (int j = seg.j0; j < seg.j1 && ok; ++j) {
          int pg = __ldg(bt + j);
          if ((unsigned)pg >= (unsigned)A.npages) pg = 0;    // a wrong table reads page 0
          const int y = (int)(((int64_t)pg * A.Hkv + seg.h) * SD_KV_PAGE);
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv, ++idx) {
            const int sl = (int)(idx % PX_SLOTS);
            if (idx >= (uint32_t)PX_SLOTS)
              ok = tc_wait(&S.empty[sl], ((idx / PX_SLOTS) - 1) & 1u, &S.abort_);
            if (!ok) break;
            tc_expect_tx(&S.full[sl], 2u * 128u * 128u);
            const void* map = kv ? (const void*)&tmv : (const void*)&tmk;
            tc_tma_2d(S.kv[sl][0], map, 0, y, &S.full[sl]);
            tc_tma_2d(S.kv[sl][1], map, 64, y, &S.full[sl]);
          }
        }
      } while (ok && px_next(seg, P));
      if (!ok) {
        // let the copies already issued land before the CTA leaves
        for (uint32_t q = idx > (uint32_t)PX_SLOTS ? idx - PX_SLOTS : 0u; q < idx; ++q) {
          int dummy = 0;
          tc_wait(&S.full[q % PX_SLOTS], (q / PX_SLOTS) & 1u, &dummy);
        }
      }
    } else if (w == 9) {
      // ---------------- MMA issuer (the whole warp): S0(0) S1(0) | PV0(i) S0(i + 1)
      // PV1(i) S1(i + 1) | ...
      constexpr uint32_t ID1 = tc_idesc(128, 128, 0, 0);     // S = Q . K^T
      constexpr uint32_t ID1H = tc_idesc(128, 64, 0, 0);     // of half a page
      constexpr uint32_t ID2 = tc_idesc(128, 128, 0, 1);     // O += P . V (V [key][d]: N-major)
      // One burst of each kind in the code: a kernel starts with cold
      // instruction caches, and each new burst (by tile, ring position) costs its
      // first execution more than the constants in it save later.
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
      do {
        const int pages = seg.j1 - seg.j0;
        dup = seg.dup;
        if (pages == 0) continue;
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
      } while (ok && px_next(seg, P));
      // every MMA this warp issued has finished before the CTA leaves
      tc_commit_warp(&S.fin);
      int dummy = 0;
      tc_wait(&S.fin, 0u, &dummy);
    }
  } else {
    // ---------------- softmax warps of tile x: thread r owns query row r
    const int x = w >> 2, r = t & 127;
    const uint32_t lrow = (uint32_t)(32 * (w & 3)) << 16;
    const uint32_t scol = tm + lrow + 128u * x, ocol = scol + 256u;
    const float sl2 = A.scale * 1.4426950408889634f;
    auto first_row = [&](const PxSeg& g) { return g.p * PX_ROWS + (g.dup ? 0 : 128 * x); };
    // slot (item + CTA) of the segment's partial, this thread's row
    auto slot_row = [&](const PxSeg& g) {
      return ((int64_t)P.g_item[g.g] + g.h * g.np + g.p + blockIdx.x) * PX_ROWS + 128 * x + r;
    };
    // on to the next segment with pages
    auto find = [&](PxSeg& g) {
      while (g.j1 == g.j0)
        if (!px_next(g, P)) return false;
      return true;
    };
    // the tile's 128 query rows (rows past the group's end compute what nobody reads)
    auto load_q = [&](const PxSeg& g) {
      if (r == 0) {
        const int y = (g.h * A.B + P.g_row0[g.g]) * A.R + first_row(g);
        tc_expect_tx(&S.qfull[x], 2u * 128u * 128u);
        tc_tma_2d(S.q[x][0], &tmq, 0, y, &S.qfull[x]);
        tc_tma_2d(S.q[x][1], &tmq, 64, y, &S.qfull[x]);
      }
    };
    uint32_t n = 0, qn = 0;                          // pages done, Q tiles asked for
    bool ok = true, more = find(seg);
    if (more) {
      load_q(seg);
      ++qn;
    }
    while (more) {
      const PxSeg cur = seg;
      more = px_next(seg, P) && find(seg);
      const int pages = cur.j1 - cur.j0, halves = cur.dup ? 1 : 2;
      float m = -CUDART_INF_F, l = 0.f;
      bool wild = false;
#pragma unroll 1
      for (int i = 0; i < pages; ++i) {
        ok = __all_sync(0xffffffffu, tc_wait(&S.sfull[x], n & 1u, &S.abort_));
        if (!ok) break;
        tc_fence_after();
        // the scores twice from TMEM, 64 columns at a time: for the maximum, then
        // for the exponentials (all 128 in registers made the loop bodies so long
        // that their first, cold pass cost 4 us)
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
        // the segment's S are all done with Q: the next segment's may come
        if (i == pages - 1 && more) {
          load_q(seg);
          ++qn;
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
        unsigned long long ls[2] = {0ULL, 0ULL};     // (0.f, 0.f)
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
          TC_ST32(scol + 32u * c, pk);               // over columns that have been read
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        tc_arrive(&S.pfull[x]);
        float la, lb;
        unpair(add2(ls[0], ls[1]), la, lb);
        l += la + lb;
        ++n;
      }
      if (!ok) break;
      // ---- the segment's partial: 32 columns of the warp's rows at a time to
      // shared memory, and from there as one 4 KB bulk copy; in a row's 128 B
      // the 16-byte chunks are permuted by the row (no bank conflicts)
      ok = __all_sync(0xffffffffu, tc_wait(&S.oready[x], (n - 1) & 1u, &S.abort_));
      if (!ok) break;
      tc_fence_after();
      const int64_t at = slot_row(cur);
      unsigned char* stage = S.out[w];
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        uint32_t o[32];
        TC_LD32(o, ocol + 32u * q);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();                                // the last copy has read the buffer
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
              make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          // [slot][tile][32-column chunk][128 rows][32 floats]
          float* dst = P.pacc + ((at - r) * PX_D + (q * 128 + 32 * (w & 3)) * 32);
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                       :: "l"(dst), "r"(smem_addr(stage)), "r"(32u * 128u) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      tc_fence_before();
      P.pml[at * 2] = m;
      P.pml[at * 2 + 1] = l;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (!ok && r == 0) {
      // let the Q tiles asked for land before the CTA leaves
      for (uint32_t q = qn > 1 ? qn - 2 : 0u; q < qn; ++q) {
        int dummy = 0;
        tc_wait(&S.qfull[x], q & 1u, &dummy);
      }
    }
  }
  tc_fence_before();
  __syncthreads();                                   // every role is done
  if (t == 0 && S.abort_) atomicOr(A.status, 1);
}

// ---------------------------------------------------------------------------
// The rows' own ranges
// ---------------------------------------------------------------------------
// A CTA's run of (row, kv head, page) units as segments, walked identically
// by every role (row-major, kv head inner; OW_OVH virtual units in front of
// each (row, kv head)'s pages).
struct OwSeg {
  int b, h, tb, off, tt, t1, ncost, n, s0, s1;       // n pages; keys [s0, s1)
  int k0, kmax;                                      // the row's own range
};
__device__ __forceinline__ void ow_bounds(OwSeg& g) {
  g.ncost = min(g.tb - g.off, g.t1 - g.tt);
  const int r0 = max(g.off, OW_OVH) - OW_OVH, r1 = g.off + g.ncost - OW_OVH;
  g.n = max(r1 - r0, 0);
  g.s0 = g.k0 + r0 * SD_KV_PAGE;
  g.s1 = min(g.kmax, g.k0 + r1 * SD_KV_PAGE);
}
__device__ __forceinline__ bool ow_next(OwSeg& g, const PrefixParams& P) {
  const AttnParams& A = P.A;
  g.tt += g.ncost;
  if (g.tt >= g.t1) return false;
  g.off = 0;
  if (++g.h == A.Hkv) {
    g.h = 0;
    do { ++g.b; } while (A.rowpre[g.b + 1] == A.rowpre[g.b]);   // units remain, so a row follows
    g.tb = A.rowpre[g.b + 1] - A.rowpre[g.b];
    g.k0 = P.rowstart[g.b];
    g.kmax = A.rowkmax[g.b];
  }
  ow_bounds(g);
  return true;
}
// The current or next segment with pages; false when none is left.
__device__ __forceinline__ bool ow_real(OwSeg& g, const PrefixParams& P) {
  while (g.n == 0)
    if (!ow_next(g, P)) return false;
  return true;
}

struct OwSmem {
  alignas(1024) unsigned char k[OW_STAGES][2][128 * 128];    // [stage][64-col box][128 keys x 128 B]
  alignas(1024) unsigned char v[OW_STAGES][2][128 * 128];
  alignas(1024) unsigned char q[2][128 * 128];               // [64-col box][128 rows x 128 B]
  alignas(8) unsigned long long full[OW_STAGES][2], empty[OW_STAGES][2];   // K, V
  // by stream and the stream's page parity (at most two phases of each are open)
  alignas(8) unsigned long long sfull[4][2], pfull[4][2], oready[4][2], qfull[4], fin;
  int first[5];                                      // the CTA's first row: b, unit, tb, k0, kmax
  int abort_;
};
static_assert(sizeof(OwSmem) + 2048 <= 227 * 1024, "shared memory, with room to align");

// A row's first unit per kv head, the next one's, first key and end of its own range
__device__ __forceinline__ int4 ow_row(const PrefixParams& P, int b) {
  return make_int4(P.A.rowpre[b], P.A.rowpre[b + 1], P.rowstart[b], P.A.rowkmax[b]);
}

// Stream-K over the pages of all (row, kv head) segments.  A segment has at
// most 128 query rows and needs 1, 2 or 4 quarters of the 128 accumulator lanes
// (P.nq): 4 / nq segments are in work at once, each on its own quarters, its own
// warps and, by the lane masks of tcgen05.mma, its own part of every
// accumulator.  Per page:
//   S[lanes, 128 keys] = Q . K^T     (all lanes multiply, the segment's are written)
//   thread = query row = lane: scores in registers, lazy reference maximum,
//   p = 2^(s - m) as bf16 over the columns of S
//   O[lanes, 128 d] += P . V
// So a segment's start and end (Q, first maximum, partial out) overlap the
// pages of the next one, no reduction crosses a thread, and K and V are read
// once whatever the number of query rows.  The idle lanes cost tensor time that
// is not the bound: 1024 cycles a page against about 2600 for its 64 KB from HBM.
// K leaves its slot when S is done, V when P . V is; slots behind a row's live
// keys that TMA brings in are zeroed in V before P . V reads them (they may hold
// NaN).  64 rows of 5 queries and 520 own keys, 32 / 8 heads (136 MB): 45 us for the
// call, 34 as a launch of its own (4 TB/s); in its middle a page takes 2130 cycles,
// the bandwidth of HBM, but the first three pages of a CTA take 10 us (cold code and
// first loads), which so short a run does not hide.
__device__ __forceinline__ void own_ranges(const PrefixParams& P, const CUtensorMap& tmk,
                                           const CUtensorMap& tmv, const CUtensorMap& tmq,
                                           int4 totals, int4 row, int cta, int chunk,
                                           const uint32_t* tmem) {
  extern __shared__ __align__(1024) unsigned char px_raw[];
  const uint32_t pad = (1024u - (smem_addr(px_raw) & 1023u)) & 1023u;   // swizzle atoms: 1024 B
  OwSmem& S = *reinterpret_cast<OwSmem*>(px_raw + pad);
  const AttnParams& A = P.A;
  const int t = threadIdx.x, w = t >> 5, lane = t & 31;
  const int total = totals.x, share = totals.z;
  if ((int64_t)cta * share >= total) return;         // no work for this CTA (uniform)
  const int t0 = cta * share, t1 = t0 + min(total - t0, share);
  const int j0 = chunk * P.qc;                       // the chunk's first query
  const int R = min(P.qc, A.qlen - j0) * A.group;    // its query rows per kv head
  const int nq = P.nq, ns = 4 / nq;                  // quarters per segment, streams
  for (int b = t; b < A.B; b += PX_THREADS) {
    if (b != t) row = ow_row(P, b);
    if (row.x * A.Hkv <= t0 && t0 < row.y * A.Hkv) {
      S.first[0] = b;
      S.first[1] = row.x * A.Hkv;
      S.first[2] = row.y - row.x;
      S.first[3] = row.z;
      S.first[4] = row.w;
    }
  }
  if (t == 0) {
    for (int i = 0; i < OW_STAGES; ++i)
      for (int kv = 0; kv < 2; ++kv) {
        tc_bar_init(&S.full[i][kv], 1);
        tc_bar_init(&S.empty[i][kv], 1);
      }
    for (int i = 0; i < 4; ++i) {
      tc_bar_init(&S.qfull[i], nq);
      for (int p = 0; p < 2; ++p) {
        tc_bar_init(&S.sfull[i][p], 1);
        tc_bar_init(&S.pfull[i][p], 32 * nq);
        tc_bar_init(&S.oready[i][p], 1);
      }
    }
    tc_bar_init(&S.fin, 1);
    S.abort_ = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = *tmem;                         // S0, S1 (128 columns each), O (128)
  OwSeg seg;
  seg.b = S.first[0];
  seg.tb = S.first[2];
  seg.k0 = S.first[3];
  seg.kmax = S.first[4];
  seg.h = (t0 - S.first[1]) / seg.tb;
  seg.off = (t0 - S.first[1]) % seg.tb;
  seg.tt = t0;
  seg.t1 = t1;
  ow_bounds(seg);
  bool more = ow_real(seg, P);

  if (w == 4) {
    // ---------------- TMA producer: pages in segment order
    if (lane == 0) {
      // a row's own pages are read by nobody else: they go first from L2, so that
      // the shared ranges' partials stay in it for the join
      const uint64_t once = tc_evict_first();
      uint32_t gi = 0, tiles = 0;                    // pages, K and V tiles asked for
      bool ok = true;
      while (more && ok) {
        for (int i = 0; i < seg.n && ok; ++i, ++gi) {
          const int st = (int)(gi % OW_STAGES);
          const int y = (int)kv_row(A, seg.b, seg.h, seg.s0 + i * SD_KV_PAGE);
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv, ++tiles) {
            if (gi >= (uint32_t)OW_STAGES)
              ok = tc_wait(&S.empty[st][kv], ((gi / OW_STAGES) - 1) & 1u, &S.abort_);
            if (!ok) break;
            tc_expect_tx(&S.full[st][kv], 2u * 128u * 128u);
            const void* map = kv ? (const void*)&tmv : (const void*)&tmk;
            unsigned char* dst = kv ? S.v[st][0] : S.k[st][0];
            tc_tma_2d(dst, map, 0, y, &S.full[st][kv], once);
            tc_tma_2d(dst + 128 * 128, map, 64, y, &S.full[st][kv], once);
          }
        }
        if (ok) more = ow_next(seg, P) && ow_real(seg, P);
      }
      if (!ok) {
        // let the copies already issued land before the CTA leaves
        constexpr uint32_t RING = 2 * OW_STAGES;
        for (uint32_t q = tiles > RING ? tiles - RING : 0u; q < tiles; ++q) {
          int dummy = 0;
          tc_wait(&S.full[q / 2 % OW_STAGES][q & 1], (q / RING) & 1u, &dummy);
        }
      }
    }
  } else if (w == 5) {
    // ---------------- MMA issuer (the whole warp): S of page a and P . V of page c,
    // each in page order, polled together; S(a) behind P . V(a - 2), whose P it
    // overwrites
    constexpr uint32_t ID1 = tc_idesc(128, 128, 0, 0);     // S = Q . K^T
    constexpr uint32_t ID2 = tc_idesc(128, 128, 0, 1);     // O += P . V (V [key][d]: N-major)
    const uint64_t dq = tc_desc(smem_addr(S.q[0]), 16, 1024, 2);
    OwSeg sa = seg, sc = seg;
    bool ma = more, mc = more;
    int ia = 0, ic = 0;                            // page of the segment
    uint32_t a = 0, c = 0, ga = 0, gc = 0;         // pages and segments issued
    uint32_t na[4] = {0u, 0u, 0u, 0u}, nc[4] = {0u, 0u, 0u, 0u};   // pages by stream
    auto lanes = [&](uint32_t (&off)[4], uint32_t g) {
      const int q0 = (int)(g % ns) * nq;
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = i >= q0 && i < q0 + nq ? 0u : 0xFFFFFFFFu;
    };
    auto count = [&](uint32_t (&n)[4], int s, bool step) -> uint32_t {
      uint32_t v = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i == s) {
          v = n[i];
          if (step) ++n[i];
        }
      return v;
    };
    long long idle0 = clock64();
    while (mc) {
      bool progressed = false;
      if (ma && a < c + 2) {
        const int st = (int)(a % OW_STAGES), s = (int)(ga % ns);
        if (__all_sync(0xffffffffu, tc_test(&S.full[st][0], (a / OW_STAGES) & 1u) &&
                                        (ia != 0 || tc_test(&S.qfull[s], (ga / ns) & 1u)))) {
          tc_fence_after();
          uint32_t off[4];
          lanes(off, ga);
          const uint32_t n = count(na, s, true);
          const uint64_t dk = tc_desc(smem_addr(S.k[st][0]), 16, 1024, 2);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {           // 16 of 128 d: 32 B, the second box 16 KB on
            const uint64_t o = (uint64_t)((ks & 3) * 2 + (ks >> 2) * 1024);
            tc_mma_lanes_warp(tm + 128u * (a & 1u), dq + o, dk + o, ID1, off, ks > 0 ? 1 : 0);
          }
          tc_commit_warp(&S.sfull[s][n & 1u]);
          tc_commit_warp(&S.empty[st][0]);
          ++a;
          if (++ia == sa.n) {
            ia = 0;
            ++ga;
            ma = ow_next(sa, P) && ow_real(sa, P);
          }
          progressed = true;
        }
      }
      if (c < a) {
        const int st = (int)(c % OW_STAGES), s = (int)(gc % ns);
        const uint32_t n = count(nc, s, false);
        if (__all_sync(0xffffffffu, tc_test(&S.pfull[s][n & 1u], (n >> 1) & 1u) &&
                                        tc_test(&S.full[st][1], (c / OW_STAGES) & 1u))) {
          tc_fence_after();
          uint32_t off[4];
          lanes(off, gc);
          count(nc, s, true);
          const uint64_t dv = tc_desc(smem_addr(S.v[st][0]), 16384, 1024, 2);
          const uint32_t pa = tm + 128u * (c & 1u);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)             // 16 keys: 2 KB
            tc_mma_ts_lanes_warp(tm + 256u, pa + 8u * ks, dv + (uint64_t)(ks * 128), ID2, off,
                                 ic > 0 || ks > 0 ? 1 : 0);
          tc_commit_warp(&S.empty[st][1]);
          tc_commit_warp(&S.oready[s][n & 1u]);
          ++c;
          if (++ic == sc.n) {
            ic = 0;
            ++gc;
            mc = ow_next(sc, P) && ow_real(sc, P);
          }
          progressed = true;
        }
      }
      if (progressed) {
        idle0 = clock64();
      } else if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&S.abort_) ||
                                             clock64() - idle0 > TC_WAIT)) {
        *reinterpret_cast<volatile int*>(&S.abort_) = 1;
        break;
      }
    }
    // every MMA this warp issued has finished before the CTA leaves
    tc_commit_warp(&S.fin);
    int dummy = 0;
    tc_wait(&S.fin, 0u, &dummy);
  } else if (w < 4) {
    // ---------------- softmax warps: lane quarter w, query row r of the chunk
    const int s = w / nq, r = (w % nq) * 32 + lane;
    const uint32_t lcol = tm + ((uint32_t)(32 * w) << 16), ocol = lcol + 256u;
    const float sl2 = A.scale * 1.4426950408889634f;
    // the warp's 32 query rows (rows past the segment's compute what nobody reads)
    auto load_q = [&](int b, int h) {
      if (lane == 0) {
        const int y = (h * A.B + b) * A.R + j0 * A.group + (w % nq) * 32;
        tc_expect_tx(&S.qfull[s], 2u * 32u * 128u);
        tc_tma_2d(S.q[0] + 32 * w * 128, &tmq, 0, y, &S.qfull[s]);
        tc_tma_2d(S.q[1] + 32 * w * 128, &tmq, 64, y, &S.qfull[s]);
      }
    };
    uint32_t qn = 0;                                 // Q tiles asked for
    uint32_t gi = 0, n = 0;                          // pages before; the stream's pages done
    int g = 0;                                       // segment
    // this stream's first segment
    auto skip = [&]() {
      while (more && g % ns != s) {
        gi += (uint32_t)seg.n;
        more = ow_next(seg, P) && ow_real(seg, P);
        ++g;
      }
    };
    skip();
    if (more) {
      load_q(seg.b, seg.h);
      ++qn;
    }
    bool ok = true;
    while (more) {
      const OwSeg cur = seg;
      const uint32_t g0 = gi;
      // the stream's next segment
      gi += (uint32_t)seg.n;
      more = ow_next(seg, P) && ow_real(seg, P);
      ++g;
      skip();
      // the row's live keys (an idle lane sees all: its result goes nowhere)
      int lim = 0x7FFFFFFF;
      if (r < R) lim = row_limit(A, cur.b, j0 + r / A.group);
      float m = -CUDART_INF_F, l = 0.f;
      bool wild = false;
      for (int i = 0; i < cur.n; ++i, ++n) {
        ok = __all_sync(0xffffffffu, tc_wait(&S.sfull[s][n & 1u], (n >> 1) & 1u, &S.abort_));
        if (!ok) break;
        tc_fence_after();
        const uint32_t scol = lcol + 128u * ((g0 + (uint32_t)i) & 1u);
        const int key0 = cur.s0 + i * SD_KV_PAGE;
        if (key0 + SD_KV_PAGE > cur.s1 || !__all_sync(0xffffffffu, key0 + SD_KV_PAGE <= lim)) {
          // The last pages: keys past a row's limit to -inf, in TMEM, 32 columns at
          // a time (a short loop: this code is cold whenever it runs).
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int k0 = key0 + 32 * c;
            if (__all_sync(0xffffffffu, k0 + 32 <= lim)) continue;
            uint32_t x[32];
            TC_LD32(x, scol + 32u * c);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = k0 + e < lim ? x[e] : 0xFF800000u;
            TC_ST32(scol + 32u * c, x);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          // past the live window the page holds other slots, maybe NaN: their V to
          // zero, four rows of a 128-byte box at a time
          const uint32_t pg = g0 + (uint32_t)i, st = pg % OW_STAGES;
          ok = __all_sync(0xffffffffu, tc_wait(&S.full[st][1], (pg / OW_STAGES) & 1u, &S.abort_));
          if (!ok) break;
          for (int kr = cur.s1 - key0 + 4 * (w % nq) + (lane >> 3); kr < 128; kr += 4 * nq) {
            const int at = kr * 128 + (lane & 7) * 16;
            *reinterpret_cast<uint4*>(S.v[st][0] + at) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(S.v[st][1] + at) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        // the scores twice from TMEM, 64 columns at a time: for the maximum, then for
        // the exponentials (all 128 in registers are too many beside 320 threads)
        uint32_t sa[32], sb[32];
        float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          TC_LD32(sa, scol + 64u * c);
          TC_LD32(sb, scol + 64u * c + 32u);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            px_max3(mx[e & 2], sa[e], sa[e + 1]);
            px_max3(mx[(e & 2) + 1], sb[e], sb[e + 1]);
          }
        }
        // the segment's S are all done with Q: the next segment's may come
        if (i == cur.n - 1 && more) {
          load_q(seg.b, seg.h);
          ++qn;
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
            ok = __all_sync(0xffffffffu,
                            tc_wait(&S.oready[s][(n - 1) & 1u], ((n - 1) >> 1) & 1u, &S.abort_));
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
        unsigned long long ls[2] = {0ULL, 0ULL};     // (0.f, 0.f)
        uint32_t pk[32];
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          TC_LD32(sa, scol + 64u * c);
          TC_LD32(sb, scol + 64u * c + 32u);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if (wild) {
            px_scale(sa, sl2);
            px_scale(sb, sl2);
          }
          px_weights(sa, pk, ls, sl22, nm2);
          px_weights(sb, pk + 16, ls, sl22, nm2);
          TC_ST32(scol + 32u * c, pk);               // over columns that have been read
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        tc_arrive(&S.pfull[s][n & 1u]);
        float la, lb;
        unpair(add2(ls[0], ls[1]), la, lb);
        l += la + lb;
      }
      if (!ok) break;
      // ---- the segment's partial: slot (chunk, row * Hkv + head + CTA)
      ok = __all_sync(0xffffffffu,
                      tc_wait(&S.oready[s][(n - 1) & 1u], ((n - 1) >> 1) & 1u, &S.abort_));
      if (!ok) break;
      tc_fence_after();
      const int64_t at = ((int64_t)chunk * P.slots + cur.b * A.Hkv + cur.h + cta) *
                             (P.qc * A.group) + r;
      float4* dst = reinterpret_cast<float4*>(A.part_acc + at * PX_D);
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        uint32_t o[32];
        TC_LD32(o, ocol + 32u * q);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (r < R) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[8 * q + e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                         __uint_as_float(o[4 * e + 2]),
                                         __uint_as_float(o[4 * e + 3]));
        }
      }
      tc_fence_before();
      if (r < R) {
        A.part_ml[at * 2] = m;
        A.part_ml[at * 2 + 1] = l;
      }
    }
    if (!ok && lane == 0) {
      // let the Q tiles asked for land before the CTA leaves
      for (uint32_t q = qn > 1 ? qn - 2 : 0u; q < qn; ++q) {
        int dummy = 0;
        tc_wait(&S.qfull[s], q & 1u, &dummy);
      }
    }
  }
  tc_fence_before();
  __syncthreads();                                   // every role is done
  if (t == 0 && S.abort_) atomicOr(A.status, 1);
}

// Both ranges in one launch, of which every CTA waits for the plan by itself: as
// many CTAs as the shared ranges need take those, the next ones the own ranges, at
// once on the SMs that the shared ones leave idle, else as SMs run out of shared
// work (a CTA's shared memory fills an SM).  As two launches, whose second would have
// to wait for the first to see the plan, 2 rows and one shared page took 24.5 us
// instead of 16.4, a step of 32 rows, 16 / 8 heads, four shared pages and up to 300
// own keys 36.7 instead of 26.0.
__global__ void __launch_bounds__(PX_THREADS, 1)
prefix_tc_kernel(const __grid_constant__ PrefixParams P, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmq,
                 const __grid_constant__ CUtensorMap tmq32) {
  __shared__ uint32_t tmem;
  const int t = threadIdx.x, w = t >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (w == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_addr(&tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the plan and the packed queries
  // one round trip for all that the start needs: what groups and rows say is on
  // its way with the totals
  const int4 totals = *P.totals;
  int4 group = make_int4(0, 0, 0, 0), row = group;
  if (t < P.G) group = px_group(P, t);
  if (t < P.A.B) row = ow_row(P, t);
  const int i = (int)blockIdx.x - (totals.y + totals.w - 1) / totals.w;
  if (i < 0)
    shared_ranges(P, tmk, tmv, tmq, totals, group, &tmem);
  else if (i < PX_CTAS * P.chunks)
    own_ranges(P, tmk, tmv, tmq32, totals, row, i % PX_CTAS, i / PX_CTAS, &tmem);
  tc_fence_before();
  __syncthreads();                                   // nobody uses TMEM any more
  if (w == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 :: "r"(tmem), "r"(512u) : "memory");
  }
}

// A warp per query row: the pieces of the shared range and of the row's own range,
// in piece order.  Bound by latency (plan, then the partials): 10240 rows of some 6
// pieces (31 MB) in 6 us behind the own ranges, 14 from HBM.  Two rows per warp and
// eight pieces on their way were slower (more code, cold, and spills), as were 6 or
// 8 CTAs per SM.
__global__ void __launch_bounds__(PX_JOIN_THREADS, PX_JOIN_CTAS) prefix_join_kernel(const PrefixParams P) {
  const AttnParams& A = P.A;
  const int lane = threadIdx.x & 31;
  const int64_t q = (int64_t)blockIdx.x * (PX_JOIN_THREADS / 32) + (threadIdx.x >> 5);
  if (q >= (int64_t)A.B * A.Hkv * A.R) return;
  const int bh = (int)q / A.R, r = (int)q - bh * A.R, b = bh / A.Hkv, h = bh - b * A.Hkv;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // what the plan says: pieces [0, n1) are of the shared range, two per CTA where
  // both tiles worked on the rows; [n1, np) of the row's own range.  Rows of partials in 32 bits: each
  // is 512 bytes of memory.
  const int status = *A.status;
  const int4 totals = *P.totals;
  const int4 j0 = P.rowjoin[2 * b], j1 = P.rowjoin[2 * b + 1];
  const PxRow row = {j0.x, j0.y, j0.z, j0.w, j1.x, j1.y, j1.z, 0};
  const int tb = row.tb, RC = P.qc * A.group, oshare = totals.z, gshare = totals.w;
  const int ou = row.pre * A.Hkv + h * tb, oc0 = (ou + OW_OVH) / oshare, jc = r / RC;
  const int at2 = (jc * P.slots + bh + oc0) * RC + r - jc * RC;
  int n1 = 0, dup = 0, at1 = 0;
  if (row.rows > 0) {
    const int rows = row.rows * A.R, gtb = row.pages + PX_OVH;
    const int f = row.place * A.R + r, p = f / PX_ROWS;
    const int it = h * ((rows + PX_ROWS - 1) / PX_ROWS) + p, u = row.unit + it * gtb;
    const int c0 = (u + PX_OVH) / gshare;
    dup = rows - p * PX_ROWS <= PX_ROWS / 2;
    n1 = ((u + gtb - 1) / gshare - c0 + 1) << dup;
    at1 = (row.item + it + c0) * PX_ROWS + f % PX_ROWS;
  }
  const int np = n1 + (tb > 0 ? (ou + tb - 1) / oshare - oc0 + 1 : 0);
  auto row_of = [&](int i) {
    return i < n1 ? at1 + (i >> dup) * PX_ROWS + (dup & i) * (PX_ROWS / 2) : at2 + (i - n1) * RC;
  };
  // this lane's 4 columns of a partial row: in the shared range's tiles column
  // chunk lane / 8, row, and the 16-byte chunk permuted by the row
  float4 v[PX_JOIN_LOADS];
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < PX_JOIN_LOADS; ++i) {
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + i >= np) continue;
      const int row = row_of(i0 + i), tr = row & 127;
      const bool own = i0 + i >= n1;
      const int64_t at = (int64_t)(own ? row : row - tr) * 32 +
                         (own ? lane : ((lane >> 3) * 128 + tr) * 8 + ((lane & 7) ^ (tr & 7)));
      v[i] = __ldcg(reinterpret_cast<const float4*>(own ? A.part_acc : P.pacc) + at);
    }
  };
  auto ml_of = [&](int i) {
    return __ldcg(reinterpret_cast<const float2*>(i < n1 ? P.pml : A.part_ml) + row_of(i));
  };
  load(0);                                           // on their way before their weights are known
  float m = -CUDART_INF_F, l = 0.f, m0 = -CUDART_INF_F;        // per lane, then over the warp
  bool nan = false;                                  // a NaN score leaves no maximum, but its sum
  for (int i = lane; i < np; i += 32) {
    const float2 ml = ml_of(i);
    if (i == lane) m0 = ml.x;
    nan |= ml.y != ml.y;
    if (ml.x != -CUDART_INF_F) {
      const float mn = fmaxf(m, ml.x);
      l = (m == -CUDART_INF_F ? 0.f : l * ex2f(m - mn)) + ml.y * ex2f(ml.x - mn);
      m = mn;
    }
  }
  const float gm = warp_max(m);
  const float L = warp_sum(m == -CUDART_INF_F ? 0.f : l * ex2f(m - gm));
  float fw = m0 == -CUDART_INF_F ? 0.f : ex2f(m0 - gm);        // piece lane's weight
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = 0; i0 < np; i0 += PX_JOIN_LOADS) {
    if (i0 > 0) {
      load(i0);
      if (i0 % 32 == 0) {
        const float mi = i0 + lane < np ? ml_of(i0 + lane).x : -CUDART_INF_F;
        fw = mi == -CUDART_INF_F ? 0.f : ex2f(mi - gm);
      }
    }
#pragma unroll
    for (int i = 0; i < PX_JOIN_LOADS; ++i) {
      const float f = __shfl_sync(0xffffffffu, fw, (i0 & 31) + i);
      if (f == 0.f) continue;                        // nothing there (maybe never written)
      a.x = fmaf(f, v[i].x, a.x); a.y = fmaf(f, v[i].y, a.y);
      a.z = fmaf(f, v[i].z, a.z); a.w = fmaf(f, v[i].w, a.w);
    }
  }
  // a wait that gave up somewhere leaves partials unwritten: say so in the output
  nan = __any_sync(0xffffffffu, nan);
  const float il = nan || status ? CUDART_NAN_F : L == 0.f ? 0.f : 1.f / L;
  const int j = r / A.group, hq = h * A.group + r - j * A.group;
  const __nv_bfloat162 y0 = __floats2bfloat162_rn(a.x * il, a.y * il);
  const __nv_bfloat162 y1 = __floats2bfloat162_rn(a.z * il, a.w * il);
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(A.out) + b * A.obs + j * A.oqs +
                       hq * A.ohs + 4 * lane;
  if (A.out_vec4) {
    uint2 pk;
    pk.x = *reinterpret_cast<const uint32_t*>(&y0);
    pk.y = *reinterpret_cast<const uint32_t*>(&y1);
    *reinterpret_cast<uint2*>(dst) = pk;
  } else {
    dst[0] = y0.x; dst[1] = y0.y; dst[2] = y1.x; dst[3] = y1.y;
  }
}

// The shapes of the tensor-core path; every other shape reads each row's pages
// by itself (bound by its arithmetic, not by the bytes that sharing saves).
static bool px_fast(int dtype, int D, int group) {
  return dtype == SD_DTYPE_BF16 && D == PX_D && group <= 128;
}

struct PxLayout {
  size_t ints, qp, acc, ml, sacc, sml, bytes;
  int max_items, qc, nq, chunks, slots;
};
static PxLayout px_layout(int B, int G, int Hq, int Hkv, int qlen) {
  PxLayout L;
  const int group = Hq / Hkv, R = qlen * group;
  // a group of two rows or more shares: no more than B / 2 of them
  L.max_items = (int)std::min<int64_t>(
      (int64_t)Hkv * ((int64_t)B * R / PX_ROWS + std::min(G, B / 2)), 1 << 28);
  L.qc = std::min(qlen, 128 / group);
  L.nq = L.qc * group <= 32 ? 1 : L.qc * group <= 64 ? 2 : 4;
  L.chunks = (qlen + L.qc - 1) / L.qc;
  L.slots = B * Hkv + PX_CTAS;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t n1 = (size_t)(L.max_items + PX_CTAS) * PX_ROWS;
  const size_t n2 = (size_t)L.chunks * L.slots * L.qc * group;
  size_t o = up((8 * (size_t)B + 4 + 5 * (size_t)G + 2 + 3 * (size_t)B + 2) * sizeof(int));
  L.ints = 0;
  L.qp = o; o = up(o + (size_t)B * Hq * qlen * PX_D * 2);
  L.acc = o; o = up(o + n1 * PX_D * sizeof(float));
  L.ml = o; o = up(o + n1 * 2 * sizeof(float));
  L.sacc = o; o = up(o + n2 * PX_D * sizeof(float));
  L.sml = o; o = up(o + n2 * 2 * sizeof(float));
  L.bytes = o;
  return L;
}

}  // namespace sd

using namespace sd;

extern "C" {

size_t sd_prefix_attn_workspace_bytes(int B, int G, int Hq, int Hkv, int D, int W, int qlen,
                                      int dtype) {
  if (B <= 0 || G < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || W <= 0 || qlen <= 0) return 0;
  if ((int64_t)W * SD_KV_PAGE > 0x7FFFFFFF) return 0;
  if (!px_fast(dtype, D, Hq / Hkv)) return 0;
  return px_layout(B, G, Hq, Hkv, qlen).bytes;
}

int sd_prefix_attn(const void* q, int64_t qbs, int64_t qhs, int64_t qqs, const void* kpool,
                   const void* vpool, const int32_t* block_table, int bt_stride, int npages,
                   const int64_t* lengths, const int64_t* valid, const int32_t* group_starts,
                   const int32_t* prefix_pages, int G, int B, int Hq, int Hkv, int D, int qlen,
                   float scale, void* out, int64_t obs, int64_t oqs, int64_t ohs, int dtype,
                   void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || G < 0 || qlen < 0) return SD_EINVAL;
  if (B == 0 || qlen == 0) return SD_OK;
  if (!q || !kpool || !vpool || !block_table || !lengths || !out) return SD_EINVAL;
  if (G > 0 && (!group_starts || !prefix_pages)) return SD_EINVAL;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || bt_stride <= 0 || npages <= 0) return SD_EINVAL;
  if (!(scale > 0.f) || scale > 3e38f) return SD_EINVAL;
  if (dtype != SD_DTYPE_BF16 && dtype != SD_DTYPE_F32) return SD_ENOTSUP;
  if ((int64_t)bt_stride * SD_KV_PAGE > 0x7FFFFFFF) return SD_ENOTSUP;
  const int group = Hq / Hkv;
  const int64_t R = (int64_t)qlen * group;
  if (R > 0x7FFFFFFF) return SD_ENOTSUP;
  PrefixParams P = {};
  AttnParams& A = P.A;
  A.q = q; A.qbs = qbs; A.qhs = qhs; A.qqs = qqs;
  A.k = kpool; A.v = vpool; A.lengths = lengths; A.valid = valid;
  A.B = B; A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.C = bt_stride * SD_KV_PAGE; A.qlen = qlen;
  A.group = group; A.R = (int)R; A.scale = scale;
  A.out = out; A.obs = obs; A.oqs = oqs; A.ohs = ohs;
  A.out_vec4 = (reinterpret_cast<uintptr_t>(out) & 7) == 0 && obs % 4 == 0 && oqs % 4 == 0 &&
               ohs % 4 == 0;
  A.bt = block_table; A.bt_stride = bt_stride; A.npages = npages;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!px_fast(dtype, D, group)) return prefix_rows(A, dtype, st);
  // 16-byte loads of q rows and TMA boxes of the pools
  if ((reinterpret_cast<uintptr_t>(q) & 15) || qbs % 8 || qhs % 8 || qqs % 8 ||
      (reinterpret_cast<uintptr_t>(kpool) & 15) || (reinterpret_cast<uintptr_t>(vpool) & 15))
    return SD_EINVAL;
  const int64_t rows = (int64_t)npages * Hkv * SD_KV_PAGE;
  if (rows >= (int64_t)1 << 31) return SD_ENOTSUP;
  // the schedules count units in 32 bits
  if (R * B * Hkv > 0x7FFFFFFF || (int64_t)B * Hkv * (bt_stride + OW_OVH) > 0x7FFFFFFF ||
      (int64_t)Hkv * (B * R / PX_ROWS + G) * (bt_stride + PX_OVH) > 0x7FFFFFFF)
    return SD_ENOTSUP;
  const PxLayout L = px_layout(B, G, Hq, Hkv, qlen);
  if (L.chunks > 65535) return SD_ENOTSUP;           // a grid dimension
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < L.bytes)
    return SD_ENOSPC;
  char* ws = reinterpret_cast<char*>(workspace);
  P.qc = L.qc; P.nq = L.nq; P.chunks = L.chunks; P.slots = L.slots;
  P.starts = group_starts; P.pages = prefix_pages; P.G = G; P.max_items = L.max_items;
  int* in = reinterpret_cast<int*>(ws + L.ints);
  P.rowjoin = reinterpret_cast<int4*>(in); in += 8 * (size_t)B;
  P.totals = reinterpret_cast<int4*>(in); in += 4;
  P.g_unit = in; in += G + 1;
  P.g_item = in; in += G + 1;
  P.g_row0 = in; in += G;
  P.g_rows = in; in += G;
  P.g_pages = in; in += G;
  P.rowstart = in; in += B;
  A.rowkmax = in; in += B;
  A.rowpre = in; in += B + 1;
  A.status = in;
  P.qp = reinterpret_cast<uint4*>(ws + L.qp);
  P.pacc = reinterpret_cast<float*>(ws + L.acc);
  P.pml = reinterpret_cast<float*>(ws + L.ml);
  A.part_acc = reinterpret_cast<float*>(ws + L.sacc);
  A.part_ml = reinterpret_cast<float*>(ws + L.sml);
  const int64_t qrows = (int64_t)B * Hq * qlen;
  CUtensorMap mk, mv, mq, mq32;
  if (!cache_map(&mk, kpool, rows) || !cache_map(&mv, vpool, rows) ||
      !cache_map(&mq, P.qp, qrows) || !cache_map(&mq32, P.qp, qrows, 32))
    return SD_ENOTSUP;
  const int sm = (int)std::max(sizeof(PxSmem), sizeof(OwSmem)) + 1024;           // room to align
  static std::atomic<uint64_t> ready{0};             // devices whose kernels may use that much
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SD_ELAUNCH;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load() & bit) || !bit) {
    if (cudaFuncSetAttribute(prefix_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) !=
        cudaSuccess)
      return SD_ELAUNCH;
    ready.fetch_or(bit);
  }
  const int64_t pack = (qrows * 16 + PX_PLAN_THREADS - 1) / PX_PLAN_THREADS;
  prefix_plan_kernel<<<(unsigned)(1 + pack), PX_PLAN_THREADS, 0, st>>>(P);
  if (cudaGetLastError() != cudaSuccess) return SD_ELAUNCH;
  // the others as programmatic dependents: launched while the one before runs
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3(PX_CTAS * ((unsigned)L.chunks + (G > 0 ? 1 : 0)));
  cfg.blockDim = dim3(PX_THREADS);
  cfg.dynamicSmemBytes = sm;
  if (cudaLaunchKernelEx(&cfg, prefix_tc_kernel, P, mk, mv, mq, mq32) != cudaSuccess)
    return SD_ELAUNCH;
  const int64_t per = PX_JOIN_THREADS / 32;          // query rows of a CTA
  cfg.gridDim = dim3((unsigned)((R * B * Hkv + per - 1) / per));
  cfg.blockDim = dim3(PX_JOIN_THREADS);
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, prefix_join_kernel, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // extern "C"
