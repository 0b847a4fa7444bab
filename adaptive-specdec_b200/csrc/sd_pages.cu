// The page table of a paged KV cache kept on the device (sm_100a): pages by
// request lengths, the slots of the new tokens, pages back after a rollback.
//
// Row b holds `owned[b]` pages in block_table[b, 0..owned[b]), the first
// shared[b] of which belong to somebody else too (a prompt that several rows
// read) and are never given back by the row.  Free pages are a stack: pages
// free[0..n_free).  With PAGE = 128 slots per page:
//   reserve: need_b = ceil((lengths[b] + new[b]) / PAGE); the o-th missing
//            page over all rows, in row-major order, is free[n_free - 1 - o];
//            slot of token i of row b = block_table[b, p / PAGE] * PAGE +
//            p % PAGE with p = lengths[b] + i, packed over the rows
//   trim:    keep_b = max(ceil(lengths[b] / PAGE), shared[b]); the o-th page
//            past the rows' keeps (of F) goes to free[n_free + F - 1 - o], so
//            a trim undoes a reserve to the entry
// A call that cannot be done for every row (a row past its table, too few
// free pages, too small a slot array, a new token in one of a row's first
// floor[b] pages) changes nothing but *err.
//
// Bytes are few; what bounds these calls is launches and the scan over the
// rows (pages and tokens packed in one 64-bit sum).  A reserve is a scan by one
// CTA and a second launch (programmatic dependent) with a warp per (row, run of
// tokens); for few tokens the scanning CTA does the second part too.  A trim is
// one cluster of CTAs: every CTA scans all rows, and behind a cluster barrier
// (all have read the state that is about to change) moves the pages of its
// share of the rows, a warp each.
#include <cuda_runtime.h>

#include <algorithm>

#include "sd_common.cuh"

namespace sd {

constexpr int PT_THREADS = 1024;
constexpr int PT_CLUSTER = 8;
// (row, run) pairs up to which the scanning CTA fills the slots itself: a launch
// less for the host, and on the device, in a CUDA graph, 3.9 us against 4.6 for
// 8 rows of 5 tokens, 5.4 against 5.0 for 64, 7.0 against 5.0 for 128.  Rows from
// which a trim takes a cluster: 3.0 us by one CTA against 3.8 by eight for 16
// rows; a trim and a reserve of 128 rows 10.3 against 9.6, of 512 rows 22 against
// 10.1 (512 rows that give back and take 32 pages each: 15 us, 2 M slots).
constexpr int PT_FUSED_WARPS = 64;
constexpr int PF_THREADS = 256;

struct PagesParams {
  int32_t* bt;
  int64_t bt_stride;
  int W, n_pages, B;
  int32_t* owned;
  const int32_t* shared;
  int32_t* free_stack;
  int32_t* n_free;
  const int64_t* lengths;
  const int64_t* add;                           // new tokens per row, or nullptr: add_all each
  int64_t add_all;
  const int32_t* floor;                         // pages per row that take no new tokens, or nullptr
  int64_t* slots;
  int64_t max_tokens;
  int32_t* starts;                              // [B + 1]
  int* err;
  int* plan;                                    // workspace: pages before row b [B], had [B], n_free, ok
  int run, runs;                                // tokens per warp of the fill, warps per row
  bool fused;                                   // the scanning CTA fills
};

// Warp w of warps: the slots of a row's tokens [run * P.run, ...) and, for run 0,
// its new table entries; the warps past the rows fill the slots behind the last
// token with -1.
__device__ __forceinline__ void reserve_fill(const PagesParams& P, const int* plan,
                                             const int32_t* starts, int64_t w, int64_t warps) {
  const int lane = threadIdx.x & 31;
  const bool ok = plan[2 * P.B + 1] != 0;
  const int top = plan[2 * P.B] - 1;
  const int64_t rows = (int64_t)P.B * P.runs;
  if (w >= rows) {
    const int64_t first = ok ? starts[P.B] : 0;
    for (int64_t i = first + (w - rows) * 32 + lane; i < P.max_tokens; i += (warps - rows) * 32)
      P.slots[i] = -1;
    return;
  }
  if (!ok) return;
  const int b = (int)(w / P.runs), run = (int)(w % P.runs);
  const int64_t len = P.lengths[b];
  const int s0 = starts[b], n = starts[b + 1] - s0;
  const int pre = plan[b], had = plan[P.B + b];
  int32_t* row = P.bt + b * P.bt_stride;
  if (run == 0) {
    const int need = (int)((len + n + SD_KV_PAGE - 1) / SD_KV_PAGE);
    for (int p = had + lane; p < need; p += 32) row[p] = P.free_stack[top - (pre + p - had)];
  }
  if (!P.slots) return;
  const int i1 = (int)min((int64_t)n, (int64_t)(run + 1) * P.run);
  for (int i = run * P.run + lane; i < i1; i += 32) {
    const int64_t pos = len + i;
    const int p = (int)(pos / SD_KV_PAGE);
    const int page = p < had ? row[p] : P.free_stack[top - (pre + p - had)];
    P.slots[(int64_t)s0 + i] =
        page < 0 ? -1 : (int64_t)page * SD_KV_PAGE + (pos & (SD_KV_PAGE - 1));
  }
}

__global__ void __launch_bounds__(PT_THREADS) pages_reserve_plan_kernel(const PagesParams P) {
  __shared__ long long red[33];
  __shared__ int bad;
  __shared__ int own_plan[2 * PT_FUSED_WARPS + 2], own_starts[PT_FUSED_WARPS + 1];
  int* plan = P.fused ? own_plan : P.plan;
  int32_t* starts = P.fused ? own_starts : P.starts;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x;
  if (t == 0) bad = 0;
  __syncthreads();
  long long carry = 0;
  for (int b0 = 0; b0 < P.B; b0 += PT_THREADS) {
    const int b = b0 + t;
    long long v = 0;
    if (b < P.B) {
      const int64_t len = P.lengths[b], add = P.add ? P.add[b] : P.add_all;
      const int had = P.owned[b];
      const int64_t cap = (int64_t)P.W * SD_KV_PAGE;
      int why = 0;
      if (len < 0 || add < 0 || len > cap || add > cap - len || had < 0) {
        why = SD_PAGES_ERR_CAPACITY;
      } else {
        const int64_t need = (len + add + SD_KV_PAGE - 1) / SD_KV_PAGE;
        v = (add & 0xFFFFFFFFLL) | ((need > had ? need - had : 0) << 32);
      }
      if (!why && P.floor && add > 0 && len < (int64_t)P.floor[b] * SD_KV_PAGE)
        why = SD_PAGES_ERR_SHARED;
      if (why) atomicOr(&bad, why);
      plan[P.B + b] = had;
    }
    long long sum;
    // (tokens in the low 32 bits, pages above)
    const long long ex = carry + block_excl_scan<long long>(v, red, &sum);
    carry += sum;
    if (b < P.B) {
      starts[b] = (int32_t)(ex & 0xFFFFFFFFLL);
      plan[b] = (int32_t)(ex >> 32);
    }
    __syncthreads();
  }
  const long long tokens = carry & 0xFFFFFFFFLL, pages = carry >> 32;
  const int had_free = *P.n_free;
  if (t == 0) starts[P.B] = (int32_t)tokens;
  int why = bad;
  if (had_free < 0 || had_free > P.n_pages) why |= SD_PAGES_ERR_CAPACITY;   // a broken table
  if (!why && pages > had_free) why = SD_PAGES_ERR_EXHAUSTED;
  if (!why && P.slots && tokens > P.max_tokens) why = SD_PAGES_ERR_SLOTS;
  __syncthreads();                                   // everybody has read n_free
  if (t == 0) {
    plan[2 * P.B] = had_free;
    plan[2 * P.B + 1] = why == 0;
    if (why)
      atomicOr(P.err, why);
    else
      *P.n_free = had_free - (int)pages;
  }
  if (!why) {
    for (int b = t; b < P.B; b += PT_THREADS) {
      const int64_t add = P.add ? P.add[b] : P.add_all;
      const int need = (int)((P.lengths[b] + add + SD_KV_PAGE - 1) / SD_KV_PAGE);
      if (need > plan[P.B + b]) P.owned[b] = need;
    }
  }
  if (!P.fused) return;
  __syncthreads();                                   // plan and starts, for the CTA's other warps
  for (int b = t; b <= P.B; b += PT_THREADS) P.starts[b] = starts[b];
  const int64_t n = (int64_t)P.B * P.runs + PT_THREADS / 32;     // the last 32: slots behind
  for (int64_t w = t >> 5; w < n; w += PT_THREADS / 32) reserve_fill(P, plan, starts, w, n);
}

__global__ void __launch_bounds__(PF_THREADS) pages_reserve_fill_kernel(const PagesParams P) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  reserve_fill(P, P.plan, P.starts, (int64_t)blockIdx.x * (PF_THREADS / 32) + (threadIdx.x >> 5),
               (int64_t)gridDim.x * (PF_THREADS / 32));
}

// The barrier of the launch's only cluster (or CTA).
__device__ __forceinline__ void grid_barrier() {
  if (gridDim.x > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
}

// Every CTA of the cluster: the rows' keeps and their scan, PT_THREADS rows at a
// time; then its warps move the pages of their share of those rows.
__global__ void __launch_bounds__(PT_THREADS) pages_trim_kernel(const PagesParams P) {
  __shared__ int red[33];
  __shared__ int pre[PT_THREADS], keep[PT_THREADS], had[PT_THREADS];
  const int t = threadIdx.x, lane = t & 31;
  const int gw = (int)blockIdx.x * (PT_THREADS / 32) + (t >> 5);       // warp of the cluster
  const int nw = (int)gridDim.x * (PT_THREADS / 32);
  const int had_free = *P.n_free;
  auto keep_of = [&](int b) {
    const int64_t len = max(P.lengths[b], (int64_t)0);
    return max((len + SD_KV_PAGE - 1) / SD_KV_PAGE, (int64_t)P.shared[b]);
  };
  // all pages first: where the stack will end decides where each page goes
  int mine = 0;
  for (int b = t; b < P.B; b += PT_THREADS)
    mine += (int)max(min(P.owned[b], P.W) - keep_of(b), (int64_t)0);
  const int all = block_sum<int>(mine, red);
  grid_barrier();                                    // everybody has read owned and n_free
  // more pages than there are: a broken table
  if (had_free < 0 || all < 0 || all > P.n_pages - had_free) {
    if (gw == 0 && lane == 0) atomicOr(P.err, SD_PAGES_ERR_CAPACITY);
    return;
  }
  int carry = 0;
  for (int b0 = 0; b0 < P.B; b0 += PT_THREADS) {
    const int b = b0 + t;
    int gone = 0, o = 0, k32 = 0;
    if (b < P.B) {
      o = min(P.owned[b], P.W);
      k32 = (int)min(keep_of(b), (int64_t)o);
      gone = o - k32;
    }
    int sum;
    const int ex = block_excl_scan<int>(gone, red, &sum);
    pre[t] = carry + ex;
    keep[t] = k32;
    had[t] = o;
    carry += sum;
    grid_barrier();                                  // these rows' state has been read by all
    const int nb = min(PT_THREADS, P.B - b0);
    for (int q = gw; q < nb; q += nw) {
      const int k = keep[q], h = had[q];
      int32_t* row = P.bt + (int64_t)(b0 + q) * P.bt_stride;
      for (int p = k + lane; p < h; p += 32) {
        P.free_stack[had_free + all - 1 - (pre[q] + p - k)] = row[p];
        row[p] = -1;
      }
      if (lane == 0 && k < h) P.owned[b0 + q] = k;
    }
    __syncthreads();                                 // pre, keep and had are rewritten next
  }
  if (gw == 0 && lane == 0) *P.n_free = had_free + all;
}

static int pages_check(const PagesParams& P) {
  if (P.B < 0) return SD_EINVAL;
  if (P.B == 0) return SD_OK;
  if (!P.bt || !P.owned || !P.free_stack || !P.n_free || !P.lengths || !P.err) return SD_EINVAL;
  if (P.W <= 0 || P.bt_stride < P.W || P.n_pages <= 0) return SD_EINVAL;
  if ((int64_t)P.W * SD_KV_PAGE > 0x7FFFFFFF) return SD_ENOTSUP;
  // a trim counts the rows' pages in 32 bits before it compares them with the pool
  if ((int64_t)P.B * P.W > 0x7FFFFFFF) return SD_ENOTSUP;
  return SD_OK;
}

}  // namespace sd

using namespace sd;

extern "C" {

size_t sd_pages_workspace_bytes(int B) {
  return B <= 0 ? 0 : (2 * (size_t)B + 2) * sizeof(int);
}

int sd_pages_reserve(int32_t* block_table, int bt_stride, int W, int32_t* owned,
                     const int32_t* free_stack, int n_pages, int32_t* n_free,
                     const int64_t* lengths, const int64_t* new_tokens, int64_t new_each,
                     const int32_t* floor_pages, int B, int64_t* slots, int64_t max_tokens, int32_t* starts,
                     int* err, void* workspace, size_t workspace_bytes, void* stream) {
  PagesParams P = {};
  P.bt = block_table; P.bt_stride = bt_stride; P.W = W; P.n_pages = n_pages; P.B = B;
  P.owned = owned; P.free_stack = const_cast<int32_t*>(free_stack); P.n_free = n_free;
  P.lengths = lengths; P.add = new_tokens; P.add_all = new_each;
  P.floor = floor_pages;
  P.slots = slots; P.max_tokens = slots ? max_tokens : 0; P.starts = starts; P.err = err;
  P.plan = reinterpret_cast<int*>(workspace);
  if (int rc = pages_check(P)) return rc;
  if (B == 0) return SD_OK;
  if (!starts || max_tokens < 0) return SD_EINVAL;
  if (!new_tokens && new_each < 0) return SD_EINVAL;
  if (max_tokens > 0x7FFFFFFF) return SD_ENOTSUP;
  // starts is int32, and the scan packs the token count in 32 bits
  if ((int64_t)B * W * SD_KV_PAGE > 0x7FFFFFFF) return SD_ENOTSUP;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
      workspace_bytes < sd_pages_workspace_bytes(B))
    return SD_ENOSPC;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t most = std::min<int64_t>(
      std::min<int64_t>(P.max_tokens, (int64_t)W * SD_KV_PAGE), new_tokens ? P.max_tokens : new_each);
  // tokens per warp: 512, or as many as leave 65536 warps (at least one per row)
  const int64_t cuts = std::max<int64_t>(1, 65536 / B);
  P.run = (int)std::max<int64_t>(512, (most + cuts - 1) / cuts);
  P.runs = (int)std::max<int64_t>(1, (most + P.run - 1) / P.run);
  P.fused = (int64_t)B * P.runs <= PT_FUSED_WARPS && P.max_tokens <= PT_FUSED_WARPS * 32;
  // some warps for the slots behind the last token
  const int64_t tail = (P.max_tokens + 4095) / 4096;
  const int64_t warps = (int64_t)B * P.runs + std::min<int64_t>(std::max<int64_t>(tail, 1), 1024);
  pages_reserve_plan_kernel<<<1, PT_THREADS, 0, st>>>(P);
  if (cudaGetLastError() != cudaSuccess) return SD_ELAUNCH;
  if (P.fused) return SD_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((warps + PF_THREADS / 32 - 1) / (PF_THREADS / 32)));
  cfg.blockDim = dim3(PF_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, pages_reserve_fill_kernel, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

int sd_pages_trim(int32_t* block_table, int bt_stride, int W, int32_t* owned,
                  const int32_t* shared, int32_t* free_stack, int n_pages, int32_t* n_free,
                  const int64_t* lengths, int B, int* err, void* stream) {
  PagesParams P = {};
  P.bt = block_table; P.bt_stride = bt_stride; P.W = W; P.n_pages = n_pages; P.B = B;
  P.owned = owned; P.shared = shared; P.free_stack = free_stack; P.n_free = n_free;
  P.lengths = lengths; P.err = err;
  if (int rc = pages_check(P)) return rc;
  if (B == 0) return SD_OK;
  if (!shared) return SD_EINVAL;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B > 2 * PT_THREADS / 32 ? PT_CLUSTER : 1);
  cfg.blockDim = dim3(PT_THREADS);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, pages_trim_kernel, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // extern "C"
