// Trees of drafted tokens (sm_100a): ancestor bits, the accepted path, and the
// cache behind it.  The host entry of tree attention is sd_tree_attn.cu's.
//
// A path p_0 = 0 < p_1 < ... of nodes (p_j >= j) becomes the row's next tokens:
// the K and V of slot base + p_j move to slot base + j in every layer.  A thread
// takes one 16-byte column of a (row, buffer, kv head) along the whole path, in
// order, so source p_j is read before any later step writes slot p_j, and no two
// threads touch the same bytes: the move is done in place, in one pass.  What it
// has to move is tiny, so it is bound by the latency of its chain: path, page,
// K / V, store.  Accept, move and lengths take 9.2 us in a graph for 32 rows and 36 layers
// (19 MB read and written), 13.4 us for 64 rows and up to 8 nodes (76 MB).
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "sd_common.cuh"
#include "sd_tree.cuh"

namespace sd {

constexpr int TREE_WORDS = SD_TREE_MAX / 32;
constexpr int COMMIT_THREADS = 128;
constexpr int COMMIT_BUFS = 256;             // buffers of one launch (their addresses are parameters)
constexpr int COMMIT_AHEAD = 8;              // path nodes whose loads are on their way at once

// One CTA per tree, one thread per node: up the parents, a bit for each.
__global__ void __launch_bounds__(SD_TREE_MAX)
tree_masks_kernel(const int32_t* __restrict__ parents, int64_t parents_bs, int N, int W,
                  int32_t* masks, int32_t* depths) {
  __shared__ int par[SD_TREE_MAX];
  const int t = threadIdx.x, tr = blockIdx.x;
  for (int i = t; i < N; i += blockDim.x) {
    const int p = parents[tr * parents_bs + i];
    par[i] = p < -1 || p >= i ? -2 : p;
  }
  __syncthreads();
  for (int i = t; i < N; i += blockDim.x) {
    uint32_t bits[TREE_WORDS];
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w) bits[w] = 0u;
    int a = i, depth = -1;
    while (a >= 0) {                                 // (a falls: at most N steps)
#pragma unroll
      for (int w = 0; w < TREE_WORDS; ++w)
        if (w == a >> 5) bits[w] |= 1u << (a & 31);
      ++depth;
      a = par[a];
    }
    const bool absent = a == -2;
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w)
      if (w < W) masks[((int64_t)tr * N + i) * W + w] = absent ? 0 : (int32_t)bits[w];
    if (depths) depths[(int64_t)tr * N + i] = absent ? 0 : depth;
  }
}

// A warp per row.
__global__ void __launch_bounds__(32)
tree_accept_kernel(const int64_t* __restrict__ tokens, int64_t tokens_bs,
                   const int64_t* __restrict__ choices, int64_t choices_bs,
                   const int32_t* __restrict__ masks, int64_t mask_bs,
                   const uint8_t* __restrict__ alive, int N, int W, int max_path, int32_t* path,
                   int64_t* n_acc, int64_t* y) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int64_t* tok = tokens + b * tokens_bs;
  const int64_t* cho = choices + b * choices_bs;
  // node lane + 32 q: its token, and its parent (the highest bit below it)
  int64_t mine[TREE_WORDS];
  int par[TREE_WORDS];
#pragma unroll
  for (int q = 0; q < TREE_WORDS; ++q) {
    const int i = lane + 32 * q;
    mine[q] = 0;
    par[q] = -1;
    if (i < N) {
      mine[q] = tok[i];
      const int32_t* m = masks + b * mask_bs + (int64_t)i * W;
#pragma unroll
      for (int w = 0; w < TREE_WORDS; ++w)
        if (w <= q) {
          uint32_t x = tree_word(m, W, N, w);
          if (w == q) x &= (1u << lane) - 1u;
          if (x) par[q] = 32 * w + 31 - __clz(x);
        }
    }
  }
  int cur = 0, n = 0;
  int64_t want = cho[0];
  const int most = alive == nullptr || alive[b] ? max_path : 1;
  if (lane == 0) path[(int64_t)b * max_path] = 0;
  while (++n < most) {
    int next = 0x7FFFFFFF;
#pragma unroll
    for (int q = TREE_WORDS - 1; q >= 0; --q)
      if (par[q] == cur && mine[q] == want) next = lane + 32 * q;
    next = __reduce_min_sync(0xffffffffu, next);
    if (next == 0x7FFFFFFF) break;
    cur = next;                                      // (a child comes after its parent: N steps at most)
    want = cho[cur];
    if (lane == 0) path[(int64_t)b * max_path + n] = cur;
  }
  for (int j = n + lane; j < max_path; j += 32) path[(int64_t)b * max_path + j] = -1;
  if (lane == 0) {
    n_acc[b] = n - 1;
    y[b] = want;
  }
}

struct CommitParams {
  const int32_t* bt;
  int bt_stride, npages;
  int64_t* lengths;
  const int32_t* path;
  int64_t path_bs;
  int path_len;
  const int64_t* n_acc;
  int N, B, H, C, cols;                      // cols: units of a (slot, head)
  int* err;
  void* bufs[COMMIT_BUFS];
};

// Whether row b can be committed: 0, or the error bits.
__device__ __forceinline__ int commit_check(const CommitParams& P, int b, int64_t* base, int* n) {
  const int64_t len = P.lengths[b], acc = P.n_acc[b];
  *base = len - P.N;
  *n = 0;
  if (*base < 0 || len > P.C) return 1;
  if (acc < 0 || acc >= P.N || acc >= P.path_len) return 32;
  *n = (int)acc + 1;
  return 0;
}
__device__ __forceinline__ bool path_ok(const CommitParams& P, const int32_t* p, int j) {
  return p[j] >= j && p[j] < P.N && (j == 0 || p[j] > p[j - 1]);
}

// Block (row, buffer): every thread its columns, along the path.
template <typename U>
__global__ void __launch_bounds__(COMMIT_THREADS)
tree_move_kernel(const __grid_constant__ CommitParams P) {
  __shared__ int32_t path[SD_TREE_MAX];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int b = blockIdx.x, t = threadIdx.x;
  int64_t base;
  int n;
  if (commit_check(P, b, &base, &n)) return;
  const int32_t* p = P.path + b * P.path_bs;
  int bad = 0, moves = 0;
  for (int j = t; j < n; j += COMMIT_THREADS) {
    path[j] = p[j];
    bad |= !path_ok(P, p, j);
    moves |= p[j] != j;
  }
  if (__syncthreads_or(bad)) return;
  if (!__syncthreads_or(moves)) return;
  U* buf = reinterpret_cast<U*>(P.bufs[blockIdx.y]);
  int first = 0;
  while (path[first] == first) ++first;              // (some node is not in place)
  // the slot's row of the buffer in units of (head, slot) = cols units; -1: no page
  auto place = [&](int64_t slot, int h) -> int64_t {
    if (P.bt == nullptr) return ((int64_t)b * P.H + h) * P.C + slot;
    const int pg = __ldg(P.bt + (int64_t)b * P.bt_stride + slot / SD_KV_PAGE);
    if ((unsigned)pg >= (unsigned)P.npages) return -1;
    return ((int64_t)pg * P.H + h) * SD_KV_PAGE + slot % SD_KV_PAGE;
  };
  for (int i = t; i < P.H * P.cols; i += COMMIT_THREADS) {
    const int h = i / P.cols, c = i - h * P.cols;
    for (int j0 = first; j0 < n; j0 += COMMIT_AHEAD) {
      U x[COMMIT_AHEAD];
      bool ok[COMMIT_AHEAD];
#pragma unroll
      for (int e = 0; e < COMMIT_AHEAD; ++e) {
        ok[e] = false;
        if (j0 + e < n) {
          const int64_t from = place(base + path[j0 + e], h);
          ok[e] = from >= 0;
          if (ok[e]) x[e] = buf[from * P.cols + c];
        }
      }
#pragma unroll
      for (int e = 0; e < COMMIT_AHEAD; ++e)
        if (ok[e]) {
          const int64_t to = place(base + j0 + e, h);
          if (to >= 0) buf[to * P.cols + c] = x[e];
        }
    }
  }
}

// The lengths, and what is wrong, once every move has read them.
__global__ void __launch_bounds__(128) tree_lengths_kernel(const __grid_constant__ CommitParams P) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = (blockIdx.x * 128 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (b >= P.B) return;
  int64_t base;
  int n, why = commit_check(P, b, &base, &n);
  if (why == 0) {
    const int32_t* p = P.path + b * P.path_bs;
    for (int j = lane; j < n; j += 32) {
      if (!path_ok(P, p, j)) {
        why |= 32;
      } else if (P.bt && p[j] != j) {
        const int32_t* row = P.bt + (int64_t)b * P.bt_stride;
        if ((unsigned)row[(base + p[j]) / SD_KV_PAGE] >= (unsigned)P.npages ||
            (unsigned)row[(base + j) / SD_KV_PAGE] >= (unsigned)P.npages)
          why |= 2;
      }
    }
  }
  why = __reduce_or_sync(0xffffffffu, why);
  if (lane == 0) {
    if (why && P.err) atomicOr(P.err, why);
    if (!(why & ~2)) P.lengths[b] = base + n;
  }
}

}  // namespace sd

using namespace sd;

extern "C" {

int sd_tree_masks(const int32_t* parents, int64_t parents_bs, int T, int N, int32_t* masks,
                  int32_t* depths, void* stream) {
  if (T < 0 || N < 0) return SD_EINVAL;
  if (T == 0 || N == 0) return SD_OK;
  if (!parents || !masks) return SD_EINVAL;
  if (N > SD_TREE_MAX) return SD_ENOTSUP;
  tree_masks_kernel<<<T, std::min((N + 31) / 32 * 32, SD_TREE_MAX), 0,
                      reinterpret_cast<cudaStream_t>(stream)>>>(parents, parents_bs, N,
                                                                (N + 31) / 32, masks, depths);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

int sd_tree_accept(const int64_t* tokens, int64_t tokens_bs, const int64_t* choices,
                   int64_t choices_bs, const int32_t* masks, int64_t mask_bs,
                   const uint8_t* alive, int B, int N, int max_path, int32_t* path,
                   int64_t* n_acc, int64_t* y, void* stream) {
  if (B < 0 || N < 1 || max_path < 1) return SD_EINVAL;
  if (B == 0) return SD_OK;
  if (!tokens || !choices || !masks || !path || !n_acc || !y) return SD_EINVAL;
  if (N > SD_TREE_MAX) return SD_ENOTSUP;
  tree_accept_kernel<<<B, 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      tokens, tokens_bs, choices, choices_bs, masks, mask_bs, alive, N, (N + 31) / 32, max_path,
      path, n_acc, y);
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

int sd_kv_commit_tree(void* const* bufs, int n_bufs, const int32_t* block_table, int bt_stride,
                      int npages, int64_t* lengths, const int32_t* path, int64_t path_bs,
                      int path_len, const int64_t* n_acc, int N, int B, int H, int C, int D,
                      int elem_bytes, int* err, void* stream) {
  if (B < 0 || n_bufs < 0 || N < 1 || H < 1 || D < 1 || path_len < 1) return SD_EINVAL;
  if (elem_bytes != 2 && elem_bytes != 4) return SD_EINVAL;
  if (B == 0) return SD_OK;
  if (!lengths || !path || !n_acc || (n_bufs > 0 && !bufs)) return SD_EINVAL;
  if (block_table && (bt_stride < 1 || npages < 1)) return SD_EINVAL;
  if (N > SD_TREE_MAX || (int64_t)H * D > 1 << 24) return SD_ENOTSUP;
  if (block_table) {
    if ((int64_t)bt_stride * SD_KV_PAGE > 0x7FFFFFFF) return SD_ENOTSUP;
    C = bt_stride * SD_KV_PAGE;
  }
  if (C < 1) return SD_EINVAL;
  CommitParams P;
  P.bt = block_table; P.bt_stride = bt_stride; P.npages = npages;
  P.lengths = lengths; P.path = path; P.path_bs = path_bs; P.path_len = path_len;
  P.n_acc = n_acc; P.N = N; P.B = B; P.H = H; P.C = C; P.err = err;
  const int row = D * elem_bytes;
  uintptr_t low = (uintptr_t)row;
  for (int i = 0; i < n_bufs; ++i) {
    if (!bufs[i]) return SD_EINVAL;
    low |= reinterpret_cast<uintptr_t>(bufs[i]);
  }
  if (low & (uintptr_t)(elem_bytes - 1)) return SD_EINVAL;
  const int unit = (low & 15) == 0 ? 16 : (low & 3) == 0 ? 4 : 2;
  P.cols = row / unit;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int i0 = 0; i0 < n_bufs; i0 += COMMIT_BUFS) {
    const int here = std::min(n_bufs - i0, COMMIT_BUFS);
    std::copy(bufs + i0, bufs + i0 + here, P.bufs);
    const dim3 grid((unsigned)B, (unsigned)here);
    if (unit == 16) tree_move_kernel<uint4><<<grid, COMMIT_THREADS, 0, st>>>(P);
    else if (unit == 4) tree_move_kernel<uint32_t><<<grid, COMMIT_THREADS, 0, st>>>(P);
    else tree_move_kernel<uint16_t><<<grid, COMMIT_THREADS, 0, st>>>(P);
    if (cudaGetLastError() != cudaSuccess) return SD_ELAUNCH;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((B + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = n_bufs > 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, tree_lengths_kernel, P) != cudaSuccess) return SD_ELAUNCH;
  return cudaGetLastError() == cudaSuccess ? SD_OK : SD_ELAUNCH;
}

}  // extern "C"
