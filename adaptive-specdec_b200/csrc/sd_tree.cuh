// What the kernels for trees of drafted tokens share: ancestor bits and what a
// node sees of the cache.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "sd_attn.cuh"

namespace sd {

struct TreeParams {
  AttnParams A;                              // valid is not used
  const int32_t* masks;                      // [T, N, W] ancestor bits
  int64_t mask_bs;                           // words between two rows' trees (0: one tree)
  int N, W, first;                           // nodes, words per node, node of query 0
};

// Word w of a node's mask without the bits from N on.
__device__ __forceinline__ uint32_t tree_valid(int N, int w) {
  const int left = N - 32 * w;
  return left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
}
__device__ __forceinline__ uint32_t tree_word(const int32_t* m, int W, int N, int w) {
  if ((unsigned)w >= (unsigned)W) return 0u;
  return (uint32_t)__ldg(m + w) & tree_valid(N, w);
}

// The tokens of row b before the tree, held in the cache's capacity (a wrong
// length reads nothing out of bounds).
__device__ __forceinline__ int tree_base(const TreeParams& P, int b) {
  const int64_t n = P.A.lengths[b] - P.first;
  return n < 0 ? 0 : n > P.A.C ? P.A.C : (int)n;
}
// The end of the slots that row b's nodes can see.
__device__ __forceinline__ int tree_end(const TreeParams& P, int base) {
  return min(base + P.N, P.A.C);
}

// Bits of the keys s0 .. s0 + 31 that a (present) node with mask m sees.
__device__ __forceinline__ uint32_t tree_sees(const int32_t* m, int W, int N, int base, int s0) {
  const int d = base - s0;
  if (d >= 32) return 0xFFFFFFFFu;
  if (d > 0) return ((1u << d) - 1u) | (tree_word(m, W, N, 0) << d);
  const int a = -d, w = a >> 5;
  return __funnelshift_r(tree_word(m, W, N, w), tree_word(m, W, N, w + 1), a & 31);
}

__device__ __forceinline__ bool tree_present(const int32_t* m, int W, int N) {
  uint32_t any = 0;
  for (int w = 0; w < W; ++w) any |= tree_word(m, W, N, w);
  return any != 0;
}

// Whether rows of `row` elements, sizes[i] of them at strides[i] (elements), share none: in
// order of the strides, each steps over all that the smaller ones reach.  (So are all views
// of a dense tensor that do not expand or unfold it; the stride of a dimension of one is any.)
template <int N>
bool rows_apart(int64_t row, const int64_t (&sizes)[N], const int64_t (&strides)[N]) {
  int order[N];
  for (int i = 0; i < N; ++i) order[i] = i;
  auto step = [&](int i) { return (__int128)(strides[i] < 0 ? -(__int128)strides[i] : strides[i]); };
  std::sort(order, order + N, [&](int a, int b) { return step(a) < step(b); });
  __int128 reach = row;
  for (int i : order) {
    if (sizes[i] <= 1) continue;
    if (step(i) < reach) return false;
    reach += (sizes[i] - 1) * step(i);
  }
  return true;
}

// sd_tree_rows.cu: tree attention on the CUDA cores, D <= 128
int tree_rows(const TreeParams& P, int dtype, cudaStream_t st);

}  // namespace sd
