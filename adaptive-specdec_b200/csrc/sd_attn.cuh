// What the attention kernels of the ragged cache share: the call's parameters
// and the addressing of a row's keys.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "specdec_b200.h"

namespace sd {

struct AttnParams {
  const void* q; int64_t qbs, qhs, qqs;
  const void* k; const void* v;
  const int64_t* lengths; const int64_t* valid;
  int B, Hq, Hkv, D, C, qlen, group, R, nsplit, nrc;
  float scale;
  void* out; int64_t obs, oqs, ohs;
  float* part_acc;   // [B, Hkv, nsplit, R, D]
  float* part_ml;    // [B, Hkv, nsplit, R, 2]
  int* split_done;   // [B, Hkv] pieces finished (tensor-core path; zeroed per call)
  int* rowpre;       // [B + 1] exclusive prefix of 64-key tiles per row (tensor-core path)
  int* rowkmax;      // [B] live-key bound of each row (tensor-core path)
  int npiece;        // partial slots per (row, kv head) on the tensor-core path
  int out_vec4;      // out is 8-byte aligned and its strides are multiples of 4 elements
  int tile_keys;     // keys per tile of the tensor-core schedule (plan kernel)
  int seg_ovh;       // schedule cost of a (row, kv head) beyond its tiles, in tiles
  int* status;       // sticky: bit 0 = a bounded wait of the tcgen05 kernel gave up
  // paged caches: k / v are pools [npages, Hkv, SD_KV_PAGE, D] and row b's key
  // s sits in page bt[b * bt_stride + s / SD_KV_PAGE]; bt == nullptr: the
  // contiguous [B, Hkv, C, D] layout
  const int32_t* bt;
  int bt_stride, npages;
};

// Offset, in rows of D elements, of key s of row b and kv head h.  A page
// index outside the pool reads page 0 (the caller's block table is wrong, but
// nothing is read out of bounds).
__device__ __forceinline__ int64_t kv_row(const AttnParams& P, int b, int h, int s) {
  if (P.bt == nullptr) return ((int64_t)b * P.Hkv + h) * P.C + s;
  int pg = __ldg(P.bt + (int64_t)b * P.bt_stride + (s / SD_KV_PAGE));
  if ((unsigned)pg >= (unsigned)P.npages) pg = 0;
  return ((int64_t)pg * P.Hkv + h) * SD_KV_PAGE + (s % SD_KV_PAGE);
}

__device__ __forceinline__ int row_limit(const AttnParams& P, int b, int j) {
  int64_t lim = P.lengths[b] + j + 1;
  if (P.valid && P.valid[b] < lim) lim = P.valid[b];
  if (lim > P.C) lim = P.C;
  return lim > 0 ? (int)lim : 0;
}

// sd_attention.cu: a 2D tensor map over a cache viewed as [rows, 128] bf16
// (boxes of box_rows rows x 64 columns, 128-byte swizzle)
bool cache_map(CUtensorMap* map, const void* base, int64_t rows, int box_rows = SD_KV_PAGE);

// sd_prefix_rows.cu: attention over a paged cache row by row, D <= 128
int prefix_rows(const AttnParams& P, int dtype, cudaStream_t st);

}  // namespace sd
