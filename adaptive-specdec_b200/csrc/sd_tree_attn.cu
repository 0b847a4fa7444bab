// Attention of a tree's nodes over the cache: host entry.
#include <cuda_runtime.h>

#include "sd_common.cuh"
#include "sd_tree.cuh"

using namespace sd;

extern "C" {

size_t sd_tree_attn_workspace_bytes(int B, int Hq, int Hkv, int D, int C, int qlen, int dtype) {
  return 0;
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
  TreeParams P = {};
  AttnParams& A = P.A;
  A.q = q; A.qbs = qbs; A.qhs = qhs; A.qqs = qqs;
  A.k = kcache; A.v = vcache; A.lengths = lengths;
  A.B = B; A.Hq = Hq; A.Hkv = Hkv; A.D = D; A.C = C; A.qlen = qlen;
  A.group = group; A.R = (int)R; A.scale = scale;
  A.out = out; A.obs = obs; A.oqs = oqs; A.ohs = ohs;
  A.bt = block_table; A.bt_stride = bt_stride; A.npages = npages;
  P.masks = masks; P.mask_bs = mask_bs; P.N = N; P.W = (N + 31) / 32; P.first = first;
  return tree_rows(P, dtype, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
