// Host checks shared by the launchers of the attention-block operators.
#pragma once
#include "block_common.cuh"
#include "dispatch.cuh"

namespace fxh {

inline int check_buckets(const fx_buckets& b) {
  if (b.num_buckets < 1 || b.num_buckets > FX_BUCKET_MAX || b.num_edges < 0) return FX_ERR_SHAPE;
  if (b.two_sided ? (b.num_buckets % 2 != 0 || b.num_edges >= b.num_buckets / 2) : b.num_edges >= b.num_buckets)
    return FX_ERR_SHAPE;
  if (b.num_edges > 0 && !b.edges) return FX_ERR_NULL;
  for (int i = 0; i < b.num_edges; ++i)
    if (b.edges[i] < (i ? b.edges[i - 1] : 1) || b.edges[i] > FX_BUCKET_MAX_EDGE) return FX_ERR_SHAPE;
  return FX_OK;
}

inline BucketArgs make_buckets(const fx_buckets& b) {
  BucketArgs B;
  B.num_buckets = b.num_buckets;
  B.two_sided = b.two_sided != 0;
  B.num_edges = b.num_edges;
  // two-sided without edges still tells d > 0 from d <= 0
  B.reach = b.num_edges ? b.edges[b.num_edges - 1] : (b.two_sided ? 1 : 0);
  for (int i = 0; i < b.num_edges; ++i) B.edges[i] = b.edges[i];
  return B;
}

// The kernel's limit of shared memory for a launch of `smem` bytes: `most`, the same in every call,
// so that a call of one thread does not lower it between another's and its launch. 48 KB, the kernel's own
// shared memory (up to 4 KB) among them, need none.
template <typename K>
int raise_smem(K kern, size_t smem, size_t most) {
  if (smem > most) return FX_ERR_SHAPE;
  if (smem > 44 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
    return FX_ERR_CUDA;
  return FX_OK;
}

constexpr size_t kMaxSpan = 2 * FX_BUCKET_MAX_EDGE + 1;  // distances that a table by distance holds, at most

}  // namespace fxh
