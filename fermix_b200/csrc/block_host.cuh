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

}  // namespace fxh
