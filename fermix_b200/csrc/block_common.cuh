// Shared pieces of the attention-block operators (residual norm, position bias, biased
// attention): float32 / bfloat16 vectors, group reductions, the position buckets.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fermix_b200_block.h"

namespace fx {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) {
  return __float2bfloat16_rn(x);
}

// N entries of T moved as one access of N * sizeof(T) bytes (2, 4, 8 or 16).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T e[N];
};

// Sum of v over the aligned groups of `width` (a power of two <= 32) lanes of a warp.
__device__ __forceinline__ float lanes_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------- position buckets
// The edges travel as a kernel argument, so that a call needs no device copy of them.
struct BucketArgs {
  int num_buckets, two_sided, num_edges, reach;  // reach: the last edge (0 without edges)
  int edges[FX_BUCKET_MAX - 1];
};

// Beyond +-reach a distance's bucket no longer changes: the table's values are looked up by
// the distance clamped to [-reach, reach], 2 reach + 1 entries.
__device__ __forceinline__ int bucket_of(const BucketArgs& B, int d) {
  const int a = B.two_sided ? abs(d) : max(-d, 0);
  int lo = 0;  // the number of edges <= a; the same edge for all threads of a step
  for (int i = 0; i < B.num_edges; ++i) lo += B.edges[i] <= a;
  return lo + (B.two_sided && d > 0 ? B.num_buckets / 2 : 0);
}

__device__ __forceinline__ int clamp_reach(int d, int reach) { return min(max(d, -reach), reach); }

}  // namespace fx
