// The bucketed position bias and its gradient:
//
//   out[b, h, i, j] = table[h, bucket(k_pos[b, j] - q_pos[b, i])]
//   dtable[h, c]    = sum over b, i, j with that bucket = c of grad[b, h, i, j]
//
// Bound: HBM, one write (one read) of the (batch, heads, q_len, k_len) array. A thread owns
// E fixed columns, so their positions sit in registers, and walks the rows of its block; the
// table of one head is laid out in shared memory by the distance clamped to the reach of the
// buckets. Where all E columns are beyond the reach on one side of the row's position the
// lookup is a single value -- most of a long lattice.
//
// The gradient adds into a histogram of its own for each thread (column `thread` of a
// buckets x threads array: no bank is shared, nothing is atomic), a run of rows beyond the
// reach into one register; the block then adds the threads' columns in order, and
// bias_finish_kernel the blocks' partial rows in order.
//
// Measured: 8 heads of 4096 x 4096 in bfloat16: forward 63 us (268 MB, 4.3 TB/s), backward 112 us
// (2.4 TB/s); 128 x 8 heads of 255 x 255 sites in float32: forward 53 us (266 MB, 5.0 TB/s), backward
// 125 us (2.1 TB/s). What binds the backward is latency, not a pipe: in the lattice, where a thread
// reaches the histogram in about 6 % of its rows, 36 % of the issue slots of a working SM and 15 % of the
// shared-memory pipe are used and two thirds of a warp's waits are for its loads; blocks on the diagonal
// do all of the histogram, and SMs work for 133 to 219 thousand cycles, 178 on average. For the sites (rows
// of 255, so 4-byte loads; 80 registers leave 19 warps an SM) it is 50 % and 28 %, the waits spread over
// loads, fixed latencies and the histogram. Joining four entries of a bucket before the update (126 and
// 151 us) and reading the next row's distances ahead (197 and 133 us) were slower.
#pragma once
#include "block_common.cuh"

namespace fx {

struct BiasArgs {
  const void *table, *grad;
  void* out;
  float* part;  // (heads, parts, num_buckets), parts = batch x row blocks x column blocks
  const int *q_pos, *k_pos;
  int64_t q_pos_stride, k_pos_stride;
  int64_t q_len, k_len;
  int tx, rows, row_blocks, col_blocks, heads, batch;  // tx threads along a row, 128 / tx rows at a time
  BucketArgs buckets;
};

constexpr int kBiasThreads = 128;
constexpr int kBiasE = 8;  // columns of a thread

// Shared-memory place of distance index d: the columns of neighbouring threads are 8 apart,
// and swapping the low bits by the bits above the bank number spreads those over the banks.
__device__ __forceinline__ int lut_at(int d) { return d ^ ((d >> 5) & 7); }

struct BiasBlock {
  int h, b, rb, cb;
};

__device__ __forceinline__ BiasBlock bias_block(const BiasArgs& A) {
  BiasBlock p;
  int64_t i = blockIdx.x;
  p.cb = (int)(i % A.col_blocks);
  i /= A.col_blocks;
  p.rb = (int)(i % A.row_blocks);
  i /= A.row_blocks;
  p.h = (int)(i % A.heads);
  p.b = (int)(i / A.heads);
  return p;
}

// The thread's columns: VEC neighbouring ones at a time, threads next to each other.
template <int VEC>
struct BiasCols {
  int64_t col[kBiasE / VEC];
  int pos[kBiasE], lo, hi;
  bool any;
  __device__ __forceinline__ BiasCols(const BiasArgs& A, const BiasBlock& p) {
    lo = INT32_MAX;
    hi = INT32_MIN;
    any = false;
#pragma unroll
    for (int v = 0; v < kBiasE / VEC; ++v) {
      col[v] = (((int64_t)p.cb * (kBiasE / VEC) + v) * A.tx + (threadIdx.x & (A.tx - 1))) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int64_t j = col[v] + e;
        int x = 0;
        if (j < A.k_len) {
          x = A.k_pos ? A.k_pos[p.b * A.k_pos_stride + j] : (int)j;
          lo = min(lo, x);
          hi = max(hi, x);
          any = true;
        }
        pos[v * VEC + e] = x;
      }
    }
    if (!any) lo = hi = 0;
  }
};

__device__ __forceinline__ int bias_row_pos(const BiasArgs& A, int b, int64_t i) {
  return A.q_pos ? A.q_pos[b * A.q_pos_stride + i] : (int)(A.k_len - A.q_len + i);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kBiasThreads) bias_fwd_kernel(const __grid_constant__ BiasArgs A) {
  extern __shared__ float lut[];
  const BiasBlock p = bias_block(A);
  const int reach = A.buckets.reach;
  const T* table = static_cast<const T*>(A.table) + (int64_t)p.h * A.buckets.num_buckets;
  for (int d = threadIdx.x; d <= 2 * reach; d += kBiasThreads)
    lut[lut_at(d)] = to_f(table[bucket_of(A.buckets, d - reach)]);
  const BiasCols<VEC> c(A, p);
  __syncthreads();
  if (!c.any) return;
  const int ty = kBiasThreads / A.tx;
  const int64_t i0 = (int64_t)p.rb * A.rows;
  const int64_t i1 = i0 + A.rows < A.q_len ? i0 + A.rows : A.q_len;
  int64_t i = i0 + threadIdx.x / A.tx;
  T* out = static_cast<T*>(A.out) + (((int64_t)p.b * A.heads + p.h) * A.q_len + i) * A.k_len;
  for (; i < i1; i += ty, out += ty * A.k_len) {
    const int q = bias_row_pos(A, p.b, i);
    T val[kBiasE];
    if (c.lo - q >= reach || c.hi - q <= -reach) {
      const T one = from_f<T>(lut[lut_at(c.lo - q >= reach ? 2 * reach : 0)]);
#pragma unroll
      for (int e = 0; e < kBiasE; ++e) val[e] = one;
    } else {
#pragma unroll
      for (int e = 0; e < kBiasE; ++e) val[e] = from_f<T>(lut[lut_at(clamp_reach(c.pos[e] - q, reach) + reach)]);
    }
#pragma unroll
    for (int v = 0; v < kBiasE / VEC; ++v) {
      if (c.col[v] < A.k_len) {
        Pack<T, VEC> k;
#pragma unroll
        for (int e = 0; e < VEC; ++e) k.e[e] = val[v * VEC + e];
        *reinterpret_cast<Pack<T, VEC>*>(out + c.col[v]) = k;
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kBiasThreads) bias_bwd_kernel(const __grid_constant__ BiasArgs A) {
  extern __shared__ float hist[];  // num_buckets x threads, then the bucket of each distance
  const BiasBlock p = bias_block(A);
  const int reach = A.buckets.reach, nb = A.buckets.num_buckets;
  int* lut = reinterpret_cast<int*>(hist + nb * kBiasThreads);
  for (int d = threadIdx.x; d <= 2 * reach; d += kBiasThreads)
    lut[lut_at(d)] = bucket_of(A.buckets, d - reach) * kBiasThreads;
  float* mine = hist + threadIdx.x;
  for (int c = 0; c < nb; ++c) mine[c * kBiasThreads] = 0.f;
  const BiasCols<VEC> c(A, p);
  __syncthreads();
  const int ty = kBiasThreads / A.tx;
  const int64_t i0 = (int64_t)p.rb * A.rows;
  const int64_t i1 = i0 + A.rows < A.q_len ? i0 + A.rows : A.q_len;
  const int64_t first = i0 + threadIdx.x / A.tx;
  const T* g = static_cast<const T*>(A.grad) + (((int64_t)p.b * A.heads + p.h) * A.q_len + first) * A.k_len;
  float above = 0.f, below = 0.f;  // beyond the reach
  if (c.any) {
#pragma unroll 4
    for (int64_t i = first; i < i1; i += ty, g += ty * A.k_len) {
      float val[kBiasE];
#pragma unroll
      for (int v = 0; v < kBiasE / VEC; ++v) {
        if (c.col[v] < A.k_len) {
          const Pack<T, VEC> k = *reinterpret_cast<const Pack<T, VEC>*>(g + c.col[v]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) val[v * VEC + e] = to_f(k.e[e]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) val[v * VEC + e] = 0.f;
        }
      }
      const int q = bias_row_pos(A, p.b, i);
      if (c.lo - q >= reach || c.hi - q <= -reach) {
        const float s = ((val[0] + val[1]) + (val[2] + val[3])) + ((val[4] + val[5]) + (val[6] + val[7]));
        if (c.lo - q >= reach) above += s;
        else below += s;
      } else {
#pragma unroll
        for (int e = 0; e < kBiasE; ++e)
          if (c.col[e / VEC] < A.k_len) mine[lut[lut_at(clamp_reach(c.pos[e] - q, reach) + reach)]] += val[e];
      }
    }
    mine[lut[lut_at(2 * reach)]] += above;
    mine[lut[lut_at(0)]] += below;
  }
  __syncthreads();
  float* out = A.part + ((((int64_t)p.h * A.batch + p.b) * A.row_blocks + p.rb) * A.col_blocks + p.cb) * nb;
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < nb; k += kBiasThreads / 32) {
    const float* r = hist + k * kBiasThreads;
    const float v = lanes_sum((r[lane] + r[lane + 32]) + (r[lane + 64] + r[lane + 96]), 32);
    if (lane == 0) out[k] = v;
  }
}

// dtable[h, c] = the sum of part[h, 0..parts, c]: a block per (32 buckets, head), its 32 warps
// over the parts in turn, added in warp order.
template <typename T>
__global__ void __launch_bounds__(1024) bias_finish_kernel(const float* part, T* dtable, int64_t parts, int nb) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, h = blockIdx.y;
  float v = 0.f;
  if (c < nb) {
    const float* src = part + (int64_t)h * parts * nb + c;
#pragma unroll 8
    for (int64_t i = warp; i < parts; i += 32) v += src[i * nb];
  }
  s[lane][warp] = v;
  __syncthreads();
  v = lanes_sum(s[warp][lane], 32);
  if (lane == 0 && blockIdx.x * 32 + warp < nb) dtable[(int64_t)h * nb + blockIdx.x * 32 + warp] = from_f<T>(v);
}

}  // namespace fx
