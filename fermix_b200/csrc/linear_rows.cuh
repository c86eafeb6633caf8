// The linear map of few rows (a token a walker): bound by the weights' bytes, which are read once, straight into
// the operand registers of the warps' tensor instructions (m16n8k16: 16 outputs by 8 rows of x). Of few outputs, and of
// small maps, likewise in float32, where the tiles of linear_tc.cuh would read and write both operands' parts besides:
// where the outputs are fewer than the rows, x and the weights change places.
//
// A block has 16 MT outputs and 8 NT rows (all of them, up to 32); its WARPS warps share k in steps of 32, and their sums
// are added in order through shared memory. The order of k within a step is free as long as both operands have it: lane t
// of a group of four takes entries 8 t .. 8 t + 7 of its row (float32: 4 t .. and 16 + 4 t .., four each), pieces of 16
// bytes next to its neighbours', which are two instructions' worth of a fragment. Each lane's pieces come through a ring of
// asynchronous copies of its own: held in registers, the loads of a few steps were not all asked for before the first
// product, and the weights came at 2 TB/s.
//
// float32 is split into three bfloat16 parts in registers, six products as in linear_tc.cuh; the instructions cut
// off what they add to an accumulator below its last bit, so each step's sum starts from zero and is added with
// rounding.
#pragma once
#include "linear_common.cuh"

namespace fx {
namespace lin {

constexpr int kRowStep = 32;

struct RowArgs {
  const void *x, *w;
  int64_t xs, ws;  // strides of a row
  int rows, inner, outer;  // of x; of both; of w
  bool swapped;            // w is the map's x and x its weights
  Epilogue e;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight entries of a row as they lie in memory: words of two bfloat16 or of a float32.
template <typename T>
struct Eight {
  uint32_t w[8 * sizeof(T) / 4];
};

// Entry e of lane t's eight of a step.
template <typename T>
__device__ __forceinline__ int entry_of(int t, int e) {
  return sizeof(T) == 2 ? t * 8 + e : e / 4 * 16 + t * 4 + e % 4;
}
// Lane t's entries of a step that has n, one by one, zeros behind.
template <typename T>
__device__ __forceinline__ Eight<T> load_row(const T* p, int t, int n) {
  Eight<T> v;
#pragma unroll
  for (int i = 0; i < 8 * (int)sizeof(T) / 4; ++i) v.w[i] = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = entry_of<T>(t, e);
    if (k < n) {
      if constexpr (sizeof(T) == 4) v.w[e] = __float_as_uint(p[k]);
      else v.w[e / 2] |= (uint32_t)__bfloat16_as_ushort(p[k]) << (e % 2 * 16);
    }
  }
  return v;
}

// The parts: o[p][i] holds entries 2 i and 2 i + 1 of part p.
template <int NP>
__device__ __forceinline__ void parts_of(const Eight<bf16>& v, uint32_t (&o)[NP][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[0][i] = v.w[i];
}
template <int NP>
__device__ __forceinline__ void parts_of(const Eight<float>& v, uint32_t (&o)[NP][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[NP];
    split_pair<NP>(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]), w);
#pragma unroll
    for (int p = 0; p < NP; ++p) o[p][i] = w[p];
  }
}

// A lane's ring: the 16-byte pieces of a step, and as many steps as a block of about 100 KB (of sixteen warps, which
// has an SM to itself, 200; of four, three of which share an SM, 72) holds. The sums take its place.
template <typename T, int MT, int NT, int WARPS>
struct RowRing {
  static constexpr int kEach = sizeof(T) / 2, kPieces = (2 * MT + NT) * kEach;
  static constexpr int kStep = kPieces * WARPS * 32 * 16, kFit = (WARPS > 8 ? 200 : WARPS > 4 ? 100 : 72) * 1024 / kStep;
  static constexpr int kDepth = kFit < 2 ? 2 : kFit > 8 ? 8 : kFit;
  static constexpr size_t kSums = (size_t)WARPS * 8 * NT * (16 * MT + 1) * sizeof(float);
  static constexpr size_t kRing = (size_t)kDepth * kStep, kSmem = kRing > kSums ? kRing : kSums;
};

// MT tiles of 16 outputs, NT of 8 rows. (16 outputs by 64 rows, whose weights' entries are split twice as often:
// 4700 x 264 x 64 21 us, so 14.)
template <typename T, int NP, int MT, int NT, int WARPS, bool ALIGNED>
__global__ void __launch_bounds__(WARPS * 32, WARPS > 4 ? 1 : 3) linear_rows_kernel(const __grid_constant__ RowArgs A) {
  constexpr int kOut = 16 * MT, kIn = 8 * NT, LD = kOut + 1;
  extern __shared__ uint4 ring[];  // (steps, pieces, threads), then the warps' sums
  float* sums = reinterpret_cast<float*>(ring);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int j0 = blockIdx.x * kOut, i0 = blockIdx.y * kIn, here = min(A.rows - i0, kIn);
  // Outputs that are not there read the last one's: what comes of them is not stored.
  const T *w[2 * MT], *x[NT];
#pragma unroll
  for (int m = 0; m < 2 * MT; ++m) w[m] = static_cast<const T*>(A.w) + (int64_t)min(j0 + m * 8 + g, A.outer - 1) * A.ws;
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = static_cast<const T*>(A.x) + (int64_t)(i0 + min(n * 8 + g, here - 1)) * A.xs;
  float acc[MT][NT][4] = {};
  const auto multiply = [&](const Eight<T> (&a)[2 * MT], const Eight<T> (&b)[NT]) {
    uint32_t ap[2 * MT][NP][4];
#pragma unroll
    for (int m = 0; m < 2 * MT; ++m) parts_of<NP>(a[m], ap[m]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t bp[NP][4];
      parts_of<NP>(b[n], bp);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (NP == 1) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            mma_bf16(acc[m][n], ap[2 * m][0][2 * h], ap[2 * m + 1][0][2 * h], ap[2 * m][0][2 * h + 1], ap[2 * m + 1][0][2 * h + 1],
                     bp[0][2 * h], bp[0][2 * h + 1]);
        } else {
          float d[2][4] = {};  // two chains of instructions
#pragma unroll
          for (int sum = NP - 1; sum >= 0; --sum)  // the smaller products first
#pragma unroll
            for (int i = 0; i <= sum; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                mma_bf16(d[h], ap[2 * m][i][2 * h], ap[2 * m + 1][i][2 * h], ap[2 * m][i][2 * h + 1], ap[2 * m + 1][i][2 * h + 1],
                         bp[sum - i][2 * h], bp[sum - i][2 * h + 1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][n][e] += d[0][e] + d[1][e];
        }
      }
    }
  };
  const int whole = ALIGNED ? A.inner / kRowStep : 0, steps = (A.inner + kRowStep - 1) / kRowStep;
  int s = warp;
  if constexpr (ALIGNED) {
    using R = RowRing<T, MT, NT, WARPS>;
    const auto fetch = [&](int slot, int step) {
      if (step < whole) {
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + slot * (R::kPieces * WARPS * 32) + threadIdx.x);
        const auto piece = [&](int p, const T* from) {
#pragma unroll
          for (int h = 0; h < R::kEach; ++h)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (p * R::kEach + h) * (WARPS * 32 * 16)),
                         "l"(reinterpret_cast<const uint4*>(from + step * kRowStep) + h * 4 + t)
                         : "memory");
        };
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m) piece(m, w[m]);
#pragma unroll
        for (int n = 0; n < NT; ++n)  // (several lanes' copies of one address are slow)
          if (n * 8 + g < here) piece(2 * MT + n, x[n]);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int d = 0; d < R::kDepth; ++d) fetch(d, s + d * WARPS);
    int slot = 0;
#pragma unroll 1
    for (; s < whole; s += WARPS) {
      asm volatile("cp.async.wait_group %0;" ::"n"(R::kDepth - 1) : "memory");
      Eight<T> a[2 * MT], b[NT];
      const uint4* from = ring + slot * (R::kPieces * WARPS * 32) + threadIdx.x;
      const auto piece = [&](int p, Eight<T>& v) {
#pragma unroll
        for (int h = 0; h < R::kEach; ++h) {
          const uint4 q = from[(p * R::kEach + h) * (WARPS * 32)];
          v.w[4 * h] = q.x;
          v.w[4 * h + 1] = q.y;
          v.w[4 * h + 2] = q.z;
          v.w[4 * h + 3] = q.w;
        }
      };
#pragma unroll
      for (int m = 0; m < 2 * MT; ++m) piece(m, a[m]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        b[n] = {};
        if (n * 8 + g < here) piece(2 * MT + n, b[n]);
      }
      fetch(slot, s + R::kDepth * WARPS);
      slot = slot + 1 == R::kDepth ? 0 : slot + 1;
      multiply(a, b);
    }
  }
#pragma unroll 1
  for (; s < steps; s += WARPS) {  // what is left, and rows off the 16-byte boundaries
    Eight<T> a[2 * MT], b[NT];
    const int k = s * kRowStep, left = A.inner - k;
#pragma unroll
    for (int m = 0; m < 2 * MT; ++m) a[m] = load_row(w[m] + k, t, left);
#pragma unroll
    for (int n = 0; n < NT; ++n) b[n] = load_row(x[n] + k, t, left);
    multiply(a, b);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[warp * (kIn * LD) + (n * 8 + t * 2 + (e & 1)) * LD + m * 16 + g + (e >> 1) * 8] = acc[m][n][e];
  __syncthreads();
  for (int v = threadIdx.x; v < kOut * kIn; v += WARPS * 32) {
    const int i = v / kOut, o = v % kOut, j = j0 + o;
    if (i >= here || j >= A.outer) continue;
    float h = sums[i * LD + o];
#pragma unroll
    for (int k = 1; k < WARPS; ++k) h += sums[k * (kIn * LD) + i * LD + o];
    if (A.swapped) store_entry<T>(A.e, j, i0 + i, A.rows, h);
    else store_entry<T>(A.e, i0 + i, j, A.outer, h);
  }
}

}  // namespace lin
}  // namespace fx
