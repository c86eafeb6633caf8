// The linear map's products: D(i, j) = sum over k of A(i, k) B(j, k), by tiles of 64 x 64 in float32.
#pragma once
#include "linear_common.cuh"

namespace fx {

struct Operand {
  const void* p;
  int64_t row, col;  // element strides of an index of the result and of k
};

struct GemmArgs {
  Operand a, b;
  int64_t rows, cols, inner;
  Epilogue e;
};

template <typename TA, typename T>
__global__ void __launch_bounds__(256) linear_kernel(GemmArgs G) {
  __shared__ float as[16][68], bs[16][68];
  const int64_t i0 = (int64_t)blockIdx.x * 64, j0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < G.inner; k0 += 16) {
    for (int t = threadIdx.x; t < 1024; t += 256) {
      const int k = t & 15, i = t >> 4;
      as[k][i] = i0 + i < G.rows && k0 + k < G.inner
                     ? to_f(static_cast<const TA*>(G.a.p)[(i0 + i) * G.a.row + (k0 + k) * G.a.col]) : 0.f;
      bs[k][i] = j0 + i < G.cols && k0 + k < G.inner
                     ? to_f(static_cast<const T*>(G.b.p)[(j0 + i) * G.b.row + (k0 + k) * G.b.col]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[k][ty * 4 + i], bs[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (i0 + ty * 4 + i < G.rows && j0 + tx * 4 + j < G.cols)
        epilogue_one<T>(G.e, i0 + ty * 4 + i, j0 + tx * 4 + j, G.cols, acc[i][j]);
}

// g = dy act'(h) in float32 (slope not NULL), and the sums over the rows, a block 32 columns.
template <typename T>
__global__ void __launch_bounds__(256) linear_slope_kernel(const void* dy, int64_t stride, const void* slope, float* g,
                                                           void* dbias, int64_t rows, int64_t cols) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (j < cols)
    for (int64_t i = w; i < rows; i += 8) {
      float d = to_f(static_cast<const T*>(dy)[i * stride + j]);
      if (slope) {
        d *= to_f(static_cast<const typename SlopeOf<T>::type*>(slope)[i * cols + j]);
        if (g) g[i * cols + j] = d;
      }
      sum += d;
    }
  sums[w][lane] = sum;
  __syncthreads();
  if (w == 0 && j < cols && dbias) {
    for (int k = 1; k < 8; ++k) sum += sums[k][lane];
    static_cast<T*>(dbias)[j] = from_f<T>(sum);
  }
}

}  // namespace fx
