// The linear map with its epilogue: checks, launch shapes, workspace.
#include "block_host.cuh"
#include "linear.cuh"

namespace {

using namespace fxh;

int check(const fx_linear_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->activation < FX_ACT_NONE || a->activation > FX_ACT_TANH || a->rows < 0 || a->rows >= INT32_MAX ||
      a->inner < 1 || a->inner >= INT32_MAX || a->outer < 1 || a->outer >= INT32_MAX || a->x_stride < 0 ||
      a->weight_stride < 0 || a->residual_stride < 0 || a->dy_stride < 0)
    return FX_ERR_SHAPE;
  return FX_OK;
}

template <typename TA, typename T>
int product(cudaStream_t s, Operand a, Operand b, int64_t rows, int64_t cols, int64_t inner, const Epilogue& e) {
  GemmArgs G{a, b, rows, cols, inner, e};
  const int64_t y = (cols + 63) / 64;
  if (y > 65535) return FX_ERR_SHAPE;
  linear_kernel<TA, T><<<dim3((unsigned)((rows + 63) / 64), (unsigned)y), 256, 0, s>>>(G);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <typename T>
int forward(cudaStream_t s, const fx_linear_args* a) {
  Epilogue e{a->activation, a->bias, a->residual, a->residual_stride, a->y, a->slope};
  return product<T, T>(s, {a->x, a->x_stride, 1}, {a->weight, a->weight_stride, 1}, a->rows, a->outer, a->inner, e);
}

template <typename TA, typename T>
int gradients(cudaStream_t s, const fx_linear_args* a, const void* g, int64_t gs) {
  int st = FX_OK;
  if (a->dx) {
    Epilogue e{FX_ACT_NONE, nullptr, nullptr, 0, a->dx, nullptr};
    st = product<TA, T>(s, {g, gs, 1}, {a->weight, 1, a->weight_stride}, a->rows, a->inner, a->outer, e);
  }
  if (!st && a->dweight) {
    Epilogue e{FX_ACT_NONE, nullptr, nullptr, 0, a->dweight, nullptr};
    st = product<TA, T>(s, {g, 1, gs}, {a->x, 1, a->x_stride}, a->outer, a->inner, a->rows, e);
  }
  return st;
}

template <typename T>
int backward(cudaStream_t s, const fx_linear_args* a, float* g) {
  const bool slope = a->activation != FX_ACT_NONE;
  if (slope || a->dbias) {
    linear_slope_kernel<T><<<(unsigned)((a->outer + 31) / 32), 256, 0, s>>>(
        a->dy, a->dy_stride, slope ? a->slope : nullptr, g, a->dbias, a->rows, a->outer);
    if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
  }
  return slope ? gradients<float, T>(s, a, g, a->outer) : gradients<T, T>(s, a, a->dy, a->dy_stride);
}

}  // namespace

extern "C" {

size_t fermix_linear_workspace_bytes(const fx_linear_args* a) {
  (void)a;
  return 0;
}

int fermix_linear(void* stream, const fx_linear_args* a, void* ws, size_t wsb) {
  (void)ws;
  (void)wsb;
  const int e = check(a);
  if (e) return e;
  if (a->rows == 0) return FX_OK;
  if (!a->x || !a->weight || !a->y) return FX_ERR_NULL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == FX_F32 ? forward<float>(s, a) : forward<bf16>(s, a);
}

size_t fermix_linear_grad_workspace_bytes(const fx_linear_args* a) {
  if (check(a) || a->activation == FX_ACT_NONE) return 0;
  return (size_t)a->rows * a->outer * sizeof(float) + 256;
}

int fermix_linear_grad(void* stream, const fx_linear_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t size = a->dtype == FX_F32 ? 4 : 2;
  if (a->rows == 0) {
    if (a->dweight && cudaMemsetAsync(a->dweight, 0, (size_t)(a->outer * a->inner) * size, s) != cudaSuccess)
      return FX_ERR_CUDA;
    if (a->dbias && cudaMemsetAsync(a->dbias, 0, (size_t)a->outer * size, s) != cudaSuccess) return FX_ERR_CUDA;
    return FX_OK;
  }
  if (!a->dy || (a->dx && !a->weight) || (a->dweight && !a->x) || (a->activation != FX_ACT_NONE && !a->slope))
    return FX_ERR_NULL;
  const size_t need = fermix_linear_grad_workspace_bytes(a);
  if (need && (!ws || wsb < need)) return FX_ERR_WORKSPACE;
  float* g = need ? reinterpret_cast<float*>(align256(reinterpret_cast<uintptr_t>(ws))) : nullptr;
  return a->dtype == FX_F32 ? backward<float>(s, a, g) : backward<bf16>(s, a, g);
}

}  // extern "C"
