// Shared pieces of the linear map: its arguments, the activations and their derivatives.
#pragma once
#include <cuda_fp16.h>

#include "token_common.cuh"

namespace fx {

// h -> (act(h), act'(h))
struct ActOut {
  float y, d;
};

template <int ACT, bool SLOPE>
__device__ __forceinline__ ActOut activate(float h) {
  ActOut o;
  o.d = 1.f;
  if constexpr (ACT == FX_ACT_NONE) {
    o.y = h;
  } else if constexpr (ACT == FX_ACT_RELU) {
    o.y = h > 0.f ? h : 0.f * h;  // a NaN stays
    o.d = h > 0.f ? 1.f : 0.f;
    if (h != h) o.d = h;
    if (h < 0.f) o.y = 0.f;
  } else if constexpr (ACT == FX_ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-h));
    o.y = h < -88.f ? 0.f : h * s;
    if (SLOPE) o.d = s * fmaf(fmaxf(h, -88.f), 1.f - s, 1.f);
  } else if constexpr (ACT == FX_ACT_GELU) {
    // the normal distribution's integral up to h: half of erfc(-h / sqrt 2), which keeps its digits where h < 0
    const float c = 0.5f * erfcf(-0.70710678118654752f * h);
    o.y = h < -14.f ? 0.f : h * c;
    if (SLOPE) o.d = fmaf(fminf(fmaxf(h, -20.f), 20.f) * 0.3989422804014327f, __expf(-0.5f * h * h), c);
  } else if constexpr (ACT == FX_ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
    const float k = 1.5957691216057308f, h2 = fminf(h * h, 1e6f);
    const float s = 1.f / (1.f + __expf(-k * h * fmaf(0.044715f, h2, 1.f)));
    o.y = h < -10.f ? 0.f : h * s;
    if (SLOPE) o.d = fabsf(h) > 12.f ? s : s * fmaf(h * (1.f - s), k * fmaf(0.134145f, h2, 1.f), 1.f);
  } else {
    o.y = tanhf(h);
    if (SLOPE) o.d = fmaf(-o.y, o.y, 1.f);
  }
  return o;
}

template <int ACT, bool SLOPE, int N>
__device__ __forceinline__ void activate_as(const float (&h)[N], float (&y)[N], float (&d)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const ActOut o = activate<ACT, SLOPE>(h[e]);
    y[e] = o.y;
    d[e] = o.d;
  }
}
template <bool SLOPE, int N>
__device__ __forceinline__ void activate_all(int act, const float (&h)[N], float (&y)[N], float (&d)[N]) {
  switch (act) {
    case FX_ACT_RELU: return activate_as<FX_ACT_RELU, SLOPE>(h, y, d);
    case FX_ACT_SILU: return activate_as<FX_ACT_SILU, SLOPE>(h, y, d);
    case FX_ACT_GELU: return activate_as<FX_ACT_GELU, SLOPE>(h, y, d);
    case FX_ACT_GELU_TANH: return activate_as<FX_ACT_GELU_TANH, SLOPE>(h, y, d);
    case FX_ACT_TANH: return activate_as<FX_ACT_TANH, SLOPE>(h, y, d);
    default: return activate_as<FX_ACT_NONE, SLOPE>(h, y, d);
  }
}

// The type the derivative is kept in: IEEE half beside bfloat16 (within +-1.2, 2^-12 of its value
// or 2^-25 where it is small, an eighth of what bfloat16's rounding would leave), float32 beside float32.
template <typename T>
struct SlopeOf {
  using type = __half;
};
template <>
struct SlopeOf<float> {
  using type = float;
};
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) {
  return __float2half_rn(x);
}

// What is done with a sum h of the product: bias, activation, derivative, residual, store.
struct Epilogue {
  int act;
  const void *bias, *residual;
  int64_t rs;  // stride of a row of the residual
  void *y, *slope;  // (rows, cols) contiguous
};

}  // namespace fx
