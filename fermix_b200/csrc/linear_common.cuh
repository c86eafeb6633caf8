// Shared pieces of the linear map: its arguments, the activations and their derivatives.
#pragma once
#include <cuda_fp16.h>

#include "token_common.cuh"

namespace fx {

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(fminf(-x, 80.f))); }

// h -> (act(h), act'(h))
struct ActOut {
  float y, d;
};

template <int ACT>
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
    const float s = sigmoid(h);
    o.y = h < -80.f ? 0.f : h * s;
    o.d = s * fmaf(fmaxf(h, -80.f), 1.f - s, 1.f);
  } else if constexpr (ACT == FX_ACT_GELU) {
    // erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + p x), x >= 0: Abramowitz and Stegun 7.1.26, off by
    // 1.5e-7 at most. With x = |h| / sqrt 2 the exponential is the normal density's.
    const float x = fabsf(h) * 0.70710678118654752f, t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f)), e = __expf(-x * x);
    const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * q * e, c = h < 0.f ? tail : 1.f - tail;
    o.y = h < -14.f ? 0.f : h * c;
    o.d = fmaf(fminf(fmaxf(h, -20.f), 20.f) * 0.3989422804014327f, e, c);
  } else if constexpr (ACT == FX_ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
    const float k = 1.5957691216057308f, h2 = fminf(h * h, 1e6f);
    const float s = sigmoid(k * h * fmaf(0.044715f, h2, 1.f));
    o.y = h < -10.f ? 0.f : h * s;
    o.d = fabsf(h) > 12.f ? s : s * fmaf(h * (1.f - s), k * fmaf(0.134145f, h2, 1.f), 1.f);
  } else {
    // tanh u = 2 sigmoid(2 u) - 1; near 0, where that cancels, its series (the next term is 5e-8 of it)
    const float h2 = h * h;
    o.y = h2 < 0.09f ? h * fmaf(h2, fmaf(h2, fmaf(h2, fmaf(h2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f)
                     : fmaf(2.f, sigmoid(2.f * h), -1.f);
    o.d = fmaf(-o.y, o.y, 1.f);
  }
  return o;
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
