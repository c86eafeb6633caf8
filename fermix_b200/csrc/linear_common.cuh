// Shared pieces of the linear map: its arguments, the activations and their derivatives.
#pragma once
#include <cuda_fp16.h>

#include "token_common.cuh"

namespace fx {

// 1 / x, to 2^-22 of the value.
__device__ __forceinline__ float fast_inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + exp(-x)), of scale x where scale is given
__device__ __forceinline__ float sigmoid(float x, float scale = 1.f) {
  return fast_inverse(1.f + fast_exp2(x * (-1.4426950408889634f * scale)));
}

// h -> (act(h), act'(h)). Finite at every finite h: where an exponential overflows, its inverse is 0. The products
// are rounded by themselves, so that act(h) has the same bits whatever is done with it.
struct ActOut {
  float y, d;
};

template <int ACT>
__device__ __forceinline__ ActOut activate(float h) {
  ActOut o;
  o.d = 1.f;
  if constexpr (ACT == FX_ACT_RELU) {
    o.y = h < 0.f ? 0.f : h;  // a NaN stays
    o.d = h > 0.f ? 1.f : h != h ? h : 0.f;
  } else if constexpr (ACT == FX_ACT_SILU) {
    const float s = sigmoid(h);
    o.y = __fmul_rn(h, s);
    o.d = fmaf(o.y, 1.f - s, s);
  } else if constexpr (ACT == FX_ACT_GELU) {
    // erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + p x), x >= 0: Abramowitz and Stegun 7.1.26, off by
    // 1.5e-7 at most. With x = |h| / sqrt 2 the exponential is the normal density's; the halves are in the a's.
    const float t = fast_inverse(fmaf(0.3275911f * 0.70710678118654752f, fabsf(h), 1.f));
    const float e = fast_exp2(h * h * (-0.5f * 1.4426950408889634f));
    const float q = fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f),
                                 0.5f * -0.284496736f), 0.5f * 0.254829592f);
    const float tail = q * (t * e), c = h < 0.f ? tail : 1.f - tail;
    o.y = __fmul_rn(h, c);
    o.d = fmaf(h * 0.3989422804014327f, e, c);
  } else if constexpr (ACT == FX_ACT_GELU_TANH) {
    // (1 + tanh u) / 2 is the sigmoid of 2 u
    const float k = 1.5957691216057308f, h2 = h * h;
    const float s = sigmoid(h * fmaf(0.044715f, h2, 1.f), k);
    o.y = __fmul_rn(h, s);
    o.d = fmaf(o.y * (1.f - s), k * fmaf(0.134145f, fminf(h2, 1e6f), 1.f), s);
  } else if constexpr (ACT == FX_ACT_TANH) {
    // tanh u = 2 sigmoid(2 u) - 1; near 0, where that cancels, its series (the next term is 5e-8 of it)
    const float h2 = h * h;
    o.y = h2 < 0.09f ? __fmul_rn(h, fmaf(h2, fmaf(h2, fmaf(h2, fmaf(h2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f))
                     : fmaf(2.f, sigmoid(h, 2.f), -1.f);
    o.d = fmaf(-o.y, o.y, 1.f);
  } else {
    o.y = h;
  }
  return o;
}

// The type the derivative is kept in: IEEE half beside bfloat16 (within +-1.2, 2^-11 of its value
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

template <int N>
__device__ __forceinline__ void unpack(const Pack<__half, N>& p, float* x) {
  if constexpr (N % 2) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_f(p.e[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p.e[e]));
      x[e] = f.x;
      x[e + 1] = f.y;
    }
  }
}

// N entries rounded into a pack, two at a time where the type has it.
template <int N>
__device__ __forceinline__ void round_into(Pack<float, N>& o, const float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) o.e[e] = x[e];
}
template <int N>
__device__ __forceinline__ void round_into(Pack<bf16, N>& o, const float (&x)[N]) {
  if constexpr (N == 1) {
    o.e[0] = __float2bfloat16_rn(x[0]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) *reinterpret_cast<__nv_bfloat162*>(&o.e[e]) = __floats2bfloat162_rn(x[e], x[e + 1]);
  }
}
template <int N>
__device__ __forceinline__ void round_into(Pack<__half, N>& o, const float (&x)[N]) {
  if constexpr (N == 1) {
    o.e[0] = __float2half_rn(x[0]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) *reinterpret_cast<__half2*>(&o.e[e]) = __floats2half2_rn(x[e], x[e + 1]);
  }
}

// What is done with a sum h of the product: bias, activation, derivative, residual, store.
struct Epilogue {
  int act;
  const void *bias, *residual;
  int64_t rs;  // stride of a row of the residual
  void *y, *slope;  // (rows, cols) contiguous
};

__device__ __forceinline__ ActOut activate_as(int act, float h) {
  switch (act) {
    case FX_ACT_RELU: return activate<FX_ACT_RELU>(h);
    case FX_ACT_SILU: return activate<FX_ACT_SILU>(h);
    case FX_ACT_GELU: return activate<FX_ACT_GELU>(h);
    case FX_ACT_GELU_TANH: return activate<FX_ACT_GELU_TANH>(h);
    case FX_ACT_TANH: return activate<FX_ACT_TANH>(h);
    default: return activate<FX_ACT_NONE>(h);
  }
}

// One entry of the sum: bias, activation, residual, stores.
template <typename T>
__device__ __forceinline__ void store_entry(const Epilogue& E, int64_t i, int64_t j, int64_t cols, float h) {
  using TS = typename SlopeOf<T>::type;
  if (E.bias) h += to_f(static_cast<const T*>(E.bias)[j]);
  ActOut a = activate_as(E.act, h);
  if (E.act != FX_ACT_NONE && E.slope) static_cast<TS*>(E.slope)[i * cols + j] = from_f<TS>(a.d);
  if (E.residual) a.y += to_f(static_cast<const T*>(E.residual)[i * E.rs + j]);
  static_cast<T*>(E.y)[i * cols + j] = from_f<T>(a.y);
}

// (a, b) -> NP packed pairs of bfloat16 whose sum is (a, b). The first is rounded to a finite number where its value is,
// which leaves the rest to the second.
template <int NP>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&o)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (NP > 1 && i == 0) asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(b), "f"(a));
    if (i + 1 < NP) {
      a -= __uint_as_float(o[i] << 16);
      b -= __uint_as_float(o[i] & 0xffff0000u);
    }
  }
}

}  // namespace fx
