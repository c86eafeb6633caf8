// Shared pieces of the operators on tokens.
#pragma once
#include "block_common.cuh"
#include "fermix_b200_token.h"

namespace fx {

// The entries of a pack as float32; bfloat16 by words, an instruction an entry.
template <int N>
__device__ __forceinline__ void unpack(const Pack<float, N>& p, float* x) {
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = p.e[e];
}
template <int N>
__device__ __forceinline__ void unpack(const Pack<bf16, N>& p, float* x) {
  if constexpr (N % 2) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_f(p.e[e]);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      x[e] = __uint_as_float(w[e / 2] << 16);
      x[e + 1] = __uint_as_float(w[e / 2] & 0xffff0000u);
    }
  }
}

// 2^x, to 2^-22 of the value.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A launch of the host's launch_next waits here, before it reads or writes anything in memory, until everything before it
// is done.
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Tokens {
  const void* p;
  int bytes, has_padding;
  int64_t padding;

  __device__ __forceinline__ int64_t at(int64_t i) const {
    switch (bytes) {
      case 1: return static_cast<const uint8_t*>(p)[i];
      case 2: return static_cast<const int16_t*>(p)[i];
      case 4: return static_cast<const int32_t*>(p)[i];
      default: return static_cast<const int64_t*>(p)[i];
    }
  }
  __device__ __forceinline__ bool padded(int64_t t) const { return has_padding && t == padding; }
  // The table's row of token i; `rows` where it has none.
  __device__ __forceinline__ int key(int64_t i, int64_t rows) const {
    const int64_t t = at(i);
    return t < 0 || t >= rows || padded(t) ? (int)rows : (int)t;
  }
};

}  // namespace fx
