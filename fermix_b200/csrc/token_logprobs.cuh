// Log probabilities of given tokens under softmax(scale logits), with entropy and the likeliest
// entries, and their gradient.
//
// One pass over a row keeps the running maximum m, S = sum of exp(scale (x - m)) and
// W = sum of exp(scale (x - m)) (x - m); then with L = log S
//   log p_t = scale (x_t - m) - L,   entropy = L - scale W / S.
// The likeliest entries are kept by each warp, one a lane in descending order; an entry that
// passes the last of them is inserted, which becomes rare after the first few hundred.
// Bound by HBM where rows are many or long. A block takes a row, or a part of one where the
// rows do not fill the device; parts are joined in order by a second kernel.
#pragma once
#include "token_common.cuh"

namespace fx {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kProbThreads = 256, kProbWarps = kProbThreads / 32;

struct ProbArgs {
  Tokens tok;
  const void* logits;
  const uint8_t* mask;
  int64_t ls, ms;  // strides of a row
  float *logp, *entropy, *top_logp;
  int64_t* top_index;
  float* stats;  // (2, rows): m, log2 S
  // parts of a row: (rows, parts) of {m, S, W, unused} and of `top` (value, index)
  float4* part;
  int2* part_top;
  int64_t rows;
  int entries, top, parts, per;  // per: entries of a part, a multiple of kProbThreads * 8
  float scale;
  // backward
  const float *glogp, *gentropy;
  void* dlogits;
};

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kNone = -INFINITY;

struct Sums {
  float m = kNone, s = 0.f, w = 0.f;

  // Everything so far to the reference `to` >= m.
  __device__ __forceinline__ void move(float to, float c) {
    if (m != kNone) {
      const float d = m - to, f = exp2_of(d * c);
      w = f * (w + fmaxf(d, -1e30f) * s);
      s *= f;
    }
    m = to;
  }
  __device__ __forceinline__ void join(float m2, float s2, float w2, float c) {
    const float to = fmaxf(m, m2);
    Sums o;
    o.m = m2;
    o.s = s2;
    o.w = w2;
    if (to != kNone) {
      move(to, c);
      o.move(to, c);
    }
    s += o.s;
    w += o.w;
  }
};

// Of a warp: entry `lane` of the list in descending order, ties to the lower index.
struct Best {
  float v = kNone;
  int i = -1;

  __device__ __forceinline__ bool before(float x, int j) const { return v > x || (v == x && (unsigned)i < (unsigned)j); }
  // (x, j), the same in all lanes, into its place.
  __device__ __forceinline__ void insert(float x, int j) {
    const int at = __popc(__ballot_sync(0xffffffffu, before(x, j)));
    const float pv = __shfl_up_sync(0xffffffffu, v, 1);
    const int pi = __shfl_up_sync(0xffffffffu, i, 1), lane = threadIdx.x & 31;
    if (lane == at) {
      v = x;
      i = j;
    } else if (lane > at) {
      v = pv;
      i = pi;
    }
  }
};

// Lists of `top` entries in src (lists after each other), joined by one warp.
template <typename Get>
__device__ __forceinline__ void best_join(Best& best, int top, int lists, Get get) {
  for (int l = 0; l < lists; ++l) {
    for (int k = 0; k < top; ++k) {
      const int2 e = get(l, k);  // descending: the first that is behind the last ends the list
      const float x = __int_as_float(e.x);
      const float lv = __shfl_sync(0xffffffffu, best.v, top - 1);
      const int li = __shfl_sync(0xffffffffu, best.i, top - 1);
      if (e.y < 0 || lv > x || (lv == x && (unsigned)li < (unsigned)e.y)) break;
      best.insert(x, e.y);
    }
  }
}

// One row's results, by a warp that holds the joined sums in every lane and the list one a lane.
template <typename T>
__device__ __forceinline__ void prob_finish(const ProbArgs& A, int64_t r, const Sums& S, const Best& best) {
  const int lane = threadIdx.x & 31;
  const bool none = S.s == 0.f;  // no entry of any probability
  const float L = logf(S.s);
  if (lane == 0) {
    const int64_t t = A.tok.at(r);
    float lp;
    if (t < 0 || t >= A.entries) {
      lp = __int_as_float(0x7fc00000);
    } else {
      const float x = to_f(static_cast<const T*>(A.logits)[r * A.ls + t]);
      const bool out = A.mask && !A.mask[r * A.ms + t];
      lp = none || out ? (S.s != S.s ? S.s : kNone) : (x - S.m) * A.scale - L;
    }
    A.logp[r] = lp;
    A.entropy[r] = none ? 0.f : fmaxf(L - A.scale * (S.w / S.s), 0.f) + 0.f * S.s;
    if (A.stats) {
      A.stats[r] = none ? 0.f : S.m;
      A.stats[A.rows + r] = none ? INFINITY : log2f(S.s);
    }
  }
  if (lane < A.top) {
    const bool nan = S.s != S.s, some = best.i >= 0 && !nan;
    A.top_logp[r * A.top + lane] = nan ? S.s : some ? (best.v - S.m) * A.scale - L : kNone;
    A.top_index[r * A.top + lane] = some ? best.i : -1;
  }
}

template <typename T, int E, bool TOP>
__global__ void __launch_bounds__(kProbThreads) prob_kernel(ProbArgs A) {
  __shared__ float4 sums[kProbWarps];
  __shared__ int2 lists[kProbWarps][32];
  const int64_t r = blockIdx.x / A.parts;
  const int part = blockIdx.x % A.parts;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (A.tok.padded(A.tok.at(r))) {
    if (part == 0) {
      if (threadIdx.x == 0) {
        A.logp[r] = A.entropy[r] = 0.f;
        if (A.stats) {
          A.stats[r] = 0.f;
          A.stats[A.rows + r] = INFINITY;
        }
      }
      if (TOP && threadIdx.x < A.top) {
        A.top_logp[r * A.top + threadIdx.x] = kNone;
        A.top_index[r * A.top + threadIdx.x] = -1;
      }
    }
    return;
  }
  const T* x = static_cast<const T*>(A.logits) + r * A.ls;
  const uint8_t* mask = A.mask ? A.mask + r * A.ms : nullptr;
  const float c = A.scale * kLog2e;
  const int begin = part * A.per, end = min(begin + A.per, A.entries);
  Sums S;
  Best best;
  float last = kNone;  // of the list
  for (int i0 = begin; i0 < end; i0 += kProbThreads * E) {  // the whole warp stays for the list
    const int i = i0 + threadIdx.x * E;
    float v[E];
    if (i < end) {
      const Pack<T, E> p = *reinterpret_cast<const Pack<T, E>*>(x + i);  // E > 1: entries are a multiple of E
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = to_f(p.e[e]);
      if (mask) {
        Pack<uint8_t, E> k = *reinterpret_cast<const Pack<uint8_t, E>*>(mask + i);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!k.e[e]) v[e] = kNone;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = kNone;
    }
    float top = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, v[e]);
    if (top > S.m) S.move(top, c);
    const float m = S.m == kNone ? 0.f : S.m;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = v[e] - m, p = exp2_of(d * c);
      S.s += p;
      S.w = fmaf(p, fmaxf(d, -1e30f), S.w);
    }
    if constexpr (TOP) {
      unsigned who = __ballot_sync(0xffffffffu, top > last);
      while (who) {
        const int src = __ffs(who) - 1;
        who &= who - 1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float y = __shfl_sync(0xffffffffu, v[e], src);
          if (y > last) {
            best.insert(y, i0 + (w * 32 + src) * E + e);
            last = __shfl_sync(0xffffffffu, best.v, A.top - 1);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    S.join(__shfl_xor_sync(0xffffffffu, S.m, o), __shfl_xor_sync(0xffffffffu, S.s, o), __shfl_xor_sync(0xffffffffu, S.w, o), c);
  if (lane == 0) sums[w] = make_float4(S.m, S.s, S.w, 0.f);
  if constexpr (TOP) lists[w][lane] = make_int2(__float_as_int(best.v), best.i);
  __syncthreads();
  if (w) return;
  for (int k = 1; k < kProbWarps; ++k) S.join(sums[k].x, sums[k].y, sums[k].z, c);
  if constexpr (TOP) best_join(best, A.top, kProbWarps - 1, [&](int l, int k) { return lists[l + 1][k]; });
  if (A.parts == 1) {
    prob_finish<T>(A, r, S, best);
  } else {
    if (lane == 0) A.part[blockIdx.x] = make_float4(S.m, S.s, S.w, 0.f);
    if (TOP && lane < A.top) A.part_top[(int64_t)blockIdx.x * A.top + lane] = make_int2(__float_as_int(best.v), best.i);
  }
}

// A warp a row.
template <typename T>
__global__ void __launch_bounds__(128) prob_join_kernel(ProbArgs A) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= A.rows || A.tok.padded(A.tok.at(r))) return;
  const float c = A.scale * kLog2e;
  Sums S;
  for (int p = lane; p < A.parts; p += 32) {
    const float4 q = A.part[r * A.parts + p];
    S.join(q.x, q.y, q.z, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    S.join(__shfl_xor_sync(0xffffffffu, S.m, o), __shfl_xor_sync(0xffffffffu, S.s, o), __shfl_xor_sync(0xffffffffu, S.w, o), c);
  Best best;
  if (A.top) {
    const int2* p = A.part_top + r * A.parts * A.top;
    if (lane < A.top) {
      const int2 q = p[lane];
      best.v = __int_as_float(q.x);
      best.i = q.y;
    }
    best_join(best, A.top, A.parts - 1, [&](int l, int k) { return p[(l + 1) * A.top + k]; });
  }
  prob_finish<T>(A, r, S, best);
}

// ---------------------------------------------------------------- gradient
// d = scale (g (hit - p) - e p (log p + H)), entry by entry: HBM.
template <typename T, int E>
__global__ void __launch_bounds__(kProbThreads) prob_grad_kernel(ProbArgs A) {
  const int64_t r = blockIdx.x / A.parts;
  const int begin = (int)(blockIdx.x % A.parts) * A.per, end = min(begin + A.per, A.entries);
  const int64_t t = A.tok.at(r);
  const bool padded = A.tok.padded(t);
  const T* x = static_cast<const T*>(A.logits) + r * A.ls;
  const uint8_t* mask = A.mask ? A.mask + r * A.ms : nullptr;
  T* out = static_cast<T*>(A.dlogits) + r * A.entries;
  const float g = A.glogp && t >= 0 && t < A.entries ? A.glogp[r] : 0.f, e = A.gentropy ? A.gentropy[r] : 0.f;
  const float m = A.stats[r], l2 = A.stats[A.rows + r], c = A.scale * kLog2e, H = A.entropy[r];
  constexpr float kLn2 = 0.6931471805599453f;
  for (int i = begin + threadIdx.x * E; i < end; i += kProbThreads * E) {
    Pack<T, E> o;
    if (padded) {
#pragma unroll
      for (int k = 0; k < E; ++k) o.e[k] = from_f<T>(0.f);
    } else {
      const Pack<T, E> p = *reinterpret_cast<const Pack<T, E>*>(x + i);
      Pack<uint8_t, E> keep;
      if (mask) keep = *reinterpret_cast<const Pack<uint8_t, E>*>(mask + i);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float q = (to_f(p.e[k]) - m) * c - l2, pr = exp2_of(q);
        // q of an entry without probability is -inf: 0 all the same
        float d = -pr * (g + e * (fmaxf(q, -300.f) * kLn2 + H));
        if (i + k == t) d += g;
        o.e[k] = from_f<T>(mask && !keep.e[k] ? 0.f : d * A.scale);
      }
    }
    *reinterpret_cast<Pack<T, E>*>(out + i) = o;
  }
}

}  // namespace fx
