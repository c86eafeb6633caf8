// Attention with the position bias, a few query rows at a time, split over the keys.
//
//   s_j = scale q . k_j + table[h, bucket(kp_j - qp)],  o = sum_j e^{s_j} v_j / sum_j e^{s_j}
//
// One pass over the keys with the running maximum and sum; exponentials in base 2 (the scale
// and the table carry the factor log2 e). A block takes up to RC rows of the queries that
// share a key head and one part of the keys; LPK lanes share a key, each with NE of its
// entries, and every group of lanes keeps a running (m, l, o) of its own, joined at the end.
// With several parts each leaves (m, l, o) in the workspace and attn_join_kernel joins them.
//
// Bound: FMA instructions and the sums over lanes (each row of a key head its own dot products). One query
// of 8 x 8 heads on 2 key heads of 4096 keys, dim 64 in float32 (34 MB): 40 us, 0.84 TB/s; 4 queries 93 us.
#pragma once
#include "block_common.cuh"

namespace fx {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowsThreads = 128;

struct AttnArgs {
  const void *q, *k, *v, *table;
  int64_t qs[3], ks[3], vs[3];  // element strides: batch, head, token
  const uint8_t* mask;
  int64_t mask_stride;
  const int *q_pos, *k_pos;
  int64_t q_pos_stride, k_pos_stride;
  void* out;
  int64_t os[3];
  float *lse, *lse_low;  // (batch, heads, q_len) each
  const void* dout;
  int64_t dos[3];
  void *dq, *dk, *dv;
  int64_t dqs[3], dks[3], dvs[3];
  float* delta;   // (batch, heads, q_len)
  float* dpart;   // partial table gradients (heads, parts, num_buckets)
  float* lut;     // table by distance, base 2 (heads, 2 reach + 1)
  float* part;    // split parts: (rows, splits, part_step(dim)): m, l, -, -, o
  int64_t Lq, Lk;
  int64_t split_keys;
  int B, H, Hk, D, causal, splits;
  uint32_t polls;  // of each bounded wait
  float scale2;  // scale log2 e
  float scale;
  BucketArgs buckets;
};

// Floats of a split part, whole 16-byte pieces.
__host__ __device__ constexpr int part_step(int dim) { return (dim + 3) / 4 * 4 + 4; }

// The table's value in base 2; finite entries stay finite.
__device__ __forceinline__ float bias2(float t) {
  const float b = t * kLog2e;
  return isfinite(t) ? fminf(fmaxf(b, -3.4028234e38f), 3.4028234e38f) : b;
}

// The logarithm of a row's sum of exponentials, l to the reference m, as two floats: beside an m of 1e9
// log2 l would be lost, and the gradient's probabilities with it. (Knuth's sum of two and its error.)
__device__ __forceinline__ void store_lse(const AttnArgs& A, int64_t row, float m, float l, bool broken = false) {
  const float g = log2f(l), hi = m + g, z = hi - m;
  A.lse[row] = broken ? NAN : l == 0.f ? -INFINITY : hi;
  if (A.lse_low) A.lse_low[row] = l == 0.f ? 0.f : (m - (hi - z)) + (g - z);
}

template <typename T, int NE, bool VECLOAD>
__device__ __forceinline__ void load_entries(const T* p, int c0, int D, float (&o)[NE]) {
  if (VECLOAD) {
    if (c0 < D) {
      const Pack<T, NE> v = *reinterpret_cast<const Pack<T, NE>*>(p + c0);
#pragma unroll
      for (int e = 0; e < NE; ++e) o[e] = to_f(v.e[e]);
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e) o[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = c0 + e < D ? to_f(p[c0 + e]) : 0.f;
  }
}

__device__ __forceinline__ int attn_q_pos(const AttnArgs& A, int b, int64_t i) {
  return A.q_pos ? A.q_pos[b * A.q_pos_stride + i] : (int)(A.Lk - A.Lq + i);
}
__device__ __forceinline__ int attn_k_pos(const AttnArgs& A, int b, int64_t j) {
  return A.k_pos ? A.k_pos[b * A.k_pos_stride + j] : (int)j;
}

// Blocks: parts of the keys, then chunks of the rows of a key head, then key heads, batches.
template <typename T, int LPK, bool VECLOAD, int RC>
__global__ void __launch_bounds__(kRowsThreads) attn_rows_kernel(const __grid_constant__ AttnArgs A) {
  constexpr int NE = 16 / sizeof(T), U = 4, GROUPS = kRowsThreads / LPK;
  extern __shared__ float lut[];  // RC x (2 reach + 1), then the joins
  const int G = A.H / A.Hk, reach = A.buckets.reach, span = 2 * reach + 1;
  const int64_t rows = (int64_t)G * A.Lq, chunks = (rows + RC - 1) / RC;
  const int part = blockIdx.x % A.splits;
  const int64_t r0 = blockIdx.x / A.splits % chunks * RC, z = blockIdx.x / A.splits / chunks;
  const int b = (int)(z / A.Hk), hk = (int)(z % A.Hk);
  const int group = threadIdx.x / LPK, gl = threadIdx.x % LPK, c0 = gl * NE;

  int qp[RC];
  float q[RC][NE], o[RC][NE], m[RC], l[RC];
#pragma unroll
  for (int r = 0; r < RC; ++r) {
    const int64_t row = r0 + r;
    qp[r] = 0;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) q[r][e] = o[r][e] = 0.f;
    if (row < rows) {
      const int h = hk * G + (int)(row / A.Lq);
      const int64_t i = row % A.Lq;
      qp[r] = attn_q_pos(A, b, i);
      load_entries<T, NE, VECLOAD>(static_cast<const T*>(A.q) + b * A.qs[0] + h * A.qs[1] + i * A.qs[2], c0, A.D,
                                   q[r]);
#pragma unroll
      for (int e = 0; e < NE; ++e) q[r][e] *= A.scale2;
      if (A.table) {
        const T* t = static_cast<const T*>(A.table) + (int64_t)h * A.buckets.num_buckets;
        for (int d = threadIdx.x; d < span; d += kRowsThreads)
          lut[r * span + d] = bias2(to_f(t[bucket_of(A.buckets, d - reach)]));
      }
    }
  }
  __syncthreads();
  const int64_t j0 = part * A.split_keys;
  const int64_t j1 = j0 + A.split_keys < A.Lk ? j0 + A.split_keys : A.Lk;
  const T* K = static_cast<const T*>(A.k) + b * A.ks[0] + hk * A.ks[1];
  const T* V = static_cast<const T*>(A.v) + b * A.vs[0] + hk * A.vs[1];
  for (int64_t base = j0; base < j1; base += GROUPS * U) {
    float k[U][NE], v[U][NE];
    int kp[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = base + u * GROUPS + group;
      live[u] = j < j1 && (!A.mask || A.mask[b * A.mask_stride + j]);
      kp[u] = 0;
      if (live[u]) {
        kp[u] = attn_k_pos(A, b, j);
        load_entries<T, NE, VECLOAD>(K + j * A.ks[2], c0, A.D, k[u]);
        load_entries<T, NE, VECLOAD>(V + j * A.vs[2], c0, A.D, v[u]);
      } else {
#pragma unroll
        for (int e = 0; e < NE; ++e) k[u][e] = v[u][e] = 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < RC; ++r) {
      float s[U], top = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) d = fmaf(q[r][e], k[u][e], d);
        s[u] = lanes_sum(d, LPK);
        if (A.table && live[u]) s[u] += lut[r * span + clamp_reach(kp[u] - qp[r], reach) + reach];
        if (!live[u] || (A.causal && kp[u] > qp[r])) s[u] = -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float ref = top == -INFINITY ? 0.f : top;
      const float f = exp2f(m[r] - ref);
      m[r] = top;
      l[r] *= f;
#pragma unroll
      for (int e = 0; e < NE; ++e) o[r][e] *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = exp2f(s[u] - ref);
        l[r] += p;
#pragma unroll
        for (int e = 0; e < NE; ++e) o[r][e] = fmaf(p, v[u][e], o[r][e]);
      }
    }
  }
  // join the groups: (m, l) and then o through shared memory, group after group
  __syncthreads();
  float* sm = lut;                      // GROUPS x RC
  float* sl = sm + GROUPS * RC;         // GROUPS x RC
  float* so = sl + GROUPS * RC;         // GROUPS x RC x LPK x NE
#pragma unroll
  for (int r = 0; r < RC; ++r) {
    if (gl == 0) {
      sm[group * RC + r] = m[r];
      sl[group * RC + r] = l[r];
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) so[((group * RC + r) * LPK + gl) * NE + e] = o[r][e];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < RC * A.D; t += kRowsThreads) {
    const int r = t / A.D, c = t % A.D;
    const int64_t row = r0 + r;
    if (row >= rows) continue;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
    for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, sm[g * RC + r]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int g = 0; g < GROUPS; ++g) {
      const float f = exp2f(sm[g * RC + r] - ref);
      sum = fmaf(sl[g * RC + r], f, sum);
      acc = fmaf(so[(g * RC + r) * LPK * NE + c], f, acc);
    }
    if (A.splits > 1) {
      float* p = A.part + ((z * rows + row) * A.splits + part) * part_step(A.D);
      p[4 + c] = acc;
      if (c == 0) {
        p[0] = top;
        p[1] = sum;
      }
    } else {
      const int h = hk * G + (int)(row / A.Lq);
      const int64_t i = row % A.Lq;
      static_cast<T*>(A.out)[b * A.os[0] + h * A.os[1] + i * A.os[2] + c] = from_f<T>(sum == 0.f ? 0.f : acc / sum);
      if (A.lse && c == 0) store_lse(A, ((int64_t)b * A.H + h) * A.Lq + i, top, sum);
    }
  }
}

// A block a row: the parts' (m, l, o) into the output. The parts' weights first, side by side,
// then a thread an entry.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) attn_join_kernel(const __grid_constant__ AttnArgs A) {
  static_assert(FX_ATTN_MAX_DIM <= kRowsThreads);
  __shared__ float red[kRowsThreads / 32], weight[kRowsThreads];
  const int G = A.H / A.Hk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = (int64_t)G * A.Lq, w = blockIdx.x, z = w / rows, row = w % rows;
  const int b = (int)(z / A.Hk), h = (int)(z % A.Hk) * G + (int)(row / A.Lq);
  const int64_t i = row % A.Lq;
  const int step = part_step(A.D);
  const float* p = A.part + w * A.splits * step;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < A.splits; s += kRowsThreads) top = fmaxf(top, p[(int64_t)s * step]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRowsThreads / 32; ++k) top = fmaxf(top, red[k]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc = 0.f;
  for (int s0 = 0; s0 < A.splits; s0 += kRowsThreads) {
    const int n = A.splits - s0 < kRowsThreads ? A.splits - s0 : kRowsThreads;
    __syncthreads();
    if (threadIdx.x < n) {
      const float* q = p + (int64_t)(s0 + threadIdx.x) * step;
      const float f = exp2f(q[0] - ref);
      weight[threadIdx.x] = f;
      sum = fmaf(q[1], f, sum);
    }
    __syncthreads();
    if (threadIdx.x < A.D) {
      const float* q = p + (int64_t)s0 * step + 4 + threadIdx.x;
#pragma unroll 8
      for (int s = 0; s < n; ++s) acc = fmaf(q[(int64_t)s * step], weight[s], acc);
    }
  }
  sum = lanes_sum(sum, 32);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < kRowsThreads / 32; ++k) sum += red[k];
  if (threadIdx.x < A.D)
    static_cast<T*>(A.out)[b * A.os[0] + h * A.os[1] + i * A.os[2] + threadIdx.x] =
        from_f<T>(sum == 0.f ? 0.f : acc / sum);
  if (A.lse && threadIdx.x == 0) store_lse(A, ((int64_t)b * A.H + h) * A.Lq + i, top, sum);
}

// The same with a warp a row, for many rows of few parts. A lane weighs a part, 32 at a time, and adds
// up to four entries of the row.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) attn_join_warp_kernel(const __grid_constant__ AttnArgs A) {
  constexpr int NE = FX_ATTN_MAX_DIM / 32;
  const int lane = threadIdx.x & 31, step = part_step(A.D);
  const int64_t w = (int64_t)blockIdx.x * (kRowsThreads / 32) + (threadIdx.x >> 5);
  if (w >= (int64_t)A.B * A.H * A.Lq) return;
  const int64_t i = w % A.Lq, bh = w / A.Lq, h = bh % A.H, b = bh / A.H;
  const float* p = A.part + w * A.splits * step;
  float top = -INFINITY;
  for (int s = lane; s < A.splits; s += 32) top = fmaxf(top, p[(int64_t)s * step]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc[NE] = {};
  for (int s0 = 0; s0 < A.splits; s0 += 32) {
    const float* q = p + (int64_t)s0 * step;
    const int n = A.splits - s0 < 32 ? A.splits - s0 : 32;
    float f = 0.f;
    if (lane < n) {
      f = exp2f(q[lane * step] - ref);
      sum = fmaf(q[lane * step + 1], f, sum);
    }
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float weight = __shfl_sync(0xffffffffu, f, s);
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (lane + 32 * e < A.D) acc[e] = fmaf(q[s * step + 4 + lane + 32 * e], weight, acc[e]);
    }
  }
  sum = lanes_sum(sum, 32);
  T* out = static_cast<T*>(A.out) + b * A.os[0] + h * A.os[1] + i * A.os[2];
#pragma unroll
  for (int e = 0; e < NE; ++e)
    if (lane + 32 * e < A.D) out[lane + 32 * e] = from_f<T>(sum == 0.f ? 0.f : acc[e] / sum);
  if (A.lse && lane == 0) store_lse(A, w, top, sum);
}

}  // namespace fx
