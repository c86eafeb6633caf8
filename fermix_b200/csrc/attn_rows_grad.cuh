// Gradient of the biased attention, a few rows (queries, then keys) at a time:
//
//   p_ij = 2^((s_ij - lse_i) - lse_low_i),  delta_i = sum_c o_ic do_ic,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//   dtable[h, c] = sum of ds_ij over the pairs of bucket c
//
// A row's ds sum to 0 exactly, and a bucket that holds all of a row's keys gets nothing from it.
// delta from the rounded output would leave its rounding there, so the table's gradient keeps
// a = sum p (do . v) and b = sum p of each row and bucket, and takes sum_i (a - b sum a / sum b).
//
// This is the float32 path above 64 entries, whose three parts of both sides do not fit shared memory.
// Bound: instructions, and few of them products: for every pair a warp walks the edges of the buckets
// (15 comparisons for 32 buckets), reads the table from global memory and takes part in ten
// shuffles beside 12 to 16 FMAs; 60 % of the issue slots are used. 8 x 4 heads of 512 x 512, dim 128: 2.6 ms for
// dk and dv, 2.6 ms for dq and the table, trained 5.2 ms (dim 96 the same), where the plain form in
// library calls takes 0.86 (0.94): the one form here that is slower than that.
//
// Nothing is added atomically: a block owns its rows of dq (or of dk and dv, over all the
// query heads that share the key head), and its groups' partial sums are added in order.
#pragma once
#include "attn_rows.cuh"

namespace fx {

__global__ void __launch_bounds__(kRowsThreads) attn_delta_kernel(const __grid_constant__ AttnArgs A) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * (kRowsThreads / 32) + (threadIdx.x >> 5);
  if (w >= (int64_t)A.B * A.H * A.Lq) return;
  const int64_t i = w % A.Lq, bh = w / A.Lq, h = bh % A.H, b = bh / A.H;
  const float* o = static_cast<const float*>(A.out) + b * A.os[0] + h * A.os[1] + i * A.os[2];
  const float* g = static_cast<const float*>(A.dout) + b * A.dos[0] + h * A.dos[1] + i * A.dos[2];
  float s = 0.f;
  for (int c = lane; c < A.D; c += 32) s = fmaf(o[c], g[c], s);
  s = lanes_sum(s, 32);
  if (lane == 0) A.delta[w] = s;
}

template <typename T>
__global__ void __launch_bounds__(256) attn_zero_kernel(const __grid_constant__ AttnArgs A) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x, token = n / A.D, c = n % A.D, j = token % A.Lk;
  const int64_t bh = token / A.Lk, hk = bh % A.Hk, b = bh / A.Hk;
  if (b >= A.B) return;
  static_cast<T*>(A.dk)[b * A.dks[0] + hk * A.dks[1] + j * A.dks[2] + c] = from_f<T>(0.f);
  static_cast<T*>(A.dv)[b * A.dvs[0] + hk * A.dvs[1] + j * A.dvs[2] + c] = from_f<T>(0.f);
}

// KEYS false: RC query rows against all keys, dq and the table; true: RC keys against all
// query rows of the group, dk and dv.
template <typename T, int LPK, bool VECLOAD, int RC, bool KEYS>
__global__ void __launch_bounds__(kRowsThreads) attn_rows_grad_kernel(const __grid_constant__ AttnArgs A) {
  constexpr int NE = 16 / sizeof(T), GROUPS = kRowsThreads / LPK;
  extern __shared__ float sm[];
  const int G = A.H / A.Hk, nb = A.buckets.num_buckets;
  const int64_t qrows = (int64_t)G * A.Lq, own = KEYS ? A.Lk : qrows, other = KEYS ? qrows : A.Lk;
  const int64_t chunks = (own + RC - 1) / RC, r0 = blockIdx.x % chunks * RC, z = blockIdx.x / chunks;
  const int b = (int)(z / A.Hk), hk = (int)(z % A.Hk);
  const int group = threadIdx.x / LPK, gl = threadIdx.x % LPK, c0 = gl * NE;
  float* hist = sm;  // GROUPS x RC x nb x (a, b)
  if (!KEYS && A.table)
    for (int t = threadIdx.x; t < 2 * GROUPS * RC * nb; t += kRowsThreads) hist[t] = 0.f;
  const T* Q = static_cast<const T*>(A.q) + b * A.qs[0] + (int64_t)hk * G * A.qs[1];
  const T* K = static_cast<const T*>(A.k) + b * A.ks[0] + hk * A.ks[1];
  const T* V = static_cast<const T*>(A.v) + b * A.vs[0] + hk * A.vs[1];
  const T* DO = static_cast<const T*>(A.dout) + b * A.dos[0] + (int64_t)hk * G * A.dos[1];
  const T* table = static_cast<const T*>(A.table) + (int64_t)hk * G * nb;
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_stride : nullptr;

  float x[RC][NE], y[RC][NE], ax[RC][NE], ay[RC][NE], lse[RC], low[RC], del[RC];
  int pos[RC], head[RC];
  bool live[RC];
#pragma unroll
  for (int r = 0; r < RC; ++r) {
    const int64_t row = r0 + r;
    live[r] = row < own && (!KEYS || !mask || mask[row]);
    pos[r] = head[r] = 0;
    lse[r] = low[r] = del[r] = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) x[r][e] = y[r][e] = ax[r][e] = ay[r][e] = 0.f;
    if (!live[r]) continue;
    if (KEYS) {
      pos[r] = attn_k_pos(A, b, row);
      load_entries<T, NE, VECLOAD>(K + row * A.ks[2], c0, A.D, x[r]);
      load_entries<T, NE, VECLOAD>(V + row * A.vs[2], c0, A.D, y[r]);
    } else {
      head[r] = (int)(row / A.Lq);
      const int64_t i = row % A.Lq, at = ((int64_t)b * A.H + hk * G + head[r]) * A.Lq + i;
      pos[r] = attn_q_pos(A, b, i);
      lse[r] = A.lse[at];
      low[r] = A.lse_low ? A.lse_low[at] : 0.f;
      del[r] = A.delta[at];
      load_entries<T, NE, VECLOAD>(Q + head[r] * A.qs[1] + i * A.qs[2], c0, A.D, x[r]);
      load_entries<T, NE, VECLOAD>(DO + head[r] * A.dos[1] + i * A.dos[2], c0, A.D, y[r]);
    }
  }
  __syncthreads();
  for (int64_t base = 0; base < other; base += GROUPS) {
    const int64_t j = base + group;
    float u[NE], w[NE], lse_j = 0.f, low_j = 0.f, del_j = 0.f;
    int pj = 0, hj = 0;
    bool there = j < other;
    if (!KEYS && there && mask) there = mask[j];
#pragma unroll
    for (int e = 0; e < NE; ++e) u[e] = w[e] = 0.f;
    if (there) {
      if (KEYS) {
        hj = (int)(j / A.Lq);
        const int64_t i = j % A.Lq, at = ((int64_t)b * A.H + hk * G + hj) * A.Lq + i;
        pj = attn_q_pos(A, b, i);
        lse_j = A.lse[at];
        low_j = A.lse_low ? A.lse_low[at] : 0.f;
        del_j = A.delta[at];
        load_entries<T, NE, VECLOAD>(Q + hj * A.qs[1] + i * A.qs[2], c0, A.D, u);
        load_entries<T, NE, VECLOAD>(DO + hj * A.dos[1] + i * A.dos[2], c0, A.D, w);
      } else {
        pj = attn_k_pos(A, b, j);
        load_entries<T, NE, VECLOAD>(K + j * A.ks[2], c0, A.D, u);
        load_entries<T, NE, VECLOAD>(V + j * A.vs[2], c0, A.D, w);
      }
    }
#pragma unroll
    for (int r = 0; r < RC; ++r) {
      float s = 0.f, dp = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        s = fmaf(x[r][e], u[e], s);
        dp = fmaf(y[r][e], w[e], dp);
      }
      s = lanes_sum(s, LPK) * A.scale2;
      dp = lanes_sum(dp, LPK);
      const int d = KEYS ? pos[r] - pj : pj - pos[r];
      const float L = KEYS ? lse_j : lse[r], de = KEYS ? del_j : del[r];
      float p = 0.f, ds = 0.f;
      if (there && live[r] && !(A.causal && d > 0) && L != -INFINITY) {
        int c = 0;
        if (A.table) {
          c = bucket_of(A.buckets, clamp_reach(d, A.buckets.reach));
          s += bias2(to_f(table[(KEYS ? hj : head[r]) * nb + c]));
        }
        p = exp2f((s - L) - (KEYS ? low_j : low[r]));
        ds = p * (dp - de);
        if (!KEYS && A.table && gl == 0) {
          hist[((group * RC + r) * nb + c) * 2] += p * dp;
          hist[((group * RC + r) * nb + c) * 2 + 1] += p;
        }
      }
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        ax[r][e] = fmaf(ds, u[e], ax[r][e]);
        if (KEYS) ay[r][e] = fmaf(p, w[e], ay[r][e]);
      }
    }
  }
  __syncthreads();
  if (!KEYS && A.table) {
    for (int t = threadIdx.x; t < 2 * RC * nb; t += kRowsThreads)
      for (int g = 1; g < GROUPS; ++g) hist[t] += hist[g * 2 * RC * nb + t];
    __syncthreads();
    for (int t = threadIdx.x; t < RC * nb; t += kRowsThreads) {
      const int64_t row = r0 + t / nb;
      if (row >= own) continue;
      float sa = 0.f, sb = 0.f;
      for (int c = 0; c < nb; ++c) {
        sa += hist[(t / nb * nb + c) * 2];
        sb += hist[(t / nb * nb + c) * 2 + 1];
      }
      const int64_t h = hk * G + row / A.Lq, i = row % A.Lq;
      A.dpart[((h * A.B + b) * A.Lq + i) * nb + t % nb] =
          sb == 0.f ? 0.f : fmaf(-hist[t * 2 + 1], sa / sb, hist[t * 2]);
    }
    __syncthreads();
  }
  float* so = sm;  // GROUPS x RC x LPK x NE
  for (int which = 0; which < (KEYS ? 2 : 1); ++which) {
#pragma unroll
    for (int r = 0; r < RC; ++r)
#pragma unroll
      for (int e = 0; e < NE; ++e) so[((group * RC + r) * LPK + gl) * NE + e] = which ? ay[r][e] : ax[r][e] * A.scale;
    __syncthreads();
    for (int t = threadIdx.x; t < RC * A.D; t += kRowsThreads) {
      const int r = t / A.D, c = t % A.D;
      const int64_t row = r0 + r;
      if (row >= own) continue;
      float v = 0.f;
      for (int g = 0; g < GROUPS; ++g) v += so[(g * RC + r) * LPK * NE + c];
      if (KEYS) {
        if (which) static_cast<T*>(A.dv)[b * A.dvs[0] + hk * A.dvs[1] + row * A.dvs[2] + c] = from_f<T>(v);
        else static_cast<T*>(A.dk)[b * A.dks[0] + hk * A.dks[1] + row * A.dks[2] + c] = from_f<T>(v);
      } else {
        const int h = hk * G + (int)(row / A.Lq);
        static_cast<T*>(A.dq)[b * A.dqs[0] + h * A.dqs[1] + (row % A.Lq) * A.dqs[2] + c] = from_f<T>(v);
      }
    }
    __syncthreads();
  }
}

}  // namespace fx
