// Gradient of the biased attention on the tensor cores, in three launches: the rows' products
// delta = o . do and the table by distance (attn_prep_kernel), then dk and dv by blocks of keys
// (attn_dkv_kernel) and dq and the table's gradient by blocks of queries (attn_dq_kernel). Each block
// owns what it writes, so nothing is added atomically; the scores are formed twice for that
// (seven products instead of five).
//
//   p = 2^(((scale2 q.k + bias2) - lse) - lse_low),  ds = p (do.v - delta)
//   dv = p^T do, dk = scale ds^T q, dq = scale ds k
//
// The bias is added first and the logarithm of the row's sum taken off as two floats, the forward's
// order: what a huge bias absorbed there is absorbed here.
//
// In both, a thread holds one row of the 128-row block (TMEM lane), p and ds go back to TMEM as
// the A operand of the second products, and the 64-row tiles of the other side stream through
// shared memory, each read K-major for the scores and MN-major for the second product.
//
// Bound: the latency of the threads' work between the matrix instructions (TMEM loads, exponentials,
// operands back to TMEM, in dq the histogram) at two blocks an SM: 0.41 (dkv) and 0.37 (dq) of the issue
// slots are used, 0.16 and 0.08 of the tensor pipe. Within a block the tensor work and the threads' work
// take turns: the next tile's scores have to wait until p and ds, which lie over this tile's, are read.
// Measured: 64 x 8 heads of 512 x 512, dim 64 in bfloat16, three quarters of the keys live: dkv 198 us, dq
// 230 us; causal 8 heads of 4095: 141 and 148 us; float32 512 x 4 heads of 128 x 128, dim 32: 201 and
// 219 us (spills of 56 and 72 bytes a thread).
//
// Fewer bits, and why: p and ds are rounded to bfloat16 for the second products, whose operands are of that
// type (three parts each in float32, which keep 24 bits). delta = o . do is formed from the output as
// stored, which spares a second pass over the values: its rounding adds up to 2^-9 |o| |do| to every dp of
// a row, so dq and dk of a row whose ds cancel (a sharp softmax over nearly equal values) carry that
// much beside their own; the table's gradient, which sums ds over whole rows, is mended for it below.
// Measured, of dq's norm: ds 1.7e-3, as much as the rounding of the result itself; delta 0.4 to 0.9e-3
// from the output and as much from the forward's p; in all 2.4 to 2.6e-3, float32 throughout 1.7e-3.
#pragma once
#include "attn_tc.cuh"

namespace fx {
namespace tc {

constexpr int kGradN = 64;  // rows of a streamed tile

// delta of every query row (LPR lanes a row), and the blocks past them: the table by distance
// in base 2, lut[h, d + reach].
template <typename T, int LPR, bool VEC>
__global__ void __launch_bounds__(256) attn_prep_kernel(const __grid_constant__ AttnArgs A, int64_t row_blocks) {
  constexpr int NE = 16 / sizeof(T);
  if ((int64_t)blockIdx.x >= row_blocks) {
    const int span = 2 * A.buckets.reach + 1, nb = A.buckets.num_buckets;
    const int64_t i = ((int64_t)blockIdx.x - row_blocks) * 256 + threadIdx.x;
    if (i < (int64_t)A.H * span)
      A.lut[i] =
          bias2(to_f(static_cast<const T*>(A.table)[i / span * nb + bucket_of(A.buckets, (int)(i % span) - A.buckets.reach)]));
    return;
  }
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const bool there = row < (int64_t)A.B * A.H * A.Lq;
  float s = 0.f;
  if (there) {
    const int64_t i = row % A.Lq, bh = row / A.Lq, h = bh % A.H, b = bh / A.H;
    float x[NE], y[NE];
    load_entries<T, NE, VEC>(static_cast<const T*>(A.out) + b * A.os[0] + h * A.os[1] + i * A.os[2],
                             threadIdx.x % LPR * NE, A.D, x);
    load_entries<T, NE, VEC>(static_cast<const T*>(A.dout) + b * A.dos[0] + h * A.dos[1] + i * A.dos[2],
                             threadIdx.x % LPR * NE, A.D, y);
#pragma unroll
    for (int e = 0; e < NE; ++e) s = fmaf(x[e], y[e], s);
  }
  s = lanes_sum(s, LPR);
  if (there && threadIdx.x % LPR == 0) A.delta[row] = s;
}

// Row r of the block from TMEM (columns col ..), times f and added to p (held) or in its place, to p (zero: 0).
template <typename T, int DIM>
__device__ __forceinline__ void store_row(uint32_t taddr, T* p, int64_t step, int dim, float f, bool held, bool zero,
                                          bool valid) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = dim % V == 0 && ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(step * sizeof(T))) & 15) == 0;
#pragma unroll
  for (int c = 0; c < DIM; c += 16) {
    if (c < dim) {
      uint32_t o[16];
      ld16(taddr + c, o);
      tmem_wait_ld();
      alignas(16) T r[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) r[e] = from_f<T>(zero ? 0.f : __uint_as_float(o[e]) * f);
      if (sizeof(T) == 4 && held && valid && !zero) {
#pragma unroll
        for (int e = 0; e < 16; e += V) {
          if (vec && c + e < dim) {
            const Pack<T, V> was = *reinterpret_cast<const Pack<T, V>*>(p + c + e);
#pragma unroll
            for (int n = 0; n < V; ++n) r[e + n] = from_f<T>(to_f(r[e + n]) + to_f(was.e[n]));
          } else if (!vec) {
#pragma unroll
            for (int n = 0; n < V; ++n)
              if (c + e + n < dim) r[e + n] = from_f<T>(to_f(r[e + n]) + to_f(p[c + e + n]));
          }
        }
      }
      if (valid) {
        if (vec) {
#pragma unroll
          for (int e = 0; e < 16; e += V)
            if (c + e < dim) *reinterpret_cast<Pack<T, V>*>(p + c + e) = *reinterpret_cast<Pack<T, V>*>(r + e);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c + e < dim) p[c + e] = r[e];
        }
      }
    }
  }
}

// ---------------------------------------------------------------- dk, dv
template <int NS, typename L, int ST>
struct DkvShape {
  static constexpr int kThreads = 384;  // 8 warps on the scores, one issuing, three loading
  static constexpr uint32_t kRow = NS * L::DC * L::RB, kOwn = 128 * kRow, kTile = kGradN * kRow;
  static constexpr uint32_t kTileBytes = 2 * kOwn + 2 * ST * kTile;
  // TMEM: scores, do.v, [third parts of p and ds], dv, dk. p and ds of 16 columns take the place of
  // those 16 once read: 8 columns a part, two parts; the third has 32 columns of its own.
  static constexpr int kDp = kGradN, kP3 = 2 * kGradN, kDs3 = kP3 + 32;
  static constexpr int kDv = NS == 1 ? 2 * kGradN : kDs3 + 32, kDk = kDv + L::kDim;
  static constexpr int kCols = kDk + L::kDim, kAlloc = kCols <= 256 ? 256 : 512;
  static constexpr int kInfo = ST + 1;
  static constexpr int kBlocks = kAlloc <= 256 && kTileBytes <= 104 * 1024 ? 2 : 1;  // an SM holds
  // Columns of a step: 8 fit 80 registers without spills; the second part of 16 columns takes the
  // place of their latter half, which has to be read by then.
  static constexpr int kStepCols = NS == 1 ? 8 : 16;
};

struct alignas(16) QueryInfo {
  TileInfo<kGradN> t;
  // the parts of -lse (-inf: a row without keys, or past the end) and -delta
  float lse[kGradN], low[kGradN], delta[kGradN];
};

template <typename T, int NS, typename L, int ST, int LOAD>
__global__ void __launch_bounds__(DkvShape<NS, L, ST>::kThreads, DkvShape<NS, L, ST>::kBlocks)
    attn_dkv_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TmaMaps M) {
  using S = DkvShape<NS, L, ST>;
  constexpr bool TMA = LOAD == LOAD_TMA, PIECES = LOAD == LOAD_PIECES;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char *sK = sm, *sV = sm + S::kOwn, *sQ = sV + S::kOwn, *sO = sQ + ST * S::kTile;
  float* lut = reinterpret_cast<float*>(sm + S::kTileBytes);
  __shared__ QueryInfo info[S::kInfo];
  __shared__ uint64_t full[ST], empty[ST], loaded[ST], own, sfull, pfull, done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = A.H / A.Hk;

  // key blocks slow, longest first under a causal order
  const int64_t heads = (int64_t)A.B * A.Hk, nk = (A.Lk + 127) / 128;
  const bool ordered = A.causal && !A.q_pos && !A.k_pos;
  const int64_t kb = ordered ? blockIdx.x / heads : blockIdx.x % nk;
  const int64_t bh = ordered ? blockIdx.x % heads : blockIdx.x / nk;
  const int b = (int)(bh / A.Hk), hk = (int)(bh % A.Hk);
  const int64_t j0 = kb * 128;
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_stride : nullptr;
  const int reach = A.buckets.reach, span = 2 * reach + 1;

  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], TMA ? 64 : 96);
      mbar_init(&empty[i], 1);
      mbar_init(&loaded[i], 2);  // the copies, and what goes with the rows
    }
    mbar_init(&own, 1);
    mbar_init(&sfull, 1);
    mbar_init(&pfull, 256);
    mbar_init(&done, 1);
    fence_mbar_init();
    if constexpr (TMA) {
      mbar_arrive_expect_tx(&own, 2 * S::kOwn);
      tma_tile<L>(sK, M, MAP_K, 128, j0, hk, b, &own);
      tma_tile<L>(sV, M, MAP_V, 128, j0, hk, b, &own);
    }
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  const auto key_live = [&](int r) { return j0 + r < A.Lk && (!mask || mask[j0 + r]); };
  if constexpr (TMA) {
    __syncthreads();
    wait(&own, 0, &abort_flag, A.polls);
    if (mask) {
      clear_rows<L>(sK, 128, tid, S::kThreads, key_live);
      clear_rows<L>(sV, 128, tid, S::kThreads, key_live);
    }
  } else {
    const T* K = static_cast<const T*>(A.k) + b * A.ks[0] + hk * A.ks[1] + j0 * A.ks[2];
    const T* V = static_cast<const T*>(A.v) + b * A.vs[0] + hk * A.vs[1] + j0 * A.vs[2];
    load_tile<T, NS, PIECES, 128, L>(sK, K, A.ks[2], A.D, tid, S::kThreads, key_live);
    load_tile<T, NS, PIECES, 128, L>(sV, V, A.vs[2], A.D, tid, S::kThreads, key_live);
  }
  fence_proxy_async_smem();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_slot, polls = A.polls;
  const int64_t nq = (A.Lq + kGradN - 1) / kGradN;
  int64_t q0 = 0;  // the first query tile that sees a key of this block
  if (ordered) {
    const int64_t i = j0 - (A.Lk - A.Lq);
    q0 = i > 0 ? i / kGradN : 0;
    if (q0 > nq) q0 = nq;
  }
  const int64_t per = nq - q0, tiles = per * G;

  if (warp < 8) {
    const int wg = warp >> 2, r = tid & 127;
    const int64_t j = j0 + r;
    const bool live = key_live(r);
    const int kp = live ? attn_k_pos(A, b, j) : 0;
    const int klo = __reduce_min_sync(0xffffffffu, live ? kp : INT32_MAX);
    const int khi = __reduce_max_sync(0xffffffffu, live ? kp : INT32_MIN);
    const uint32_t base = tmem + ((uint32_t)(warp & 3) << 21);
    // the sums so far to dv (or dk)
    const auto keep = [&](float f, bool held, bool zero) {
      const bool dv = wg == 0;
      const int64_t* st = dv ? A.dvs : A.dks;
      T* p = static_cast<T*>(dv ? A.dv : A.dk) + b * st[0] + hk * st[1] + j * st[2];
      store_row<T, L::kDim>(base + (dv ? S::kDv : S::kDk), p, st[2], A.D, dv ? f : f * A.scale, held, zero, j < A.Lk);
    };
    for (int64_t it = 0; it < tiles; ++it) {
      if (A.table && it % per == 0) {  // the next head's table
        named_barrier(2, 256);
        const float* src = A.lut + (int64_t)(hk * G + it / per) * span;
        for (int d = tid; d < span; d += 256) lut[d] = src[d];
        named_barrier(2, 256);
      }
      const QueryInfo& I = info[it % S::kInfo];
      wait(&sfull, it & 1, &abort_flag, polls);
      fence_after_sync();
      if (NS > 1 && it > 0 && starts<NS>(it)) keep(1.f, it > kRest, false);
      const int qlo = I.t.lo[wg], qhi = I.t.hi[wg];
      const bool some = I.t.live[wg] != 0 && klo <= khi;
      const bool above = (int64_t)klo - qhi >= reach, below = (int64_t)khi - qlo <= -reach;
      const bool each = some && ((A.table && !above && !below) || (A.causal && khi > qlo));
      const float flat = A.table && some && !each ? lut[above ? 2 * reach : 0] : 0.f;
#pragma unroll 1  // one copy of the code, to stay in the instruction cache
      for (int c = 0; c < 32; c += S::kStepCols) {
        const int col = wg * 32 + c;
        uint32_t s[S::kStepCols], dp[S::kStepCols];
        ld_cols<S::kStepCols>(base + col, s);
        ld_cols<S::kStepCols>(base + S::kDp + col, dp);
        tmem_wait_ld();
        uint32_t wp[NS][S::kStepCols / 2], wd[NS][S::kStepCols / 2];
        float bias[S::kStepCols];
#pragma unroll
        for (int e = 0; e < S::kStepCols; ++e) bias[e] = flat;
        if (each) {
          int q[S::kStepCols];
#pragma unroll
          for (int e = 0; e < S::kStepCols; e += 4) {
            const int4 v = *reinterpret_cast<const int4*>(&I.t.pos[col + e]);
            q[e] = v.x;
            q[e + 1] = v.y;
            q[e + 2] = v.z;
            q[e + 3] = v.w;
          }
          if (A.table) {
#pragma unroll
            for (int e = 0; e < S::kStepCols; ++e) bias[e] = lut[__vimin_s32_relu(kp + reach - q[e], 2 * reach)];
          }
          if (A.causal) {
#pragma unroll
            for (int e = 0; e < S::kStepCols; ++e)
              if (kp > q[e]) bias[e] = -INFINITY;
          }
        }
        const uint64_t ss = both(A.scale2, A.scale2);
#pragma unroll
        for (int e = 0; e < S::kStepCols; e += 4) {
          const float4 de = *reinterpret_cast<const float4*>(&I.delta[col + e]);
          const float4 hi = *reinterpret_cast<const float4*>(&I.lse[col + e]);
          const float4 lo = *reinterpret_cast<const float4*>(&I.low[col + e]);
          const uint64_t d2[2] = {both(de.x, de.y), both(de.z, de.w)};
          const uint64_t h2[2] = {both(hi.x, hi.y), both(hi.z, hi.w)}, l2[2] = {both(lo.x, lo.y), both(lo.z, lo.w)};
#pragma unroll
          for (int f = 0; f < 4; f += 2) {
            const int i0 = e + f;
            float v0, v1;
            const uint64_t sc =
                fma_both(both(__uint_as_float(s[i0]), __uint_as_float(s[i0 + 1])), ss, both(bias[i0], bias[i0 + 1]));
            halves(add_both(add_both(sc, h2[f / 2]), l2[f / 2]), v0, v1);
            const float p0 = ex2(v0), p1 = ex2(v1);
            float d0, d1;
            halves(mul_both(both(p0, p1),
                            add_both(both(__uint_as_float(dp[i0]), __uint_as_float(dp[i0 + 1])), d2[f / 2])),
                   d0, d1);
            uint32_t o[NS];
            split2<NS>(p0, p1, o);
#pragma unroll
            for (int i = 0; i < NS; ++i) wp[i][i0 / 2] = o[i];
            split2<NS>(d0, d1, o);
#pragma unroll
            for (int i = 0; i < NS; ++i) wd[i][i0 / 2] = o[i];
          }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          // place within the 16 columns' 8 of a part
          const int at = (col & ~15) + (col & 15) / 2;
          st_cols<S::kStepCols / 2>(base + (i < 2 ? at + i * 8 : S::kP3 + col / 2), wp[i]);
          st_cols<S::kStepCols / 2>(base + (i < 2 ? S::kDp + at + i * 8 : S::kDs3 + col / 2), wd[i]);
        }
      }
      tmem_wait_st();
      fence_before_sync();
      arrive(&pfull);
    }
    if (tiles > 0) {
      wait(&sfull, tiles & 1, &abort_flag, polls);
      fence_after_sync();
    }
    keep(abort_flag ? NAN : 1.f, NS > 1 && tiles > kRest, !live || tiles == 0);
  } else if (warp == 8) {
    if (lane == 0 && tiles > 0) {
      const uint32_t id_s = idesc_bf16(128, kGradN, false), id_o = idesc_bf16(128, (A.D + 15) / 16 * 16, true);
      const uint32_t aK = smem_u32(sK), aV = smem_u32(sV);
      const auto p_at = [=](int part, int k) { return tmem + (part < 2 ? k * 16 + part * 8 : S::kP3 + k * 8); };
      const auto ds_at = [=](int part, int k) {
        return tmem + (part < 2 ? S::kDp + k * 16 + part * 8 : S::kDs3 + k * 8);
      };
      for (int64_t it = 0; it < tiles; ++it) {
        const int st = (int)(it % ST);
        const uint32_t aQ = smem_u32(sQ) + st * S::kTile, aO = smem_u32(sO) + st * S::kTile;
        wait(&full[st], (it / ST) & 1, &abort_flag, polls);
        scores<NS, 128, kGradN, L>(tmem, aK, aQ, A.D, id_s);
        scores<NS, 128, kGradN, L>(tmem + S::kDp, aV, aO, A.D, id_s);
        mma_commit(&sfull);
        wait(&pfull, it & 1, &abort_flag, polls);
        fence_after_sync();
        values<NS, kGradN, L>(tmem + S::kDv, aO, id_o, !starts<NS>(it), p_at);
        values<NS, kGradN, L>(tmem + S::kDk, aQ, id_o, !starts<NS>(it), ds_at);
        mma_commit(&empty[st]);
      }
      mma_commit(&sfull);
      mma_commit(&done);
      mbar_wait(&done, 0, kDrainPolls);
    }
  } else {
    const int t = tid - 288, w = t >> 5;
    // lse, delta and positions of 32 rows of a tile, by a warp
    const auto fill = [&](int64_t it, int sub) {
      QueryInfo& I = info[it % S::kInfo];
      const int64_t i0 = (q0 + it % per) * kGradN, row = ((int64_t)b * A.H + hk * G + it / per) * A.Lq;
      const int e = sub * kSub + lane;
      const float ls = i0 + e < A.Lq ? A.lse[row + i0 + e] : -INFINITY;
      const uint32_t bits = fill_info<kGradN>(
          I.t, sub, [&](int) { return ls != -INFINITY; }, [&](int x) { return attn_q_pos(A, b, i0 + x); });
      const bool ok = (bits >> lane) & 1u;
      I.lse[e] = ok ? -ls : -INFINITY;
      I.low[e] = ok && A.lse_low ? -A.lse_low[row + i0 + e] : 0.f;
      I.delta[e] = ok ? -A.delta[row + i0 + e] : 0.f;
    };
    if constexpr (TMA) {
      if (w == 0) {
        int64_t asked = 0;
        for (int64_t it = 0; it < tiles; ++it) {
          const int st = (int)(it % ST), h = (int)(hk * G + it / per);
          const int64_t i0 = (q0 + it % per) * kGradN;
          if (it >= ST) wait(&empty[st], (it / ST - 1) & 1, &abort_flag, polls);
          if (__any_sync(0xffffffffu, abort_flag)) break;
          ++asked;
          if (lane == 0) {
            mbar_arrive_expect_tx(&loaded[st], 2 * S::kTile);
            tma_tile<L>(sQ + st * S::kTile, M, MAP_Q, kGradN, i0, h, b, &loaded[st]);
            tma_tile<L>(sO + st * S::kTile, M, MAP_DO, kGradN, i0, h, b, &loaded[st]);
          }
          for (int sub = 0; sub < kGradN / kSub; ++sub) fill(it, sub);
          __syncwarp();
          if (lane == 0) arrive(&loaded[st]);
        }
        mbar_wait(&own, 0, kDrainPolls);
        drain(loaded, asked);
      } else {
        for (int64_t it = 0; it < tiles; ++it) {
          const int st = (int)(it % ST);
          const QueryInfo& I = info[it % S::kInfo];
          wait(&loaded[st], (it / ST) & 1, &abort_flag, polls);
          if ((I.t.live[0] & I.t.live[1]) != 0xffffffffu) {
            const auto row_live = [&](int r) { return (I.t.live[r >> 5] >> (r & 31)) & 1u; };
            clear_rows<L>(sQ + st * S::kTile, kGradN, t - 32, 64, row_live);
            clear_rows<L>(sO + st * S::kTile, kGradN, t - 32, 64, row_live);
            fence_proxy_async_smem();
          }
          arrive(&full[st]);
        }
      }
    } else {
      for (int64_t it = 0; it < tiles; ++it) {
        const int st = (int)(it % ST), h = (int)(hk * G + it / per);
        const int64_t i0 = (q0 + it % per) * kGradN;
        const QueryInfo& I = info[it % S::kInfo];
        if (it >= ST) wait(&empty[st], (it / ST - 1) & 1, &abort_flag, polls);
        if (w < kGradN / kSub) fill(it, w);
        named_barrier(1, 96);
        const auto row_live = [&](int r) { return (I.t.live[r >> 5] >> (r & 31)) & 1u; };
        load_tile<T, NS, PIECES, kGradN, L>(
            sQ + st * S::kTile, static_cast<const T*>(A.q) + b * A.qs[0] + h * A.qs[1] + i0 * A.qs[2], A.qs[2], A.D, t, 96,
            row_live);
        load_tile<T, NS, PIECES, kGradN, L>(
            sO + st * S::kTile, static_cast<const T*>(A.dout) + b * A.dos[0] + h * A.dos[1] + i0 * A.dos[2], A.dos[2], A.D,
            t, 96, row_live);
        fence_proxy_async_smem();
        arrive(&full[st]);
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (warp == 0) tmem_dealloc(tmem, S::kAlloc);
}

// ---------------------------------------------------------------- dq, dtable
template <int NS, typename L, int ST>
struct DqShape {
  static constexpr int kThreads = 256;  // 4 warps on the scores, one issuing, three loading
  static constexpr uint32_t kRow = NS * L::DC * L::RB, kOwn = 128 * kRow, kTile = kGradN * kRow;
  static constexpr uint32_t kTileBytes = 2 * kOwn + 2 * ST * kTile;
  // TMEM: scores, do.v, dq. ds of 16 columns takes the place of those once read: 8 columns a part,
  // two parts over the scores, the third over do.v.
  static constexpr int kDp = kGradN, kDq = 2 * kGradN;
  static constexpr int kCols = kDq + L::kDim, kAlloc = kCols <= 256 ? 256 : 512;
  static constexpr int kInfo = ST + 1;
  static constexpr int kBlocks = kAlloc <= 256 && kTileBytes <= 104 * 1024 ? 2 : 1;  // an SM holds
};

// The table's gradient: a row's ds sum to 0, and a bucket that holds all of a row's keys gets
// nothing from it. delta from the rounded output would leave its rounding there. So each
// thread keeps a = sum p (do.v) and b = sum p of its row by bucket, in columns of its own in
// shared memory (beyond the reach in registers), and the row gives a - b (sum a / sum b). Tables
// of more than kWindow buckets take a launch for every kWindow of them.
constexpr int kWindow = 64;

template <typename T, int NS, typename L, int ST, int LOAD>
__global__ void __launch_bounds__(DqShape<NS, L, ST>::kThreads, DqShape<NS, L, ST>::kBlocks)
    attn_dq_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TmaMaps M, int w0, int wn) {
  using S = DqShape<NS, L, ST>;
  constexpr bool TMA = LOAD == LOAD_TMA, PIECES = LOAD == LOAD_PIECES;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char *sQ = sm, *sO = sm + S::kOwn, *sK = sO + S::kOwn, *sV = sK + ST * S::kTile;
  float2* hist = reinterpret_cast<float2*>(sm + S::kTileBytes);  // wn x 128 (a, b)
  int2* lut = reinterpret_cast<int2*>(hist + wn * 128);           // (bias, column of its bucket or -1)
  __shared__ TileInfo<kGradN> info[S::kInfo];
  __shared__ uint64_t full[ST], empty[ST], loaded[ST], own, sfull, pfull, done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ int last_live;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int64_t heads = (int64_t)A.B * A.H, nq = (A.Lq + 127) / 128;
  const bool ordered = A.causal && !A.q_pos && !A.k_pos;
  const int64_t qb = ordered ? nq - 1 - blockIdx.x / heads : blockIdx.x % nq;
  const int64_t bh = ordered ? blockIdx.x % heads : blockIdx.x / nq;
  const int b = (int)(bh / A.H), h = (int)(bh % A.H), hk = h / (A.H / A.Hk);
  const int64_t i0 = qb * 128;
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_stride : nullptr;
  const int reach = A.buckets.reach, span = 2 * reach + 1;
  const float* lse = A.lse + bh * A.Lq;

  if (tid == 0) {
    abort_flag = 0;
    last_live = mask ? 0 : (int)A.Lk;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], TMA ? 64 : 96);
      mbar_init(&empty[i], 1);
      mbar_init(&loaded[i], 2);  // the copies, and what goes with the rows
    }
    mbar_init(&own, 1);
    mbar_init(&sfull, 1);
    mbar_init(&pfull, 128);
    mbar_init(&done, 1);
    fence_mbar_init();
    if constexpr (TMA) {
      mbar_arrive_expect_tx(&own, 2 * S::kOwn);
      tma_tile<L>(sQ, M, MAP_Q, 128, i0, h, b, &own);
      tma_tile<L>(sO, M, MAP_DO, 128, i0, h, b, &own);
    }
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  const auto row_live = [&](int r) { return i0 + r < A.Lq && lse[i0 + r] != -INFINITY; };
  if constexpr (!TMA) {
    load_tile<T, NS, PIECES, 128, L>(sQ, static_cast<const T*>(A.q) + b * A.qs[0] + h * A.qs[1] + i0 * A.qs[2], A.qs[2],
                                     A.D, tid, S::kThreads, row_live);
    load_tile<T, NS, PIECES, 128, L>(sO, static_cast<const T*>(A.dout) + b * A.dos[0] + h * A.dos[1] + i0 * A.dos[2],
                                     A.dos[2], A.D, tid, S::kThreads, row_live);
  }
  if (A.table) {
    for (int d = tid; d < span; d += S::kThreads) {
      const int c = bucket_of(A.buckets, d - reach) - w0;
      lut[d] = make_int2(__float_as_int(A.lut[(int64_t)h * span + d]), c >= 0 && c < wn ? c * 128 : -1);
    }
    for (int i = tid; i < wn * 128; i += S::kThreads) hist[i] = make_float2(0.f, 0.f);
  }
  if constexpr (TMA) {
    __syncthreads();
    wait(&own, 0, &abort_flag, A.polls);
    clear_rows<L>(sQ, 128, tid, S::kThreads, row_live);
    clear_rows<L>(sO, 128, tid, S::kThreads, row_live);
  }
  fence_proxy_async_smem();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (mask) {  // the keys after the last live one are not visited
    int last = 0;
    for (int j = tid; j < (int)A.Lk; j += S::kThreads)
      if (mask[j]) last = j + 1;
    if (last) atomicMax(&last_live, last);
    __syncthreads();
  }
  int64_t keys = last_live;
  if (ordered) {
    const int64_t end = i0 + 128 < A.Lq ? i0 + 128 : A.Lq, seen = A.Lk - A.Lq + end;
    keys = seen < keys ? (seen > 0 ? seen : 0) : keys;
  }
  const int tiles = (int)((keys + kGradN - 1) / kGradN);
  const uint32_t tmem = tmem_slot, polls = A.polls;

  if (warp < 4) {
    const int64_t i = i0 + tid;
    const bool valid = i < A.Lq, live = row_live(tid);
    const int qp = live ? attn_q_pos(A, b, i) : 0;
    const float lse_i = live ? lse[i] : INFINITY, low_i = live && A.lse_low ? A.lse_low[bh * A.Lq + i] : 0.f, delta = live ? A.delta[bh * A.Lq + i] : 0.f;
    const int qlo = __reduce_min_sync(0xffffffffu, live ? qp : INT32_MAX);
    const int qhi = __reduce_max_sync(0xffffffffu, live ? qp : INT32_MIN);
    const uint32_t base = tmem + ((uint32_t)(warp & 3) << 21);
    float2* mine = hist + tid;
    float ta = 0.f, tb = 0.f;                      // all of the row
    float ha = 0.f, hb = 0.f, la = 0.f, lb = 0.f;  // beyond the reach, above and below
    const bool windows = A.table && wn < A.buckets.num_buckets;
    // the sums so far to dq
    const auto keep = [&](float f, bool held, bool zero) {
      store_row<T, L::kDim>(base + S::kDq, static_cast<T*>(A.dq) + b * A.dqs[0] + h * A.dqs[1] + i * A.dqs[2], A.dqs[2], A.D,
                            f, held, zero, valid);
    };
    for (int j = 0; j < tiles; ++j) {
      const TileInfo<kGradN>& I = info[j % S::kInfo];
      wait(&sfull, j & 1, &abort_flag, polls);
      fence_after_sync();
      if (NS > 1 && w0 == 0 && j > 0 && starts<NS>(j)) keep(A.scale, j > kRest, false);
#pragma unroll 1  // one copy of the code: four no longer stay in the instruction cache
      for (int c = 0; c < kGradN; c += 16) {
        const int sub = c / kSub;
        const uint32_t bits = I.live[sub] >> (c % kSub);
        const int klo = I.lo[sub], khi = I.hi[sub];
        const bool some = I.live[sub] != 0 && qlo <= qhi;
        const bool above = (int64_t)klo - qhi >= reach, below = (int64_t)khi - qlo <= -reach;
        const bool near = some && A.table && !above && !below, later = some && A.causal && khi > qlo;
        uint32_t s[16], dp[16], wd[NS][8];
        ld16(base + c, s);
        ld16(base + S::kDp + c, dp);
        tmem_wait_ld();
        const uint64_t ss = both(A.scale2, A.scale2), nd = both(-delta, -delta);
        const uint64_t nh = both(-lse_i, -lse_i), nl = both(-low_i, -low_i);
        uint64_t sa = 0, sb = 0;  // pairs of zeros
        if (near || later) {
          // everything that is read before the first histogram is written: the compiler may not
          // move a lookup over a store
          int k[16], at[16];
          float bias[16];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const int4 v = *reinterpret_cast<const int4*>(&I.pos[c + e]);
            k[e] = v.x;
            k[e + 1] = v.y;
            k[e + 2] = v.z;
            k[e + 3] = v.w;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            int2 t = make_int2(0, -1);
            if (A.table) t = lut[__vimin_s32_relu(k[e] + reach - qp, 2 * reach)];
            bias[e] = __int_as_float(t.x);
            if ((A.causal && k[e] > qp) || !((bits >> e) & 1u)) bias[e] = -INFINITY;
            at[e] = t.y;
          }
          float pr[16], px[16];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float v0, v1, x0, x1, y0, y1;
            const uint64_t sc = fma_both(both(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), ss, both(bias[e], bias[e + 1]));
            halves(add_both(add_both(sc, nh), nl), v0, v1);
            pr[e] = ex2(v0);
            pr[e + 1] = ex2(v1);
            const uint64_t pp = both(pr[e], pr[e + 1]), dd = both(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1]));
            const uint64_t xx = mul_both(pp, dd);
            halves(xx, x0, x1);
            px[e] = x0;
            px[e + 1] = x1;
            halves(mul_both(pp, add_both(dd, nd)), y0, y1);
            s[e] = __float_as_uint(y0);
            s[e + 1] = __float_as_uint(y1);
            sa = add_both(sa, xx);
            sb = add_both(sb, pp);
          }
          if (A.table) {
            // four columns at a time: runs of one bucket joined, the rest read together, unless a
            // bucket comes back after another (positions in any order)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const int o0 = at[e], o1 = at[e + 1], o2 = at[e + 2], o3 = at[e + 3];
              const bool j1 = o1 == o0, j2 = o2 == o1, j3 = o3 == o2;
              const bool back = (o2 == o0 && !j1) || (o3 == o1 && !j2) || (o3 == o0 && !(j1 && j2 && j3) && !(o2 == o0));
              float a0 = px[e], a1 = px[e + 1], a2 = px[e + 2], a3 = px[e + 3];
              float b0 = pr[e], b1 = pr[e + 1], b2 = pr[e + 2], b3 = pr[e + 3];
              if (!__any_sync(0xffffffffu, back)) {
                if (j1) a1 += a0, b1 += b0;
                if (j2) a2 += a1, b2 += b1;
                if (j3) a3 += a2, b3 += b2;
                const bool w0 = !j1 && o0 >= 0, w1 = !j2 && o1 >= 0, w2 = !j3 && o2 >= 0, w3 = o3 >= 0;
                float2 h0, h1, h2, h3;
                if (w0) h0 = mine[o0];
                if (w1) h1 = mine[o1];
                if (w2) h2 = mine[o2];
                if (w3) h3 = mine[o3];
                if (w0) mine[o0] = make_float2(h0.x + a0, h0.y + b0);
                if (w1) mine[o1] = make_float2(h1.x + a1, h1.y + b1);
                if (w2) mine[o2] = make_float2(h2.x + a2, h2.y + b2);
                if (w3) mine[o3] = make_float2(h3.x + a3, h3.y + b3);
              } else {
                const int o[4] = {o0, o1, o2, o3};
                const float a[4] = {a0, a1, a2, a3}, bb[4] = {b0, b1, b2, b3};
#pragma unroll
                for (int n = 0; n < 4; ++n)
                  if (o[n] >= 0) {
                    float2 v = mine[o[n]];
                    v.x += a[n];
                    v.y += bb[n];
                    mine[o[n]] = v;
                  }
              }
            }
          }
        } else {
          const float flat = A.table && some ? __int_as_float(lut[above ? 2 * reach : 0].x) : 0.f;
          const uint64_t bb = both(flat, flat);
          const bool whole = (bits & 0xffffu) == 0xffffu;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float v0, v1, y0, y1;
            const uint64_t sc = fma_both(both(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), ss, bb);
            halves(add_both(add_both(sc, nh), nl), v0, v1);
            if (!whole) {
              if (!((bits >> e) & 1u)) v0 = -INFINITY;
              if (!((bits >> (e + 1)) & 1u)) v1 = -INFINITY;
            }
            const uint64_t pp = both(ex2(v0), ex2(v1)), dd = both(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1]));
            sa = fma_both(pp, dd, sa);
            sb = add_both(sb, pp);
            halves(mul_both(pp, add_both(dd, nd)), y0, y1);
            s[e] = __float_as_uint(y0);
            s[e + 1] = __float_as_uint(y1);
          }
        }
        {
          float x0, x1, y0, y1;
          halves(sa, x0, x1);
          halves(sb, y0, y1);
          x0 += x1;
          y0 += y1;
          if (!(near || later)) {
            if (above) {
              ha += x0;
              hb += y0;
            } else {
              la += x0;
              lb += y0;
            }
          }
          ta += x0;
          tb += y0;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t o[NS];
          split2<NS>(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]), o);
#pragma unroll
          for (int n = 0; n < NS; ++n) wd[n][e] = o[n];
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) st8(base + c + (n < 2 ? n * 8 : S::kDp), wd[n]);
      }
      tmem_wait_st();
      fence_before_sync();
      arrive(&pfull);
    }
    if (tiles > 0) {
      wait(&sfull, tiles & 1, &abort_flag, polls);
      fence_after_sync();
    }
    const float broken = abort_flag ? NAN : 0.f;
    if (w0 == 0) keep(A.scale + broken, NS > 1 && tiles > kRest, !live || tiles == 0);
    if (A.table) {
      const int hi = lut[2 * reach].y, lo = lut[0].y;
      if (hi >= 0) {
        mine[hi].x += ha;
        mine[hi].y += hb;
      }
      if (lo >= 0) {
        mine[lo].x += la;
        mine[lo].y += lb;
      }
      if (!windows) {
        ta = tb = 0.f;
#pragma unroll 8
        for (int c = 0; c < wn; ++c) {
          const float2 v = mine[c * 128];
          ta += v.x;
          tb += v.y;
        }
      }
      const float mean = live && tb != 0.f ? ta / tb : 0.f;
      for (int c = 0; c < wn; c += 8) {
        float2 v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < wn) v[e] = mine[(c + e) * 128];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < wn) mine[(c + e) * 128].x = live ? fmaf(-v[e].y, mean, v[e].x) + broken : 0.f;
      }
      named_barrier(2, 128);
      float* part = A.dpart + (((int64_t)h * A.B + b) * nq + qb) * A.buckets.num_buckets + w0;
#pragma unroll 4
      for (int c = warp; c < wn; c += 4) {
        const float2* r = hist + c * 128 + lane;
        const float v = lanes_sum((r[0].x + r[32].x) + (r[64].x + r[96].x), 32);
        if (lane == 0) part[c] = v;
      }
    }
  } else if (warp == 4) {
    if (lane == 0 && tiles > 0) {
      const uint32_t id_s = idesc_bf16(128, kGradN, false), id_o = idesc_bf16(128, (A.D + 15) / 16 * 16, true);
      const uint32_t aQ = smem_u32(sQ), aO = smem_u32(sO);
      for (int j = 0; j < tiles; ++j) {
        const int st = j % ST;
        const uint32_t aK = smem_u32(sK) + st * S::kTile, aV = smem_u32(sV) + st * S::kTile;
        wait(&full[st], (j / ST) & 1, &abort_flag, polls);
        scores<NS, 128, kGradN, L>(tmem, aQ, aK, A.D, id_s);
        scores<NS, 128, kGradN, L>(tmem + S::kDp, aO, aV, A.D, id_s);
        mma_commit(&sfull);
        wait(&pfull, j & 1, &abort_flag, polls);
        fence_after_sync();
        values<NS, kGradN, L>(tmem + S::kDq, aK, id_o, !starts<NS>(j),
                              [=](int part, int k) { return tmem + k * 16 + (part < 2 ? part * 8 : S::kDp); });
        mma_commit(&empty[st]);
      }
      mma_commit(&sfull);
      mma_commit(&done);
      mbar_wait(&done, 0, kDrainPolls);
    }
  } else {
    const int t = tid - 160, w = t >> 5;
    const auto fill = [&](int j, int sub) {
      const int64_t j0 = (int64_t)j * kGradN;
      fill_info<kGradN>(
          info[j % S::kInfo], sub, [&](int e) { return j0 + e < A.Lk && (!mask || mask[j0 + e]); },
          [&](int e) { return attn_k_pos(A, b, j0 + e); });
    };
    if constexpr (TMA) {
      if (w == 0) {
        int64_t asked = 0;
        for (int j = 0; j < tiles; ++j) {
          const int st = j % ST;
          if (j >= ST) wait(&empty[st], (j / ST - 1) & 1, &abort_flag, polls);
          if (__any_sync(0xffffffffu, abort_flag)) break;
          ++asked;
          if (lane == 0) {
            mbar_arrive_expect_tx(&loaded[st], 2 * S::kTile);
            tma_tile<L>(sK + st * S::kTile, M, MAP_K, kGradN, (int64_t)j * kGradN, hk, b, &loaded[st]);
            tma_tile<L>(sV + st * S::kTile, M, MAP_V, kGradN, (int64_t)j * kGradN, hk, b, &loaded[st]);
          }
          for (int sub = 0; sub < kGradN / kSub; ++sub) fill(j, sub);
          __syncwarp();
          if (lane == 0) arrive(&loaded[st]);
        }
        mbar_wait(&own, 0, kDrainPolls);
        drain(loaded, asked);
      } else {
        for (int j = 0; j < tiles; ++j) {
          const int st = j % ST;
          const TileInfo<kGradN>& I = info[j % S::kInfo];
          wait(&loaded[st], (j / ST) & 1, &abort_flag, polls);
          if (mask && (I.live[0] & I.live[1]) != 0xffffffffu) {
            const auto live = [&](int r) { return (I.live[r >> 5] >> (r & 31)) & 1u; };
            clear_rows<L>(sK + st * S::kTile, kGradN, t - 32, 64, live);
            clear_rows<L>(sV + st * S::kTile, kGradN, t - 32, 64, live);
            fence_proxy_async_smem();
          }
          arrive(&full[st]);
        }
      }
    } else {
      const T* K = static_cast<const T*>(A.k) + b * A.ks[0] + hk * A.ks[1];
      const T* V = static_cast<const T*>(A.v) + b * A.vs[0] + hk * A.vs[1];
      for (int j = 0; j < tiles; ++j) {
        const int st = j % ST;
        const int64_t j0 = (int64_t)j * kGradN;
        const TileInfo<kGradN>& I = info[j % S::kInfo];
        if (j >= ST) wait(&empty[st], (j / ST - 1) & 1, &abort_flag, polls);
        if (w < kGradN / kSub) fill(j, w);
        named_barrier(1, 96);
        const auto live = [&](int r) { return (I.live[r >> 5] >> (r & 31)) & 1u; };
        load_tile<T, NS, PIECES, kGradN, L>(sK + st * S::kTile, K + j0 * A.ks[2], A.ks[2], A.D, t, 96, live);
        load_tile<T, NS, PIECES, kGradN, L>(sV + st * S::kTile, V + j0 * A.vs[2], A.vs[2], A.D, t, 96, live);
        fence_proxy_async_smem();
        arrive(&full[st]);
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (warp == 0) tmem_dealloc(tmem, S::kAlloc);
}

}  // namespace tc
}  // namespace fx
