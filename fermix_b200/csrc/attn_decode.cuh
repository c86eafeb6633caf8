// Attention of few queries over a long bfloat16 cache, split over the keys. A block takes up to 16 query
// rows that share a key head (one new token of a group of heads, or a few).
//
// Bound: HBM, each live key and value once; the arithmetic has to stay out of the way. With FMA
// instructions four rows a key head already took eight times as long as the bytes (1222 us for
// 807 MB: conversions, dot products over lanes), so the products run as 16 x 8 x 16 tensor
// instructions on register fragments loaded straight from global memory: a warp takes 16 keys a
// step. The order of the entries within a dot product is free, so a lane's 16-byte piece of a key
// serves two k-steps as it is (the queries are permuted alike), and the order of the output's
// columns is free, so a lane's 16-byte piece of a value row serves eight column tiles after two
// byte permutations each. The scores' fragment is the probabilities' operand fragment. tcgen05
// would need the cache staged through shared memory for 16 rows of 128.
//
// A lane copies the pieces it will use into a ring of its own in shared memory (cp.async), three
// steps ahead: 96 KB a block on the way without registers (with the loads in registers, one step
// at a time, 217 us for 64 key heads of 65536 keys, three quarters live; with the ring 190 us,
// 4.2 TB/s of the live keys' bytes, 0.65 of a copy's rate; all live 4.5 TB/s). What is left is not the
// ring's depth, two blocks have 130 KB of an SM on the way: caches of different live lengths leave SMs idle
// at the end (233 to 339 thousand cycles of work, 295 on average), and while they work 16 warps use
// half of the issue slots and wait for fixed latencies (1.8 of 7 an instruction), shared memory (1.2) and
// the positions' and mask's loads (0.6).
//
// The probabilities are rounded to bfloat16 for the second product, the tensor instruction's operand
// type, and are summed unrounded: each entry of the output takes up to 2^-9 of the values' size, as much as the
// rounding of the output itself.
#pragma once
#include "attn_rows.cuh"

namespace fx {

constexpr int kDecodeThreads = 256, kDecodeWarps = 8;
constexpr int kDecodeRows = 16;       // query rows of a block
constexpr int kDecodeStages = 3;

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Entries [c, c + 8) of a token, zero past D, into a slot of the ring. VEC: tokens start on 16-byte
// boundaries and are whole pieces; else entry by entry, in the same places, so that the results
// have the same bits.
template <bool VEC>
__device__ __forceinline__ void fetch8(uint4* slot, const bf16* p, int c, int D, bool ok) {
  if (VEC) {
    const int bytes = ok && c < D ? 16 : 0;  // 0: zeros, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(slot))),
                 "l"(bytes ? p + c : p), "r"(bytes)
                 : "memory");
    return;
  }
  Pack<bf16, 8> k;
#pragma unroll
  for (int e = 0; e < 8; ++e) k.e[e] = ok && c + e < D ? p[c + e] : from_f<bf16>(0.f);
  *slot = *reinterpret_cast<const uint4*>(&k);
}

// A block: one part of the keys of one (batch, key head): of every `splits` runs of 128 keys one,
// so that the parts of a cache whose end is masked have the same number of live keys. DB: 64-entry blocks of the head
// dimension. Entries beyond D are zero.
template <int DB, bool VEC>
__global__ void __launch_bounds__(kDecodeThreads, DB == 1 ? 2 : 1) attn_decode_kernel(const __grid_constant__ AttnArgs A) {
  constexpr int S = kDecodeStages, P = 8 * DB;  // pieces of a lane and step: keys 4 DB, values 4 DB
  extern __shared__ uint4 ring_mem[];  // the ring (after the keys, the warps' joins), the table by distance
  float* sm = reinterpret_cast<float*>(ring_mem + S * P * kDecodeThreads);
  const int G = A.H / A.Hk, reach = A.buckets.reach, span = A.table ? 2 * reach + 1 : 0;
  // this block's rows [row0, row0 + rows) of the key head's G Lq, of the query heads h0 and following
  const int all = G * (int)A.Lq, chunks = (all + kDecodeRows - 1) / kDecodeRows;
  const int part = blockIdx.x % A.splits, cz = blockIdx.x / A.splits, z = cz / chunks, b = z / A.Hk, hk = z % A.Hk;
  const int row0 = cz % chunks * kDecodeRows, rows = all - row0 < kDecodeRows ? all - row0 : kDecodeRows;
  const int h0 = row0 / (int)A.Lq, heads = (row0 + rows - 1) / (int)A.Lq - h0 + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t j0 = part * (kDecodeWarps * 16), kStep = (int64_t)A.splits * (kDecodeWarps * 16);
  const int64_t count = A.Lk - j0;

  const bf16* K = static_cast<const bf16*>(A.k) + b * A.ks[0] + hk * A.ks[1] + j0 * A.ks[2];
  const bf16* V = static_cast<const bf16*>(A.v) + b * A.vs[0] + hk * A.vs[1] + j0 * A.vs[2];
  uint4* slots = ring_mem + (warp * S * P) * 32 + lane;  // slot (stage, piece) at (stage * P + piece) * 32
  // Live keys of this warp's groups of 16: lane n holds group first + n, 32 groups at a time.
  const auto group_bits = [&](int first) -> uint32_t {
    const int64_t base = warp * 16 + (first + lane) * kStep;
    if (base >= count) return 0u;
    const int n = count - base < 16 ? (int)(count - base) : 16;
    if (!A.mask) return (1u << n) - 1u;
    const uint8_t* p = A.mask + b * A.mask_stride + j0 + base;
    uint32_t bits = 0;
    if (n == 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 16; ++e) bits |= ((w[e / 4] >> (e % 4 * 8)) & 0xffu ? 1u : 0u) << e;
    } else {
      for (int e = 0; e < n; ++e) bits |= (p[e] ? 1u : 0u) << e;
    }
    return bits;
  };
  uint32_t mine = group_bits(0), after = 0;  // of groups [first, first + 32) and the 32 after them
  int first = 0;
  const auto bits_of = [&](int n) { return __shfl_sync(0xffffffffu, n - first < 32 ? mine : after, n & 31); };
  // keys base + g and base + 8 + g; values of keys base + {2t, 2t + 1, 2t + 8, 2t + 9}
  const auto fetch = [&](int n_group, int stage) {
    const uint32_t bits = bits_of(n_group);
    const int64_t base = warp * 16 + n_group * kStep;
    if (bits != 0) {
      uint4* slot = slots + stage * P * 32;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int e = n * 8 + g;
#pragma unroll
        for (int c = 0; c < 2 * DB; ++c)
          fetch8<VEC>(slot + (n * 2 * DB + c) * 32, K + (base + e) * A.ks[2], c * 32 + t * 8, A.D, (bits >> e) & 1u);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int e = 2 * t + (n & 1) + (n >> 1) * 8;
#pragma unroll
        for (int c = 0; c < DB; ++c)
          fetch8<VEC>(slot + (4 * DB + n * DB + c) * 32, V + (base + e) * A.vs[2], c * 64 + g * 8, A.D,
                      (bits >> e) & 1u);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int n = 0; n < S - 1; ++n) fetch(n, n);
  if (A.table) {
    const bf16* table = static_cast<const bf16*>(A.table) + ((int64_t)hk * G + h0) * A.buckets.num_buckets;
    for (int i = threadIdx.x; i < heads * span; i += kDecodeThreads)
      sm[i] = bias2(to_f(table[i / span * A.buckets.num_buckets + bucket_of(A.buckets, i % span - reach)]));
  }
  // this lane's two rows, g and g + 8
  uint4 q[2][2 * DB];
  int qp[2], lut[2];
  bool row_ok[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = g + 8 * r;
    row_ok[r] = row < rows;
    const int h = row_ok[r] ? (row0 + row) / (int)A.Lq : h0, i = row_ok[r] ? (row0 + row) % (int)A.Lq : 0;
    qp[r] = attn_q_pos(A, b, i);
    lut[r] = (h - h0) * span;
    const bf16* p = static_cast<const bf16*>(A.q) + b * A.qs[0] + (hk * G + h) * A.qs[1] + i * A.qs[2];
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) {
      Pack<bf16, 8> x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x.e[e] = row_ok[r] && c * 32 + t * 8 + e < A.D ? p[c * 32 + t * 8 + e] : from_f<bf16>(0.f);
      q[r][c] = *reinterpret_cast<const uint4*>(&x);
    }
  }
  const int rows_hi = rows > 8;
  __syncthreads();

  float o[8 * DB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 8 * DB; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;

  int stage = 0;
  const int groups = (int)((count - warp * 16 + kStep - 1) / kStep);  // <= 0: none
  for (int n_group = 0; n_group < groups; ++n_group, stage = stage == S - 1 ? 0 : stage + 1) {
    const int64_t base = warp * 16 + n_group * kStep;
    if ((n_group & 31) == 16) after = group_bits(n_group - 16 + 32);
    if (n_group - first == 32) {
      mine = after;
      first = n_group;
    }
    fetch(n_group + S - 1, stage == 0 ? S - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    const uint32_t bits = bits_of(n_group);
    if (bits == 0) continue;
    const uint4* slot = slots + stage * P * 32;
    uint4 k[2][2 * DB], v[4][DB];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int c = 0; c < 2 * DB; ++c) k[n][c] = slot[(n * 2 * DB + c) * 32];
    bool ok[4];
    int kp[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int e = 2 * t + (n & 1) + (n >> 1) * 8;
      ok[n] = (bits >> e) & 1u;
      kp[n] = ok[n] ? attn_k_pos(A, b, j0 + base + e) : 0;
#pragma unroll
      for (int c = 0; c < DB; ++c) v[n][c] = slot[(4 * DB + n * DB + c) * 32];
    }
    float s[2][4] = {};  // s[n]: rows g, g + 8 of keys n * 8 + 2t, + 1
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma_16816(s[n], q[0][c].x, q[1][c].x, q[0][c].y, q[1][c].y, k[n][c].x, k[n][c].y);
        mma_16816(s[n], q[0][c].z, q[1][c].z, q[0][c].w, q[1][c].w, k[n][c].z, k[n][c].w);
      }
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r && !rows_hi) break;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int d = kp[n] - qp[r];
        const float bias = A.table ? sm[lut[r] + clamp_reach(d, reach) + reach] : 0.f;
        float& x = s[n >> 1][2 * r + (n & 1)];
        x = fmaf(x, A.scale2, bias);
        if (!ok[n] || (A.causal && d > 0)) x = -INFINITY;
        top = fmaxf(top, x - (m[r] == -INFINITY ? (x == -INFINITY ? 0.f : -INFINITY) : m[r]));
      }
    }
    // a score more than 2^20 above a row's reference, or a row without one: the references move
    if (__any_sync(0xffffffffu, top > 20.f)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        if (r && !rows_hi) x = -INFINITY;
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        x = fmaxf(x, m[r]);
        const float f = x == -INFINITY ? 1.f : exp2f(m[r] - x);
        m[r] = x;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < 8 * DB; ++e) {
          o[e][2 * r] *= f;
          o[e][2 * r + 1] *= f;
        }
      }
    }
    uint32_t p[2][2];  // [n][r]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float x = 0.f, y = 0.f;
        if (r == 0 || rows_hi) {
          x = exp2f(s[n][2 * r] - ref);
          y = exp2f(s[n][2 * r + 1] - ref);
        }
        l[r] += x + y;
        const __nv_bfloat162 w = __floats2bfloat162_rn(x, y);
        p[n][r] = *reinterpret_cast<const uint32_t*>(&w);
      }
    }
#pragma unroll
    for (int c = 0; c < DB; ++c) {
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&v[0][c]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&v[1][c]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&v[2][c]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&v[3][c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
        mma_16816(o[c * 8 + e], p[0][0], p[0][1], p[1][0], p[1][1], __byte_perm(v0[e / 2], v1[e / 2], sel),
                  __byte_perm(v2[e / 2], v3[e / 2], sel));
      }
    }
  }
  // join the warps: (m, l) and the outputs of each, entry c = block * 64 + 8 n + e of tile e, column n
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* wm = reinterpret_cast<float*>(ring_mem);                                  // warps x 16
  float* wl = wm + kDecodeWarps * kDecodeRows;     // warps x 16
  float* wo = wl + kDecodeWarps * kDecodeRows;     // warps x rows x (64 DB + 1)
  constexpr int W = 64 * DB + 1;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (!row_ok[r]) continue;
    const int row = g + 8 * r;
    if (t == 0) {
      wm[warp * kDecodeRows + row] = m[r];
      wl[warp * kDecodeRows + row] = l[r];
    }
    float* w = wo + (warp * rows + row) * W;
#pragma unroll
    for (int e = 0; e < 8 * DB; ++e)
#pragma unroll
      for (int n = 0; n < 2; ++n) w[(e / 8) * 64 + 8 * (2 * t + n) + e % 8] = o[e][2 * r + n];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * A.D; i += kDecodeThreads) {
    const int row = i / A.D, c = i - row * A.D;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, wm[w * kDecodeRows + row]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      const float f = exp2f(wm[w * kDecodeRows + row] - ref);
      sum = fmaf(wl[w * kDecodeRows + row], f, sum);
      acc = fmaf(wo[(w * rows + row) * W + c], f, acc);
    }
    if (A.splits > 1) {
      float* p = A.part + (((int64_t)z * all + row0 + row) * A.splits + part) * part_step(A.D);
      p[4 + c] = acc;
      if (c == 0) {
        p[0] = top;
        p[1] = sum;
      }
    } else {
      const int h = hk * G + (row0 + row) / (int)A.Lq;
      const int64_t q_i = (row0 + row) % (int)A.Lq;
      static_cast<bf16*>(A.out)[b * A.os[0] + h * A.os[1] + q_i * A.os[2] + c] =
          from_f<bf16>(sum == 0.f ? 0.f : acc / sum);
      if (A.lse && c == 0) store_lse(A, ((int64_t)b * A.H + h) * A.Lq + q_i, top, sum);
    }
  }
}

}  // namespace fx
