// Tensor-core (tcgen05) pieces of the biased attention, and its forward kernel.
//
// Operands sit in shared memory in the 128-byte swizzled layout: a tile is chunks of 64
// head-dimension entries, a chunk R rows of 128 bytes, the 16-byte piece c of row r at
// r * 128 + ((c ^ (r & 7)) << 4). Read along the rows it is a K-major operand (scores), read
// across them an MN-major one (products with the values), so each tile is stored once.
//
// float32 runs on the same bfloat16 instructions: x = x1 + x2 + x3, each part the rest rounded
// to bfloat16, holds 24 bits exactly, and the six products with index sum <= 4 leave out
// terms of 2^-24 -- the accuracy of a float32 product at a sixth of the bfloat16 rate (three
// TF32 products cost the same and keep 22 bits). bfloat16 keeps float32's exponent range, so
// neither the parts nor the score gradients need a scale.
//
// Loading is by threads (cp.async, or through registers where a type is split or an address
// is not on 16 bytes), not by tensor maps: a masked key's row must be zero whatever it
// holds, rows end anywhere, and strides are the caller's.
#pragma once
#include "attn_rows.cuh"
#include "umma.cuh"

namespace fx {
namespace tc {

using namespace umma;

constexpr int kSub = 32;  // keys (or queries) whose positions are summarised together

// K-major / MN-major operand in the 128-byte swizzle. lbo: bytes between chunks of 64 entries
// (MN-major only), groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16, bfloat16 operands, float32 accumulator
__device__ __forceinline__ uint32_t idesc_bf16(int M, int N, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}

#define FX_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define FX_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void ld32(uint32_t a, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : FX_R8(v, 0), FX_R8(v, 8), FX_R8(v, 16), FX_R8(v, 24)
      : "r"(a));
}
__device__ __forceinline__ void ld16(uint32_t a, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : FX_R8(v, 0), FX_R8(v, 8)
      : "r"(a));
}
__device__ __forceinline__ void st16(uint32_t a, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      FX_I8(v, 0), FX_I8(v, 8));
}
__device__ __forceinline__ void st8(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), FX_I8(v, 0));
}
#undef FX_R8
#undef FX_I8

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// (a, b) -> NS packed pairs whose sum is (a, b)
template <int NS>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&o)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    o[i] = pack2(a, b);
    if (i + 1 < NS) {
      a -= __uint_as_float(o[i] << 16);
      b -= __uint_as_float(o[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void arrive(uint64_t* m) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(m)) : "memory");
}
// A bounded wait. After a first one ran out (abort flag, status word) every further wait of the
// block returns at once: the block runs to its end on whatever is there and frees its TMEM.
__device__ __forceinline__ void wait(uint64_t* m, uint32_t parity, volatile int* abort, uint32_t polls) {
  const uint32_t a = smem_u32(m);
  for (uint32_t it = 0; it < polls; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return;
    if ((it & 63) == 63 && *abort) return;
  }
  if (!*abort) {
    record_status(FX_ERR_TIMEOUT);
    *abort = 1;
  }
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows [0, R) of a tile from p (element strides `step` a row, dim entries a row, entries
// beyond dim up to the next multiple of 16 zero), row r only if live(r), by `n` threads of index
// t. Parts of a split type are R * chunks * 128 bytes apart. cp.async copies are left open.
template <typename T, int NS, bool VEC, int R, typename Live>
__device__ __forceinline__ void load_tile(unsigned char* dst, const T* p, int64_t step, int dim, int chunks, int t,
                                          int n, Live live) {
  const int pieces = (dim + 15) / 16 * 2;  // of 8 entries
  const uint32_t part = (uint32_t)R * 128u * (uint32_t)chunks;
  for (int i = t; i < R * pieces; i += n) {
    const int r = i / pieces, c = i - r * pieces;
    const bool ok = live(r);
    unsigned char* d = dst + (uint32_t)(c >> 3) * (R * 128u) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    if constexpr (NS == 1 && VEC && sizeof(T) == 2) {
      const bool has = ok && c * 8 < dim;
      cp16(smem_u32(d), has ? p + r * step + c * 8 : p, has ? 16 : 0);
    } else {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
      if (ok) {
        const T* s = p + r * step + c * 8;
        if constexpr (VEC) {
          constexpr int V = 16 / sizeof(T);
#pragma unroll
          for (int h = 0; h < 8; h += V) {
            if (c * 8 + h < dim) {
              const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(s + h);
#pragma unroll
              for (int e = 0; e < V; ++e) x[h + e] = to_f(k.e[e]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c * 8 + e < dim) x[e] = to_f(s[e]);
        }
      }
      uint32_t w[4][NS];
#pragma unroll
      for (int e = 0; e < 4; ++e) split2<NS>(x[2 * e], x[2 * e + 1], w[e]);
#pragma unroll
      for (int s = 0; s < NS; ++s)
        *reinterpret_cast<uint4*>(d + s * part) = make_uint4(w[0][s], w[1][s], w[2][s], w[3][s]);
    }
  }
}

// D (+)= A B^T over `steps` k-steps of 16 entries, both K-major tiles of RA / RB rows.
template <int NS, int RA, int RB>
__device__ __forceinline__ void scores(uint32_t d, uint32_t a, uint32_t b, int dim, int chunks, uint32_t idesc) {
  const int steps = (dim + 15) / 16;
  bool acc = false;
  // the smaller products first
#pragma unroll
  for (int sum = NS - 1; sum >= 0; --sum) {
#pragma unroll
    for (int i = 0; i <= sum; ++i) {
      const uint32_t ap = a + i * (RA * 128u * chunks), bp = b + (sum - i) * (RB * 128u * chunks);
      for (int k = 0; k < steps; ++k) {
        mma_ss(d, desc_sw128(ap + (k >> 2) * (RA * 128u) + (k & 3) * 32u, 16),
               desc_sw128(bp + (k >> 2) * (RB * 128u) + (k & 3) * 32u, 16), idesc, acc);
        acc = true;
      }
    }
  }
}

// D (+)= A B, A in TMEM (NS parts, `apart` columns apart; k-step kk at a + acol(kk)), B the
// MN-major view of a tile of RB rows (the contraction's index).
template <int NS, int RB, typename Col>
__device__ __forceinline__ void values(uint32_t d, uint32_t a, uint32_t apart, uint32_t b, int chunks, uint32_t idesc,
                                       bool acc, Col acol) {
#pragma unroll
  for (int sum = NS - 1; sum >= 0; --sum) {
#pragma unroll
    for (int i = 0; i <= sum; ++i) {
      const uint32_t bp = b + (sum - i) * (RB * 128u * chunks);
#pragma unroll
      for (int k = 0; k < RB / 16; ++k) {
        mma_ts(d, a + i * apart + acol(k), desc_sw128(bp + k * 2048u, RB * 128u), idesc, acc);
        acc = true;
      }
    }
  }
}

// Positions and liveness of up to R keys (or queries) of a tile.
template <int R>
struct alignas(16) TileInfo {  // positions are read four at a time
  int pos[R];
  int lo[R / kSub], hi[R / kSub];
  uint32_t live[R / kSub];
};

// Entries [sub * 32, sub * 32 + 32) of the tile, by one warp; returns the live ones' bits.
template <int R, typename Live, typename Pos>
__device__ __forceinline__ uint32_t fill_info(TileInfo<R>& I, int sub, Live live, Pos pos) {
  const int lane = threadIdx.x & 31, e = sub * kSub + lane;
  const bool ok = live(e);
  const int x = ok ? pos(e) : 0;
  const uint32_t bits = __ballot_sync(0xffffffffu, ok);
  const int lo = __reduce_min_sync(0xffffffffu, ok ? x : INT32_MAX);
  const int hi = __reduce_max_sync(0xffffffffu, ok ? x : INT32_MIN);
  I.pos[e] = x;
  if (lane == 0) {
    I.lo[sub] = lo;
    I.hi[sub] = hi;
    I.live[sub] = bits;
  }
  return bits;
}

// ---------------------------------------------------------------- forward
// A block takes QT tiles of 128 query rows of one head (thread = row = TMEM lane) and walks the
// keys BN at a time. Warps 4 t .. 4 t + 3 hold the running maximum and sum of tile t; the next
// warp issues the tensor instructions, the last three load. With QT = 2 one tile's
// exponentials run while the other's products do. The probabilities overwrite (QT = 2) or
// follow the scores in TMEM and are the A operand of the second product. The output is
// rescaled only when the maximum has grown by more than 2^8.
template <typename T, int NS, int QT, int BN, int DC, int ST>
struct FwdShape {
  static constexpr int kThreads = 128 * QT + 128;
  static constexpr uint32_t kQ = NS * DC * 16384u, kKV = NS * DC * BN * 128u;
  static constexpr int kInfo = ST + 1;
  static constexpr uint32_t kTileBytes = QT * kQ + 2 * ST * kKV;
  // TMEM columns of a tile: scores, then (NS > 1) the probabilities' parts, then the output
  static constexpr int kP = NS == 1 ? 0 : BN;
  static constexpr int kO = NS == 1 ? BN : BN + NS * BN / 2;
  static constexpr int kCols = QT * (kO + 64 * DC);
  static constexpr int kAlloc = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
};

template <typename T, int NS, int QT, int BN, int DC, int ST, bool VEC>
__global__ void __launch_bounds__(FwdShape<T, NS, QT, BN, DC, ST>::kThreads, QT == 1 && DC == 1 ? 2 : 1)
    attn_fwd_kernel(const __grid_constant__ AttnArgs A) {
  using S = FwdShape<T, NS, QT, BN, DC, ST>;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char *sQ = sm, *sK = sm + QT * S::kQ, *sV = sK + ST * S::kKV;
  float* lut = reinterpret_cast<float*>(sm + S::kTileBytes);
  __shared__ TileInfo<BN> info[S::kInfo];
  __shared__ uint64_t kfull[ST], vfull[ST], kempty[ST], vempty[ST], sfull[QT], pfull[QT], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ int last_live;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // block -> (batch, head, query block); late query blocks first (causal: the longest)
  int64_t blk = blockIdx.x;
  const int64_t nq = (A.Lq + 128 * QT - 1) / (128 * QT);
  const int64_t qb = nq - 1 - blk % nq;
  blk /= nq;
  const int h = (int)(blk % A.H), b = (int)(blk / A.H), hk = h / (A.H / A.Hk);
  const int64_t i0 = qb * 128 * QT;
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_stride : nullptr;
  const int reach = A.buckets.reach;

  if (tid == 0) {
    abort_flag = 0;
    last_live = mask ? 0 : (int)A.Lk;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kfull[i], 96);
      mbar_init(&vfull[i], 96);
      mbar_init(&kempty[i], 1);
      mbar_init(&vempty[i], 1);
    }
    for (int t = 0; t < QT; ++t) {
      mbar_init(&sfull[t], 1);
      mbar_init(&pfull[t], 128);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  const T* Q = static_cast<const T*>(A.q) + b * A.qs[0] + h * A.qs[1];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int64_t first = i0 + t * 128;
    load_tile<T, NS, VEC, 128>(sQ + t * S::kQ, Q + first * A.qs[2], A.qs[2], A.D, DC, tid, S::kThreads,
                               [&](int r) { return first + r < A.Lq; });
  }
  if (A.table) {
    const T* t = static_cast<const T*>(A.table) + (int64_t)h * A.buckets.num_buckets;
    for (int d = tid; d <= 2 * reach; d += S::kThreads) lut[d] = bias2(to_f(t[bucket_of(A.buckets, d - reach)]));
  }
  cp_commit();
  cp_wait<0>();
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
  if (A.causal && !A.q_pos && !A.k_pos) {
    const int64_t end = i0 + 128 * QT < A.Lq ? i0 + 128 * QT : A.Lq;
    const int64_t seen = A.Lk - A.Lq + end;
    keys = seen < keys ? (seen > 0 ? seen : 0) : keys;
  }
  const int tiles = (int)((keys + BN - 1) / BN);
  const uint32_t tmem = tmem_slot;
  const uint32_t polls = A.polls;

  if (warp < 4 * QT) {
    // -------------------------------------------------------- softmax
    const int t = warp >> 2;
    const int64_t i = i0 + t * 128 + (tid & 127);
    const bool valid = i < A.Lq;
    const int qp = valid ? attn_q_pos(A, b, i) : 0;
    const int qlo = __reduce_min_sync(0xffffffffu, valid ? qp : INT32_MAX);
    const int qhi = __reduce_max_sync(0xffffffffu, valid ? qp : INT32_MIN);
    const uint32_t base = tmem + ((uint32_t)(warp & 3) << 21) + t * (S::kO + 64 * DC);
    float m = -INFINITY, l = 0.f;  // m: the reference the exponentials are taken to
    for (int j = 0; j < tiles; ++j) {
      const TileInfo<BN>& I = info[j % S::kInfo];
      wait(&sfull[t], j & 1, &abort_flag, polls);
      fence_after_sync();
      uint32_t s[BN];
#pragma unroll
      for (int c = 0; c < BN; c += 32) ld32(base + c, s + c);
      tmem_wait_ld();
      float top = m;
#pragma unroll
      for (int sub = 0; sub < BN / kSub; ++sub) {
        uint32_t* x = s + sub * kSub;
        const uint32_t bits = I.live[sub];
        const int lo = I.lo[sub], hi = I.hi[sub];
        const bool later = A.causal && hi > qlo;
        if (bits != 0 && valid | (qlo <= qhi)) {
          const bool near = A.table && !((int64_t)lo - qhi >= reach || (int64_t)hi - qlo <= -reach);
          if (near || later) {
#pragma unroll
            for (int c = 0; c < kSub; c += 4) {
              const int4 kp = *reinterpret_cast<const int4*>(&I.pos[sub * kSub + c]);
              const int k4[4] = {kp.x, kp.y, kp.z, kp.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int d = k4[e] - qp;
                const float bias = A.table ? lut[clamp_reach(d, reach) + reach] : 0.f;
                float v = fmaf(__uint_as_float(x[c + e]), A.scale2, bias);
                if (A.causal && d > 0) v = -INFINITY;
                x[c + e] = __float_as_uint(v);
              }
            }
          } else {
            const float bias = !A.table ? 0.f : lut[(int64_t)lo - qhi >= reach ? 2 * reach : 0];
#pragma unroll
            for (int c = 0; c < kSub; ++c) x[c] = __float_as_uint(fmaf(__uint_as_float(x[c]), A.scale2, bias));
          }
          if (bits != 0xffffffffu) {
#pragma unroll
            for (int c = 0; c < kSub; ++c)
              if (!((bits >> c) & 1u)) x[c] = 0xff800000u;
          }
        } else {
#pragma unroll
          for (int c = 0; c < kSub; ++c) x[c] = 0xff800000u;
        }
#pragma unroll
        for (int c = 0; c < kSub; ++c) top = fmaxf(top, __uint_as_float(x[c]));
      }
      // the reference moves when it must: NaN and the first finite maximum included
      const bool move = !(top - m <= 8.f) && top != -INFINITY;
      if (__any_sync(0xffffffffu, move)) {
        const float f = move ? ex2(m - top) : 1.f;
        if (move) m = top;
        l *= f;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < 64 * DC; c += 16) {
            if (c < A.D) {
              uint32_t o[16];
              ld16(base + S::kO + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              st16(base + S::kO + c, o);
            }
          }
        }
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int c = 0; c < BN; c += 32) {
        uint32_t w[NS][16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = ex2(__uint_as_float(s[c + 2 * e]) - ref), p1 = ex2(__uint_as_float(s[c + 2 * e + 1]) - ref);
          l += p0 + p1;
          uint32_t o[NS];
          split2<NS>(p0, p1, o);
#pragma unroll
          for (int i2 = 0; i2 < NS; ++i2) w[i2][e] = o[i2];
        }
#pragma unroll
        for (int i2 = 0; i2 < NS; ++i2) st16(base + S::kP + i2 * (BN / 2) + c / 2, w[i2]);
      }
      tmem_wait_st();
      fence_before_sync();
      arrive(&pfull[t]);
    }
    // -------------------------------------------------------- output
    if (tiles > 0) {
      wait(&sfull[t], tiles & 1, &abort_flag, polls);
      fence_after_sync();
    }
    const bool broken = abort_flag != 0;
    const float inv = broken ? NAN : l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(A.out) + b * A.os[0] + h * A.os[1] + i * A.os[2];
    constexpr int V = 16 / sizeof(T);
    const bool ovec =
        A.D % V == 0 && ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(A.os[2] * sizeof(T))) & 15) == 0;
#pragma unroll
    for (int c = 0; c < 64 * DC; c += 16) {
      if (c < A.D) {
        uint32_t o[16];
        if (tiles > 0) {
          ld16(base + S::kO + c, o);
          tmem_wait_ld();
        }
        alignas(16) T r[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = from_f<T>(l == 0.f ? 0.f : __uint_as_float(o[e]) * inv);
        if (valid) {
          if (ovec) {
#pragma unroll
            for (int e = 0; e < 16; e += V)
              if (c + e < A.D) *reinterpret_cast<Pack<T, V>*>(out + c + e) = *reinterpret_cast<Pack<T, V>*>(r + e);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c + e < A.D) out[c + e] = r[e];
          }
        }
      }
    }
    if (valid && A.lse)
      A.lse[((int64_t)b * A.H + h) * A.Lq + i] = broken ? NAN : l == 0.f ? -INFINITY : m + log2f(l);
  } else if (warp == 4 * QT) {
    // -------------------------------------------------------- tensor instructions
    if (lane == 0 && tiles > 0) {
      const uint32_t id_s = idesc_bf16(128, BN, false), id_o = idesc_bf16(128, (A.D + 15) / 16 * 16, true);
      const uint32_t aQ = smem_u32(sQ), aK = smem_u32(sK), aV = smem_u32(sV);
      wait(&kfull[0], 0, &abort_flag, polls);
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        scores<NS, 128, BN>(tmem + t * (S::kO + 64 * DC), aQ + t * S::kQ, aK, A.D, DC, id_s);
        mma_commit(&sfull[t]);
      }
      mma_commit(&kempty[0]);
      for (int j = 0; j < tiles; ++j) {
        const int st = j % ST, sn = (j + 1) % ST;
        wait(&vfull[st], (j / ST) & 1, &abort_flag, polls);
        if (j + 1 < tiles) wait(&kfull[sn], ((j + 1) / ST) & 1, &abort_flag, polls);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const uint32_t d = tmem + t * (S::kO + 64 * DC);
          wait(&pfull[t], j & 1, &abort_flag, polls);
          fence_after_sync();
          values<NS, BN>(d + S::kO, d + S::kP, BN / 2, aV + st * S::kKV, DC, id_o, j > 0, [](int k) { return k * 8; });
          if (t == QT - 1) mma_commit(&vempty[st]);
          if (j + 1 < tiles) scores<NS, 128, BN>(d, aQ + t * S::kQ, aK + sn * S::kKV, A.D, DC, id_s);
          mma_commit(&sfull[t]);  // after the last keys: the output is whole
        }
        if (j + 1 < tiles) mma_commit(&kempty[sn]);
      }
      if (abort_flag) {  // nothing may be in flight when the TMEM is freed
        mma_commit(&done);
        mbar_wait(&done, 0, polls);
      }
    }
  } else {
    // -------------------------------------------------------- loads
    const int t = tid - 128 * QT - 32, w = t >> 5;
    const T* K = static_cast<const T*>(A.k) + b * A.ks[0] + hk * A.ks[1];
    const T* V = static_cast<const T*>(A.v) + b * A.vs[0] + hk * A.vs[1];
    constexpr bool ASYNC = NS == 1 && VEC && sizeof(T) == 2;
    for (int j = 0; j < tiles; ++j) {
      const int st = j % ST;
      const int64_t j0 = (int64_t)j * BN;
      TileInfo<BN>& I = info[j % S::kInfo];
      if (j >= ST) wait(&kempty[st], (j / ST - 1) & 1, &abort_flag, polls);
      for (int sub = w; sub < BN / kSub; sub += 3)
        fill_info<BN>(
            I, sub, [&](int e) { return j0 + e < A.Lk && (!mask || mask[j0 + e]); },
            [&](int e) { return attn_k_pos(A, b, j0 + e); });
      named_barrier(1, 96);
      const auto live = [&](int r) { return (I.live[r >> 5] >> (r & 31)) & 1u; };
      load_tile<T, NS, VEC, BN>(sK + st * S::kKV, K + j0 * A.ks[2], A.ks[2], A.D, DC, t, 96, live);
      if constexpr (ASYNC) {
        cp_commit();
        if (j > 0) {  // the values of the tile before have landed
          cp_wait<1>();
          fence_proxy_async_smem();
          arrive(&vfull[(j - 1) % ST]);
        }
        cp_wait<0>();
      }
      fence_proxy_async_smem();
      arrive(&kfull[st]);
      if (j >= ST) wait(&vempty[st], (j / ST - 1) & 1, &abort_flag, polls);
      load_tile<T, NS, VEC, BN>(sV + st * S::kKV, V + j0 * A.vs[2], A.vs[2], A.D, DC, t, 96, live);
      if constexpr (ASYNC) {
        cp_commit();
        if (j + 1 < tiles) continue;
        cp_wait<0>();
      }
      fence_proxy_async_smem();
      arrive(&vfull[st]);
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (warp == 0) tmem_dealloc(tmem, S::kAlloc);
}

}  // namespace tc
}  // namespace fx
