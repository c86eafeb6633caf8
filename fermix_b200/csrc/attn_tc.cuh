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
// bfloat16 tiles on 16-byte boundaries come by tensor maps (one thread issues a tile's copies;
// rows and entries past the ends are filled with zeros); two more warps then clear the rows
// of masked keys, whatever those hold, before the tensor cores may read the tile. float32 is split
// on the way and unaligned storage has no map: those tiles are loaded by the threads.
//
// The forward: a block holds one tile of 128 queries (two that share the keys, bfloat16 above 64
// entries), two threads a row, half the columns each; scores and probabilities live in TMEM. A row's
// reference is its first tile's maximum and moves only when a score is 2^64 above it, which the sum of
// the exponentials shows: no maximum is taken on the way. Few blocks of queries split the keys over
// blocks. Bound: the softmax's latency at two blocks an SM, what TMEM and registers allow: 0.44 of the
// issue slots are used, warps wait for TMEM loads, fixed latencies and each other (64 x 8 heads of
// 512 x 512, dim 64, three quarters of the keys live: 154 us, 167 TFLOP/s of live pairs; 2 x 16 heads of
// 4096 x 4096, dim 128: 406 us a call, 676 TFLOP/s, 0.42 of the library's matrix rate). float32, 512 x 4
// heads of 128 x 128, dim 32: 142 us; its forward up to 64 entries spills 40 registers' worth (152 to
// 160 bytes a thread) at the 80 that two blocks an SM leave.
//
// Fewer bits, and why: in bfloat16 the probabilities are rounded to the operand type of the second
// product (their sum is not), 2^-9 of the values' size at most, as much as the output's own rounding.
// Its sums stay in the accumulator over all keys, which cuts off towards zero below its last bit: 1.6e-8 of
// the sum for every 16 keys by the figure at kRest, 1e-3, half of the output's rounding, after a
// million keys in one part. In float32 the products of parts with index sum 5 and 6 are left out (2^-24
// of a product), the exponential is the approximate instruction (2^-22 of its value), and an
// infinite entry, whose parts are inf - inf, gives NaN in the rows that read it.
#pragma once
#include <cuda.h>

#include "attn_rows.cuh"
#include "umma.cuh"

namespace fx {
namespace tc {

using namespace umma;

constexpr int kSub = 32;  // keys (or queries) whose positions are summarised together

// A tile's layout: chunks of RB bytes a row (128, or 64 for float32's parts of up to 32 entries, which
// halves what they take), DC of them. The 16-byte piece c of row r is at piece
// c ^ (r & 7) (RB = 128) or c ^ (r / 2 & 3) (RB = 64) of its row.
template <int RB_, int DC_>
struct Rows {
  static constexpr int RB = RB_, DC = DC_, kDim = RB / 2 * DC;  // bytes, chunks, entries
  static __device__ __forceinline__ uint32_t at(int rows, int r, int c) {
    constexpr int P = RB / 16;
    return (uint32_t)(c / P) * (uint32_t)(rows * RB) + r * RB + (((c % P) ^ (RB == 128 ? r & 7 : (r >> 1) & 3)) << 4);
  }
};

// K-major / MN-major operand. lbo: bytes between chunks (MN-major only); groups of 8 rows follow
// each other.
template <int RB>
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 | (uint64_t)(RB * 8 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)(RB == 128 ? 2 : 4) << 61;
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
__device__ __forceinline__ void st4(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]));
}
template <int N>
__device__ __forceinline__ void ld_cols(uint32_t a, uint32_t (&v)[N]) {
  static_assert(N == 8 || N == 16);
  if constexpr (N == 8) tmem_ld8(a, v);
  else ld16(a, v);
}
template <int N>
__device__ __forceinline__ void st_cols(uint32_t a, const uint32_t (&v)[N]) {
  static_assert(N == 4 || N == 8);
  if constexpr (N == 4) st4(a, v);
  else st8(a, v);
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
// two float32 operations in one instruction
__device__ __forceinline__ uint64_t both(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void halves(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_both(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_both(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t mul_both(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
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
// After a wait that ran out no more copies are asked for. The threads that asked for the copies and the
// tensor instructions wait for the last of them (of the last ST of n tiles) before they go, with a
// bound of their own and whatever the flag says: another thread's wait may run out after they have
// looked at it, and nothing may be under way when the block ends and its TMEM is freed.
constexpr uint32_t kDrainPolls = 1u << 20;
template <int ST>
__device__ __forceinline__ void drain(uint64_t (&bar)[ST], int64_t n) {
  for (int64_t j = n > ST ? n - ST : 0; j < n; ++j) mbar_wait(&bar[j % ST], (uint32_t)(j / ST) & 1u, kDrainPolls);
}

// How a tile is brought in: by the threads, entry by entry or in 16-byte pieces, or by a tensor map.
enum { LOAD_ENTRIES, LOAD_PIECES, LOAD_TMA };

// Tensor maps of q, k, v and dout: (entry, token, head, batch), boxes of one chunk by BN or 128
// tokens. A dimension the tensor is expanded along has one entry in its map (mul 0).
struct alignas(64) TmaMaps {
  CUtensorMap m[4];
  int head_mul[4], batch_mul[4];
};
enum { MAP_Q, MAP_K, MAP_V, MAP_DO };

// One tile (DC chunks of `rows` rows from token i0) by one thread; the mbarrier was told the bytes.
template <typename L>
__device__ __forceinline__ void tma_tile(unsigned char* dst, const TmaMaps& M, int which, int rows, int64_t i0, int h, int b,
                                         uint64_t* mbar) {
#pragma unroll
  for (int c = 0; c < L::DC; ++c)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_u32(dst) + (uint32_t)(c * rows * L::RB)),
        "l"(&M.m[which]), "r"(c * 64), "r"((int)i0), "r"(h * M.head_mul[which]), "r"(b * M.batch_mul[which]),
        "r"(smem_u32(mbar))
        : "memory");
}

// Zeros in the rows of a tile that are not live, by `n` threads of index t.
template <typename L, typename Live>
__device__ __forceinline__ void clear_rows(unsigned char* dst, int rows, int t, int n, Live live) {
  for (int i = t; i < rows * L::DC; i += n) {
    const int r = i % rows, c = i / rows;
    if (!live(r)) {
      uint4* p = reinterpret_cast<uint4*>(dst + (uint32_t)(c * rows + r) * L::RB);
#pragma unroll
      for (int e = 0; e < L::RB / 16; ++e) p[e] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// Rows [0, R) of a tile from p (element strides `step` a row, dim entries a row, entries
// beyond dim up to the next multiple of 16 zero), row r only if live(r), by `n` threads of index
// t, through registers. Parts of a split type follow each other.
template <typename T, int NS, bool PIECES, int R, typename L, typename Live>
__device__ __forceinline__ void load_tile(unsigned char* dst, const T* p, int64_t step, int dim, int t, int n, Live live) {
  const int pieces = (dim + 15) / 16 * 2;  // of 8 entries
  const int dr = n / pieces, dc = n - dr * pieces;
  int r = t / pieces, c = t - r * pieces;
  constexpr int U = 4;  // pieces on the way at a time
  while (r < R) {
    float x[U][8];
    unsigned char* d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      d[u] = r < R ? dst + L::at(R, r, c) : nullptr;
      const bool ok = r < R && live(r);
      const T* s = p + (ok ? r * step + c * 8 : 0);
      if constexpr (PIECES) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8; h += V) {
          Pack<T, V> k;
#pragma unroll
          for (int e = 0; e < V; ++e) k.e[e] = from_f<T>(0.f);
          if (ok && c * 8 + h < dim) k = *reinterpret_cast<const Pack<T, V>*>(s + h);
#pragma unroll
          for (int e = 0; e < V; ++e) x[u][h + e] = to_f(k.e[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u][e] = ok && c * 8 + e < dim ? to_f(s[e]) : 0.f;
      }
      r += dr;
      c += dc;
      if (c >= pieces) {
        c -= pieces;
        ++r;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (d[u] == nullptr) continue;
      uint32_t w[4][NS];
#pragma unroll
      for (int e = 0; e < 4; ++e) split2<NS>(x[u][2 * e], x[u][2 * e + 1], w[e]);
#pragma unroll
      for (int s = 0; s < NS; ++s)
        *reinterpret_cast<uint4*>(d[u] + s * (R * L::RB * L::DC)) = make_uint4(w[0][s], w[1][s], w[2][s], w[3][s]);
    }
  }
}

// D (+)= A B^T over the k-steps of 16 entries, both K-major tiles of RA / RB rows.
template <int NS, int RA, int RB, typename L>
__device__ __forceinline__ void scores(uint32_t d, uint32_t a, uint32_t b, int dim, uint32_t idesc) {
  // One thread issues all of a block's tensor instructions, one after the other: building a
  // descriptor for each took longer than the product, so they are stepped. Addresses are below
  // 2^18 and stay in their field.
  const int steps = (dim + 15) / 16;
  constexpr int K = L::RB / 32;  // steps of a chunk
  bool acc = false;
  // the smaller products first
#pragma unroll
  for (int sum = NS - 1; sum >= 0; --sum) {
#pragma unroll
    for (int i = 0; i <= sum; ++i) {
      uint64_t da = desc<L::RB>(a + i * (RA * L::RB * L::DC), 16);
      uint64_t db = desc<L::RB>(b + (sum - i) * (RB * L::RB * L::DC), 16);
#pragma unroll 1
      for (int k = 1; k <= steps; ++k) {
        mma_ss(d, da, db, idesc, acc);
        acc = true;
        da += 2;
        db += 2;
        if (L::DC > 1 && k % K == 0) {  // the next chunk
          da += (RA * L::RB >> 4) - 2 * K;
          db += (RB * L::RB >> 4) - 2 * K;
        }
      }
    }
  }
}

// D (+)= A B, A in TMEM (8 columns a part and k-step, from acol(part, k)), B the MN-major view
// of a tile of RB rows (the contraction's index).
template <int NS, int RB, typename L, typename Col>
__device__ __forceinline__ void values(uint32_t d, uint32_t b, uint32_t idesc, bool acc, Col acol) {
#pragma unroll
  for (int sum = NS - 1; sum >= 0; --sum) {
#pragma unroll
    for (int i = 0; i <= sum; ++i) {
      const uint32_t bp = b + (sum - i) * (RB * L::RB * L::DC);
#pragma unroll
      for (int k = 0; k < RB / 16; ++k) {
        mma_ts(d, acol(i, k), desc<L::RB>(bp + k * 16u * L::RB, RB * L::RB), idesc, acc);
        acc = true;
      }
    }
  }
}

// The tensor cores cut off what they add to an accumulator below its last bit, always towards zero:
// a float32 sum over 1165 keys (six products of 16 keys each) was off by 7e-6 of the result. So
// float32 sums are moved on after kRest tiles of 64, added to the output in memory, which the thread
// owns, with rounding; the accumulator starts anew.
constexpr int kRest = 4;
template <int NS>
__device__ __forceinline__ bool starts(int64_t tile) {  // the tile starts a sum
  return NS == 1 ? tile == 0 : tile % kRest == 0;
}

// Up to 8 entries of a sum (n of them are there) from the accumulator to p, added to what is there or
// in its place.
__device__ __forceinline__ void hold8(float* p, int n, bool vec, bool add, bool zero, const uint32_t (&o)[8]) {
  if (vec) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      if (e >= n) break;
      float4 v = add ? *reinterpret_cast<const float4*>(p + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      v.x += __uint_as_float(o[e]);
      v.y += __uint_as_float(o[e + 1]);
      v.z += __uint_as_float(o[e + 2]);
      v.w += __uint_as_float(o[e + 3]);
      *reinterpret_cast<float4*>(p + e) = zero ? make_float4(0.f, 0.f, 0.f, 0.f) : v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = zero ? 0.f : (add ? p[e] : 0.f) + __uint_as_float(o[e]);
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
// A block takes QT tiles of 128 query rows of one head and walks the keys BN at a time. A row
// (TMEM lane) of a tile belongs to two threads, each with half of the columns: a warp's
// exponentials, lookups and conversions are chains that four warps a scheduler cover and two do
// not (measured: 5.1 thousand cycles for 128 columns with one warp a scheduler, 3.2 with two).
// Warps 8 t .. 8 t + 7 work on tile t, the next one issues the tensor instructions, the last three
// load. With QT = 2 one tile's exponentials run while the other's products do.
//
// The exponentials are taken to a reference per row, set from the first tile that holds a live
// key and kept until a score passes it by more than 2^64, which shows in the sums. float32 sums and
// bfloat16 probabilities have the exponent range for that, so the usual pass over the scores
// for their maximum, and the rescaling of the output when it grows, are left to the rare case. (Its
// code is loops, not unrolled: it runs about once a block, and instructions fetched for one use
// cost more than they do.) The reference is taken off after the bias is added, so that what a bias
// of the type's lowest value absorbs stays absorbed. The probabilities go back to TMEM as the A
// operand of the second product: over the scores where TMEM is full (QT = 2, 128 entries), else
// to columns of their own, which lets the next scores be formed before this tile's second product.
struct FwdLane {
  uint32_t base;     // TMEM of the tile, this warp's lanes
  int qp, qlo, qhi;  // this row's position, the warp's rows' least and greatest
  bool valid;
};

// The greatest of the W scores from column c0 of a tile.
template <int BN, int W>
__device__ __forceinline__ float fwd_top(const AttnArgs& A, const TileInfo<BN>& I, const float* lut, const FwdLane& F,
                                         int c0) {
  const int reach = A.buckets.reach;
  float top = -INFINITY;
#pragma unroll 1
  for (int c = c0; c < c0 + W; c += 8) {
    uint32_t x[8];
    tmem_ld8(F.base + c, x);
    tmem_wait_ld();
    const uint32_t bits = I.live[c / kSub] >> (c % kSub);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = I.pos[c + e];
      const float bias = A.table ? lut[clamp_reach(k - F.qp, reach) + reach] : 0.f;
      const float v = fmaf(__uint_as_float(x[e]), A.scale2, bias);
      if (((bits >> e) & 1u) && !(A.causal && k > F.qp)) top = fmaxf(top, v);
    }
  }
  return top;
}

// NS parts of the probabilities of 32 columns into p, their sum back: x the raw scores, ref the
// reference with its sign turned.
template <int NS, int BN>
__device__ __forceinline__ float fwd_columns(const AttnArgs& A, const TileInfo<BN>& I, const float* lut, const FwdLane& F,
                                             int sub, float ref, uint32_t* x, uint32_t (*p)[16]) {
  const int reach = A.buckets.reach, far = 2 * reach;
  const uint32_t bits = I.live[sub];
  const int lo = I.lo[sub], hi = I.hi[sub];
  const bool above = lo - (int64_t)F.qhi >= reach, below = hi - (int64_t)F.qlo <= -reach;
  if (bits == 0 || F.qlo > F.qhi) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) p[n][e] = 0u;
    return 0.f;
  }
  if ((A.table && !above && !below) || (A.causal && hi > F.qlo)) {
    const int qoff = F.qp - reach, qlim = A.causal ? F.qp : INT32_MAX;
#pragma unroll
    for (int c = 0; c < kSub; c += 8) {
      int k[8];
      float bias[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const int4 v = *reinterpret_cast<const int4*>(&I.pos[sub * kSub + c + e]);
        k[e] = v.x;
        k[e + 1] = v.y;
        k[e + 2] = v.z;
        k[e + 3] = v.w;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[e] = A.table ? lut[__vimin_s32_relu(k[e] - qoff, far)] : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = fmaf(__uint_as_float(x[c + e]), A.scale2, bias[e]) + ref;
        x[c + e] = k[e] > qlim ? 0xff800000u : __float_as_uint(v);
      }
    }
  } else {
    const float bias = A.table ? lut[above ? far : 0] : 0.f;
    const uint64_t bb = both(bias, bias), ss = both(A.scale2, A.scale2), rr = both(ref, ref);
#pragma unroll
    for (int c = 0; c < kSub; c += 2) {
      float v0, v1;
      halves(add_both(fma_both(both(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), ss, bb), rr), v0, v1);
      x[c] = __float_as_uint(v0);
      x[c + 1] = __float_as_uint(v1);
    }
  }
  if (bits != 0xffffffffu) {
#pragma unroll
    for (int c = 0; c < kSub; ++c)
      if (!((bits >> c) & 1u)) x[c] = 0xff800000u;
  }
  uint64_t sum[2] = {0, 0};  // pairs of zeros
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float p0 = ex2(__uint_as_float(x[2 * e])), p1 = ex2(__uint_as_float(x[2 * e + 1]));
    sum[e & 1] = add_both(sum[e & 1], both(p0, p1));
    uint32_t o[NS];
    split2<NS>(p0, p1, o);
#pragma unroll
    for (int n = 0; n < NS; ++n) p[n][e] = o[n];
  }
  float a0, a1;
  halves(add_both(sum[0], sum[1]), a0, a1);
  return a0 + a1;
}

template <int NS, int QT, int BN, typename L, int ST>
struct FwdShape {
  static constexpr int kThreads = 256 * QT + 128;
  static constexpr int kHalf = BN / 2;  // columns of a thread
  static constexpr uint32_t kRow = NS * L::DC * L::RB, kQ = 128 * kRow, kKV = BN * kRow;
  static constexpr int kInfo = ST + 1;
  static constexpr uint32_t kTileBytes = QT * kQ + 2 * ST * kKV;
  // TMEM columns of a tile: scores, the probabilities' parts, the output
  static constexpr bool kOver = QT * (BN + NS * BN / 2 + L::kDim) > 512;  // probabilities over the scores
  static constexpr int kP = kOver ? 0 : BN;
  static constexpr int kO = kOver ? BN : BN + NS * BN / 2;
  static_assert(!kOver || NS == 1);
  static constexpr int kTile = kO + L::kDim;
  static constexpr int kCols = QT * kTile;
  static constexpr int kAlloc = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  // blocks an SM holds by TMEM and shared memory (float32's parts of 128 entries: one)
  static constexpr int kBlocks = QT == 1 && kAlloc <= 256 && kTileBytes <= 104 * 1024 ? 2 : 1;
};

template <typename T, int NS, int QT, int BN, typename L, int ST, int LOAD>
__global__ void __launch_bounds__(FwdShape<NS, QT, BN, L, ST>::kThreads, FwdShape<NS, QT, BN, L, ST>::kBlocks)
    attn_fwd_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TmaMaps M) {
  using S = FwdShape<NS, QT, BN, L, ST>;
  constexpr bool TMA = LOAD == LOAD_TMA, PIECES = LOAD == LOAD_PIECES;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char *sQ = sm, *sK = sm + QT * S::kQ, *sV = sK + ST * S::kKV;
  float* lut = reinterpret_cast<float*>(sm + S::kTileBytes);
  __shared__ TileInfo<BN> info[S::kInfo];
  __shared__ uint64_t kfull[ST], vfull[ST], kempty[ST], vempty[ST], kraw[ST], vraw[ST], qraw, sfull[QT], pfull[QT],
      ofull[QT], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ int last_live, moving[QT][2];
  __shared__ float shared_row[QT][2][128];  // what the two threads of a row tell each other
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // block -> (batch, head, query block, part of the keys); under a causal order the longest blocks first
  const int64_t nq = (A.Lq + 128 * QT - 1) / (128 * QT), heads = (int64_t)A.B * A.H;
  const bool ordered = A.causal && !A.q_pos && !A.k_pos;
  const int part = blockIdx.x % A.splits;
  const int64_t block = blockIdx.x / A.splits;
  const int64_t qb = ordered ? nq - 1 - block / heads : block % nq;
  const int64_t bh = ordered ? block % heads : block / nq;
  const int h = (int)(bh % A.H), b = (int)(bh / A.H), hk = h / (A.H / A.Hk);
  const int64_t i0 = qb * 128 * QT;
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_stride : nullptr;
  const int reach = A.buckets.reach;

  if (tid == 0) {
    abort_flag = 0;
    last_live = mask ? 0 : (int)A.Lk;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kfull[i], TMA ? 64 : 96);
      mbar_init(&vfull[i], TMA ? 64 : 96);
      mbar_init(&kempty[i], 1);
      mbar_init(&vempty[i], 1);
      mbar_init(&kraw[i], 2);  // the copies, and the positions
      mbar_init(&vraw[i], 1);
    }
    mbar_init(&qraw, 1);
    for (int t = 0; t < QT; ++t) {
      mbar_init(&sfull[t], 1);
      mbar_init(&pfull[t], 256);
      mbar_init(&ofull[t], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
    if constexpr (TMA) {
      mbar_arrive_expect_tx(&qraw, QT * S::kQ);
      for (int t = 0; t < QT; ++t) tma_tile<L>(sQ + t * S::kQ, M, MAP_Q, 128, i0 + t * 128, h, b, &qraw);
    }
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, S::kAlloc);
    tmem_relinquish();
  }
  if constexpr (!TMA) {
    const T* Q = static_cast<const T*>(A.q) + b * A.qs[0] + h * A.qs[1];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int64_t first = i0 + t * 128;
      load_tile<T, NS, PIECES, 128, L>(sQ + t * S::kQ, Q + first * A.qs[2], A.qs[2], A.D, tid, S::kThreads,
                                       [&](int r) { return first + r < A.Lq; });
    }
  }
  if (A.table) {
    const T* t = static_cast<const T*>(A.table) + (int64_t)h * A.buckets.num_buckets;
    for (int d = tid; d <= 2 * reach; d += S::kThreads) lut[d] = bias2(to_f(t[bucket_of(A.buckets, d - reach)]));
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
    const int64_t end = i0 + 128 * QT < A.Lq ? i0 + 128 * QT : A.Lq;
    const int64_t seen = A.Lk - A.Lq + end;
    keys = seen < keys ? (seen > 0 ? seen : 0) : keys;
  }
  // this part's tiles [first, first + tiles), numbered from 0 below
  const int all = (int)((keys + BN - 1) / BN), per = (all + A.splits - 1) / A.splits;
  const int first = part * per < all ? part * per : all, tiles = all - first < per ? all - first : per;
  const uint32_t tmem = tmem_slot;
  const uint32_t polls = A.polls;

  if (warp < 8 * QT) {
    // -------------------------------------------------------- softmax
    const int t = warp >> 3, half = (warp >> 2) & 1, r = tid & 127;
    const int64_t i = i0 + t * 128 + r;
    const bool valid = i < A.Lq;
    const int qp = valid ? attn_q_pos(A, b, i) : 0;
    const FwdLane F{tmem + ((uint32_t)(warp & 3) << 21) + t * S::kTile, qp,
                    __reduce_min_sync(0xffffffffu, valid ? qp : INT32_MAX),
                    __reduce_max_sync(0xffffffffu, valid ? qp : INT32_MIN), valid};
    const uint32_t base = F.base;
    float m = -INFINITY, l = 0.f;  // the reference (-inf before the first key), the sum of this half
    // Where this row's sums are held (float32), entries [16 half, 16 half + 16) and every 32 on.
    const auto held_row = [&]() -> float* {
      if (A.splits > 1) return A.part + ((((int64_t)b * A.H + h) * A.Lq + i) * A.splits + part) * part_step(A.D) + 4;
      return static_cast<float*>(A.out) + b * A.os[0] + h * A.os[1] + i * A.os[2];
    };
    const bool held = NS > 1 && tiles > kRest;
    if ((tid & 255) < 2) moving[t][tid & 255] = 0;
    named_barrier(2 + t, 256);
    for (int j = 0; j < tiles; ++j) {
      const TileInfo<BN>& I = info[j % S::kInfo];
      wait(&sfull[t], j & 1, &abort_flag, polls);
      fence_after_sync();
      uint32_t p[S::kOver ? S::kHalf / kSub : 1][NS][16];
      bool free_p = S::kOver || j == 0;
      float sum = 0.f;
      if constexpr (NS > 1) {
        if (j > 0 && starts<NS>(j)) {
          wait(&ofull[t], (j - 1) & 1, &abort_flag, polls);
          fence_after_sync();
          free_p = true;
          float* row = held_row();
          const bool held_vec = A.splits > 1 || (A.D % 4 == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0);
          const int entries = A.splits > 1 ? (A.D + 3) / 4 * 4 : A.D;
#pragma unroll 1
          for (int c = half * 16; c < A.D; c += c & 8 ? 24 : 8) {
            uint32_t o[8];
            tmem_ld8(base + S::kO + c, o);
            tmem_wait_ld();
            if (valid) hold8(row + c, entries - c, held_vec, j > kRest, false, o);
          }
        }
      }
      bool moved = false;
      for (;;) {
        bool low = __any_sync(0xffffffffu, valid && m == -INFINITY);
        if (!low || moved) {
          const float ref = m == -INFINITY ? 0.f : -m;
          sum = 0.f;
          if constexpr (S::kOver) {  // held until both halves have read the scores
#pragma unroll
            for (int c = 0; c < S::kHalf / kSub; ++c) {
              const int sub = half * (S::kHalf / kSub) + c;
              uint32_t x[kSub];
              ld32(base + sub * kSub, x);
              tmem_wait_ld();
              sum += fwd_columns<NS, BN>(A, I, lut, F, sub, ref, x, p[c]);
            }
          } else {
#pragma unroll 1  // one copy of the code: the score loops have to stay in the instruction cache
            for (int sub = half * (S::kHalf / kSub); sub < (half + 1) * (S::kHalf / kSub); ++sub) {
              uint32_t x[kSub];
              ld32(base + sub * kSub, x);
              tmem_wait_ld();
              sum += fwd_columns<NS, BN>(A, I, lut, F, sub, ref, x, p[0]);
              if (!free_p) {  // the last tile's second product has read the probabilities
                wait(&ofull[t], (j - 1) & 1, &abort_flag, polls);
                free_p = true;
              }
#pragma unroll
              for (int n = 0; n < NS; ++n) st16(base + S::kP + n * (BN / 2) + sub * (kSub / 2), p[0][n]);
            }
          }
          low = __any_sync(0xffffffffu, valid && !(sum <= 1.8446744e19f));
        }
        if (moved) break;
        // both halves of all rows agree on whether references move (two flags in turn)
        if (low && lane == 0) moving[t][j & 1] = 1;
        named_barrier(2 + t, 256);
        if (!moving[t][j & 1]) break;
        shared_row[t][half][r] = fwd_top<BN, S::kHalf>(A, I, lut, F, half * S::kHalf);
        if (!free_p) {  // the output is at rest
          wait(&ofull[t], (j - 1) & 1, &abort_flag, polls);
          free_p = true;
        }
        fence_after_sync();
        named_barrier(2 + t, 256);
        if ((tid & 255) == 0) moving[t][j & 1] = 0;
        const float top = fmaxf(shared_row[t][0][r], shared_row[t][1][r]);
        float f = 1.f;
        if (m == -INFINITY ? top > -INFINITY : top - m > 64.f) {
          f = m == -INFINITY ? 0.f : ex2(m - top);
          m = top;
        }
        l *= f;
        if (j > 0 && __any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
          for (int c = half * 8; c < A.D; c += 16) {
            uint32_t o[8];
            tmem_ld8(base + S::kO + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st8(base + S::kO + c, o);
          }
        }
        if constexpr (NS > 1) {
          if (j >= kRest && valid && f != 1.f) {
            float* row = held_row();
#pragma unroll 1
            for (int c = half * 16; c < A.D; c += (c & 15) == 15 ? 17 : 1) row[c] *= f;
          }
        }
        moved = true;
      }
      l += sum;
      if constexpr (S::kOver) {
        named_barrier(2 + t, 256);  // both halves have read the scores
#pragma unroll
        for (int c = 0; c < S::kHalf / kSub; ++c)
          st16(base + S::kP + (half * S::kHalf + c * kSub) / 2, p[c][0]);
      }
      tmem_wait_st();
      fence_before_sync();
      arrive(&pfull[t]);
    }
    shared_row[t][half][r] = l;
    named_barrier(2 + t, 256);
    l = shared_row[t][0][r] + shared_row[t][1][r];
    // -------------------------------------------------------- output
    if (tiles > 0) {
      wait(&ofull[t], (tiles - 1) & 1, &abort_flag, polls);
      fence_after_sync();
    }
    const bool broken = abort_flag != 0;
    if (A.splits > 1) {  // (m, l, o) of this part for attn_join_kernel
      float* p = A.part + ((((int64_t)b * A.H + h) * A.Lq + i) * A.splits + part) * part_step(A.D);
#pragma unroll 1
      for (int c = half * 16; c < A.D; c += c & 8 ? 24 : 8) {
        uint32_t o[8];
        if (tiles > 0) {
          tmem_ld8(base + S::kO + c, o);
          tmem_wait_ld();
        }
        if (valid) hold8(p + 4 + c, (A.D + 3) / 4 * 4 - c, true, held, l == 0.f, o);
      }
      if (valid && half == 0) {
        p[0] = m;
        p[1] = broken ? NAN : l;
      }
    } else {
      const bool empty = l == 0.f && !broken;
      const float inv = broken ? NAN : 1.f / l;
      T* out = static_cast<T*>(A.out) + b * A.os[0] + h * A.os[1] + i * A.os[2];
      constexpr int V = 16 / sizeof(T);
      const bool ovec =
          A.D % V == 0 && ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(A.os[2] * sizeof(T))) & 15) == 0;
#pragma unroll
      for (int c = half * 16; c < L::kDim; c += 32) {
        if (c < A.D) {
          uint32_t o[16];
          if (tiles > 0) {
            ld16(base + S::kO + c, o);
            tmem_wait_ld();
          }
          if constexpr (NS > 1) {
            if (held && valid) {
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                if (c + e >= A.D) break;
                Pack<T, 4> v;
                if (ovec) v = *reinterpret_cast<const Pack<T, 4>*>(out + c + e);
                else
#pragma unroll
                  for (int n = 0; n < 4; ++n) v.e[n] = c + e + n < A.D ? out[c + e + n] : 0.f;
#pragma unroll
                for (int n = 0; n < 4; ++n) o[e + n] = __float_as_uint(__uint_as_float(o[e + n]) + v.e[n]);
              }
            }
          }
          alignas(16) T r[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] = from_f<T>(empty ? 0.f : __uint_as_float(o[e]) * inv);
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
      if (valid && half == 0 && A.lse) store_lse(A, ((int64_t)b * A.H + h) * A.Lq + i, m, l, broken);
    }
  } else if (warp == 8 * QT) {
    // -------------------------------------------------------- tensor instructions
    if constexpr (TMA) wait(&qraw, 0, &abort_flag, polls);  // also where there are no keys: nothing is left under way
    if (lane == 0 && tiles > 0) {
      const uint32_t id_s = idesc_bf16(128, BN, false), id_o = idesc_bf16(128, (A.D + 15) / 16 * 16, true);
      const uint32_t aQ = smem_u32(sQ), aK = smem_u32(sK), aV = smem_u32(sV);
      wait(&kfull[0], 0, &abort_flag, polls);
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        scores<NS, 128, BN, L>(tmem + t * S::kTile, aQ + t * S::kQ, aK, A.D, id_s);
        mma_commit(&sfull[t]);
      }
      mma_commit(&kempty[0]);
      for (int j = 0; j < tiles; ++j) {
        const int st = j % ST, sn = (j + 1) % ST;
        const bool more = j + 1 < tiles;
        if (more) wait(&kfull[sn], ((j + 1) / ST) & 1, &abort_flag, polls);
        if (S::kOver) wait(&vfull[st], (j / ST) & 1, &abort_flag, polls);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const uint32_t d = tmem + t * S::kTile;
          wait(&pfull[t], j & 1, &abort_flag, polls);
          fence_after_sync();
          if (!S::kOver && more) {
            scores<NS, 128, BN, L>(d, aQ + t * S::kQ, aK + sn * S::kKV, A.D, id_s);
            mma_commit(&sfull[t]);
            if (t == QT - 1) mma_commit(&kempty[sn]);
          }
          if (!S::kOver && t == 0) wait(&vfull[st], (j / ST) & 1, &abort_flag, polls);
          values<NS, BN, L>(d + S::kO, aV + st * S::kKV, id_o, !starts<NS>(j),
                            [=](int part, int k) { return d + S::kP + part * (BN / 2) + k * 8; });
          mma_commit(&ofull[t]);
          if (t == QT - 1) mma_commit(&vempty[st]);
          if (S::kOver && more) {
            scores<NS, 128, BN, L>(d, aQ + t * S::kQ, aK + sn * S::kKV, A.D, id_s);
            mma_commit(&sfull[t]);
            if (t == QT - 1) mma_commit(&kempty[sn]);
          }
        }
      }
      mma_commit(&done);
      mbar_wait(&done, 0, kDrainPolls);
    }
  } else {
    // -------------------------------------------------------- loads
    const int t = tid - 256 * QT - 32, w = t >> 5;
    const auto fill = [&](int j, int sub) {
      const int64_t j0 = (int64_t)(first + j) * BN;
      fill_info<BN>(
          info[j % S::kInfo], sub, [&](int e) { return j0 + e < A.Lk && (!mask || mask[j0 + e]); },
          [&](int e) { return attn_k_pos(A, b, j0 + e); });
    };
    if constexpr (TMA) {
      if (w == 0) {
        int keys_asked = 0, values_asked = 0;
        for (int j = 0; j < tiles; ++j) {
          const int st = j % ST;
          if (j >= ST) wait(&kempty[st], (j / ST - 1) & 1, &abort_flag, polls);
          if (__any_sync(0xffffffffu, abort_flag)) break;
          ++keys_asked;
          if (lane == 0) {
            mbar_arrive_expect_tx(&kraw[st], S::kKV);
            tma_tile<L>(sK + st * S::kKV, M, MAP_K, BN, (int64_t)(first + j) * BN, hk, b, &kraw[st]);
          }
          for (int sub = 0; sub < BN / kSub; ++sub) fill(j, sub);
          __syncwarp();
          if (lane == 0) arrive(&kraw[st]);
          if (j >= ST) wait(&vempty[st], (j / ST - 1) & 1, &abort_flag, polls);
          if (__any_sync(0xffffffffu, abort_flag)) break;
          ++values_asked;
          if (lane == 0) {
            mbar_arrive_expect_tx(&vraw[st], S::kKV);
            tma_tile<L>(sV + st * S::kKV, M, MAP_V, BN, (int64_t)(first + j) * BN, hk, b, &vraw[st]);
          }
        }
        mbar_wait(&qraw, 0, kDrainPolls);
        drain(kraw, keys_asked);
        drain(vraw, values_asked);
      } else {
        for (int j = 0; j < tiles; ++j) {
          const int st = j % ST;
          const TileInfo<BN>& I = info[j % S::kInfo];
          const auto live = [&](int r) { return (I.live[r >> 5] >> (r & 31)) & 1u; };
          if (mask) wait(&vraw[st], (j / ST) & 1, &abort_flag, polls);
          wait(&kraw[st], (j / ST) & 1, &abort_flag, polls);
          if (mask) {
            clear_rows<L>(sK + st * S::kKV, BN, t - 32, 64, live);
            clear_rows<L>(sV + st * S::kKV, BN, t - 32, 64, live);
            fence_proxy_async_smem();
          }
          arrive(&kfull[st]);
          if (!mask) wait(&vraw[st], (j / ST) & 1, &abort_flag, polls);
          arrive(&vfull[st]);
        }
      }
    } else {
      const T* K = static_cast<const T*>(A.k) + b * A.ks[0] + hk * A.ks[1];
      const T* V = static_cast<const T*>(A.v) + b * A.vs[0] + hk * A.vs[1];
      for (int j = 0; j < tiles; ++j) {
        const int st = j % ST;
        const int64_t j0 = (int64_t)(first + j) * BN;
        TileInfo<BN>& I = info[j % S::kInfo];
        if (j >= ST) wait(&kempty[st], (j / ST - 1) & 1, &abort_flag, polls);
        for (int sub = w; sub < BN / kSub; sub += 3) fill(j, sub);
        named_barrier(1, 96);
        const auto live = [&](int r) { return (I.live[r >> 5] >> (r & 31)) & 1u; };
        load_tile<T, NS, PIECES, BN, L>(sK + st * S::kKV, K + j0 * A.ks[2], A.ks[2], A.D, t, 96, live);
        fence_proxy_async_smem();
        arrive(&kfull[st]);
        if (j >= ST) wait(&vempty[st], (j / ST - 1) & 1, &abort_flag, polls);
        load_tile<T, NS, PIECES, BN, L>(sV + st * S::kKV, V + j0 * A.vs[2], A.vs[2], A.D, t, 96, live);
        fence_proxy_async_smem();
        arrive(&vfull[st]);
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
