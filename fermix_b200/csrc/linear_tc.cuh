// The linear map's products on the tensor cores: D(i, j) = sum over k of A(i, k) B(j, k), the
// forward (x, W), dx (g, W) and dW (g, x) alike. Each operand is read as it is stored, along k
// (K-major) or across it (MN-major).
//
// A pair of SMs holds a tile of 256 x 256: each brings 128 rows of A and 128 of B by tensor maps (64
// entries of k a stage) and keeps 128 rows of the sum in its TMEM, twice, so that one tile's epilogue
// runs under the next tile's products. The grid is persistent.
//
// float32 runs on the same bfloat16 instructions: x = x1 + x2 + x3, each part the rest rounded to
// bfloat16, holds 24 bits, and the six products with index sum <= 4 leave out terms of 2^-24. The
// tensor cores cut off what they add to an accumulator below its last bit, always towards zero, so
// float32 sums are moved on to registers, with rounding, every kChunk blocks of k. In bfloat16 the
// whole sum stays in the accumulator: 1.6e-8 of it is lost for every 16 entries of k, which reaches
// half of the output's rounding (2e-3) after a million.
//
// Tiles that do not fill the device, or the last round of many, split k over pairs of SMs; the parts are
// float32 sums in the workspace, added in order by linear_join_kernel, which then does the epilogue.
//
// Bound by the tensor cores where the result is large beside k, else by the epilogue's bytes. Measured: bfloat16 8192 x
// 2048 -> 8192 with gelu and its slope 226 us, 1216 TFLOP/s, the two gradients 411 us, 1338 TFLOP/s (the library's
// product of the same sizes 180 us, 1527); float32 65536 x 256 -> 512 with silu 115 us, the two gradients 162 us, in
// bfloat16 products 896 and 1272 TFLOP/s, besides 27 and 106 us for the layout.
#pragma once
#include <cuda.h>

#include "linear_common.cuh"
#include "umma.cuh"

namespace fx {
namespace lin {

using namespace umma;

constexpr int kTile = 256, kHalf = 128, kBlockK = 64;  // of a pair, of an SM, of a stage
constexpr int kWarps = 16;                             // of the epilogue: 32 rows, 64 columns each
constexpr int kThreads = 64 + 32 * kWarps;             // and one warp for the copies, one for the products
constexpr uint32_t kOperand = kHalf * kBlockK * 2;     // bytes of an SM's rows of an operand

template <int NP>
struct Shape {
  static constexpr int kStages = NP == 1 ? 5 : 2;
  static constexpr int kStore = NP == 1 ? 32 : 16;  // columns that a warp stores at a time
  static constexpr uint32_t kBlock = 32 * kStore * 4;
  static constexpr uint32_t kStage = 2 * NP * kOperand;  // the parts of A, the parts of B
  static constexpr uint32_t kSmem = kStages * kStage + kWarps * kBlock + 1024;
  static constexpr int kChunk = 2;  // blocks of k in an accumulator (three parts)
};

// One product, cut into units: tiles that a pair does alone, then parts of the others.
struct Args {
  int64_t rows, cols;      // of the result
  int blocks, tm, tn;      // blocks of k, tiles
  int whole, splits, per;  // tiles done alone; parts of each other tile, blocks of k of a part
  int a_mn, b_mn, vec;     // vec: rows of y, slope, residual and bias are whole pieces of 16 bytes
  float* part;             // of the tiles from `whole` on: (tile, part, 256, 256)
  Epilogue e;

  __host__ __device__ int joined() const { return tm * tn - whole; }
  __host__ __device__ int units() const { return whole + joined() * splits; }
};

// The products of a launch: one, or a backward pass' two, whose tiles fill the device together. Its units are of two
// lengths, `longs` long ones (of one product its whole tiles, of two the first product's units) and then `shorts` short
// ones. The pairs of SMs take the long ones in turn; those left without one in the last round do `ahead` rounds of
// short ones meanwhile, then all pairs take the other short ones in turn.
struct Group {
  Args p[2];
  int longs, shorts, ahead;
  uint32_t polls;
  // a backward pass' sums of g over blocks of rows, (sum_blocks, sum_cols), and where their sums go
  const float* sums;
  void* dbias;
  int sum_blocks;
  int64_t sum_cols;
};
struct alignas(64) Maps {
  CUtensorMap m[4];  // A and B of each product
};

// ---------------------------------------------------------------- instructions of a pair
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// True in one lane of the warp, which is converged: the same one every time.
__device__ __forceinline__ bool elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
// The address of the pair's first block's copy of a shared variable.
__device__ __forceinline__ uint32_t first_block(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
// An arrival that orders TMEM reads alone (with the fence before it): a release to the cluster would wait for the
// epilogue's stores to memory too, which took most of its time.
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}
// Arrival at both blocks' copies of the barrier when the products issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void alloc_pair(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void dealloc_pair(uint32_t t) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(t));
}
#define FX_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
__device__ __forceinline__ void ld32(uint32_t a, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : FX_R8(v, 0), FX_R8(v, 8), FX_R8(v, 16), FX_R8(v, 24)
      : "r"(a));
}
__device__ __forceinline__ void ld16(uint32_t a, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : FX_R8(v, 0), FX_R8(v, 8)
      : "r"(a));
}
#define FX_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void st16(uint32_t a, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      FX_I8(v, 0), FX_I8(v, 8));
}
#undef FX_I8
#undef FX_R8

// 128-byte swizzled operand: rows of 64 entries of k, or, MN-major, rows of 64 entries across k, 64 of
// them (of k) a chunk, chunks of 8 KB after each other.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, bool mn) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(mn ? 8192 >> 4 : 1) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// A bounded wait. One that runs out is recorded (the block's outputs become NaN) and waits once
// more, with a limit of its own, so that nothing is under way that the block does not know of; if that
// runs out too, the block's threads wait and issue no more, and its tiles are filled with NaN.
enum { RUNS = 0, LATE = 1, DEAD = 2 };
constexpr uint32_t kLastPolls = 1u << 22;
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* state, uint32_t polls) {
  const uint32_t few = polls < 32 ? polls : 32;
  if (mbar_wait(bar, parity, few)) return true;
  if (*state == DEAD) return false;
  if (mbar_wait(bar, parity, polls - few)) return true;
  record_status(8);  // FX_ERR_TIMEOUT
  if (*state == RUNS) *state = LATE;
  if (mbar_wait(bar, parity, kLastPolls)) return true;
  *state = DEAD;
  return false;
}
// The same for a whole warp, whose lanes poll for themselves: instructions that need all of them follow, so they take one
// way, on where the wait ended for every lane.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* state, uint32_t polls) {
  return __all_sync(0xffffffffu, wait(bar, parity, state, polls));
}
__device__ __forceinline__ bool warp_runs(volatile int* state) { return __all_sync(0xffffffffu, *state != DEAD); }

// ---------------------------------------------------------------- epilogue
// NaN in the place of sums that a wait did not end for.
template <int C>
__device__ __forceinline__ void spoil(int state, uint32_t (&v)[C]) {
  if (state != RUNS) {
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = 0x7fc00000u;
  }
}

// N entries of a row: activation, residual, stores.
template <typename T, int ACT, int N, bool RES, bool SLOPE>
__device__ __forceinline__ void finish(const float (&h)[N], const Pack<T, N>& residual, T* y, typename SlopeOf<T>::type* slope) {
  float v[N], d[N], res[N];
  unpack<N>(residual, res);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const ActOut a = activate<ACT>(h[e]);
    v[e] = RES ? a.y + res[e] : a.y;
    d[e] = a.d;
  }
  Pack<T, N> o;
  round_into<N>(o, v);
  *reinterpret_cast<Pack<T, N>*>(y) = o;
  if constexpr (SLOPE) {
    Pack<typename SlopeOf<T>::type, N> s;
    round_into<N>(s, d);
    *reinterpret_cast<Pack<typename SlopeOf<T>::type, N>*>(slope) = s;
  }
}

// A warp's staging block holds 32 rows of C entries; the 16-byte piece p of row r is at piece
// p ^ (r & 7) of its row (C = 32) or p ^ (r >> 1 & 3) (C = 16).
template <int C>
__device__ __forceinline__ uint32_t staged(int r, int p) {
  return r * (C * 4) + ((C == 32 ? p ^ (r & 7) : p ^ (r >> 1 & 3)) << 4);
}

// Of 32 x C staged entries of the sum, N entries of a row a lane (16 bytes of the result, or, where rows are
// not whole pieces, one), so that stores cover whole sectors; R rows at a time. y, slope and residual are this
// lane's, `last` is the number of rows from its first on.
template <typename T, int ACT, int C, int N, bool RES, bool SLOPE>
__device__ __forceinline__ void store_rows(const Args& G, const unsigned char* stage, T* y, typename SlopeOf<T>::type* slope,
                                           const T* residual, const Pack<T, N>& bias, int last) {
  constexpr int L = C / N, R = 32 / L, U = N == 1 ? 8 : 2;  // U: residuals read ahead
  const int lane = threadIdx.x & 31, c = lane % L * N, r0 = lane / L;
  const int64_t step = R * G.cols, rstep = R * G.e.rs;
  float b[N];
  unpack<N>(bias, b);
#pragma unroll (N == 1 ? 1 : 32)
  for (int k0 = 0; k0 < 32; k0 += U * R) {
    Pack<T, N> res[U] = {};
    if constexpr (RES) {
#pragma unroll
      for (int u = 0; u < U; ++u, residual += rstep)
        if (k0 + u * R < last) res[u] = *reinterpret_cast<const Pack<T, N>*>(residual);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float h[N];
      if constexpr (N == 1) {
        h[0] = *reinterpret_cast<const float*>(stage + staged<C>(k0 + u * R + r0, c / 4) + (c & 3) * 4);
      } else {
        static_assert(R % 8 == 0);  // the swizzle is the same every time
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const float4 x = *reinterpret_cast<const float4*>(stage + (k0 + u * R) * (C * 4) + staged<C>(r0, (c + e) / 4));
          h[e] = x.x;
          h[e + 1] = x.y;
          h[e + 2] = x.z;
          h[e + 3] = x.w;
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) h[e] += b[e];
      if (k0 + u * R < last) finish<T, ACT, N, RES, SLOPE>(h, res[u], y, slope);
      y += step;
      if constexpr (SLOPE) slope += step;
    }
  }
}

// A warp's 32 rows and 64 columns of a tile: where its lanes' entries go.
template <typename T, int C, int N>
struct Lines {
  using TS = typename SlopeOf<T>::type;
  T* y;
  TS* slope;
  const T *residual, *bias;
  int last;      // rows
  int64_t left;  // columns from this lane's first on

  __device__ __forceinline__ Lines(const Args& G, int64_t i0, int64_t j0) {
    constexpr int L = C / N;
    const int lane = threadIdx.x & 31;
    const int64_t i = i0 + lane / L, j = j0 + lane % L * N;
    last = (int)(G.rows - i < 32 ? G.rows - i : 32);
    left = G.cols - j;
    y = static_cast<T*>(G.e.y) + i * G.cols + j;
    slope = G.e.slope ? static_cast<TS*>(G.e.slope) + i * G.cols + j : nullptr;
    residual = G.e.residual ? static_cast<const T*>(G.e.residual) + i * G.e.rs + j : nullptr;
    bias = G.e.bias ? static_cast<const T*>(G.e.bias) + j : nullptr;
  }
  template <int ACT>
  __device__ __forceinline__ void store(const Args& G, const unsigned char* stage) {  // and on to the next C columns
    if (left > 0) {
      Pack<T, N> b = {};
      if (bias) b = *reinterpret_cast<const Pack<T, N>*>(bias);
      if (ACT != FX_ACT_NONE && slope) {
        if (residual) store_rows<T, ACT, C, N, true, true>(G, stage, y, slope, residual, b, last);
        else store_rows<T, ACT, C, N, false, true>(G, stage, y, slope, residual, b, last);
      } else {
        if (residual) store_rows<T, ACT, C, N, true, false>(G, stage, y, slope, residual, b, last);
        else store_rows<T, ACT, C, N, false, false>(G, stage, y, slope, residual, b, last);
      }
    }
    y += C;
    if (slope) slope += C;
    if (residual) residual += C;
    if (bias) bias += C;
    left -= C;
  }
};

// The sums themselves, to a row-major tile of 256 columns.
template <int C>
__device__ __forceinline__ void store_part(float* out, const unsigned char* stage) {
  constexpr int L = C / 4, R = 32 / L;
  const int lane = threadIdx.x & 31, r0 = lane / L;
  out += r0 * kTile + lane % L * 4;
#pragma unroll
  for (int k = 0; k < 32; k += R)
    *reinterpret_cast<float4*>(out + k * kTile) = *reinterpret_cast<const float4*>(stage + staged<C>(k + r0, lane % L));
}

struct Unit {
  int q, m, n, part, first, last;  // product, tile, place among the parts (-1: whole), blocks of k
};
// Tiles in groups of 8 rows of tiles, down the columns of a group, so that what runs at a time shares
// rows and columns; the parts of a tile next to each other.
__device__ __forceinline__ Unit unit_of(const Args& G, int u) {
  Unit U;
  int t = u;
  U.q = 0;
  U.part = -1;
  U.first = 0;
  U.last = G.blocks;
  if (u >= G.whole) {
    U.part = u - G.whole;
    const int v = U.part / G.splits;
    t = G.whole + v;
    U.first = (U.part - v * G.splits) * G.per;
    U.last = min(U.first + G.per, G.blocks);
  }
  const int group = t / (8 * G.tn), in = t - group * 8 * G.tn;
  const int rows = min(8, G.tm - group * 8);
  U.n = rows == 8 ? in >> 3 : in / rows;
  U.m = group * 8 + in - U.n * rows;
  return U;
}
// Pair `pair`'s i-th unit of a launch by `pairs`; false behind its last.
__device__ __forceinline__ bool unit_of(const Group& G, int pair, int pairs, int i, Unit& U) {
  const int rounds = G.longs / pairs, rest = G.longs - rounds * pairs;
  int u;
  if (i < rounds + (pair < rest)) {
    u = i * pairs + pair;
  } else {
    i -= rounds;
    int v;
    if (pair >= rest && i < G.ahead) v = i * (pairs - rest) + pair - rest;
    else v = G.ahead * (pairs - rest) + (i - (pair < rest ? 1 : G.ahead)) * pairs + pair;
    if (v >= G.shorts) return false;
    u = G.longs + v;
  }
  const int first = G.p[0].units(), q = u >= first;
  U = unit_of(G.p[q], u - (q ? first : 0));
  U.q = q;
  return true;
}

// The epilogue of a warp's 32 rows and 64 columns of a tile, in TMEM from `from` on, C columns at a time through the
// warp's staging block.
template <typename T, int ACT, int C>
__device__ __forceinline__ void epilogue(const Args& G, const Unit& U, unsigned char* stage, int row, int col, uint32_t from,
                                         volatile int* state) {
  constexpr int B = 64 / C, UNROLL = C == 32 ? B : 1;  // float32 needs the registers
  const int lane = threadIdx.x & 31;
  const int64_t i0 = (int64_t)U.m * kTile + row, j0 = (int64_t)U.n * kTile + col;
  const auto bring = [&](int c) {
    uint32_t v[C];
    if constexpr (C == 32) ld32(from + c * C, v);
    else ld16(from + c * C, v);
    tmem_wait_ld();
    spoil(*state, v);
    __syncwarp();
#pragma unroll
    for (int p = 0; p < C / 4; ++p)
      *reinterpret_cast<uint4*>(stage + staged<C>(lane, p)) = make_uint4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
    __syncwarp();
  };
  if (U.part >= 0) {
    float* out = G.part + ((int64_t)U.part * kTile + row) * kTile + col;
#pragma unroll UNROLL
    for (int c = 0; c < B; ++c, out += C) {
      bring(c);
      store_part<C>(out, stage);
    }
  } else if (G.vec) {
    Lines<T, C, 16 / sizeof(T)> lines(G, i0, j0);
#pragma unroll UNROLL
    for (int c = 0; c < B; ++c) {
      if (j0 + c * C >= G.cols) break;
      bring(c);
      lines.template store<ACT>(G, stage);
    }
  } else {
    Lines<T, C, 1> lines(G, i0, j0);
#pragma unroll 1
    for (int c = 0; c < B; ++c) {
      if (j0 + c * C >= G.cols) break;
      bring(c);
      lines.template store<ACT>(G, stage);
    }
  }
}

// The sums of g over the rows from those of blocks of rows, in order: 32 columns a warp.
template <typename T>
__device__ __forceinline__ void bias_sums(const float* sums, int blocks, int64_t cols, void* dbias, int64_t warp, int64_t warps) {
  for (int64_t j = warp * 32 + (threadIdx.x & 31); j < cols; j += warps * 32) {
    float s = 0.f;
#pragma unroll 16
    for (int b = 0; b < blocks; ++b) s += sums[b * cols + j];
    static_cast<T*>(dbias)[j] = from_f<T>(s);
  }
}

// NaN for a block's 128 rows of its units, by the epilogue's warps. (Not inlined: its registers would be the epilogue's.)
template <typename T>
__device__ __noinline__ void fill_nan(const Group& G, int first_row) {
  using TS = typename SlopeOf<T>::type;
  const float nan = __int_as_float(0x7fc00000);
  Unit U;
  for (int n = 0; unit_of(G, blockIdx.x >> 1, gridDim.x >> 1, n, U); ++n) {
    const Args& A = G.p[U.q];
    for (int e = threadIdx.x - 64; e < kHalf * kTile; e += 32 * kWarps) {
      const int r = first_row + e / kTile, c = e % kTile;
      const int64_t i = (int64_t)U.m * kTile + r, j = (int64_t)U.n * kTile + c;
      if (U.part >= 0) {
        A.part[((int64_t)U.part * kTile + r) * kTile + c] = nan;
      } else if (i < A.rows && j < A.cols) {
        static_cast<T*>(A.e.y)[i * A.cols + j] = from_f<T>(nan);
        if (A.e.slope) static_cast<TS*>(A.e.slope)[i * A.cols + j] = from_f<TS>(nan);
      }
    }
  }
}

template <typename T, int NP, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_tc_kernel(const __grid_constant__ Group G, const __grid_constant__ Maps M) {
  using S = Shape<NP>;
  constexpr int ST = S::kStages;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[ST], empty[ST], sum_full[2], sum_empty[2];
  __shared__ uint32_t slot;
  __shared__ volatile int state;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cta_rank();
  if (tid == 0) {
    state = RUNS;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sum_full[i], 1);
      mbar_init(&sum_empty[i], 2 * kWarps);  // the epilogue's warps of both blocks
    }
    fence_mbar_init();
  }
  if (warp == 2) alloc_pair(&slot);
  fence_before_sync();
  __syncthreads();
  cluster_sync();
  fence_after_sync();
  wait_for_last();
  const uint32_t tmem = slot;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  Unit U;
  constexpr int kAll = 1 << 30;
  constexpr int chunk = NP == 1 ? kAll : S::kChunk;  // blocks of k in an accumulator

  if (warp == 0) {
    // -------------------------------------------------------- copies, one thread of each block
    if (lane == 0) {
      int it = 0;
      for (int n = 0; state != DEAD && unit_of(G, pair, pairs, n, U); ++n) {
        const CUtensorMap *ma = &M.m[2 * U.q], *mb = ma + 1;
        const bool a_mn = G.p[U.q].a_mn, b_mn = G.p[U.q].b_mn;
        const int i0 = U.m * kTile + rank * kHalf, j0 = U.n * kTile + rank * kHalf;
        for (int kb = U.first; kb < U.last; ++kb, ++it) {
          const int st = it % ST;
          if (!wait(&empty[st], (it / ST & 1) ^ 1, &state, G.polls)) break;
          const uint32_t bar = first_block(&full[st]), at = smem_u32(sm) + st * S::kStage;
          if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * S::kStage);
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            const uint32_t a = at + p * kOperand, b = at + (NP + p) * kOperand;
            if (a_mn) {
              tma_box(a, ma, i0, kb * kBlockK, p, bar);
              tma_box(a + 8192, ma, i0 + 64, kb * kBlockK, p, bar);
            } else {
              tma_box(a, ma, kb * kBlockK, i0, p, bar);
            }
            if (b_mn) {
              tma_box(b, mb, j0, kb * kBlockK, p, bar);
              tma_box(b + 8192, mb, j0 + 64, kb * kBlockK, p, bar);
            } else {
              tma_box(b, mb, kb * kBlockK, j0, p, bar);
            }
          }
        }
      }
      // after a wait that ran out: the copies asked for, with a bound (the second block's are counted by the first's
      // barriers: it waits its limit)
      if (state == DEAD)
        for (int j = it > ST ? it - ST : 0; j < it; ++j) mbar_wait(&full[j % ST], j / ST & 1, 1u << 20);
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- products, one warp of the pair
    // The whole warp runs the loops, so that descriptors stay in uniform registers, and one lane issues.
    if (rank == 0) {
      int st = 0, ch = 0, issued = 0;  // blocks of k
      uint32_t phase = 0;
      for (int n = 0; warp_runs(&state) && unit_of(G, pair, pairs, n, U); ++n) {
        const bool a_mn = G.p[U.q].a_mn, b_mn = G.p[U.q].b_mn;
        const uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
                               (uint32_t)(kTile >> 3) << 17 | (uint32_t)(kTile >> 4) << 24;
        const uint32_t sa = a_mn ? 128 : 2, sb = b_mn ? 128 : 2;  // 16 entries of k further, in 16 bytes
        const uint64_t a0 = desc(smem_u32(sm), a_mn), b0 = desc(smem_u32(sm) + NP * kOperand, b_mn);
        for (int k0 = U.first; k0 < U.last; k0 += chunk, ++ch) {
          const int buf = ch % 2;
          if (!wait_warp(&sum_empty[buf], (ch / 2 & 1) ^ 1, &state, G.polls)) break;
          fence_after_sync();
          const uint32_t d = tmem + buf * kTile;
          const int k1 = min(k0 + chunk, U.last);
          for (int kb = k0; kb < k1; ++kb) {
            if (!wait_warp(&full[st], phase, &state, G.polls)) break;
            fence_after_sync();
            if (elected()) {
              const uint64_t a1 = a0 + (uint32_t)(st * (S::kStage >> 4)), b1 = b0 + (uint32_t)(st * (S::kStage >> 4));
#pragma unroll
              for (int sum = NP - 1; sum >= 0; --sum) {  // the smaller products first
#pragma unroll
                for (int i = 0; i <= sum; ++i) {
#pragma unroll
                  for (int k = 0; k < kBlockK / 16; ++k)
                    mma_pair(d, a1 + i * (kOperand >> 4) + k * sa, b1 + (sum - i) * (kOperand >> 4) + k * sb, idesc,
                             kb > k0 || sum < NP - 1 || i > 0 || k > 0);
                }
              }
              commit_pair(&empty[st]);
              if (kb == k1 - 1) commit_pair(&sum_full[buf]);
            }
            __syncwarp();
            ++issued;
            if (++st == ST) {
              st = 0;
              phase ^= 1;
            }
          }
        }
      }
      // after a wait that ran out: the products issued, which read shared memory and write TMEM, with a bound
      if (!warp_runs(&state))
        for (int j = issued > ST ? issued - ST : 0; j < issued; ++j) mbar_wait(&empty[j % ST], j / ST & 1, 1u << 20);
    }
  } else {
    // -------------------------------------------------------- epilogue
    if (G.dbias)  // while the first tile's products run
      bias_sums<T>(G.sums, G.sum_blocks, G.sum_cols, G.dbias, blockIdx.x * kWarps + warp - 2, gridDim.x * kWarps);
    constexpr int C = 16, B = 64 / C;
    const int quarter = warp & 3, strip = (warp - 2) >> 2, row = rank * kHalf + quarter * 32, col = strip * 64;
    unsigned char* stage = sm + ST * S::kStage + (warp - 2) * S::kBlock;
    const uint32_t lanes = tmem + ((uint32_t)quarter << 21) + col;
    int ch = 0;
    for (int n = 0; warp_runs(&state) && unit_of(G, pair, pairs, n, U); ++n) {
      float acc[NP == 1 ? 1 : B][C];
      for (int k0 = U.first; k0 < U.last; k0 += chunk, ++ch) {
        const int buf = ch % 2;
        if (!wait_warp(&sum_full[buf], ch / 2 & 1, &state, G.polls)) break;
        fence_after_sync();
        const uint32_t from = lanes + buf * kTile;
        const bool last = NP == 1 || k0 + chunk >= U.last;
        if constexpr (NP > 1) {
          // The sums so far are in registers; with the last of them they go back to TMEM, from where they are stored.
          const bool more = k0 > U.first;
          if (more || !last) {
#pragma unroll
            for (int c = 0; c < B; ++c) {
              uint32_t v[C];
              ld16(from + c * C, v);
              tmem_wait_ld();
              if (more) {
#pragma unroll
                for (int e = 0; e < C; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + acc[c][e]);
              }
              if (last) {
                st16(from + c * C, v);
              } else {
#pragma unroll
                for (int e = 0; e < C; ++e) acc[c][e] = __uint_as_float(v[e]);
              }
            }
            if (last) tmem_wait_st();
          }
        }
        if (last) epilogue<T, ACT, S::kStore>(G.p[U.q], U, stage, row, col, from, &state);
        fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_at(first_block(&sum_empty[buf]));
      }
    }
  }
  __syncwarp();
  fence_before_sync();
  cluster_sync();
  fence_after_sync();
  if (warp == 2) dealloc_pair(tmem);
  if (warp >= 2 && state == DEAD) fill_nan<T>(G, rank * kHalf);
}

// ---------------------------------------------------------------- around the products
// The parts of the split tiles in order, then the epilogue; N columns a thread, P * 256 threads a tile. Both
// products' tiles, one after the other.
template <typename T, int ACT, int N>
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ Group H) {
  wait_for_last();
  constexpr int P = kTile / N;  // pieces of a row
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int v = (int)(t / (P * kTile));
  const int second = v >= H.p[0].joined();
  const Args& G = H.p[second];
  if (second) v -= H.p[0].joined();
  const int row = (int)(t / P) % kTile, col = (int)(t % P) * N;
  const Unit U = unit_of(G, G.whole + v * G.splits);
  const int64_t i = (int64_t)U.m * kTile + row, j = (int64_t)U.n * kTile + col;
  if (i >= G.rows || j >= G.cols) return;
  const float* p = G.part + ((int64_t)v * G.splits * kTile + row) * kTile + col;
  float h[N] = {};
#pragma unroll 4
  for (int s = 0; s < G.splits; ++s, p += kTile * kTile) {
    if constexpr (N == 1) {
      h[0] += *p;
    } else {
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 x = *reinterpret_cast<const float4*>(p + e);
        h[e] += x.x;
        h[e + 1] += x.y;
        h[e + 2] += x.z;
        h[e + 3] += x.w;
      }
    }
  }
  using TS = typename SlopeOf<T>::type;
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (G.e.bias) h[e] += to_f(static_cast<const T*>(G.e.bias)[j + e]);
  T* y = static_cast<T*>(G.e.y) + i * G.cols + j;
  TS* slope = G.e.slope ? static_cast<TS*>(G.e.slope) + i * G.cols + j : nullptr;
  Pack<T, N> res = {};
  if (G.e.residual) {
    res = *reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(G.e.residual) + i * G.e.rs + j);
    if (ACT != FX_ACT_NONE && slope) finish<T, ACT, N, true, true>(h, res, y, slope);
    else finish<T, ACT, N, true, false>(h, res, y, slope);
  } else {
    if (ACT != FX_ACT_NONE && slope) finish<T, ACT, N, false, true>(h, res, y, slope);
    else finish<T, ACT, N, false, false>(h, res, y, slope);
  }
}

template <typename T>
__device__ __forceinline__ void load_eight(const T* p, int64_t n, bool vec, float (&x)[8]) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
#pragma unroll
    for (int h = 0; h < 8; h += V) {
      if (h < n) {
        unpack<V>(*reinterpret_cast<const Pack<T, V>*>(p + h), x + h);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[h + e] = 0.f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < n ? to_f(p[e]) : 0.f;
  }
}

template <int NP>
__device__ __forceinline__ void store_parts(uint16_t* out, int64_t plane, const float (&x)[8]) {
  uint32_t w[4][NP];
#pragma unroll
  for (int e = 0; e < 4; ++e) split_pair<NP>(x[2 * e], x[2 * e + 1], w[e]);
#pragma unroll
  for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4*>(out + p * plane) = make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]);
}

// What is laid out anew for the products: up to two operands as NP planes of bfloat16, (NP, rows, ld), ld a multiple
// of 8, and g = dy act'(h) likewise (out not NULL) with each block's sums over its rows (sums not NULL): `tpr` threads
// share a row of g, eight columns each, `per` rows a block. In bfloat16 g is rounded to it here, as the products' operand
// has to be (its sums are not): both gradients are then off by two roundings, 2.3e-3 of them in the norm, in the place of
// one, 1.7e-3. A second part of g would keep that and double the products (411 us of 8192 x 2048 -> 8192).
struct Layout {
  const void* src;
  int64_t stride, rows, cols, ld;
  uint16_t* out;
  int vec, blocks;  // blocks of the launch that work on it
};
struct PrepArgs {
  Layout g, o[2];
  const void* slope;
  float* sums;  // (blocks of rows, cols)
  int64_t per;
  int tpr, strips;
};

template <typename T, int NP>
__device__ __forceinline__ void lay_out(const Layout& A, int block) {
  const int64_t eights = A.ld / 8, n = A.rows * eights;
  for (int64_t t = (int64_t)block * 256 + threadIdx.x; t < n; t += (int64_t)A.blocks * 256) {
    const int64_t i = t / eights, j = (t - i * eights) * 8;
    float x[8];
    load_eight<T>(static_cast<const T*>(A.src) + i * A.stride + j, A.cols - j, A.vec, x);
    store_parts<NP>(A.out + i * A.ld + j, A.rows * A.ld, x);
  }
}

// One row a thread at a time and five blocks an SM: 8192 x 8192 bfloat16 with their slopes 78 us, 5.2 TB/s. Rows ahead cost
// the blocks that hide as much: four rows unrolled 90 to 120 us, two loaded before the first is stored 97 (four blocks an
// SM), six blocks, whose registers spill, 81.
constexpr int kPrepBlocks = 5;

template <typename T, int NP>
__global__ void __launch_bounds__(256, kPrepBlocks) linear_prep_kernel(const __grid_constant__ PrepArgs P) {
  using TS = typename SlopeOf<T>::type;
  __shared__ float share[8][256];
  int block = blockIdx.x;
  if (block >= P.g.blocks) {
    block -= P.g.blocks;
    if (block < P.o[0].blocks) lay_out<T, NP>(P.o[0], block);
    else lay_out<T, NP>(P.o[1], block - P.o[0].blocks);
    return;
  }
  const Layout& A = P.g;
  const int strip = block % P.strips, rows = block / P.strips;
  const int groups = 256 / P.tpr, g = threadIdx.x / P.tpr, col = threadIdx.x & (P.tpr - 1);
  const int64_t j = ((int64_t)strip * P.tpr + col) * 8, r0 = rows * P.per;
  const int64_t end = r0 + P.per < A.rows ? r0 + P.per : A.rows;
  float sum[8] = {};
  if (j < A.cols) {
#pragma unroll 1
    for (int64_t i = r0 + g; i < end; i += groups) {
      float x[8];
      load_eight<T>(static_cast<const T*>(A.src) + i * A.stride + j, A.cols - j, A.vec, x);
      if (P.slope) {
        float d[8];
        load_eight<TS>(static_cast<const TS*>(P.slope) + i * A.cols + j, A.cols - j, A.vec, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], d[e]);  // the same g whether it is stored or only summed
      }
      if (A.out) store_parts<NP>(A.out + i * A.ld + j, A.rows * A.ld, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += x[e];
    }
  }
  if (!P.sums) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) share[e][threadIdx.x] = sum[e];
  __syncthreads();
  // the groups' sums in order, a column a thread
  for (int c = threadIdx.x; c < P.tpr * 8; c += 256) {
    const int64_t jj = (int64_t)strip * P.tpr * 8 + c;
    if (jj >= A.cols) break;
    float s = 0.f;
    for (int k = 0; k < groups; ++k) s += share[c & 7][k * P.tpr + (c >> 3)];
    P.sums[rows * A.cols + jj] = s;
  }
}

// The sums alone, where no product follows.
template <typename T>
__global__ void __launch_bounds__(256) linear_bias_kernel(const float* sums, int blocks, int64_t cols, void* dbias) {
  wait_for_last();
  bias_sums<T>(sums, blocks, cols, dbias, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8);
}

}  // namespace lin
}  // namespace fx
