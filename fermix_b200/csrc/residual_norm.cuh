// The gated residual between two blocks of a network, with the norms on both sides of it:
//
//   nf = (f - mean f) / sqrt(mean (f - mean f)^2 + eps)      (kind 1; kind 0 leaves the mean in)
//   u  = nf post_w + post_b,   r = x + scale gate u,
//   nr = the same norm of r,   z = nr pre_w + pre_b
//
// and its gradient. With the total gradient of r
//   t  = dr + inv_r (a - mean(a) [kind 1] - nr mean(a nr)),  a = dz pre_w
// it is dx = t, du = t scale gate, df = inv_f (b - mean(b) [kind 1] - nf mean(b nf)) with
// b = du post_w; dgate = t scale u and dscale = t gate u summed over what they are shared by;
// dpost_w = sum du nf, dpost_b = sum du, dpre_w = sum dz nr, dpre_b = sum dz over the rows. The
// three that belong to f need two sums only, P = sum t gate nf and Q = sum t gate:
// dpost_w = scale P, dpost_b = scale Q, dscale = post_w P + post_b Q; and a gate shared by rows has
// dgate = scale (post_w sum t nf + post_b sum t).
//
// Bound: HBM. A row is read once and held in registers by a group of TPR threads (a part of a
// warp for narrow rows, a block for wide ones), E entries a thread. The mean and the centred squares
// come from one reduction, of the sums of v - c and (v - c)^2 about an entry c of the row, so that
// nothing of a large mean cancels. The backward recomputes
// nf, r and nr from x, f and gate -- the same bytes that the saved statistics and r would
// be, and r unrounded -- and keeps the sums over rows in registers while a block walks its
// rows; each block writes one partial row per parameter and norm_finish_kernel adds those in
// block order. While a row is worked on (up to four reductions in a row, each a wait), the next
// rows are under way: a thread copies its own entries of them into a ring in shared memory
// (cp.async), which no other thread reads, so the ring needs no barrier.
//
// Measured: 524288 rows of 128 in float32, a gate for each entry: forward 232 us (1.34 GB, 5.8 TB/s,
// 0.88 of a copy's rate), backward 370 us (2.15 GB with the inputs read again, 5.8 TB/s): HBM. 31293 rows
// of 1000 in bfloat16, centred, a gate for each group: forward 89 us (250 MB, 2.8 TB/s), backward
// 160 us (376 MB, 2.4 TB/s): instructions, of the two norms and their reductions over a block. Rows of 999,
// off the 16-byte boundaries: 182 us a call forward, 484 us trained, where 1000 take 90 and 250. Rows of more
// than 512 chunks give a thread two or four, which at 128 registers spill in the backward (1.0 to 1.6 KB a
// thread in bfloat16 and from 4096 float32 entries on): 4096 rows of 8192, trained: float32 467 us (2.6
// TB/s of what the inputs, results and gradients take), bfloat16 353 us (1.7 TB/s), unaligned bfloat16
// 646 us; rows of 4096: 186 and 174 us.
#pragma once
#include "block_common.cuh"

namespace fx {

struct NormArgs {
  const void *x, *f, *gate, *scale, *pw, *pb, *rw, *rb;  // p: post (of f), r: pre (of r)
  void *r, *z;
  const void *gr, *gz;
  void *dx, *df, *dgate;
  float* part;   // (4, grid, W): P, Q, dpre_w, dpre_b
  float* gpart;  // (grid + groups, W): slot block + group, gate_mode 3
  int64_t N, R;  // all rows, rows of a group
  int64_t per;   // rows of a block
  float eps;
  int W, layer, gate_mode, dgate_f32, tpr;
};

constexpr int kNormThreads = 256;  // block of the sub-warp groups; wider rows: one row a block
constexpr int kNormSums = 4;

// Sums over the TPR threads of a row. Blocks that hold one row go through shared memory,
// alternating between two buffers so that one barrier a sum is enough.
// WIDE: more than a warp a row.
template <bool WIDE>
struct RowSum {
  float* red;  // 2 x 32 x 4
  int tpr, flip;
  float inv_w;  // 1 / width
  __device__ __forceinline__ float4* put(float a, float b, float c) {
    float4* buf = reinterpret_cast<float4*>(red) + flip * 32;
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float4(a, b, c, 0.f);
    __syncthreads();
    return buf;
  }
  __device__ __forceinline__ void lanes(float& a, float& b) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      if (WIDE || o < tpr) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
  }
  // the means of a and b
  __device__ __forceinline__ float2 mean2(float a, float b) {
    lanes(a, b);
    if (WIDE) {
      const float4* buf = put(a, b, 0.f);
      const int nw = tpr >> 5;
      a = b = 0.f;
#pragma unroll 4
      for (int i = 0; i < nw; ++i) {
        const float2 v = *reinterpret_cast<const float2*>(&buf[i]);
        a += v.x;
        b += v.y;
      }
    }
    return make_float2(a * inv_w, b * inv_w);
  }
  __device__ __forceinline__ float mean(float a) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      if (WIDE || o < tpr) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (WIDE) {
      const float4* buf = put(a, 0.f, 0.f);
      const int nw = tpr >> 5;
      a = 0.f;
#pragma unroll 4
      for (int i = 0; i < nw; ++i) a += buf[i].x;
    }
    return a * inv_w;
  }
  // (mean, mean of the centred squares) from the sums a of v - c and b of (v - c)^2 over the
  // 1 / inv_count entries of the warp (or group): c is an entry, so nothing of a large mean
  // cancels; the warps are joined about the first one's mean.
  __device__ __forceinline__ float2 moments(float a, float b, float c, float count, float inv_count) {
    lanes(a, b);
    const float m = a * inv_count, sq = fmaxf(fmaf(-m, a, b), 0.f);
    if (!WIDE) return make_float2(c + m, sq * inv_w);
    const float4* buf = put(c + m, sq, count);
    const int nw = tpr >> 5;
    const float base = buf[0].x;
    float s = 0.f, q = 0.f, d2 = 0.f;
#pragma unroll 4
    for (int i = 0; i < nw; ++i) {
      const float4 v = buf[i];
      const float d = v.x - base, nd = v.z * d;
      s += nd;
      d2 = fmaf(nd, d, d2);
      q += v.y;
    }
    const float shift = s * inv_w;
    return make_float2(base + shift, (q + fmaxf(fmaf(-shift, s, d2), 0.f)) * inv_w);
  }
};

// L1: the neighbour reads the same piece (unaligned rows).
template <bool L1>
__device__ __forceinline__ void cp_async16(uint4* dst, const void* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if (L1) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
}

// A thread's part of a row: NV chunks of 16 bytes, neighbouring threads next to each other.
// The mapping does not depend on alignment, so the sums (and the results' bits) do not
// either. ALIGNED: every row and parameter starts on a 16-byte boundary and the width is whole
// chunks. Otherwise a chunk is cut out of the two aligned 16-byte pieces around it, and stored
// as aligned pieces joined with the neighbour's entries.
template <typename T, int NV, bool ALIGNED, bool WIDE>
struct NormRow {
  static constexpr int C = 16 / sizeof(T), E = C * NV;
  int t, tpr, W;
  float count, inv_count;  // entries of the row that this warp (or group) holds
  float kept[ALIGNED ? NV : E];  // 1 within the row, 0 past its end
  __device__ __forceinline__ int at(int v) const { return (v * tpr + t) * C; }
  __device__ __forceinline__ float keep(int e) const { return kept[ALIGNED ? e / C : e]; }
  __device__ __forceinline__ bool in(int e) const { return at(e / C) + (ALIGNED ? 0 : e % C) < W; }
  static constexpr int P = ALIGNED ? 1 : 2;  // aligned pieces that hold a chunk
  // Whether the aligned pieces around entries [c, c + C) of the row at p lie in [begin, end).
  struct Where {
    const T* a;
    uint32_t off;  // bytes of the first piece before the chunk
    bool two, whole;
  };
  __device__ __forceinline__ Where where(const T* p, int c, const T* begin, const T* end) const {
    Where w;
    w.off = (uint32_t)(reinterpret_cast<uintptr_t>(p + c) & 15);
    w.a = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(p + c) - w.off);
    const int got = C - (int)(w.off / sizeof(T));
    w.two = got < C && c + got < W;
    w.whole = w.a >= begin && w.a + (w.two ? 2 * C : C) <= end;
    return w;
  }
  static __device__ __forceinline__ uint4 shifted(uint4 u, uint4 x, uint32_t off) {
    const bool w2 = off & 8, w1 = off & 4;
    const uint32_t a0 = w2 ? u.z : u.x, a1 = w2 ? u.w : u.y, a2 = w2 ? x.x : u.z, a3 = w2 ? x.y : u.w,
                   a4 = w2 ? x.z : x.x, a5 = w2 ? x.w : x.y;
    const uint32_t b0 = w1 ? a1 : a0, b1 = w1 ? a2 : a1, b2 = w1 ? a3 : a2, b3 = w1 ? a4 : a3, b4 = w1 ? a5 : a4;
    const uint32_t sh = (off & 2) * 8;
    return make_uint4(__funnelshift_r(b0, b1, sh), __funnelshift_r(b1, b2, sh), __funnelshift_r(b2, b3, sh),
                      __funnelshift_r(b3, b4, sh));
  }
  __device__ __forceinline__ Pack<T, C> entrywise(const T* p, int c) const {
    Pack<T, C> k;
#pragma unroll
    for (int e = 0; e < C; ++e) k.e[e] = c + e < W ? p[c + e] : from_f<T>(0.f);
    return k;
  }
  __device__ __forceinline__ void unpack(const Pack<T, C>& k, int v, float (&o)[E], float fill) const {
#pragma unroll
    for (int e = 0; e < C; ++e) o[v * C + e] = in(v * C + e) ? to_f(k.e[e]) : fill;
  }
  // The row at p, a part of the array [begin, end) (not there, past the width: fill).
  __device__ __forceinline__ void load(const T* p, const T* begin, const T* end, bool there, float (&o)[E],
                                       float fill) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (there && at(v) < W) {
        Pack<T, C> k;
        if constexpr (ALIGNED) {
          k = *reinterpret_cast<const Pack<T, C>*>(p + at(v));
        } else {
          const Where w = where(p, at(v), begin, end);
          if (w.whole) {
            const uint4 u = *reinterpret_cast<const uint4*>(w.a);
            const uint4 x = w.two ? *reinterpret_cast<const uint4*>(w.a + C) : make_uint4(0u, 0u, 0u, 0u);
            const uint4 r = shifted(u, x, w.off);
            k = *reinterpret_cast<const Pack<T, C>*>(&r);
          } else {
            k = entrywise(p, at(v));
          }
        }
        unpack(k, v, o, fill);
      } else {
#pragma unroll
        for (int e = 0; e < C; ++e) o[v * C + e] = fill;
      }
    }
  }
  // a parameter of W entries (nullptr: fill)
  __device__ __forceinline__ void load(const T* p, float (&o)[E], float fill) const {
    load(p, p, p + W, p != nullptr, o, fill);
  }
  // The row at p, a part of the array [begin, end), into this thread's slots: pieces `stride`
  // apart. An array's own ends are fetched entry by entry, already shifted.
  __device__ __forceinline__ void fetch(uint4* slot, int stride, const T* p, const T* begin, const T* end) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (at(v) < W) {
        if constexpr (ALIGNED) {
          cp_async16<false>(slot + v * stride, p + at(v));
        } else {
          const Where w = where(p, at(v), begin, end);
          if (w.whole) {
            cp_async16<true>(slot + 2 * v * stride, w.a);
            if (w.two) cp_async16<true>(slot + (2 * v + 1) * stride, w.a + C);
          } else {
            const Pack<T, C> k = entrywise(p, at(v));
            slot[2 * v * stride] = *reinterpret_cast<const uint4*>(&k);
          }
        }
      }
    }
  }
  // What fetch left in the slots (a row that is not there: 0).
  __device__ __forceinline__ void take(const uint4* slot, int stride, const T* p, const T* begin, const T* end,
                                       bool there, float (&o)[E]) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      uint4 r = make_uint4(0u, 0u, 0u, 0u);
      if (there && at(v) < W) {
        if constexpr (ALIGNED) {
          r = slot[v * stride];
        } else {
          const Where w = where(p, at(v), begin, end);
          r = slot[2 * v * stride];
          if (w.whole) r = shifted(r, w.two ? slot[(2 * v + 1) * stride] : make_uint4(0u, 0u, 0u, 0u), w.off);
        }
      }
      const Pack<T, C> k = *reinterpret_cast<const Pack<T, C>*>(&r);
#pragma unroll
      for (int e = 0; e < C; ++e) o[v * C + e] = ALIGNED || in(v * C + e) ? to_f(k.e[e]) : 0.f;
    }
  }
  // Every lane of the warp calls this; a row that is not there is not written.
  __device__ __forceinline__ void store(T* p, const float (&o)[E], bool there) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = at(v);
      Pack<T, C> k;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < C; e += 2)
          *reinterpret_cast<__nv_bfloat162*>(&k.e[e]) = __floats2bfloat162_rn(o[v * C + e], o[v * C + e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < C; ++e) k.e[e] = from_f<T>(o[v * C + e]);
      }
      if constexpr (ALIGNED) {
        if (there && c < W) *reinterpret_cast<Pack<T, C>*>(p + c) = k;
      } else {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15);  // c is whole chunks
        const int back = (int)(off / sizeof(T));                               // entries in the piece before
        const uint4 u = *reinterpret_cast<const uint4*>(&k);
        uint4 l;  // the left neighbour's chunk
        l.x = __shfl_up_sync(0xffffffffu, u.x, 1);
        l.y = __shfl_up_sync(0xffffffffu, u.y, 1);
        l.z = __shfl_up_sync(0xffffffffu, u.z, 1);
        l.w = __shfl_up_sync(0xffffffffu, u.w, 1);
        if (!there || c >= W) continue;
        const int lane = threadIdx.x & 31;
        const bool left = t > 0 && lane > 0, right = t + 1 < tpr && lane < 31 && c + C < W;
        // the aligned piece that ends in this chunk: (left chunk, this chunk) moved back by off
        const uint32_t d = 16 - off;  // bytes to drop from the left chunk
        const bool w2 = d & 8, w1 = d & 4;
        const uint32_t a0 = w2 ? l.z : l.x, a1 = w2 ? l.w : l.y, a2 = w2 ? u.x : l.z, a3 = w2 ? u.y : l.w,
                       a4 = w2 ? u.z : u.x, a5 = w2 ? u.w : u.y;
        const uint32_t b0 = w1 ? a1 : a0, b1 = w1 ? a2 : a1, b2 = w1 ? a3 : a2, b3 = w1 ? a4 : a3, b4 = w1 ? a5 : a4;
        const uint32_t sh = (d & 2) * 8;
        uint4 r = make_uint4(__funnelshift_r(b0, b1, sh), __funnelshift_r(b1, b2, sh), __funnelshift_r(b2, b3, sh),
                             __funnelshift_r(b3, b4, sh));
        if (off == 0) r = u;
        T* q = p + c - back;
        if ((left || back == 0) && c + C - back <= W) {
          *reinterpret_cast<uint4*>(q) = r;
        } else {
          const Pack<T, C> m = *reinterpret_cast<const Pack<T, C>*>(&r);
#pragma unroll
          for (int e = 0; e < C; ++e)
            if ((e >= back || left) && c - back + e < W) q[e] = m.e[e];
        }
        if (!right) {
#pragma unroll
          for (int e = 0; e < C; ++e)
            if (e >= C - back && c + e < W) p[c + e] = k.e[e];
        }
      }
    }
  }
  // v <- normalised v (entries outside the row are 0 and stay so), returns 1 / rms; 0 of a row that is
  // not there, whose own would be infinite without eps and make NaN of its zeros.
  __device__ __forceinline__ float normalise(float (&v)[E], bool there, bool layer, float eps, RowSum<WIDE>& sum) const {
    if (!layer) {
      float q = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) q = fmaf(v[e], v[e], q);
      const float rms = rsqrtf(sum.mean(q) + eps), inv = there ? rms : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] *= inv;
      return inv;
    }
    const float c = __shfl_sync(0xffffffffu, v[0], WIDE ? 0 : threadIdx.x & 31 & ~(tpr - 1));
    float a = 0.f, q = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = fmaf(-c, keep(e), v[e]);
      a += d;
      q = fmaf(d, d, q);
    }
    const float2 m = sum.moments(a, q, c, count, inv_count);
    const float inv = there ? rsqrtf(m.y + eps) : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fmaf(-m.x, keep(e), v[e]) * inv;
    return inv;
  }
  // a <- the gradient through normalise(): inv (a - mean(a) [layer] - n mean(a n))
  __device__ __forceinline__ void back(float (&a)[E], const float (&n)[E], float inv, bool layer, RowSum<WIDE>& sum) const {
    float s = 0.f, d = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (layer) s += a[e];
      d = fmaf(a[e], n[e], d);
    }
    const float2 m = layer ? sum.mean2(s, d) : make_float2(0.f, sum.mean(d));
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = inv * fmaf(-m.x, keep(e), fmaf(-n[e], m.y, a[e]));
  }
};

template <typename Row>
__device__ __forceinline__ Row make_row(int t, int tpr, int W) {
  Row row;
  row.t = t;
  row.tpr = tpr;
  row.W = W;
  float n = 0.f;
#pragma unroll
  for (int e = 0; e < Row::E; ++e) {
    n += row.in(e) ? 1.f : 0.f;
    row.kept[sizeof(row.kept) / 4 == Row::E ? e : e / Row::C] = row.in(e) ? 1.f : 0.f;
  }
  row.count = lanes_sum(n, tpr < 32 ? tpr : 32);
  row.inv_count = row.count > 0.f ? 1.f / row.count : 0.f;
  return row;
}

// The arrays of a row (nullptr: not there), and this thread's ring of their entries: three rows
// deep, two where the pieces are twice as many. Rows of several chunks a thread that would not
// fit are loaded when they are needed.
template <typename T, int NV, bool ALIGNED, bool WIDE, int K>
struct NormRing {
  using Row = NormRow<T, NV, ALIGNED, WIDE>;
  static constexpr int S = NV == 1 ? (ALIGNED ? 3 : 2) : NV == 2 && ALIGNED ? 2 : 0;
  static constexpr int kThreadBytes = S * K * NV * Row::P * 16;
  const T* array[K];
  uint4* slots;  // + threadIdx.x
  const T* last[K];
  int64_t W;
  __device__ __forceinline__ uint4* slot(int stage, int k) const {
    return slots + (stage * K + k) * (NV * Row::P) * (int)blockDim.x;
  }
  __device__ __forceinline__ int next(int stage) const { return S == 0 || stage == S - 1 ? 0 : stage + 1; }
  // Row i, S - 1 steps before it is taken.
  __device__ __forceinline__ void fetch(const Row& row, int stage, int64_t i, bool there) const {
    if (S == 0) return;
    if (there) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (array[k]) row.fetch(slot(stage, k), blockDim.x, array[k] + i * W, array[k], last[k]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void wait() const {
    if (S > 0) asm volatile("cp.async.wait_group %0;" ::"n"(S > 0 ? S - 1 : 0) : "memory");
  }
  __device__ __forceinline__ void take(const Row& row, int stage, int k, int64_t i, bool there,
                                       float (&o)[Row::E]) const {
    if constexpr (S == 0)
      row.load(array[k] + i * W, array[k], last[k], there && array[k], o, 0.f);
    else
    row.take(slot(stage, k), blockDim.x, array[k] + i * W, array[k], last[k], there && array[k], o);
  }
};

// The rows of a block in steps of rpb, each step within one group of the gate (gate_mode 3);
// counted from the block's first row.
struct NormWalk {
  int base, end, last, rpb;
  bool grouped;
  int64_t first, R;
  __device__ __forceinline__ int segment_end(int i) const {
    if (!grouped) return last;
    const int64_t e = ((first + i) / R + 1) * R - first;
    return e < last ? (int)e : last;
  }
  __device__ __forceinline__ NormWalk(const NormArgs& A, int rpb_)
      : base(0), rpb(rpb_), grouped(A.gate_mode == FX_GATE_GROUP), first((int64_t)blockIdx.x * A.per), R(A.R) {
    last = (int)(first + A.per < A.N ? A.per : A.N - first);
    end = segment_end(0);
  }
  __device__ __forceinline__ void step() {
    base += rpb;
    if (base >= end && end < last) {
      base = end;
      end = segment_end(base);
    }
  }
};

// Threads an SM holds of the forward: eight entries a thread with the weights take 80 registers.
template <typename T, int NV>
constexpr int kNormFwdResident = NV > 1 ? 512 : sizeof(T) == 4 ? 1024 : 768;

template <typename T, int NV, bool ALIGNED, bool WIDE>
__global__ void __launch_bounds__(kNormFwdResident<T, NV>) norm_fwd_kernel(const __grid_constant__ NormArgs A) {
  using Row = NormRow<T, NV, ALIGNED, WIDE>;
  constexpr int E = Row::E;
  extern __shared__ uint4 ring_mem[];
  __shared__ __align__(16) float red[256];
  const int tpr = A.tpr, W = A.W, rpb = WIDE ? 1 : blockDim.x / tpr;
  const int sub = WIDE ? 0 : threadIdx.x / tpr;
  const Row row = make_row<Row>((int)threadIdx.x - sub * tpr, tpr, W);
  RowSum<WIDE> sum{red, tpr, 0, 1.f / (float)W};
  const T* gate = static_cast<const T*>(A.gate);
  using Ring = NormRing<T, NV, ALIGNED, WIDE, 3>;
  Ring ring;
  ring.array[0] = static_cast<const T*>(A.f);
  ring.array[1] = static_cast<const T*>(A.x);
  ring.array[2] = A.gate_mode == FX_GATE_FULL ? gate : nullptr;
  ring.slots = ring_mem + threadIdx.x;
  ring.W = W;
#pragma unroll
  for (int k = 0; k < 3; ++k) ring.last[k] = ring.array[k] + A.N * W;
  // scale folded into the first norm's weights: scale u = nf s1 + b1
  float s1[E], b1[E], w2[E], b2[E], g[E];
  row.load(static_cast<const T*>(A.scale), g, 1.f);
  row.load(static_cast<const T*>(A.pw), s1, 0.f);
  row.load(static_cast<const T*>(A.pb), b1, 0.f);
  row.load(static_cast<const T*>(A.rw), w2, 0.f);
  row.load(static_cast<const T*>(A.rb), b2, 0.f);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s1[e] *= g[e];
    b1[e] *= g[e];
    g[e] = 1.f;
  }
  NormWalk now(A, rpb), ahead = now;
  int seg = -1;
#pragma unroll
  for (int n = 0; n < Ring::S - 1; ++n) {
    ring.fetch(row, n, ahead.first + ahead.base + sub, ahead.base + sub < ahead.end);
    ahead.step();
  }
  int stage = 0;
  for (; now.base < now.last; now.step()) {
    const int64_t i = now.first + now.base + sub;
    const bool there = now.base + sub < now.end;
    ring.fetch(row, stage == 0 ? Ring::S - 1 : stage - 1, ahead.first + ahead.base + sub,
               ahead.base + sub < ahead.end);
    ahead.step();
    ring.wait();
    float f[E], x[E];
    ring.take(row, stage, 0, i, there, f);
    ring.take(row, stage, 1, i, there, x);
    if (A.gate_mode == FX_GATE_FULL) {
      ring.take(row, stage, 2, i, there, g);
    } else if (A.gate_mode == FX_GATE_ROW) {
      const float g1 = there ? to_f(gate[i]) : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = g1;
    } else if (now.grouped && now.end != seg) {
      seg = now.end;
      row.load(gate + (now.first + now.base) / A.R * W, g, 0.f);
    }
    stage = ring.next(stage);
    row.normalise(f, there, A.layer, A.eps, sum);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaf(g[e], fmaf(f[e], s1[e], b1[e]), x[e]);
    row.store(static_cast<T*>(A.r) + (there ? i * W : 0), x, there);
    row.normalise(x, there, A.layer, A.eps, sum);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaf(x[e], w2[e], b2[e]);
    row.store(static_cast<T*>(A.z) + (there ? i * W : 0), x, there);
  }
}

// The block's sum of acc over its rows to out[0..W): over the warp's groups by shuffles,
// over the warps through buf (8 x W floats), in warp order.
template <typename Row>
__device__ __forceinline__ void norm_block_sum(float (&acc)[Row::E], const Row& row, float* buf, float* out) {
  const int tpr = row.tpr, W = row.W;
  if (tpr > 32) {
#pragma unroll
    for (int e = 0; e < Row::E; ++e)
      if (row.in(e)) out[row.at(e / Row::C) + e % Row::C] = acc[e];
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < Row::E; ++e) {
    float v = acc[e];
    for (int o = tpr; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane < tpr && row.in(e)) buf[warp * W + row.at(e / Row::C) + e % Row::C] = v;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < W; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < kNormThreads / 32; ++w) s += buf[w * W + i];
    out[i] = s;
  }
  __syncthreads();
}

// Registers for 768 threads an SM with four entries a thread, 512 with eight (the sums over rows).
template <typename T, int NV>
constexpr int kNormBwdResident = sizeof(T) == 4 && NV == 1 ? 768 : 512;

template <typename T, int NV, bool ALIGNED, bool WIDE, bool LAYER>
__global__ void __launch_bounds__(kNormBwdResident<T, NV>) norm_bwd_kernel(const __grid_constant__ NormArgs A) {
  using Row = NormRow<T, NV, ALIGNED, WIDE>;
  constexpr int E = Row::E;
  extern __shared__ uint4 ring_mem[];
  __shared__ __align__(16) float red[256];
  const int tpr = A.tpr, W = A.W, rpb = WIDE ? 1 : blockDim.x / tpr;
  const int sub = WIDE ? 0 : threadIdx.x / tpr;
  const Row row = make_row<Row>((int)threadIdx.x - sub * tpr, tpr, W);
  RowSum<WIDE> sum{red, tpr, 0, 1.f / (float)W};
  const T* gate = static_cast<const T*>(A.gate);
  using Ring = NormRing<T, NV, ALIGNED, WIDE, 5>;
  Ring ring;
  ring.array[0] = static_cast<const T*>(A.f);
  ring.array[1] = static_cast<const T*>(A.x);
  ring.array[2] = static_cast<const T*>(A.gz);
  ring.array[3] = static_cast<const T*>(A.gr);
  ring.array[4] = A.gate_mode == FX_GATE_FULL ? gate : nullptr;
  ring.slots = ring_mem + threadIdx.x;
  ring.W = W;
#pragma unroll
  for (int k = 0; k < 5; ++k) ring.last[k] = ring.array[k] + A.N * W;
  float* block_buf = reinterpret_cast<float*>(ring_mem + Ring::kThreadBytes / 16 * blockDim.x);  // past the ring
  // scale u = nf s1 + b1; P, Q: sums of t gate nf and t gate (of a shared gate: of t nf and t
  // within its segment, times the gate after it)
  float s1[E], b1[E], w2[E], g[E], P[E], Q[E], aw[E], ab[E];
  row.load(static_cast<const T*>(A.scale), g, 1.f);
  row.load(static_cast<const T*>(A.pw), s1, 0.f);
  row.load(static_cast<const T*>(A.pb), b1, 0.f);
  row.load(static_cast<const T*>(A.rw), w2, 0.f);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s1[e] *= g[e];
    b1[e] *= g[e];
    g[e] = 1.f;
    P[e] = Q[e] = aw[e] = ab[e] = 0.f;
  }
  NormWalk now(A, rpb), ahead = now;
#pragma unroll
  for (int n = 0; n < Ring::S - 1; ++n) {
    ring.fetch(row, n, ahead.first + ahead.base + sub, ahead.base + sub < ahead.end);
    ahead.step();
  }
  int stage = 0;
  while (now.base < now.last) {
    float Pg[E], Qg[E];  // of a segment
    const int64_t grp = now.grouped ? (now.first + now.base) / A.R : 0;
    const int end = now.end;
    if (now.grouped) {
      row.load(gate + grp * W, g, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) Pg[e] = P[e], Qg[e] = Q[e], P[e] = Q[e] = 0.f;
    }
    for (; now.base < end && now.end == end; now.step()) {
      const int64_t i = now.first + now.base + sub;
      const bool there = now.base + sub < end;
      const int64_t o = there ? i * W : 0;
      ring.fetch(row, stage == 0 ? Ring::S - 1 : stage - 1, ahead.first + ahead.base + sub,
               ahead.base + sub < ahead.end);
      ahead.step();
      ring.wait();
      float f[E], x[E], t[E], a[E];
      ring.take(row, stage, 0, i, there, f);
      ring.take(row, stage, 1, i, there, x);
      if (A.gate_mode == FX_GATE_FULL) {
        ring.take(row, stage, 4, i, there, g);
      } else if (A.gate_mode == FX_GATE_ROW) {
        const float g1 = there ? to_f(gate[i]) : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) g[e] = g1;
      }
      // f becomes nf, x becomes nr
      const float inv_f = row.normalise(f, there, LAYER, A.eps, sum);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = fmaf(g[e], fmaf(f[e], s1[e], b1[e]), x[e]);
      const float inv_r = row.normalise(x, there, LAYER, A.eps, sum);
      ring.take(row, stage, 2, i, there, a);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        aw[e] = fmaf(a[e], x[e], aw[e]);
        ab[e] += a[e];
        a[e] *= w2[e];
      }
      row.back(a, x, inv_r, LAYER, sum);
      ring.take(row, stage, 3, i, there, t);
      stage = ring.next(stage);
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] += a[e];  // 0 past the width and in rows that are not there
      row.store(static_cast<T*>(A.dx) + o, t, there);
      if (A.gate_mode == FX_GATE_FULL || A.gate_mode == FX_GATE_ROW) {
        float rowg = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          a[e] = t[e] * fmaf(f[e], s1[e], b1[e]);
          rowg += a[e];
        }
        if (A.gate_mode == FX_GATE_ROW) {
          rowg = sum.mean(rowg) * (float)W;
          if (there && row.t == 0) static_cast<T*>(A.dgate)[i] = from_f<T>(rowg);
        } else if (A.dgate_f32) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (there && row.in(e)) static_cast<float*>(A.dgate)[o + row.at(e / Row::C) + e % Row::C] = a[e];
        } else {
          row.store(static_cast<T*>(A.dgate) + o, a, there);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float tg = t[e] * g[e], sum_of = now.grouped ? t[e] : tg;
        P[e] = fmaf(sum_of, f[e], P[e]);
        Q[e] += sum_of;
        t[e] = tg * s1[e];
      }
      row.back(t, f, inv_f, LAYER, sum);
      row.store(static_cast<T*>(A.df) + o, t, there);
    }
    if (now.grouped) {
      // blocks and groups both ascend along the rows, so block + group names a segment
      float d[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        d[e] = fmaf(s1[e], P[e], b1[e] * Q[e]);
        P[e] = fmaf(g[e], P[e], Pg[e]);
        Q[e] = fmaf(g[e], Q[e], Qg[e]);
      }
      norm_block_sum(d, row, block_buf, A.gpart + ((int64_t)blockIdx.x + grp) * W);
    }
  }
  const int64_t stride = (int64_t)gridDim.x * W;
  float* out = A.part + (int64_t)blockIdx.x * W;
  norm_block_sum(P, row, block_buf, out);
  norm_block_sum(Q, row, block_buf, out + stride);
  norm_block_sum(aw, row, block_buf, out + 2 * stride);
  norm_block_sum(ab, row, block_buf, out + 3 * stride);
}

struct NormFinish {
  const float *part, *gpart;
  const void *pw, *pb, *scale;
  void *dpw, *dpb, *drw, *drb, *dscale;  // dpb, drb, dscale may be nullptr
  void* dgate;
  int64_t groups, R, per;
  int blocks, W, cols, dgate_f32;  // cols: ceil(W / 32)
};

// The blocks' partial sums into the channel gradients: blocks [0, cols) take 32 columns of P and
// Q (post_*, scale), [cols, 2 cols) of the pre_* sums; the 32 warps take the partial rows in
// turn and are added in warp order. Blocks past 2 cols: the gate's vectors, group by group over
// the blocks that held its rows.
template <typename T>
__global__ void __launch_bounds__(1024) norm_finish_kernel(const __grid_constant__ NormFinish F) {
  __shared__ float2 s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= 2 * F.cols) {
    const int64_t i = (int64_t)(blockIdx.x - 2 * F.cols) * 1024 + threadIdx.x;
    if (i >= F.groups * F.W) return;
    const int64_t g = i / F.W, c = i - g * F.W;
    const int64_t b0 = g * F.R / F.per, b1 = ((g + 1) * F.R - 1) / F.per;
    float v = 0.f;
    for (int64_t b = b0; b <= b1; ++b) v += F.gpart[(b + g) * F.W + c];
    if (F.dgate_f32) static_cast<float*>(F.dgate)[i] = v;
    else static_cast<T*>(F.dgate)[i] = from_f<T>(v);
    return;
  }
  const bool pre = blockIdx.x >= F.cols;
  const int c = (blockIdx.x - (pre ? F.cols : 0)) * 32 + lane;
  float2 v = make_float2(0.f, 0.f);
  if (c < F.W) {
    const int64_t plane = (int64_t)F.blocks * F.W;
    const float* src = F.part + (pre ? 2 * plane : 0) + c;
#pragma unroll 4
    for (int b = warp; b < F.blocks; b += 32) {
      v.x += src[(int64_t)b * F.W];
      v.y += src[plane + (int64_t)b * F.W];
    }
  }
  s[lane][warp] = v;
  __syncthreads();
  v = s[warp][lane];
  v.x = lanes_sum(v.x, 32);
  v.y = lanes_sum(v.y, 32);
  const int o = c - lane + warp;  // this warp's column
  if (lane != 0 || o >= F.W) return;
  if (pre) {
    static_cast<T*>(F.drw)[o] = from_f<T>(v.x);
    if (F.drb) static_cast<T*>(F.drb)[o] = from_f<T>(v.y);
  } else {
    const float sc = F.scale ? to_f(static_cast<const T*>(F.scale)[o]) : 1.f;
    const float pb = F.pb ? to_f(static_cast<const T*>(F.pb)[o]) : 0.f;
    static_cast<T*>(F.dpw)[o] = from_f<T>(sc * v.x);
    if (F.dpb) static_cast<T*>(F.dpb)[o] = from_f<T>(sc * v.y);
    if (F.dscale)
      static_cast<T*>(F.dscale)[o] = from_f<T>(fmaf(to_f(static_cast<const T*>(F.pw)[o]), v.x, pb * v.y));
  }
}

}  // namespace fx
