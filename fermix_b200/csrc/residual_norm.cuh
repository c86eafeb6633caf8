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
// dpost_w = sum du nf, dpost_b = sum du, dpre_w = sum dz nr, dpre_b = sum dz over the rows.
//
// Bound: HBM. A row is read once and held in registers by a group of TPR threads (a part of a
// warp for narrow rows, a block for wide ones), E entries a thread, so that the statistics
// are two-pass (mean, then centred squares) without reading again. The backward recomputes
// nf, r and nr from x, f and gate -- the same bytes that the saved statistics and r would
// be, and r unrounded -- and keeps the sums over rows in registers while a block walks its
// rows; each block writes one partial row per parameter and norm_finish_kernel adds those in
// block order.
#pragma once
#include "block_common.cuh"

namespace fx {

struct NormArgs {
  const void *x, *f, *gate, *scale, *pw, *pb, *rw, *rb;  // p: post (of f), r: pre (of r)
  void *r, *z;
  const void *gr, *gz;
  void *dx, *df, *dgate;
  float* part;   // (5, grid, W): dpost_w, dpost_b, dpre_w, dpre_b, dscale
  float* gpart;  // (grid + groups, W): slot block + group, gate_mode 3
  int64_t N, R;  // all rows, rows of a group
  int64_t per;   // rows of a block
  float eps;
  int W, layer, gate_mode, dgate_f32, tpr;
};

constexpr int kNormThreads = 256;  // block of the sub-warp groups; wider rows: one row a block
constexpr int kNormParams = 5;

// Sums over the TPR threads of a row. Blocks that hold one row go through shared memory,
// alternating between two buffers so that one barrier a sum is enough.
struct RowSum {
  float* red;  // 2 x 64
  int tpr, flip;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    if (tpr <= 32) return make_float2(lanes_sum(a, tpr), lanes_sum(b, tpr));
    a = lanes_sum(a, 32);
    b = lanes_sum(b, 32);
    float* buf = red + flip * 64;
    flip ^= 1;
    const int w = threadIdx.x >> 5, nw = tpr >> 5;
    if ((threadIdx.x & 31) == 0) {
      buf[w] = a;
      buf[32 + w] = b;
    }
    __syncthreads();
    a = b = 0.f;
    for (int i = 0; i < nw; ++i) {
      a += buf[i];
      b += buf[32 + i];
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float operator()(float a) {
    return tpr <= 32 ? lanes_sum(a, tpr) : (*this)(a, 0.f).x;
  }
};

// A thread's part of a row: NV chunks of 16 bytes, neighbouring threads next to each other.
// The mapping does not depend on alignment, so the sums (and the results' bits) do not
// either. ALIGNED: every row and parameter starts on a 16-byte boundary and the width is whole
// chunks. Otherwise a chunk is cut out of the two aligned 16-byte pieces around it, and stored
// as aligned pieces joined with the neighbour's entries.
template <typename T, int NV, bool ALIGNED>
struct NormRow {
  static constexpr int C = 16 / sizeof(T), E = C * NV;
  int t, tpr, W;
  __device__ __forceinline__ int at(int v) const { return (v * tpr + t) * C; }
  __device__ __forceinline__ bool in(int e) const { return at(e / C) + e % C < W; }
  // entries [c, c + C) of the row at p, a part of the array [begin, end)
  __device__ __forceinline__ Pack<T, C> piece(const T* p, int c, const T* begin, const T* end) const {
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p + c) & 15);  // bytes past a boundary
    const T* a = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(p + c) - off);
    const int got = C - (int)(off / sizeof(T));  // entries in the first piece
    const bool two = got < C && c + got < W;
    if (a >= begin && a + (two ? 2 * C : C) <= end) {
      const uint4 u = *reinterpret_cast<const uint4*>(a);
      const uint4 x = two ? *reinterpret_cast<const uint4*>(a + C) : make_uint4(0u, 0u, 0u, 0u);
      const bool w2 = off & 8, w1 = off & 4;
      const uint32_t a0 = w2 ? u.z : u.x, a1 = w2 ? u.w : u.y, a2 = w2 ? x.x : u.z, a3 = w2 ? x.y : u.w,
                     a4 = w2 ? x.z : x.x, a5 = w2 ? x.w : x.y;
      const uint32_t b0 = w1 ? a1 : a0, b1 = w1 ? a2 : a1, b2 = w1 ? a3 : a2, b3 = w1 ? a4 : a3, b4 = w1 ? a5 : a4;
      const uint32_t sh = (off & 2) * 8;
      const uint4 r = make_uint4(__funnelshift_r(b0, b1, sh), __funnelshift_r(b1, b2, sh),
                                 __funnelshift_r(b2, b3, sh), __funnelshift_r(b3, b4, sh));
      return *reinterpret_cast<const Pack<T, C>*>(&r);
    }
    Pack<T, C> k;  // the array's own ends
#pragma unroll
    for (int e = 0; e < C; ++e) k.e[e] = c + e < W ? p[c + e] : from_f<T>(0.f);
    return k;
  }
  // entries of the row at p (nullptr, a row that is not there or past the width: fill)
  __device__ __forceinline__ void load(const T* p, float (&o)[E], float fill, bool there, const T* begin,
                                       const T* end) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (p != nullptr && there && at(v) < W) {
        Pack<T, C> k;
        if constexpr (ALIGNED) k = *reinterpret_cast<const Pack<T, C>*>(p + at(v));
        else k = piece(p, at(v), begin, end);
#pragma unroll
        for (int e = 0; e < C; ++e) o[v * C + e] = in(v * C + e) ? to_f(k.e[e]) : fill;
      } else {
#pragma unroll
        for (int e = 0; e < C; ++e) o[v * C + e] = fill;
      }
    }
  }
  // a parameter of W entries
  __device__ __forceinline__ void load(const T* p, float (&o)[E], float fill) const { load(p, o, fill, true, p, p + W); }
  // Every lane of the warp calls this; a row that is not there is not written.
  __device__ __forceinline__ void store(T* p, const float (&o)[E], bool there) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = at(v);
      Pack<T, C> k;
#pragma unroll
      for (int e = 0; e < C; ++e) k.e[e] = from_f<T>(o[v * C + e]);
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
  // v <- normalised v (entries outside the row are 0), returns 1 / rms
  __device__ __forceinline__ float normalise(float (&v)[E], bool layer, float eps, RowSum& sum) const {
    if (layer) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += v[e];
      const float mean = sum(s) / (float)W;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (in(e)) v[e] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) q = fmaf(v[e], v[e], q);
    const float inv = rsqrtf(sum(q) / (float)W + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= inv;
    return inv;
  }
  // a <- the gradient through normalise(): inv (a - mean(a) [layer] - n mean(a n))
  __device__ __forceinline__ void back(float (&a)[E], const float (&n)[E], float inv, bool layer, RowSum& sum) const {
    float s = 0.f, d = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s += a[e];
      d = fmaf(a[e], n[e], d);
    }
    float2 m;
    if (layer) m = sum(s, d);
    else m = make_float2(0.f, sum(d));
    const float ms = m.x / (float)W, md = m.y / (float)W;
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = inv * (a[e] - ms - n[e] * md);
  }
};

template <typename T, int NV, bool ALIGNED>
__global__ void __launch_bounds__(512) norm_fwd_kernel(NormArgs A) {
  using Row = NormRow<T, NV, ALIGNED>;
  constexpr int E = Row::E;
  __shared__ float red[128];
  const int tpr = A.tpr, W = A.W, rpb = tpr > 32 ? 1 : blockDim.x / tpr;
  const int sub = tpr > 32 ? 0 : threadIdx.x / tpr;
  const Row row{(int)threadIdx.x - sub * tpr, tpr, W};
  RowSum sum{red, tpr, 0};
  const int64_t all = A.N * W;
  for (int64_t base = (int64_t)blockIdx.x * rpb; base < A.N; base += (int64_t)gridDim.x * rpb) {
    const int64_t i = base + sub;
    const bool there = i < A.N;
    const int64_t o = there ? i * W : 0;
    auto load = [&](const void* p, float(&v)[E]) {
      const T* q = static_cast<const T*>(p);
      row.load(q ? q + o : nullptr, v, 0.f, there, q, q + all);
    };
    float f[E], x[E], g[E], w[E];
    load(A.f, f);
    load(A.x, x);
    const T* gate = static_cast<const T*>(A.gate);
    if (A.gate_mode == FX_GATE_FULL) {
      load(A.gate, g);
    } else if (A.gate_mode == FX_GATE_GROUP) {
      row.load(gate + (there ? i / A.R : 0) * W, g, 0.f);
    } else {
      const float g1 = A.gate_mode == FX_GATE_ROW && there ? to_f(gate[i]) : 1.f;
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = g1;
    }
    row.normalise(f, A.layer, A.eps, sum);
    row.load(static_cast<const T*>(A.pw), w, 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= w[e];
    if (A.pb != nullptr) {
      row.load(static_cast<const T*>(A.pb), w, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] += w[e];
    }
    if (A.scale != nullptr) {
      row.load(static_cast<const T*>(A.scale), w, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (row.in(e)) x[e] = fmaf(g[e], f[e], x[e]);
    row.store(static_cast<T*>(A.r) + o, x, there);
    row.normalise(x, A.layer, A.eps, sum);
    row.load(static_cast<const T*>(A.rw), w, 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] *= w[e];
    if (A.rb != nullptr) {
      row.load(static_cast<const T*>(A.rb), w, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += w[e];
    }
    row.store(static_cast<T*>(A.z) + o, x, there);
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

template <typename T, int NV, bool ALIGNED>
__global__ void __launch_bounds__(512) norm_bwd_kernel(NormArgs A) {
  using Row = NormRow<T, NV, ALIGNED>;
  constexpr int E = Row::E;
  extern __shared__ float buf[];
  __shared__ float red[128];
  const int tpr = A.tpr, W = A.W, rpb = tpr > 32 ? 1 : blockDim.x / tpr;
  const int sub = tpr > 32 ? 0 : threadIdx.x / tpr;
  const Row row{(int)threadIdx.x - sub * tpr, tpr, W};
  RowSum sum{red, tpr, 0};
  const int64_t all = A.N * W;
  float apw[E], apb[E], arw[E], arb[E], asc[E], agt[E];
#pragma unroll
  for (int e = 0; e < E; ++e) apw[e] = apb[e] = arw[e] = arb[e] = asc[e] = agt[e] = 0.f;
  const int64_t first = (int64_t)blockIdx.x * A.per;
  const int64_t last = first + A.per < A.N ? first + A.per : A.N;
  // one segment a group of the gate (gate_mode 3), else one segment
  for (int64_t seg = first; seg < last;) {
    const int64_t grp = A.gate_mode == FX_GATE_GROUP ? seg / A.R : 0;
    int64_t end = last;
    if (A.gate_mode == FX_GATE_GROUP && (grp + 1) * A.R < end) end = (grp + 1) * A.R;
    for (int64_t base = seg; base < end; base += rpb) {
      const int64_t i = base + sub;
      const bool there = i < end;
      const int64_t o = there ? i * W : 0;
      auto load = [&](const void* p, float(&v)[E]) {
        const T* q = static_cast<const T*>(p);
        row.load(q ? q + o : nullptr, v, 0.f, there, q, q + all);
      };
      float f[E], x[E], g[E], t[E], dz[E], w[E];
      load(A.f, f);
      load(A.x, x);
      load(A.gz, dz);
      load(A.gr, t);
      const T* gate = static_cast<const T*>(A.gate);
      if (A.gate_mode == FX_GATE_FULL) {
        load(A.gate, g);
      } else if (A.gate_mode == FX_GATE_GROUP) {
        row.load(gate + grp * W, g, 0.f);
      } else {
        const float g1 = A.gate_mode == FX_GATE_ROW && there ? to_f(gate[i]) : 1.f;
#pragma unroll
        for (int e = 0; e < E; ++e) g[e] = g1;
      }
      float sc[E], u[E];
      row.load(static_cast<const T*>(A.scale), sc, 1.f);
      // f becomes nf, x becomes nr
      const float inv_f = row.normalise(f, A.layer, A.eps, sum);
      row.load(static_cast<const T*>(A.pw), w, 0.f);
      if (A.pb != nullptr) {
        row.load(static_cast<const T*>(A.pb), u, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = fmaf(f[e], w[e], u[e]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = f[e] * w[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (row.in(e)) x[e] = fmaf(g[e] * sc[e], u[e], x[e]);
      const float inv_r = row.normalise(x, A.layer, A.eps, sum);
      float a[E];
      row.load(static_cast<const T*>(A.rw), a, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        a[e] *= dz[e];
        arw[e] = fmaf(dz[e], x[e], arw[e]);
        arb[e] += dz[e];
      }
      row.back(a, x, inv_r, A.layer, sum);
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = row.in(e) && there ? t[e] + a[e] : 0.f;
      row.store(static_cast<T*>(A.dx) + o, t, there);
      float rowg = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float tu = t[e] * u[e];
        asc[e] = fmaf(tu, g[e], asc[e]);
        a[e] = tu * sc[e];  // the gate's gradient
        rowg += a[e];
        agt[e] += a[e];
        t[e] *= sc[e] * g[e];  // du
        apw[e] = fmaf(t[e], f[e], apw[e]);
        apb[e] += t[e];
        t[e] *= w[e];
      }
      if (A.gate_mode == FX_GATE_FULL) {
        if (A.dgate_f32) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (there && row.in(e)) static_cast<float*>(A.dgate)[o + row.at(e / Row::C) + e % Row::C] = a[e];
        } else {
          row.store(static_cast<T*>(A.dgate) + o, a, there);
        }
      }
      if (A.gate_mode == FX_GATE_ROW) {
        rowg = sum(rowg);
        if (there && row.t == 0) static_cast<T*>(A.dgate)[i] = from_f<T>(rowg);
      }
      row.back(t, f, inv_f, A.layer, sum);
      row.store(static_cast<T*>(A.df) + o, t, there);
    }
    if (A.gate_mode == FX_GATE_GROUP) {
      // blocks and groups both ascend along the rows, so block + group names a segment
      norm_block_sum(agt, row, buf, A.gpart + ((int64_t)blockIdx.x + grp) * W);
#pragma unroll
      for (int e = 0; e < E; ++e) agt[e] = 0.f;
    }
    seg = end;
  }
  const int64_t stride = (int64_t)gridDim.x * W;
  float* out = A.part + (int64_t)blockIdx.x * W;
  norm_block_sum(apw, row, buf, out);
  if (A.pb != nullptr) norm_block_sum(apb, row, buf, out + stride);
  norm_block_sum(arw, row, buf, out + 2 * stride);
  if (A.rb != nullptr) norm_block_sum(arb, row, buf, out + 3 * stride);
  if (A.scale != nullptr) norm_block_sum(asc, row, buf, out + 4 * stride);
}

struct NormFinish {
  const float *part, *gpart;
  void* out[kNormParams];  // nullptr: not wanted
  void* dgate;
  int64_t groups, R, per;
  int blocks, W, cols, dgate_f32;  // cols: ceil(W / 32)
};

// dst[i] = the sum of the blocks' partial rows: 32 columns a block, the 8 warps take the
// partial rows in turn and are added in warp order. Blocks past 5 cols: the gate's vectors,
// group by group over the blocks that held its rows.
template <typename T>
__global__ void __launch_bounds__(256) norm_finish_kernel(NormFinish F) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= kNormParams * F.cols) {
    const int64_t i = (int64_t)(blockIdx.x - kNormParams * F.cols) * 256 + threadIdx.x;
    if (i >= F.groups * F.W) return;
    const int64_t g = i / F.W, c = i - g * F.W;
    const int64_t b0 = g * F.R / F.per, b1 = ((g + 1) * F.R - 1) / F.per;
    float v = 0.f;
    for (int64_t b = b0; b <= b1; ++b) v += F.gpart[(b + g) * F.W + c];
    if (F.dgate_f32) static_cast<float*>(F.dgate)[i] = v;
    else static_cast<T*>(F.dgate)[i] = from_f<T>(v);
    return;
  }
  const int p = blockIdx.x / F.cols, c = (blockIdx.x - p * F.cols) * 32 + lane;
  T* out = static_cast<T*>(F.out[p]);
  if (out == nullptr) return;
  float v = 0.f;
  if (c < F.W) {
    const float* src = F.part + (int64_t)p * F.blocks * F.W + c;
#pragma unroll 8
    for (int b = warp; b < F.blocks; b += 8) v += src[(int64_t)b * F.W];
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < F.W) {
    for (int w = 1; w < 8; ++w) v += s[w][lane];
    out[c] = from_f<T>(v);
  }
}

}  // namespace fx
