// Log probabilities of given tokens under softmax(scale logits), with entropy and the likeliest
// entries, and their gradient.
//
// One pass over a row keeps a reference m near its maximum, S = sum of exp(scale (x - m)) and
// W = sum of exp(scale (x - m)) log2(the same); then with L = log S
//   log p_t = scale (x_t - m) - L,   entropy = L - W / (S log2 e).
// A lane's reference moves when an entry is 2^kRise above it, not with every new maximum: in a row of 16 pieces a lane some
// lane of a warp has one at every piece.
// A lane takes a 16-byte piece at a time, on its boundary wherever the row begins, through a ring of asynchronous copies
// of its own, four pieces deep: bytes on the way cost no registers (with two pieces ahead in registers, which halved the
// threads, 8191 x 32000 bfloat16 took 197 us, with one and no ring 154, so 119). The likeliest entries are kept by each
// warp, one a lane in descending order: of the pieces at hand the largest entries are taken one by one (a warp-wide
// maximum each) while they pass the last of the list, which few do after the first; lists are joined by sorting networks.
// The forward is bound by its instructions, about 14 an entry (those rows, 524 MB, 119 us, 4.4 TB/s at 87% of the issue
// slots), the gradient by HBM (1.05 GB, 162 us, 6.5 TB/s). With a mask a row is loaded entry by entry, without the ring:
// those rows 264 us forward, 238 the gradient. A warp takes a row
// of up to 1024 entries, a block a longer one, or a part of it where the rows do not fill the device; parts are joined in
// order by a second kernel.
#pragma once
#include "token_common.cuh"

namespace fx {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kProbThreads = 128, kProbWarps = kProbThreads / 32;

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
  int entries, top, parts, per;  // per: 16-byte pieces of a part
  float scale;
  // backward
  const float *glogp, *gentropy;
  void* dlogits;
};

constexpr float kNone = -INFINITY;
constexpr float kRise = 8.f;
constexpr float kFar = -1e30f;  // in the place of log2(0), whose product with 0 it leaves 0

// c = scale log2 e.
struct Sums {
  float m = kNone, s = 0.f, w = 0.f;

  // Everything so far to the reference `to` >= m.
  __device__ __forceinline__ void move(float to, float c) {
    if (m != kNone) {
      const float t = fmaxf((m - to) * c, kFar), f = fast_exp2((m - to) * c);
      w = f * (w + t * s);
      s *= f;
    }
    m = to;
  }
  // The lanes' sums, in every lane.
  __device__ __forceinline__ void join_lanes(float c) {
    float to = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
    if (to != kNone) move(to, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      w += __shfl_xor_sync(0xffffffffu, w, o);
    }
  }
};

// Order of floats as unsigned numbers; NaN is not asked for.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Of a warp: entry `lane` of the list in descending order, ties to the lower index; index -1: none.
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
  // The 32 first of this list and another, whose entries come in ascending order: lane k has entry 31 - k. Of each pair the
  // better one is among them, and the result rises to its maximum and falls again: five steps sort it.
  __device__ __forceinline__ void merge(float x, int j) {
    if (!before(x, j)) {
      v = x;
      i = j;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, v, o);
      const int oi = __shfl_xor_sync(0xffffffffu, i, o);
      const bool low = (threadIdx.x & o) == 0;  // keeps the better one
      if (before(ov, oi) != low) {
        v = ov;
        i = oi;
      }
    }
  }
};

// N entries of each lane, entry e of index at(e), which rises with e and (for the same e) with the lane: those that belong in the first
// `top` of the list. `last` is entry top - 1.
template <int N, typename At>
__device__ __forceinline__ void take_best(Best& best, float& last, int top, float (&x)[N], At at) {
  for (;;) {
    float m = x[0];
    int e = 0;
#pragma unroll
    for (int k = 1; k < N; ++k)
      if (x[k] > m) {  // the first of equal ones
        m = x[k];
        e = k;
      }
    if (!(m > last)) m = kNone;  // NaN and what the list has no room for
    const unsigned own = ordered(m + 0.f), key = __reduce_max_sync(0xffffffffu, own);  // -0 + 0 is +0: the zeros are equal
    if (key == ordered(kNone)) return;
    const unsigned mine = own == key ? (unsigned)at(e) : 0xffffffffu, j = __reduce_min_sync(0xffffffffu, mine);
    const int src = __ffs(__ballot_sync(0xffffffffu, mine == j)) - 1;
    best.insert(__shfl_sync(0xffffffffu, m, src), (int)j);
    last = __shfl_sync(0xffffffffu, best.v, top - 1);
    if ((threadIdx.x & 31) == src) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k == e) x[k] = kNone;
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
    A.entropy[r] = none ? 0.f : fmaxf(L - 0.6931471805599453f * (S.w / S.s), 0.f) + 0.f * S.s;
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

// The sums and lists of a block's warps, in warp 0. Called by the whole block.
template <bool TOP>
__device__ __forceinline__ void prob_join_warps(Sums& S, Best& best, float c) {
  __shared__ float4 sums[kProbWarps];
  __shared__ int2 lists[kProbWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (lane == 0) sums[w] = make_float4(S.m, S.s, S.w, 0.f);
  if (TOP) lists[w][lane] = make_int2(__float_as_int(best.v), best.i);
  __syncthreads();
  if (w) return;
  const float4 q = lane < kProbWarps ? sums[lane] : make_float4(kNone, 0.f, 0.f, 0.f);
  S.m = q.x;
  S.s = q.y;
  S.w = q.z;
  S.join_lanes(c);
  if (TOP)
    for (int k = 1; k < kProbWarps; ++k) {
      const int2 e = lists[k][31 - lane];
      best.merge(__int_as_float(e.x), e.y);
    }
}

// A row as pieces of E entries on 16-byte boundaries; piece 0 may begin before the row, the last end behind it.
template <typename T>
struct PieceRow {
  static constexpr int E = 16 / sizeof(T);
  const T* base;  // of piece 0
  int off, entries;  // entries of piece 0 before the row
  int whole, end;    // pieces [whole, end) lie in the row

  __device__ __forceinline__ PieceRow(const T* x, int V) {
    off = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    base = x - off;
    entries = V;
    whole = off > 0;
    end = (int)(((int64_t)V + off) / E);
  }
  __device__ __forceinline__ int pieces() const { return end + (((int64_t)entries + off) % E != 0); }
  __device__ __forceinline__ int first(int k) const { return k * E - off; }  // entry of the row
  __device__ __forceinline__ bool has(int e) const { return e >= 0 && e < entries; }

  // Piece k to a slot of this thread's; entries outside the row -inf.
  __device__ __forceinline__ void bring(Pack<T, E>* slot, int k) const {
    if (k >= whole && k < end) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(slot)),
                   "l"(base + (int64_t)k * E)
                   : "memory");
    } else {
      Pack<T, E> p;
#pragma unroll
      for (int e = 0; e < E; ++e) p.e[e] = has(first(k) + e) ? base[(int64_t)k * E + e] : from_f<T>(kNone);
      *slot = p;
    }
  }
  // Bit e: entry e of piece k is in the row and its byte of the mask is not 0.
  __device__ __forceinline__ unsigned kept(const uint8_t* mask, bool aligned, int k) const {
    unsigned keep = 0;
    const int e0 = first(k);
    if (aligned && k >= whole && k < end) {
      const Pack<uint8_t, E> b = *reinterpret_cast<const Pack<uint8_t, E>*>(mask + e0);
#pragma unroll
      for (int e = 0; e < E; ++e) keep |= (b.e[e] ? 1u : 0u) << e;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (has(e0 + e) && mask[e0 + e]) keep |= 1u << e;
    }
    return keep;
  }
};

constexpr int kRing = 4;
template <int N>
__device__ __forceinline__ void ring_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// A row (or one of its parts) by WARPS warps.
template <typename T, bool TOP, int WARPS>
__global__ void __launch_bounds__(kProbThreads, TOP ? 8 : 12) prob_kernel(ProbArgs A) {
  using Row = PieceRow<T>;
  constexpr int E = Row::E, STEP = WARPS * 32;
  __shared__ Pack<T, E> ring[kRing][kProbThreads];
  const int lane = threadIdx.x & 31;
  const int64_t r = WARPS == 1 ? (int64_t)blockIdx.x * kProbWarps + (threadIdx.x >> 5) : blockIdx.x / A.parts;
  const int part = WARPS == 1 ? 0 : (int)(blockIdx.x % A.parts), t = WARPS == 1 ? lane : threadIdx.x;
  if (r >= A.rows) return;
  if (A.tok.has_padding && A.tok.padded(A.tok.at(r))) {
    if (part == 0) {
      if (t == 0) {
        A.logp[r] = A.entropy[r] = 0.f;
        if (A.stats) {
          A.stats[r] = 0.f;
          A.stats[A.rows + r] = INFINITY;
        }
      }
      if (TOP && t < A.top) {
        A.top_logp[r * A.top + t] = kNone;
        A.top_index[r * A.top + t] = -1;
      }
    }
    return;
  }
  const Row row(static_cast<const T*>(A.logits) + r * A.ls, A.entries);
  const uint8_t* mask = A.mask ? A.mask + r * A.ms : nullptr;
  const bool mask_aligned = (reinterpret_cast<uintptr_t>(mask) - row.off) % E == 0;
  const float c = A.scale * kLog2e, rise = fminf(kRise / c, 3e38f);
  const int begin = part * A.per, end = min(begin + A.per, row.pieces());
  Sums S;
  float s2[2] = {}, w2[2] = {};  // two sums each
  Best best;
  float last = kNone;  // of the list
  float m = 0.f;  // the reference, 0 before the first entry
  // The entries of piece k (its first is the row's entry `from`), -inf where there are none; by whole warps. (Two entries an
  // instruction, f32x2, took twice the instructions: the pairs have to be moved together.)
  const auto take = [&](float (&v)[E], float top, int from) {
    if (top > S.m + rise) {
      S.s = s2[0] + s2[1];
      S.w = w2[0] + w2[1];
      S.move(top, c);
      s2[0] = S.s;
      w2[0] = S.w;
      s2[1] = w2[1] = 0.f;
      m = top;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float a = (v[e] - m) * c, p = fast_exp2(a);
      s2[e & 1] += p;
      w2[e & 1] = fmaf(p, fmaxf(a, kFar), w2[e & 1]);
    }
    if constexpr (TOP) {
      if (__any_sync(0xffffffffu, top > last)) take_best(best, last, A.top, v, [&](int e) { return from + e; });
    }
  };
  const auto greatest = [](const float (&v)[E]) {
    float top = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, v[e]);
    return top;
  };
  // piece k by lane 0, the others without entries; where it is not whole, or masked
  const auto take_checked = [&](int k, bool has) {
    float v[E];
    const unsigned keep = !has ? 0u : mask ? row.kept(mask, mask_aligned, k) : 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; ++e)
      v[e] = (keep >> e & 1u) && row.has(row.first(k) + e) ? to_f(row.base[(int64_t)k * E + e]) : kNone;
    take(v, greatest(v), row.first(k));
  };
  if (mask) {
#pragma unroll 1
    for (int i = begin; i < end; i += STEP) take_checked(i + t, i + t < end);
  } else {
    // pieces [b0, e0) are whole, a round of them every lane's but for the last; the one before and the one behind are the
    // row's ends
    const int b0 = max(begin, row.whole), e0 = min(end, row.end), rounds = max(e0 - b0, 0) / STEP;
    const bool more = b0 + rounds * STEP + t < e0;
    const T* from = row.base + (int64_t)(b0 + t) * E;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&ring[0][threadIdx.x]);
    const auto fetch = [&](int slot, int j) {
      if (j < rounds || (j == rounds && more))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + slot * (kProbThreads * 16)),
                     "l"(from + (int64_t)j * (STEP * E))
                     : "memory");
      ring_commit();
    };
    const auto piece = [&](float (&v)[E], int slot) {  // its greatest
      const Pack<T, E> p = ring[slot][threadIdx.x];
      unpack<E>(p, v);
      if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162* q = reinterpret_cast<const __nv_bfloat162*>(&p);
        const float2 m = __bfloat1622float2(__hmax2(__hmax2(q[0], q[1]), __hmax2(q[2], q[3])));
        return fmaxf(m.x, m.y);
      } else {
        return greatest(v);
      }
    };
#pragma unroll
    for (int d = 0; d < kRing; ++d) fetch(d, d);
    if (begin < b0) take_checked(begin, t == 0);
    int slot = 0;
#pragma unroll 1
    for (int j = 0; j < rounds; ++j) {
      float v[E];
      ring_wait<kRing - 1>();
      const float top = piece(v, slot);
      fetch(slot, j + kRing);
      slot = (slot + 1) % kRing;
      take(v, top, row.first(b0 + t + j * STEP));
    }
    if (b0 + rounds * STEP < e0) {
      float v[E], top = kNone;
      ring_wait<0>();
      if (more) {
        top = piece(v, slot);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = kNone;
      }
      take(v, top, row.first(b0 + t + rounds * STEP));
    }
    if (e0 < end && e0 >= b0) take_checked(e0, t == 0);  // not the piece before, where that is the only one
  }
  S.s = s2[0] + s2[1];
  S.w = w2[0] + w2[1];
  S.join_lanes(c);
  if constexpr (WARPS > 1) {
    prob_join_warps<TOP>(S, best, c);
    if (threadIdx.x >= 32) return;
  }
  if (WARPS == 1 || A.parts == 1) {
    prob_finish<T>(A, r, S, best);
  } else {
    if (lane == 0) A.part[blockIdx.x] = make_float4(S.m, S.s, S.w, 0.f);
    if (TOP && lane < A.top) A.part_top[(int64_t)blockIdx.x * A.top + lane] = make_int2(__float_as_int(best.v), best.i);
  }
}

// A block a row: its parts in order by stretches of them a warp.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kProbThreads) prob_join_kernel(ProbArgs A) {
  wait_for_last();
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (A.tok.padded(A.tok.at(r))) return;
  const float c = A.scale * kLog2e;
  const int per = (A.parts + kProbWarps - 1) / kProbWarps, first = w * per, end = min(first + per, A.parts);
  Sums S;
  for (int p = first + lane; p - lane < end; p += 32) {  // what is there so far counts as lane 0's
    const float4 q = p < end ? A.part[r * A.parts + p] : make_float4(kNone, 0.f, 0.f, 0.f);
    Sums one;
    one.m = q.x;
    one.s = q.y;
    one.w = q.z;
    one.join_lanes(c);
    Sums both = lane ? one : S;
    if (lane > 1) both = Sums{};
    both.join_lanes(c);
    S = both;
  }
  Best best;
  if constexpr (TOP) {
    const int2* p = A.part_top + r * A.parts * A.top;
    constexpr int kAhead = 4;
    for (int l = first; l < end; l += kAhead) {
      int2 q[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        q[u] = l + u < end && 31 - lane < A.top ? p[(l + u) * A.top + 31 - lane] : make_int2(__float_as_int(kNone), -1);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (l + u < end) best.merge(__int_as_float(q[u].x), q[u].y);
    }
  }
  prob_join_warps<TOP>(S, best, c);
  if (w == 0) prob_finish<T>(A, r, S, best);
}

// ---------------------------------------------------------------- gradient
// d = scale (g (hit - p) - e p (log p + H)), entry by entry: HBM.
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> prob_round(const float (&d)[E]) {
  Pack<T, E> o;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < E; ++e) o.e[e] = d[e];
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<__nv_bfloat162*>(&o.e[e]) = __floats2bfloat162_rn(d[e], d[e + 1]);
  }
  return o;
}

template <typename T, int WARPS>
__global__ void __launch_bounds__(kProbThreads, 12) prob_grad_kernel(ProbArgs A) {
  using Row = PieceRow<T>;
  constexpr int E = Row::E, STEP = WARPS * 32;
  __shared__ Pack<T, E> ring[kRing][kProbThreads];
  const int64_t r = WARPS == 1 ? (int64_t)blockIdx.x * kProbWarps + (threadIdx.x >> 5) : blockIdx.x / A.parts;
  const int part = WARPS == 1 ? 0 : (int)(blockIdx.x % A.parts), lane = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x;
  if (r >= A.rows) return;
  const Row row(static_cast<const T*>(A.logits) + r * A.ls, A.entries);
  const uint8_t* mask = A.mask ? A.mask + r * A.ms : nullptr;
  const bool mask_aligned = (reinterpret_cast<uintptr_t>(mask) - row.off) % E == 0;
  T* out = static_cast<T*>(A.dlogits) + r * A.entries - row.off;  // of piece 0
  const bool out_aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const int begin = part * A.per + lane, end = min(part * A.per + A.per, row.pieces());
  const auto store = [&](int k, const Pack<T, E>& o) {
    if (out_aligned && k >= row.whole && k < row.end) {
      *reinterpret_cast<Pack<T, E>*>(out + (int64_t)k * E) = o;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (row.has(row.first(k) + e)) out[(int64_t)k * E + e] = o.e[e];
    }
  };
  const int64_t t = A.tok.at(r);
  if (A.tok.padded(t)) {
    const float zero[E] = {};
    for (int k = begin; k < end; k += STEP) store(k, prob_round<T, E>(zero));
    return;
  }
#pragma unroll
  for (int d = 0; d < kRing; ++d) {
    if (begin + d * STEP < end) row.bring(&ring[d][threadIdx.x], begin + d * STEP);
    ring_commit();
  }
  const bool given = t >= 0 && t < A.entries;
  const float g = A.glogp && given ? A.glogp[r] : 0.f, ent = A.gentropy ? A.gentropy[r] : 0.f;
  const float m = A.stats[r], l2 = A.stats[A.rows + r], c = A.scale * kLog2e;
  // - scale p (g + e (log p + H)), log p = ln2 q; a row without an entry of any probability has no hit either
  const float gs = -A.scale * (g + ent * A.entropy[r]), es = -A.scale * ent * 0.6931471805599453f;
  const float hit = l2 == INFINITY ? 0.f : A.scale * g;
  const int at = given ? (int)t : -E;  // the token's entry
  int slot = 0;
#pragma unroll 1
  for (int k = begin; k < end; k += STEP) {
    ring_wait<kRing - 1>();
    const Pack<T, E> v = ring[slot][threadIdx.x];
    if (k + kRing * STEP < end) row.bring(&ring[slot][threadIdx.x], k + kRing * STEP);
    ring_commit();
    slot = slot + 1 == kRing ? 0 : slot + 1;
    float d[E];
    unpack<E>(v, d);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float q = fmaf(d[e] - m, c, -l2);
      // an entry without probability has log2 p = -inf: 0 all the same
      d[e] = fast_exp2(q) * fmaf(es, fmaxf(q, -300.f), gs);
    }
    const unsigned here = (unsigned)(at - row.first(k));
    if (here < (unsigned)E) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((unsigned)e == here) d[e] += hit;
    }
    if (mask) {
      const unsigned keep = row.kept(mask, mask_aligned, k);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(keep >> e & 1u)) d[e] = 0.f;
    }
    store(k, prob_round<T, E>(d));
  }
}

}  // namespace fx
