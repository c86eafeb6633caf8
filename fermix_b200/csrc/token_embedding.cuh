// Embedding of tokens: out[i] = scale weight[token[i]], and its gradient
// dweight[v] = scale * sum of grad[i] over the i with token[i] = v.
//
// The forward is a gather, bound by HBM: each thread has four rows' 16-byte pieces on the way.
//
// The gradient adds in a fixed order, so the tokens are sorted first (stable, by digits of up
// to 11 bits: counts per block, their sums over the blocks, then every block places its
// tokens), which costs 12 bytes a token and pass beside the rows' `width` entries. The
// sorted list is cut into windows of equal length, one group of threads each, whatever
// the tokens' frequencies: a run of one token within a window is final, one that crosses
// into another window leaves a float32 partial sum there, and a last kernel adds those in
// order and fills the rows that no token names.
#pragma once
#include "token_common.cuh"

namespace fx {

constexpr int kEmbedThreads = 256;

template <typename T, int E>
struct EmbedVec {
  using P = Pack<T, E>;
};

struct EmbedFwd {
  Tokens tok;
  const void* weight;
  void* out;
  int64_t count, rows, width;
  int chunks, tpr;  // pieces of a row; threads of a row (a power of two)
  float scale;
};

constexpr int kEmbedRows = 4;  // rows a thread has on the way

// A persistent grid: the next rows' tokens are read before this round's rows are.
template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads) embed_fwd_kernel(EmbedFwd A) {
  using P = Pack<T, E>;
  const int rpb = kEmbedThreads / A.tpr, lane = threadIdx.x & (A.tpr - 1);
  const int64_t step = (int64_t)gridDim.x * rpb * kEmbedRows;
  int64_t r0 = (int64_t)blockIdx.x * (rpb * kEmbedRows) + threadIdx.x / A.tpr;
  int64_t next[kEmbedRows];
#pragma unroll
  for (int u = 0; u < kEmbedRows; ++u) next[u] = r0 + u * rpb < A.count ? A.tok.at(r0 + u * rpb) : 0;
  for (; r0 < A.count; r0 += step) {
    const P* src[kEmbedRows];
    float other[kEmbedRows];  // what a row without a source holds
#pragma unroll
    for (int u = 0; u < kEmbedRows; ++u) {
      const int64_t t = next[u], r = r0 + step + u * rpb;
      const bool ok = t >= 0 && t < A.rows && !A.tok.padded(t);
      src[u] = ok ? reinterpret_cast<const P*>(static_cast<const T*>(A.weight) + t * A.width) : nullptr;
      other[u] = A.tok.padded(t) ? 0.f : __int_as_float(0x7fc00000);
      next[u] = r < A.count ? A.tok.at(r) : 0;
    }
    for (int c = lane; c < A.chunks; c += A.tpr) {
      P v[kEmbedRows];
#pragma unroll
      for (int u = 0; u < kEmbedRows; ++u)
        if (src[u]) v[u] = src[u][c];
#pragma unroll
      for (int u = 0; u < kEmbedRows; ++u) {
        const int64_t r = r0 + u * rpb;
        if (r >= A.count) break;
        P o;
#pragma unroll
        for (int e = 0; e < E; ++e) o.e[e] = from_f<T>(src[u] ? to_f(v[u].e[e]) * A.scale : other[u]);
        reinterpret_cast<P*>(static_cast<T*>(A.out) + r * A.width)[c] = o;
      }
    }
  }
}

// ---------------------------------------------------------------- sort by token
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kSortRounds = 4;
constexpr int kSortTile = kSortThreads * kSortRounds;  // tokens of a block
constexpr int kSortBits = 11;

struct SortArgs {
  Tokens tok;           // first pass
  const int *keys, *pos;  // later passes
  int *keys_out, *pos_out;
  int* hist;    // (digits, blocks)
  int* total;   // (digits)
  int* start;   // one pass only: first place of each token, (rows + 1)
  int64_t rows;
  int count, blocks, shift, bits;
};

// Token (or key) e = warp's first + 32 round + lane, and its digit; -1 behind the last.
__device__ __forceinline__ void sort_load(const SortArgs& A, int (&key)[kSortRounds], int base) {
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int e = base + 32 * i;
    key[i] = e >= A.count ? -1 : A.keys ? A.keys[e] : A.tok.key(e, A.rows);
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs A) {
  extern __shared__ int hist[];
  const int digits = 1 << A.bits, lane = threadIdx.x & 31;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  int key[kSortRounds];
  sort_load(A, key, blockIdx.x * kSortTile + (threadIdx.x >> 5) * (32 * kSortRounds) + lane);
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int d = key[i] < 0 ? -1 : (key[i] >> A.shift) & (digits - 1);
    const unsigned same = __match_any_sync(0xffffffffu, d);  // one addition for equal digits
    if (d >= 0 && lane == __ffs(same) - 1) atomicAdd(&hist[d], __popc(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) A.hist[(int64_t)d * A.blocks + blockIdx.x] = hist[d];
}

// Counts of a digit -> first place within the digit for each block; a warp a digit.
__global__ void __launch_bounds__(256) sort_scan_kernel(SortArgs A) {
  const int d = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (d >= 1 << A.bits) return;
  int* h = A.hist + (int64_t)d * A.blocks;
  int sum = 0;
  for (int b = 0; b < A.blocks; b += 32) {
    const int n = b + lane < A.blocks ? h[b + lane] : 0;
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (b + lane < A.blocks) h[b + lane] = sum + s - n;
    sum += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) A.total[d] = sum;
}

__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortArgs A) {
  extern __shared__ int at[];  // (warps, digits), then the digits' first places
  __shared__ int sums[kSortWarps];
  const int digits = 1 << A.bits, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int* first = at + kSortWarps * digits;
  for (int i = threadIdx.x; i < kSortWarps * digits; i += kSortThreads) at[i] = 0;
  // first places of the digits: a thread sums a run of them
  const int per = (digits + kSortThreads - 1) / kSortThreads, d0 = threadIdx.x * per;
  int own = 0;
  for (int d = d0; d < d0 + per && d < digits; ++d) own += A.total[d];
  int s = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) sums[w] = s;
  __syncthreads();
  int run = s - own;
  for (int i = 0; i < w; ++i) run += sums[i];
  for (int d = d0; d < d0 + per && d < digits; ++d) {
    first[d] = run;
    if (A.start && blockIdx.x == 0 && d <= A.rows) A.start[d] = run;
    run += A.total[d];
  }
  // each warp counts its own tokens
  int key[kSortRounds];
  const int base = blockIdx.x * kSortTile + w * (32 * kSortRounds) + lane;
  sort_load(A, key, base);
  int* mine = at + w * digits;
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int d = key[i] < 0 ? -1 : (key[i] >> A.shift) & (digits - 1);
    const unsigned same = __match_any_sync(0xffffffffu, d);
    if (d >= 0 && lane == __ffs(same) - 1) mine[d] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
    int p = first[d] + A.hist[(int64_t)d * A.blocks + blockIdx.x];
    for (int i = 0; i < kSortWarps; ++i) {
      const int n = at[i * digits + d];
      at[i * digits + d] = p;
      p += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int d = key[i] < 0 ? -1 : (key[i] >> A.shift) & (digits - 1);
    const unsigned same = __match_any_sync(0xffffffffu, d);
    int p = 0;
    if (d >= 0) p = mine[d] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (d >= 0 && lane == __ffs(same) - 1) mine[d] += __popc(same);
    __syncwarp();
    if (d >= 0) {
      const int e = base + 32 * i;
      A.keys_out[p] = key[i];
      A.pos_out[p] = A.pos ? A.pos[e] : e;
    }
  }
}

// start[v]: the first place of a token >= v in the sorted list.
__global__ void sort_start_kernel(const int* keys, int count, int* start, int64_t rows) {
  const int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (v > rows) return;
  int lo = 0, hi = count;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (keys[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  start[v] = lo;
}

// ---------------------------------------------------------------- gradient
struct EmbedGrad {
  const int *keys, *pos, *start;
  const void* grad;
  void* dweight;
  float* part;  // (windows, 2, chunks * E)
  int64_t rows, width;
  int count, window, windows, chunks, tpr, rpb;
  float scale;
};

constexpr int kEmbedAhead = 4;  // rows a thread has on the way

template <typename T, int E>
__device__ __forceinline__ void embed_write(const EmbedGrad& A, int64_t v, int c, const float (&acc)[E]) {
  Pack<T, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) o.e[e] = from_f<T>(acc[e] * A.scale);
  reinterpret_cast<Pack<T, E>*>(static_cast<T*>(A.dweight) + v * A.width)[c] = o;
}

// A group of tpr threads sums the runs of one window, a piece of the columns a thread.
template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads, 4) embed_window_kernel(EmbedGrad A) {
  using P = Pack<T, E>;
  const int w = blockIdx.x * (kEmbedThreads / A.tpr) + threadIdx.x / A.tpr;
  const int c = blockIdx.y * A.tpr + (threadIdx.x & (A.tpr - 1));
  if (w >= A.windows || c >= A.chunks) return;
  const int begin = w * A.window, end = min(begin + A.window, A.count);
  const int before = begin > 0 ? A.keys[begin - 1] : -1;
  const int after = end < A.count ? A.keys[end] : -1;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  int cur = -1;  // the run's token
  bool head = false;
  auto leave = [&](bool tail) {
    if (cur < 0 || cur >= A.rows) return;
    if (!head && !tail) {
      embed_write<T, E>(A, cur, c, acc);
    } else {
      float* p = A.part + ((int64_t)w * 2 + (head ? 0 : 1)) * ((int64_t)A.chunks * E) + (int64_t)c * E;
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = acc[e];
    }
  };
  int key[kEmbedAhead], pos[kEmbedAhead];  // of the rows to come
  const auto look = [&](int i) {
#pragma unroll
    for (int u = 0; u < kEmbedAhead; ++u) {
      key[u] = i + u < end ? A.keys[i + u] : (int)A.rows;
      pos[u] = i + u < end ? A.pos[i + u] : 0;
    }
  };
  look(begin);
  const P* grad = reinterpret_cast<const P*>(A.grad) + c;
  for (int i = begin; i < end; i += kEmbedAhead) {
    P x[kEmbedAhead];
    int now[kEmbedAhead];
#pragma unroll
    for (int u = 0; u < kEmbedAhead; ++u) {
      now[u] = key[u];
      if (now[u] < A.rows) x[u] = grad[(int64_t)pos[u] * A.chunks];
    }
    look(i + kEmbedAhead);
#pragma unroll
    for (int u = 0; u < kEmbedAhead; ++u) {
      if (i + u >= end) break;
      if (now[u] != cur) {
        leave(false);
        cur = now[u];
        head = i + u == begin && cur == before;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
      }
      if (now[u] < A.rows) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += to_f(x[u].e[e]);
      }
    }
  }
  leave(cur == after);
}

// Rows without a token, and rows whose run crosses windows, whose parts are added in order: by a group of tpr
// threads a row, or, where a row has `kFew` parts or more, by all groups of the block, each a run of them.
// `rpb` rows a block at a time: as many as it has groups, or one, where the rows have many tokens.
template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads) embed_join_kernel(EmbedGrad A) {
  constexpr int kFew = 4;
  __shared__ float share[kEmbedThreads * E];
  const int groups = kEmbedThreads / A.tpr, g = threadIdx.x / A.tpr, lane = threadIdx.x & (A.tpr - 1);
  const int c = blockIdx.y * A.tpr + lane;
  const int64_t line = (int64_t)A.chunks * E;
  auto add = [&](float (&acc)[E], int first, int last, int w0) {
#pragma unroll 4
    for (int w = first; w <= last; ++w) {
      const Pack<float, E> p = *reinterpret_cast<const Pack<float, E>*>(A.part + ((int64_t)w * 2 + (w == w0 ? 1 : 0)) * line + (int64_t)c * E);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += p.e[e];
    }
  };
  for (int64_t v0 = (int64_t)blockIdx.x * A.rpb; v0 < A.rows; v0 += (int64_t)gridDim.x * A.rpb) {
    bool many = false;
    const int64_t v = v0 + g;
    if (g < A.rpb && v < A.rows) {
      const int s = A.start[v], e = A.start[v + 1], w0 = s / A.window, w1 = (e - 1) / A.window;
      float acc[E];
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] = 0.f;
      if (s == e) {
        if (c < A.chunks) embed_write<T, E>(A, v, c, acc);
      } else if (w1 > w0) {
        many = groups > 1 && w1 - w0 >= kFew;
        if (!many && c < A.chunks) {
          add(acc, w0, w1, w0);
          embed_write<T, E>(A, v, c, acc);
        }
      }
    }
    if (groups == 1 || !__syncthreads_or(many)) continue;
    for (int k = 0; k < A.rpb && v0 + k < A.rows; ++k) {  // the whole block on one row
      const int s = A.start[v0 + k], e = A.start[v0 + k + 1], w0 = s / A.window, w1 = (e - 1) / A.window;
      if (s == e || w1 - w0 < kFew) continue;
      float acc[E];
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] = 0.f;
      const int per = (w1 - w0 + groups) / groups, first = w0 + g * per;
      if (c < A.chunks) add(acc, first, min(first + per - 1, w1), w0);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i) share[i * kEmbedThreads + threadIdx.x] = acc[i];
      __syncthreads();
      if (g == 0 && c < A.chunks) {
        for (int j = 1; j < groups; ++j)
#pragma unroll
          for (int i = 0; i < E; ++i) acc[i] += share[i * kEmbedThreads + j * A.tpr + lane];
        embed_write<T, E>(A, v0 + k, c, acc);
      }
    }
  }
}

// Few tokens: one launch. A block takes a row of the table, lists its tokens' places in order
// and sums them.
constexpr int kScanTokens = 4096;

template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads) embed_scan_kernel(EmbedGrad A, Tokens tok) {
  using P = Pack<T, E>;
  constexpr int per = kScanTokens / kEmbedThreads;
  __shared__ uint16_t list[kScanTokens];
  __shared__ int sums[kEmbedThreads / 32];
  __shared__ float share[kEmbedThreads * E];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, v = blockIdx.x;
  const int each = (A.count + kEmbedThreads - 1) / kEmbedThreads, first = threadIdx.x * each;
  unsigned hits = 0;
#pragma unroll
  for (int i = 0; i < per; ++i)
    if (i < each && first + i < A.count && tok.key(first + i, A.rows) == v) hits |= 1u << i;
  int s = __popc(hits);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) sums[w] = s;
  __syncthreads();
  int at = s - __popc(hits), n = 0;
  for (int i = 0; i < kEmbedThreads / 32; ++i) {
    if (i < w) at += sums[i];
    n += sums[i];
  }
  for (unsigned h = hits; h; h &= h - 1) list[at++] = (uint16_t)(first + __ffs(h) - 1);
  __syncthreads();
  const int groups = kEmbedThreads / A.tpr, g = threadIdx.x / A.tpr, col = threadIdx.x & (A.tpr - 1);
  for (int c0 = 0; c0 < A.chunks; c0 += A.tpr) {
    const int c = c0 + col;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    if (c < A.chunks) {
#pragma unroll 4
      for (int i = g; i < n; i += groups) {
        const P x = reinterpret_cast<const P*>(static_cast<const T*>(A.grad) + (int64_t)list[i] * A.width)[c];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += to_f(x.e[e]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) share[e * kEmbedThreads + threadIdx.x] = acc[e];
    __syncthreads();
    if (g == 0 && c < A.chunks) {
      for (int j = 1; j < groups; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += share[e * kEmbedThreads + j * A.tpr + col];
      embed_write<T, E>(A, v, c, acc);
    }
  }
}

}  // namespace fx
