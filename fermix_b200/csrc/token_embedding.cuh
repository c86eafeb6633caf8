// Embedding of tokens: out[i] = scale weight[token[i]], and its gradient
// dweight[v] = scale * sum of grad[i] over the i with token[i] = v.
//
// The forward is a gather, bound by HBM: each thread has four rows' 16-byte pieces on the way (4096 x 128 tokens of 128
// float32: 48 us for the 268 MB that it writes, 5.6 TB/s).
//
// The gradient adds in a fixed order, so the tokens are sorted first (stable, by digits of up
// to 11 bits: counts per block, their sums over the blocks, then every block places its
// tokens), which costs 12 bytes a token and pass beside the rows' `width` entries. The
// sorted list is cut into windows of equal length, one group of threads each, whatever
// the tokens' frequencies: a run of one token within a window is final, one that crosses
// into another window leaves a float32 partial sum there, and a last kernel adds those in
// order and fills the rows that no token names. Of the same tokens over 512 rows: sort 31 us (bound by the latency of the
// digits' counts in shared memory), windows 48 (268 MB, HBM), join 10.
#pragma once
#include "token_common.cuh"

namespace fx {

constexpr int kEmbedThreads = 256;

struct EmbedFwd {
  Tokens tok;
  const void* weight;
  void* out;
  int64_t count, rows;
  int chunks, tpr;  // pieces of a row; threads of a row (a power of two)
  float scale;
};

// A warp takes 32 rows at a time, whose tokens its lanes look up, one each (a token's row for every lane of a row
// took as many instructions as the rest). tpr <= 32: 32 / tpr rows at a time; above that tpr / 32 warps share the rows.
constexpr int kEmbedAhead = 4;  // rows a thread has on the way

template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads) embed_fwd_kernel(EmbedFwd A) {
  using P = Pack<T, E>;
  const int lane = threadIdx.x & 31, wpr = A.tpr > 32 ? A.tpr / 32 : 1, lpr = A.tpr < 32 ? A.tpr : 32;
  const int warp = threadIdx.x >> 5, c0 = (warp % wpr) * 32 + lane % lpr, rows = 32 / lpr, sub = lane / lpr;
  const int64_t per = kEmbedThreads / 32 / wpr, r0 = ((int64_t)blockIdx.x * per + warp / wpr) * 32;
  int mine = -1;  // the row of token r0 + lane; -1: zeros, -2: none
  if (r0 + lane < A.count) {
    const int64_t t = A.tok.at(r0 + lane);
    mine = A.tok.padded(t) ? -1 : t >= 0 && t < A.rows ? (int)t : -2;
  }
  const int n = (int)(A.count - r0 < 32 ? A.count - r0 : 32);
  for (int c = c0; c - lane % lpr < A.chunks; c += A.tpr) {
    const P* in = static_cast<const P*>(A.weight) + c;
    P* out = static_cast<P*>(A.out) + (r0 + sub) * A.chunks + c;
    const int64_t step = (int64_t)rows * A.chunks;
    for (int k = 0; k < 32; k += kEmbedAhead * rows) {
      P v[kEmbedAhead];
      int row[kEmbedAhead];
#pragma unroll
      for (int u = 0; u < kEmbedAhead; ++u) {
        row[u] = __shfl_sync(0xffffffffu, mine, (k + u * rows + sub) & 31);
        if (row[u] >= 0 && k + u * rows + sub < n && c < A.chunks) v[u] = in[(int64_t)row[u] * A.chunks];
      }
#pragma unroll
      for (int u = 0; u < kEmbedAhead; ++u, out += step) {
        if (k + u * rows + sub >= n || c >= A.chunks) continue;
        P o;
        if (row[u] >= 0) {
          float x[E];
          unpack<E>(v[u], x);
#pragma unroll
          for (int e = 0; e < E; ++e) o.e[e] = from_f<T>(x[e] * A.scale);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) o.e[e] = from_f<T>(row[u] == -1 ? 0.f : __int_as_float(0x7fc00000));
        }
        *out = o;
      }
    }
  }
}

// ---------------------------------------------------------------- sort by token
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kSortRounds = 4;
constexpr int kSortTile = kSortThreads * kSortRounds;  // tokens of a block
constexpr int kSortBits = 11;

struct SortArgs {
  Tokens tok;             // first pass
  const int *keys, *pos;  // later passes
  int *keys_out, *pos_out;
  int* hist;    // (digits, blocks)
  int* total;   // (digits)
  int* start;   // one pass only: first place of each token, (rows + 1)
  int64_t rows;
  int count, blocks, shift, digits;  // digits: that occur
  int mask;
};

// Places behind the last token may pass 2^31 - 1, where the count itself does not: they are unsigned.
__device__ __forceinline__ void sort_load(const SortArgs& A, int (&key)[kSortRounds], unsigned base) {
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const unsigned e = base + 32 * i;
    key[i] = e >= (unsigned)A.count ? -1 : A.keys ? A.keys[e] : A.tok.key(e, A.rows);
  }
}
__device__ __forceinline__ int sort_digit(const SortArgs& A, int key) { return key < 0 ? -1 : (key >> A.shift) & A.mask; }

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs A) {
  wait_for_last();
  extern __shared__ int hist[];
  const int lane = threadIdx.x & 31;
  for (int d = threadIdx.x; d < A.digits; d += kSortThreads) hist[d] = 0;
  int key[kSortRounds];
  sort_load(A, key, blockIdx.x * kSortTile + (threadIdx.x >> 5) * (32 * kSortRounds) + lane);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int d = sort_digit(A, key[i]);
    const unsigned same = __match_any_sync(0xffffffffu, d);  // one addition for equal digits
    if (d >= 0 && lane == __ffs(same) - 1) atomicAdd(&hist[d], __popc(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < A.digits; d += kSortThreads) A.hist[(int64_t)d * A.blocks + blockIdx.x] = hist[d];
}

// Counts of a digit -> first place within the digit for each block; a warp a digit.
__global__ void __launch_bounds__(256) sort_scan_kernel(SortArgs A) {
  wait_for_last();
  const int d = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (d >= A.digits) return;
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

// Every token to its place: the digit's first, those of earlier blocks, of the block's earlier warps, of the warp's
// earlier rounds and lanes.
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortArgs A) {
  wait_for_last();
  extern __shared__ int first[];  // (digits), then 16-bit counts (warps, digits)
  __shared__ int sums[kSortWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, wide = (A.digits + 1) / 2 * 2;
  uint16_t* at = reinterpret_cast<uint16_t*>(first + wide);
  for (int i = threadIdx.x; i < kSortWarps * wide / 2; i += kSortThreads) reinterpret_cast<int*>(at)[i] = 0;
  int key[kSortRounds];
  const unsigned base = blockIdx.x * kSortTile + w * (32 * kSortRounds) + lane;
  sort_load(A, key, base);
  // first places of the digits: a thread sums a run of them
  const int per = (A.digits + kSortThreads - 1) / kSortThreads, d0 = threadIdx.x * per;
  int own = 0;
  for (int d = d0; d < d0 + per && d < A.digits; ++d) own += A.total[d];
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
  for (int d = d0; d < d0 + per && d < A.digits; ++d) {
    first[d] = run + A.hist[(int64_t)d * A.blocks + blockIdx.x];
    if (A.start && blockIdx.x == 0 && d <= A.rows) A.start[d] = run;
    run += A.total[d];
  }
  // each warp counts its own tokens
  uint16_t* mine = at + w * wide;
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int d = sort_digit(A, key[i]);
    const unsigned same = __match_any_sync(0xffffffffu, d);
    if (d >= 0 && lane == __ffs(same) - 1) mine[d] += (uint16_t)__popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < A.digits; d += kSortThreads) {
    int p = 0;
    for (int i = 0; i < kSortWarps; ++i) {
      const int n = at[i * wide + d];
      at[i * wide + d] = (uint16_t)p;
      p += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int d = sort_digit(A, key[i]);
    const unsigned same = __match_any_sync(0xffffffffu, d);
    int p = 0;
    if (d >= 0) p = first[d] + mine[d] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (d >= 0 && lane == __ffs(same) - 1) mine[d] += (uint16_t)__popc(same);
    __syncwarp();
    if (d >= 0) {
      const unsigned e = base + 32 * i;
      A.keys_out[p] = key[i];
      A.pos_out[p] = A.pos ? A.pos[e] : (int)e;
    }
  }
}

// Up to kSortSmall tokens in one launch: one block, all passes (of 8 bits) in shared memory.
constexpr int kSmallThreads = 1024, kSmallWarps = kSmallThreads / 32, kSmallRounds = 8, kSmallDigits = 256;
constexpr int kSortSmall = kSmallThreads * kSmallRounds;
constexpr size_t kSmallSmem = 2 * kSortSmall * sizeof(int) + kSmallDigits * (sizeof(int) + kSmallWarps * sizeof(uint16_t));

__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(SortArgs A, int passes) {
  extern __shared__ int keys[];  // and places, the digits' first places, 16-bit counts (warps, digits)
  __shared__ int sums[kSmallDigits / 32];
  int *pos = keys + kSortSmall, *first = pos + kSortSmall;
  uint16_t* at = reinterpret_cast<uint16_t*>(first + kSmallDigits);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, base = w * (32 * kSmallRounds) + lane;
  int key[kSmallRounds], from[kSmallRounds];
#pragma unroll
  for (int i = 0; i < kSmallRounds; ++i) {
    from[i] = base + 32 * i;
    key[i] = from[i] < A.count ? A.tok.key(from[i], A.rows) : -1;
  }
  for (int p = 0; p < passes; ++p) {
    for (int i = threadIdx.x; i < kSmallDigits * kSmallWarps / 2; i += kSmallThreads) reinterpret_cast<int*>(at)[i] = 0;
    __syncthreads();
    uint16_t* mine = at + w * kSmallDigits;
#pragma unroll
    for (int i = 0; i < kSmallRounds; ++i) {
      const int d = key[i] < 0 ? -1 : key[i] >> (8 * p) & (kSmallDigits - 1);
      const unsigned same = __match_any_sync(0xffffffffu, d);
      if (d >= 0 && lane == __ffs(same) - 1) mine[d] += (uint16_t)__popc(same);
      __syncwarp();
    }
    __syncthreads();
    int total = 0, s = 0;
    if (threadIdx.x < kSmallDigits) {
      for (int i = 0; i < kSmallWarps; ++i) {
        const int n = at[i * kSmallDigits + threadIdx.x];
        at[i * kSmallDigits + threadIdx.x] = (uint16_t)total;
        total += n;
      }
      s = total;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (lane == 31) sums[w] = s;
    }
    __syncthreads();
    if (threadIdx.x < kSmallDigits) {
      int run = s - total;
      for (int i = 0; i < w; ++i) run += sums[i];
      first[threadIdx.x] = run;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallRounds; ++i) {
      const int d = key[i] < 0 ? -1 : key[i] >> (8 * p) & (kSmallDigits - 1);
      const unsigned same = __match_any_sync(0xffffffffu, d);
      int to = 0;
      if (d >= 0) to = first[d] + mine[d] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (d >= 0 && lane == __ffs(same) - 1) mine[d] += (uint16_t)__popc(same);
      __syncwarp();
      if (d >= 0) {
        keys[to] = key[i];
        pos[to] = from[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallRounds; ++i)
      if (base + 32 * i < A.count) {
        key[i] = keys[base + 32 * i];
        from[i] = pos[base + 32 * i];
      }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kSmallRounds; ++i)
    if (base + 32 * i < A.count) {
      A.keys_out[base + 32 * i] = key[i];
      A.pos_out[base + 32 * i] = from[i];
    }
}

// start[v]: the first place of a token >= v in the sorted list; a warp 32 places, each fills the tokens
// between its own and the one before.
__global__ void __launch_bounds__(256) sort_start_kernel(const int* keys, int count, int* start, int rows) {
  wait_for_last();
  const int lane = threadIdx.x & 31;
  const int64_t base = ((int64_t)blockIdx.x * 256 + threadIdx.x) - lane, i = base + lane;
  const int to = i < count ? keys[i] : rows, from = i == 0 ? -1 : i <= count ? keys[i - 1] : rows;
  unsigned steps = __ballot_sync(0xffffffffu, i <= count && to > from);
  while (steps) {
    const int src = __ffs(steps) - 1;
    steps &= steps - 1;
    const int a = __shfl_sync(0xffffffffu, from, src), b = __shfl_sync(0xffffffffu, to, src);
    for (int64_t v = (int64_t)a + 1 + lane; v <= b; v += 32) start[v] = (int)(base + src);
  }
}

// ---------------------------------------------------------------- gradient
struct EmbedGrad {
  const int *keys, *pos, *start;
  const void* grad;
  void* dweight;
  float* part;  // (windows, 2, chunks * E)
  int64_t rows, width;
  int count, shift, windows, chunks, tpr;  // windows of 1 << shift tokens
  float scale;
};

template <typename T, int E>
__device__ __forceinline__ void embed_write(const EmbedGrad& A, int64_t v, int c, const float (&acc)[E]) {
  Pack<T, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) o.e[e] = from_f<T>(acc[e] * A.scale);
  reinterpret_cast<Pack<T, E>*>(static_cast<T*>(A.dweight) + v * A.width)[c] = o;
}

// A group of tpr threads sums the runs of one window, a piece of the columns a thread.
template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads, E > 4 ? 3 : 4) embed_window_kernel(EmbedGrad A) {
  wait_for_last();
  using P = Pack<T, E>;
  const int w = blockIdx.x * (kEmbedThreads / A.tpr) + threadIdx.x / A.tpr;
  const int c = blockIdx.y * A.tpr + (threadIdx.x & (A.tpr - 1));
  if (w >= A.windows || c >= A.chunks) return;
  // unsigned: of the last window the look ahead, and the end of a whole one, may pass 2^31 - 1
  const unsigned begin = (unsigned)w << A.shift, count = A.count, end = min(begin + (1u << A.shift), count);
  const int before = begin > 0 ? A.keys[begin - 1] : -1;
  const int after = end < count ? A.keys[end] : -1;
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
  const auto look = [&](unsigned i) {
#pragma unroll
    for (int u = 0; u < kEmbedAhead; ++u) {
      key[u] = i + u < end ? A.keys[i + u] : (int)A.rows;
      pos[u] = i + u < end ? A.pos[i + u] : 0;
    }
  };
  look(begin);
  const P* grad = reinterpret_cast<const P*>(A.grad) + c;
  for (unsigned i = begin; i < end; i += kEmbedAhead) {
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
        float y[E];
        unpack<E>(x[u], y);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += y[e];
      }
    }
  }
  leave(cur == after);
}

// Rows without a token, and rows whose run crosses windows, whose parts are added in order: up to kFew of them by a
// warp a row, which looks 32 rows up at a time; longer runs by a block, whose groups of tpr threads have a stretch of
// the windows each.
template <typename T, int E>
__global__ void __launch_bounds__(kEmbedThreads) embed_join_kernel(EmbedGrad A) {
  wait_for_last();
  constexpr int kFew = 4;
  __shared__ float share[kEmbedThreads * E];
  const int lane = threadIdx.x & 31, last_token = (int)A.rows;
  const int64_t line = (int64_t)A.chunks * E;
  float acc[E];
  // acc = the parts of the run that begins in window w0, those of windows [first, last], of piece c
  auto add = [&](int c, int first, int last, int w0) {
    constexpr int kAhead = E > 4 ? 4 : 8;
    const float* part = A.part + (int64_t)c * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int w = first; w <= last; w += kAhead) {
      Pack<float, E> p[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (w + u <= last) p[u] = *reinterpret_cast<const Pack<float, E>*>(part + ((int64_t)(w + u) * 2 + (w + u == w0 ? 1 : 0)) * line);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (w + u <= last) {
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += p[u].e[e];
        }
    }
  };
  // The runs of more windows: a lane looks at one window each, whether the run that goes on behind it began in it.
  for (int64_t base = blockIdx.x; base < A.windows; base += (int64_t)32 * gridDim.x) {
    const int64_t mine = base + (int64_t)lane * gridDim.x, place = (mine + 1) << A.shift;
    int row = mine < A.windows && place < A.count ? A.keys[place] : last_token, end = 0;
    if (row < A.rows) {
      end = (A.start[row + 1] - 1) >> A.shift;
      if (A.start[row] >> A.shift != mine || end - mine < kFew) row = last_token;
    }
    unsigned found = __ballot_sync(0xffffffffu, row < A.rows);  // the same in every warp
    while (found) {
      const int src = __ffs(found) - 1, groups = kEmbedThreads / A.tpr, g = threadIdx.x / A.tpr;
      found &= found - 1;
      const int w = (int)(base + (int64_t)src * gridDim.x), w1 = __shfl_sync(0xffffffffu, end, src);
      const int v = __shfl_sync(0xffffffffu, row, src);
      const int per = (w1 - w + groups) / groups, first = w + g * per;
      for (int c0 = 0; c0 < A.chunks; c0 += A.tpr) {
        const int c = c0 + (threadIdx.x & (A.tpr - 1));
        if (c < A.chunks) add(c, first, min(first + per - 1, w1), w);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i) share[i * kEmbedThreads + threadIdx.x] = acc[i];
        __syncthreads();
        if (g == 0 && c < A.chunks) {
          for (int j = 1; j < groups; ++j)
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] += share[i * kEmbedThreads + j * A.tpr + threadIdx.x];
          embed_write<T, E>(A, v, c, acc);
        }
      }
    }
  }
  // a warp's rows are far from each other: the frequent tokens, whose rows cross, often are not
  const int64_t warps = (int64_t)gridDim.x * (kEmbedThreads / 32);
  for (int64_t base = (int64_t)blockIdx.x * (kEmbedThreads / 32) + (threadIdx.x >> 5); base < A.rows; base += warps * 32) {
    const int64_t mine = base + lane * warps;
    const bool in = mine < A.rows;
    const int s = in ? A.start[mine] : 0, e = in ? A.start[mine + 1] : 0;
    const int w0 = s >> A.shift, w1 = (e - 1) >> A.shift;
    unsigned empty = __ballot_sync(0xffffffffu, in && s == e);
    unsigned cross = __ballot_sync(0xffffffffu, in && s < e && w1 > w0 && w1 - w0 < kFew);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    for (; empty; empty &= empty - 1)
      for (int c = lane; c < A.chunks; c += 32) embed_write<T, E>(A, base + (__ffs(empty) - 1) * warps, c, acc);
    for (; cross; cross &= cross - 1) {
      const int src = __ffs(cross) - 1, a = __shfl_sync(0xffffffffu, w0, src), b = __shfl_sync(0xffffffffu, w1, src);
      for (int c = lane; c < A.chunks; c += 32) {
        add(c, a, b, a);
        embed_write<T, E>(A, base + src * warps, c, acc);
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
