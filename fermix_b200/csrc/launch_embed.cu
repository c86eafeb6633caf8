// Embedding of tokens (token_embedding.cuh): checks, launch shapes, workspace.
#include "token_embedding.cuh"
#include "token_host.cuh"

namespace {

using namespace fxh;

int check(const fx_embed_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->token_bytes != 1 && a->token_bytes != 2 && a->token_bytes != 4 && a->token_bytes != 8) return FX_ERR_DTYPE;
  if (a->count < 0 || a->count >= INT32_MAX || a->rows < 1 || a->rows >= INT32_MAX || a->width < 1 ||
      a->width > FX_EMBED_MAX_WIDTH)
    return FX_ERR_SHAPE;
  if (a->rows > (int64_t{1} << 60) / a->width || a->count > (int64_t{1} << 60) / a->width) return FX_ERR_SHAPE;
  return FX_OK;
}

Tokens tokens_of(const fx_embed_args* a) { return {a->tokens, a->token_bytes, a->has_padding != 0, a->padding}; }

// Pieces of a row, the largest up to 16 bytes that rows are whole pieces of, on boundaries of theirs, and the threads
// that share a row.
struct Shape {
  int entries, chunks, tpr;
};

Shape shape_of(const fx_embed_args* a, const void* p, const void* q) {
  const int size = a->dtype == FX_F32 ? 4 : 2;
  const uintptr_t m = (uintptr_t)(a->width * size) | reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q);
  int piece = 16;
  while (piece > size && m % piece) piece /= 2;
  Shape s;
  s.entries = piece / size;
  s.chunks = (int)(a->width / s.entries);
  s.tpr = 1;
  while (s.tpr < s.chunks && s.tpr < kEmbedThreads) s.tpr *= 2;
  return s;
}

// f.template operator()<T, E>() for the type and the entries of a piece.
template <typename F>
int by_piece(int dtype, int entries, F f) {
  if (dtype == FX_F32) {
    if (entries == 4) return f.template operator()<float, 4>();
    return entries == 2 ? f.template operator()<float, 2>() : f.template operator()<float, 1>();
  }
  if (entries == 8) return f.template operator()<bf16, 8>();
  if (entries == 4) return f.template operator()<bf16, 4>();
  return entries == 2 ? f.template operator()<bf16, 2>() : f.template operator()<bf16, 1>();
}

// Few tokens and rows are listed row by row in one launch: rows x count comparisons.
// Otherwise the tokens are sorted. (The rule does not see how few blocks a small table starts: trained, 4096 tokens over 64 x
// 64 float32 16 us, over 2 x 4096 3.0 ms; 16384 tokens, which are sorted, over 2 x 4096 184 us.)
bool scans(const fx_embed_args* a) {
  return a->count <= kScanTokens && a->rows <= 16384 && a->rows * a->count <= (int64_t{1} << 22);
}

// Tokens of a window (a power of two): as many as leave every thread slot of the device a window's columns.
int shift_of(const fx_embed_args* a, const Shape& s, int sms) {
  int w = 7;
  while (w > 4 && (a->count >> w) * s.chunks < (int64_t)sms * 1024) --w;
  return w;
}

struct SortPlan {
  int passes, bits, blocks, shift, windows;
  size_t keys, hist, total, start, part, bytes;  // offsets
};

SortPlan plan_of(const fx_embed_args* a, const Shape& s, int sms) {
  SortPlan P;
  int bits = 1;
  while (a->rows >> bits) ++bits;  // keys are 0 .. rows
  P.passes = (bits + kSortBits - 1) / kSortBits;
  P.bits = (bits + P.passes - 1) / P.passes;
  P.blocks = (int)((a->count + kSortTile - 1) / kSortTile);
  P.shift = shift_of(a, s, sms);
  P.windows = (int)((a->count + (1 << P.shift) - 1) >> P.shift);
  P.keys = 0;  // keys and places, two of each
  P.hist = align256((size_t)(P.passes > 1 ? 4 : 2) * a->count * sizeof(int));
  P.total = P.hist + align256(((size_t)P.blocks << P.bits) * sizeof(int));
  P.start = P.total + align256((size_t{1} << P.bits) * sizeof(int));
  P.part = P.start + align256((size_t)(a->rows + 1) * sizeof(int));
  P.bytes = P.part + align256((size_t)P.windows * 2 * s.chunks * s.entries * sizeof(float));
  return P;
}

struct Fwd {
  cudaStream_t s;
  const EmbedFwd& A;
  template <typename T, int E>
  int operator()() const {
    const int64_t per = 32 * (kEmbedThreads / 32) / (A.tpr > 32 ? A.tpr / 32 : 1);  // rows of a block
    embed_fwd_kernel<T, E><<<(unsigned)((A.count + per - 1) / per), kEmbedThreads, 0, s>>>(A);
    return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
  }
};

struct Scan {
  cudaStream_t s;
  const EmbedGrad& A;
  const Tokens& tok;
  template <typename T, int E>
  int operator()() const {
    embed_scan_kernel<T, E><<<(unsigned)A.rows, kEmbedThreads, 0, s>>>(A, tok);
    return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
  }
};

struct SumRuns {
  cudaStream_t s;
  const EmbedGrad& A;
  int sms;
  template <typename T, int E>
  int operator()() const {
    const int groups = kEmbedThreads / A.tpr;
    const dim3 windows((A.windows + groups - 1) / groups, (unsigned)((A.chunks + A.tpr - 1) / A.tpr));
    const int st = launch_next(embed_window_kernel<T, E>, windows, kEmbedThreads, 0, s, A);
    if (st) return st;
    // the join: a warp for every row of the table, a block for every window that a long run may begin in, as far as the
    // device holds them
    const int64_t blocks = (A.rows + 7) / 8, want = blocks > A.windows ? blocks : A.windows, most = (int64_t)sms * 4;
    return launch_next(embed_join_kernel<T, E>, (unsigned)(want < most ? want : most), kEmbedThreads, 0, s, A);
  }
};

int sort(cudaStream_t s, const fx_embed_args* a, const SortPlan& P, unsigned char* ws, EmbedGrad& A) {
  int* lists = reinterpret_cast<int*>(ws + P.keys);
  SortArgs S{};
  S.tok = tokens_of(a);
  S.rows = a->rows;
  S.count = (int)a->count;
  S.blocks = P.blocks;
  S.hist = reinterpret_cast<int*>(ws + P.hist);
  S.total = reinterpret_cast<int*>(ws + P.total);
  int* start = reinterpret_cast<int*>(ws + P.start);
  S.mask = (1 << P.bits) - 1;
  S.digits = P.passes == 1 ? (int)a->rows + 1 : 1 << P.bits;
  constexpr size_t each = sizeof(int) + kSortWarps * sizeof(uint16_t);  // a digit's
  const size_t smem = (size_t)(S.digits + 1) * each;
  if (a->count <= kSortSmall) {
    int bits = 1;
    while (a->rows >> bits) ++bits;
    S.keys_out = lists;
    S.pos_out = lists + a->count;
    if (raise_smem(sort_small_kernel, kSmallSmem, kSmallSmem)) return FX_ERR_CUDA;
    sort_small_kernel<<<1, kSmallThreads, kSmallSmem, s>>>(S, (bits + 7) / 8);
    if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
    A.keys = S.keys_out;
    A.pos = S.pos_out;
    A.start = start;
    return launch_next(sort_start_kernel, (unsigned)((a->count + 256) / 256), 256, 0, s, S.keys_out, S.count, start, (int)a->rows);
  }
  if (raise_smem(sort_place_kernel, smem, each << (kSortBits + 1))) return FX_ERR_CUDA;
  for (int p = 0; p < P.passes; ++p) {
    S.keys_out = lists + (size_t)(p & 1) * 2 * a->count;
    S.pos_out = S.keys_out + a->count;
    S.shift = p * P.bits;
    S.start = P.passes == 1 ? start : nullptr;
    int st = FX_OK;
    if (p) {
      st = launch_next(sort_count_kernel, P.blocks, kSortThreads, S.digits * sizeof(int), s, S);
    } else {  // the call's first: behind everything before it
      sort_count_kernel<<<P.blocks, kSortThreads, S.digits * sizeof(int), s>>>(S);
      if (cudaGetLastError() != cudaSuccess) st = FX_ERR_CUDA;
    }
    if (!st) st = launch_next(sort_scan_kernel, (S.digits + 7) / 8, 256, 0, s, S);
    if (!st) st = launch_next(sort_place_kernel, P.blocks, kSortThreads, smem, s, S);
    if (st) return st;
    S.keys = S.keys_out;
    S.pos = S.pos_out;
  }
  A.keys = S.keys;
  A.pos = S.pos;
  A.start = start;
  if (P.passes == 1) return FX_OK;
  return launch_next(sort_start_kernel, (unsigned)((a->count + 256) / 256), 256, 0, s, S.keys, S.count, start, (int)a->rows);
}

}  // namespace

extern "C" {

int fermix_token_embedding(void* stream, const fx_embed_args* a) {
  const int e = check(a);
  if (e) return e;
  if (a->count == 0) return FX_OK;
  if (!a->tokens || !a->weight || !a->out) return FX_ERR_NULL;
  const Shape h = shape_of(a, a->weight, a->out);
  EmbedFwd A{tokens_of(a), a->weight, a->out, a->count, a->rows, h.chunks, h.tpr, a->scale};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_piece(a->dtype, h.entries, Fwd{s, A});
}

// Without the pointers the larger of the two forms counts: entry by entry, fewer windows never
// need more.
size_t fermix_token_embedding_grad_workspace_bytes(const fx_embed_args* a) {
  const DevInfo* D = dev_info();
  if (check(a) || !D || a->count == 0 || scans(a)) return 0;
  return plan_of(a, shape_of(a, a->grad, a->dweight), D->sms).bytes + 256;
}

int fermix_token_embedding_grad(void* stream, const fx_embed_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  if (!a->dweight) return FX_ERR_NULL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->count == 0)
    return cudaMemsetAsync(a->dweight, 0, (size_t)(a->rows * a->width) * (a->dtype == FX_F32 ? 4 : 2), s) == cudaSuccess
               ? FX_OK
               : FX_ERR_CUDA;
  if (!a->tokens || !a->grad) return FX_ERR_NULL;
  const Shape h = shape_of(a, a->grad, a->dweight);
  EmbedGrad A{};
  A.grad = a->grad;
  A.dweight = a->dweight;
  A.rows = a->rows;
  A.width = a->width;
  A.count = (int)a->count;
  A.chunks = h.chunks;
  A.tpr = h.tpr;
  A.scale = a->scale;
  if (scans(a)) {
    const Tokens t = tokens_of(a);
    return by_piece(a->dtype, h.entries, Scan{s, A, t});
  }
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  const SortPlan P = plan_of(a, h, D->sms);
  if (!ws || wsb < P.bytes + 256) return FX_ERR_WORKSPACE;
  unsigned char* base = reinterpret_cast<unsigned char*>(align256(reinterpret_cast<uintptr_t>(ws)));
  A.shift = P.shift;
  A.windows = P.windows;
  A.part = reinterpret_cast<float*>(base + P.part);
  const int st = sort(s, a, P, base, A);
  if (st) return st;
  return by_piece(a->dtype, h.entries, SumRuns{s, A, D->sms});
}

}  // extern "C"
