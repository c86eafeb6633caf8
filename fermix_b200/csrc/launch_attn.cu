// Attention with the position bias: checks, choice of kernel, launch shapes, workspace.
#include "attn_decode.cuh"
#include "attn_host.cuh"
#include "attn_rows_grad.cuh"
#include "position_bias.cuh"

namespace {

using namespace fxh;

constexpr int kRC = 4;          // query rows of a block (attn_rows.cuh)
constexpr int kMinSplit = 128;  // keys of a part, at least

int check(const fx_attn_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->batch < 0 || a->heads < 0 || a->kv_heads < 0 || a->q_len < 0 || a->k_len < 0 || a->dim < 1 ||
      a->dim > FX_ATTN_MAX_DIM)
    return FX_ERR_SHAPE;
  if (a->batch > (1 << 30) || a->heads > 65535 || a->q_len > (1 << 30) || a->k_len > (1 << 30)) return FX_ERR_SHAPE;
  if (a->heads > 0 && (a->kv_heads == 0 || a->heads % a->kv_heads)) return FX_ERR_SHAPE;
  return a->table ? check_buckets(a->buckets) : FX_OK;
}

bool no_rows(const fx_attn_args* a) { return a->batch == 0 || a->heads == 0 || a->q_len == 0; }

void copy3(int64_t* d, const int64_t* s) {
  for (int i = 0; i < 3; ++i) d[i] = s[i];
}

AttnArgs make(const fx_attn_args* a) {
  AttnArgs A{};
  A.q = a->q;
  A.k = a->k;
  A.v = a->v;
  A.table = a->table;
  copy3(A.qs, a->q_stride);
  copy3(A.ks, a->k_stride);
  copy3(A.vs, a->v_stride);
  copy3(A.os, a->out_stride);
  copy3(A.dos, a->dout_stride);
  copy3(A.dqs, a->dq_stride);
  copy3(A.dks, a->dk_stride);
  copy3(A.dvs, a->dv_stride);
  A.mask = a->key_mask;
  A.mask_stride = a->mask_stride;
  A.q_pos = a->buckets.q_pos;
  A.k_pos = a->buckets.k_pos;
  A.q_pos_stride = a->buckets.q_pos_stride;
  A.k_pos_stride = a->buckets.k_pos_stride;
  A.out = a->out;
  A.lse = a->lse;
  A.lse_low = a->lse_low;
  A.dout = a->dout;
  A.dq = a->dq;
  A.dk = a->dk;
  A.dv = a->dv;
  A.Lq = a->q_len;
  A.Lk = a->k_len;
  A.B = (int)a->batch;
  A.H = (int)a->heads;
  A.Hk = (int)a->kv_heads;
  A.D = (int)a->dim;
  A.causal = a->causal != 0;
  A.scale = a->scale;
  A.scale2 = a->scale * kLog2e;
  A.splits = 1;
  A.polls = wait_polls();
  if (a->table) A.buckets = make_buckets(a->buckets);
  return A;
}

// Whether every token of these tensors starts on a 16-byte boundary and is whole vectors.
bool aligned(const fx_attn_args* a, bool grad) {
  const int size = a->dtype == FX_F32 ? 4 : 2;
  uintptr_t m = (uintptr_t)a->dim * size;
  auto add = [&](const void* p, const int64_t* s, int64_t heads, int64_t len) {
    const int64_t n[3] = {a->batch, heads, len};
    m |= reinterpret_cast<uintptr_t>(p);
    for (int i = 0; i < 3; ++i)
      if (n[i] > 1) m |= (uintptr_t)(s[i] * size);
  };
  add(a->q, a->q_stride, a->heads, a->q_len);
  add(a->k, a->k_stride, a->kv_heads, a->k_len);
  add(a->v, a->v_stride, a->kv_heads, a->k_len);
  if (grad) {
    add(a->dout, a->dout_stride, a->heads, a->q_len);
    add(a->out, a->out_stride, a->heads, a->q_len);
  }
  return m % 16 == 0;
}

// Lanes of a key: 16 bytes each, a power of two, eight at least.
int lanes_of(const fx_attn_args* a) {
  const int need = (int)((a->dim * (a->dtype == FX_F32 ? 4 : 2) + 15) / 16);
  return need <= 8 ? 8 : need <= 16 ? 16 : 32;
}

// Query heads whose distances a block of the fragment kernel holds: its rows are of that many at most.
constexpr int decode_lut_most(bool wide) { return wide ? 8192 : 4096; }  // their entries
int decode_heads(int64_t shared) { return (int)(shared < kDecodeRows ? shared : kDecodeRows); }
int64_t decode_chunks(const fx_attn_args* a) {
  return (a->heads / a->kv_heads * a->q_len + kDecodeRows - 1) / kDecodeRows;
}

// Which kernel, by the queries of a head: few of them leave the tensor-core kernel's tile of 128 rows
// empty, and the heads that share keys each read them again. Measured for 1, 2, 4, 8, 16, 32 queries
// of 8 x 8 heads on 2 key heads of 4096 keys, us: bfloat16 dim 64 21, 24, 26, 28, 42, 60 by fragments
// and 40 to 44 by tiles; dim 128 28, 28, 32, 46, 62, 93 and 48 to 54; float32 dim 32 30, 42, 60, 99, 165
// by rows and 79 to 81 by tiles; dim 64 40, 62, 93, 175 and 136; dim 128 62, 101, 167, 332, 646 and
// 369. The same places for 64 batches of 128 and 512 keys. The table by distance has to fit beside
// two (one above 64 entries) of the fragment kernel's rings of 96 KB (192 KB) an SM: 16 (32) KB.
// Where it does not, tiles are no slower than bfloat16 rows were, from one query on (48 us by rows).
enum Kind { ROWS, DECODE, TC };

Kind kind_of(const fx_attn_args* a) {
  const bool wide = a->dim > 64;
  if (a->dtype == FX_F32) return a->q_len <= (wide ? 8 : 4) ? ROWS : TC;
  const bool fits = !a->table || decode_heads(a->heads / a->kv_heads) * (2 * make_buckets(a->buckets).reach + 1) <=
                                     decode_lut_most(wide);
  return fits && a->q_len <= (wide ? 8 : 16) ? DECODE : TC;
}

// Parts of the keys. Rows kernel: eight blocks an SM, parts of 128 keys at least. Fragment kernel:
// two rounds of the two blocks an SM holds (one above 64 entries), 512 keys a part at least; more
// and shorter parts spend more time on a block's start (measured for 64 key heads of 65536 keys:
// 37 parts 205 us, 9 parts 186 us). Tiles: attn_tc_splits.
void split_keys(const fx_attn_args* a, Kind kind, int sms, AttnArgs& A) {
  if (kind == TC) {
    A.splits = attn_tc_splits(A, a->dtype == FX_F32, sms);
    return;
  }
  if (kind == DECODE) {
    const int64_t blocks = decode_chunks(a) * a->batch * a->kv_heads;
    const int64_t want = (int64_t{a->dim <= 64 ? 4 : 2} * sms) / blocks;
    const int64_t most = (a->k_len + 511) / 512, splits = want < most ? want : most;
    A.splits = splits < 1 ? 1 : (int)splits;
    return;
  }
  const int64_t rows = a->heads / a->kv_heads * a->q_len;
  const int64_t blocks = (rows + kRC - 1) / kRC * a->batch * a->kv_heads;
  int64_t splits = (int64_t{8} * sms + blocks - 1) / blocks;
  const int64_t most = (a->k_len + kMinSplit - 1) / kMinSplit;
  splits = splits < most ? splits : most;
  if (splits < 1) splits = 1;
  A.split_keys = ((a->k_len + splits - 1) / splits + 31) / 32 * 32;
  A.splits = A.split_keys ? (int)((a->k_len + A.split_keys - 1) / A.split_keys) : 1;
  if (A.splits < 1) A.splits = 1;
}

size_t part_bytes(const fx_attn_args* a, const AttnArgs& A) {
  return A.splits > 1 ? (size_t)(a->batch * a->heads * a->q_len) * A.splits * part_step((int)a->dim) * sizeof(float) + 256 : 0;
}

// A block a row joins the most parts at a time (256 rows of 9 parts: 5 us, 7 with a warp a row; 8 rows
// of 128: 15 us less than with a warp); from 1024 rows on a warp each (8192 rows of 2 parts: 6 and 12 us).
template <typename T>
int join_parts(cudaStream_t s, const AttnArgs& A) {
  const int64_t rows = (int64_t)A.B * A.H * A.Lq;
  if (rows > kMaxGrid) return FX_ERR_SHAPE;
  if (rows >= 1024)
    attn_join_warp_kernel<T><<<(unsigned)((rows + kRowsThreads / 32 - 1) / (kRowsThreads / 32)), kRowsThreads, 0, s>>>(A);
  else
    attn_join_kernel<T><<<(unsigned)rows, kRowsThreads, 0, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <int LPK, bool VL>
int launch_fwd(cudaStream_t s, const AttnArgs& A) {
  constexpr int NE = 4, GROUPS = kRowsThreads / LPK;
  const size_t lut = A.table ? (size_t)kRC * (2 * A.buckets.reach + 1) * 4 : 0;
  constexpr size_t join = (size_t)GROUPS * kRC * (2 + LPK * NE) * 4;
  const size_t smem = lut > join ? lut : join;
  constexpr size_t lut_most = kRC * kMaxSpan * 4, most = lut_most > join ? lut_most : join;
  auto kern = attn_rows_kernel<float, LPK, VL, kRC>;
  if (raise_smem(kern, smem, most)) return FX_ERR_CUDA;
  const int64_t rows = (int64_t)(A.H / A.Hk) * A.Lq;
  const int64_t blocks = (rows + kRC - 1) / kRC * A.B * A.Hk * A.splits;
  if (blocks > kMaxGrid) return FX_ERR_SHAPE;
  kern<<<(unsigned)blocks, kRowsThreads, smem, s>>>(A);
  if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
  return A.splits > 1 ? join_parts<float>(s, A) : FX_OK;
}

template <int DB, bool VEC>
int launch_decode(cudaStream_t s, const AttnArgs& A) {
  const size_t lut = A.table ? (size_t)decode_heads(A.H / A.Hk) * (2 * A.buckets.reach + 1) * 4 : 0;
  const size_t ring = (size_t)kDecodeStages * 8 * DB * kDecodeThreads * 16;
  static_assert(kDecodeWarps * (2 * kDecodeRows + kDecodeRows * (64 * DB + 1)) * 4 <=
                kDecodeStages * 8 * DB * kDecodeThreads * 16);
  const size_t smem = ring + lut;
  auto kern = attn_decode_kernel<DB, VEC>;
  if (raise_smem(kern, smem, ring + decode_lut_most(DB > 1) * 4)) return FX_ERR_CUDA;
  const int64_t chunks = ((int64_t)(A.H / A.Hk) * A.Lq + kDecodeRows - 1) / kDecodeRows;
  const int64_t blocks = (int64_t)A.B * A.Hk * chunks * A.splits;
  if (blocks > kMaxGrid) return FX_ERR_SHAPE;
  kern<<<(unsigned)blocks, kDecodeThreads, smem, s>>>(A);
  if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
  return A.splits > 1 ? join_parts<bf16>(s, A) : FX_OK;
}

// float32 above 64 entries: 32 lanes a row.
template <bool VL>
int launch_bwd(cudaStream_t s, const AttnArgs& A) {
  constexpr int LPK = 32, NE = 4, GROUPS = kRowsThreads / LPK;
  constexpr size_t join = (size_t)GROUPS * kRC * LPK * NE * 4;
  const size_t hist = A.table ? (size_t)GROUPS * kRC * A.buckets.num_buckets * 8 : 0;
  const size_t smem = hist > join ? hist : join;
  constexpr size_t hist_most = (size_t)GROUPS * kRC * FX_BUCKET_MAX * 8, most = hist_most > join ? hist_most : join;
  const int64_t qrows = (int64_t)(A.H / A.Hk) * A.Lq;
  auto kq = attn_rows_grad_kernel<float, LPK, VL, kRC, false>;
  auto kk = attn_rows_grad_kernel<float, LPK, VL, kRC, true>;
  if (raise_smem(kq, smem, most) || raise_smem(kk, join, join)) return FX_ERR_CUDA;
  const int64_t qblocks = (qrows + kRC - 1) / kRC * A.B * A.Hk, kblocks = (A.Lk + kRC - 1) / kRC * A.B * A.Hk;
  if (qblocks > kMaxGrid || kblocks > kMaxGrid || (int64_t)A.B * A.H * A.Lq > kMaxGrid) return FX_ERR_SHAPE;
  attn_delta_kernel<<<(unsigned)(((int64_t)A.B * A.H * A.Lq + 3) / 4), kRowsThreads, 0, s>>>(A);
  kq<<<(unsigned)qblocks, kRowsThreads, smem, s>>>(A);
  if (A.Lk > 0) kk<<<(unsigned)kblocks, kRowsThreads, join, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

int fwd(cudaStream_t s, const AttnArgs& A, int lanes, bool vec) {
  if (lanes == 8) return vec ? launch_fwd<8, true>(s, A) : launch_fwd<8, false>(s, A);
  if (lanes == 16) return vec ? launch_fwd<16, true>(s, A) : launch_fwd<16, false>(s, A);
  return vec ? launch_fwd<32, true>(s, A) : launch_fwd<32, false>(s, A);
}

// Without queries dk and dv are zero.
template <typename T>
int no_queries(cudaStream_t s, const AttnArgs& A) {
  const int64_t blocks = ((int64_t)A.B * A.Hk * A.Lk * A.D + 255) / 256;
  if (blocks > kMaxGrid) return FX_ERR_SHAPE;
  if (blocks > 0) attn_zero_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

// The tensor-core gradient holds both sides of a block in shared memory: float32's three parts
// fit to a head dimension of 64.
bool use_tc_grad(const fx_attn_args* a) { return a->dtype != FX_F32 || a->dim <= 64; }

struct GradWorkspace {
  size_t lut, dpart, total;  // offsets behind delta
  int64_t parts;
};

GradWorkspace grad_workspace(const fx_attn_args* a) {
  GradWorkspace w;
  const size_t rows = (size_t)(a->batch * a->heads * a->q_len);
  w.parts = a->batch * (use_tc_grad(a) ? (a->q_len + 127) / 128 : a->q_len);
  const int reach = a->table ? make_buckets(a->buckets).reach : 0;
  w.lut = align256(rows * 4);
  w.dpart = w.lut + (a->table ? align256((size_t)a->heads * (2 * reach + 1) * 4) : 0);
  w.total = w.dpart + (a->table ? (size_t)a->heads * w.parts * a->buckets.num_buckets * 4 : 0) + 256;
  return w;
}

}  // namespace

extern "C" {

size_t fermix_biased_attention_workspace_bytes(const fx_attn_args* a) {
  const DevInfo* D = dev_info();
  if (check(a) || !D || no_rows(a)) return 0;
  AttnArgs A = make(a);
  split_keys(a, kind_of(a), D->sms, A);
  return part_bytes(a, A);
}

int fermix_biased_attention(void* stream, const fx_attn_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  if (no_rows(a)) return FX_OK;
  if (!a->q || !a->out || (a->k_len > 0 && (!a->k || !a->v))) return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  AttnArgs A = make(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool vec = aligned(a, false);
  const Kind kind = kind_of(a);
  split_keys(a, kind, D->sms, A);
  const size_t need = part_bytes(a, A);
  if (need) {
    if (!ws || wsb < need) return FX_ERR_WORKSPACE;
    A.part = reinterpret_cast<float*>(align256(reinterpret_cast<uintptr_t>(ws)));
  }
  if (kind == TC) {
    const int st = launch_attn_tc_fwd(s, A, a->dtype == FX_F32, vec);
    return st || A.splits == 1 ? st : a->dtype == FX_F32 ? join_parts<float>(s, A) : join_parts<bf16>(s, A);
  }
  if (kind == DECODE) {
    if (a->dim <= 64) return vec ? launch_decode<1, true>(s, A) : launch_decode<1, false>(s, A);
    return vec ? launch_decode<2, true>(s, A) : launch_decode<2, false>(s, A);
  }
  return fwd(s, A, lanes_of(a), vec);
}

size_t fermix_biased_attention_grad_workspace_bytes(const fx_attn_args* a) {
  if (check(a) || no_rows(a)) return 0;
  return grad_workspace(a).total;
}

int fermix_biased_attention_grad(void* stream, const fx_attn_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->batch == 0 || a->heads == 0) {
    if (a->table && a->heads > 0) {
      if (!a->dtable) return FX_ERR_NULL;
      if (cudaMemsetAsync(a->dtable, 0, (size_t)a->heads * a->buckets.num_buckets * (a->dtype == FX_F32 ? 4 : 2),
                          s) != cudaSuccess)
        return FX_ERR_CUDA;
    }
    return FX_OK;
  }
  if ((a->q_len > 0 && (!a->q || !a->dout || !a->out || !a->lse || !a->dq)) ||
      (a->k_len > 0 && (!a->k || !a->v || !a->dk || !a->dv)) || (a->table && !a->dtable))
    return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  AttnArgs A = make(a);
  const GradWorkspace w = grad_workspace(a);
  if (!no_rows(a) && (!ws || wsb < w.total)) return FX_ERR_WORKSPACE;
  unsigned char* p = reinterpret_cast<unsigned char*>(align256(reinterpret_cast<uintptr_t>(ws)));
  A.delta = reinterpret_cast<float*>(p);
  A.lut = reinterpret_cast<float*>(p + w.lut);
  A.dpart = reinterpret_cast<float*>(p + w.dpart);
  const bool vec = aligned(a, true), f32 = a->dtype == FX_F32;
  const int st = no_rows(a)       ? (f32 ? no_queries<float>(s, A) : no_queries<bf16>(s, A))
                 : use_tc_grad(a) ? launch_attn_tc_bwd(s, A, f32, vec)
                 : vec            ? launch_bwd<true>(s, A)
                                  : launch_bwd<false>(s, A);
  if (st || !a->table) return st;
  const int nb = a->buckets.num_buckets;
  const dim3 grid((nb + 31) / 32, A.H);
  const int64_t parts = w.parts;
  if (a->dtype == FX_F32)
    bias_finish_kernel<float><<<grid, 1024, 0, s>>>(A.dpart, static_cast<float*>(a->dtable), parts, nb);
  else
    bias_finish_kernel<bf16><<<grid, 1024, 0, s>>>(A.dpart, static_cast<bf16*>(a->dtable), parts, nb);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

}  // extern "C"
