// The tcgen05 kernels of the biased attention (attn_tc.cuh): launch shapes.
#include "attn_host.cuh"
#include "attn_tc.cuh"
#include "attn_tc_grad.cuh"

namespace fxh {

namespace {


using tc::LOAD_ENTRIES;
using tc::LOAD_PIECES;
using tc::LOAD_TMA;
using Narrow = tc::Rows<64, 1>;   // dim <= 32 (float32)
using Half = tc::Rows<128, 1>;    // dim <= 64
using Whole = tc::Rows<128, 2>;   // dim <= 128

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// The map of a bfloat16 tensor (batch, head, token) by element strides: boxes of 64 entries by
// `rows` tokens. false: no such map (the caller loads by the threads).
bool make_map(tc::TmaMaps& M, int which, const void* p, const int64_t* stride, int B, int H, int64_t L, int D, int rows) {
  if (p == nullptr || L == 0) {  // no token is asked for
    M.m[which] = M.m[tc::MAP_Q];
    return true;
  }
  const int64_t n[3] = {L, H, B}, st[3] = {stride[2], stride[1], stride[0]};
  cuuint64_t dims[4] = {(cuuint64_t)D, 1, 1, 1}, bytes[3];
  for (int i = 0; i < 3; ++i) {
    const bool one = n[i] == 1 || st[i] == 0;  // a dimension of one entry takes any stride
    if (i == 0 && st[0] == 0 && L > 1) return false;
    dims[i + 1] = one ? 1 : (cuuint64_t)n[i];
    bytes[i] = one ? (cuuint64_t)((D * 2 + 15) / 16 * 16) : (cuuint64_t)st[i] * 2;
    if (bytes[i] >= (cuuint64_t{1} << 40)) return false;
  }
  M.head_mul[which] = dims[2] > 1;
  M.batch_mul[which] = dims[3] > 1;
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, ones[4] = {1, 1, 1, 1};
  return encode_tiled()(&M.m[which], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, bytes, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int NS, int QT, int BN, typename L, int ST, int LOAD>
int fwd(cudaStream_t s, const AttnArgs& A) {
  using S = tc::FwdShape<NS, QT, BN, L, ST>;
  tc::TmaMaps M{};
  if constexpr (LOAD == LOAD_TMA) {
    if (!encode_tiled() || !make_map(M, tc::MAP_Q, A.q, A.qs, A.B, A.H, A.Lq, A.D, 128) ||
        !make_map(M, tc::MAP_K, A.k, A.ks, A.B, A.Hk, A.Lk, A.D, BN) ||
        !make_map(M, tc::MAP_V, A.v, A.vs, A.B, A.Hk, A.Lk, A.D, BN))
      return fwd<T, NS, QT, BN, L, ST, LOAD_ENTRIES>(s, A);
  }
  const size_t smem = S::kTileBytes + 1024 + (A.table ? (2 * A.buckets.reach + 1) * sizeof(float) : 0);
  auto kern = tc::attn_fwd_kernel<T, NS, QT, BN, L, ST, LOAD>;
  if (raise_smem(kern, smem, S::kTileBytes + 1024 + kMaxSpan * sizeof(float))) return FX_ERR_CUDA;
  const int64_t blocks = (A.Lq + 128 * QT - 1) / (128 * QT) * A.H * A.B * A.splits;
  if (blocks > kMaxGrid) return FX_ERR_SHAPE;
  kern<<<(unsigned)blocks, S::kThreads, smem, s>>>(A, M);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <int LOAD>
int fwd_f32(cudaStream_t s, const AttnArgs& A) {
  if (A.D <= 32) return fwd<float, 3, 1, 64, Narrow, 2, LOAD>(s, A);
  return A.D <= 64 ? fwd<float, 3, 1, 64, Half, 1, LOAD>(s, A) : fwd<float, 3, 1, 64, Whole, 1, LOAD>(s, A);
}

// Up to 64 entries two blocks of one query tile an SM, above that one block of two tiles that share
// the keys (one tile where there is only one). Measured, us: 64 x 8 heads x 512, dim 64: 152 and 161
// with the other; 8 heads x 4095 causal: 78 and 89; 2 x 16 heads x 4096, dim 128: 478 and 420.
template <int LOAD>
int fwd_bf16(cudaStream_t s, const AttnArgs& A) {
  if (A.D <= 64) return fwd<bf16, 1, 1, 128, Half, 2, LOAD>(s, A);
  return A.Lq <= 128 ? fwd<bf16, 1, 1, 64, Whole, 2, LOAD>(s, A) : fwd<bf16, 1, 2, 128, Whole, 2, LOAD>(s, A);
}

template <typename T, int LPR, bool VEC>
int prep(cudaStream_t s, const AttnArgs& A) {
  const int64_t rows = ((int64_t)A.B * A.H * A.Lq + 256 / LPR - 1) / (256 / LPR);
  const int64_t lut = A.table ? ((int64_t)A.H * (2 * A.buckets.reach + 1) + 255) / 256 : 0;
  if (rows + lut > kMaxGrid) return FX_ERR_SHAPE;
  if (rows + lut == 0) return FX_OK;
  tc::attn_prep_kernel<T, LPR, VEC><<<(unsigned)(rows + lut), 256, 0, s>>>(A, rows);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <typename T, int NS, typename L, int ST, int LOAD>
int bwd(cudaStream_t s, const AttnArgs& A) {
  tc::TmaMaps rows128{}, rows64{};  // of the blocks' own rows, of the streamed tiles
  if constexpr (LOAD == LOAD_TMA) {
    bool ok = encode_tiled() != nullptr;
    for (int own = 0; own < 2 && ok; ++own) {
      tc::TmaMaps& M = own ? rows128 : rows64;
      const int n = own ? 128 : tc::kGradN;
      ok = make_map(M, tc::MAP_Q, A.q, A.qs, A.B, A.H, A.Lq, A.D, n) &&
           make_map(M, tc::MAP_K, A.k, A.ks, A.B, A.Hk, A.Lk, A.D, n) &&
           make_map(M, tc::MAP_V, A.v, A.vs, A.B, A.Hk, A.Lk, A.D, n) &&
           make_map(M, tc::MAP_DO, A.dout, A.dos, A.B, A.H, A.Lq, A.D, n);
    }
    if (!ok) return bwd<T, NS, L, ST, LOAD_ENTRIES>(s, A);
  }
  constexpr bool VEC = LOAD != LOAD_ENTRIES;
  const int lanes = (A.D * (int)sizeof(T) + 15) / 16;
  int st = lanes <= 8 ? prep<T, 8, VEC>(s, A) : prep<T, 16, VEC>(s, A);  // 16 at most
  if (st) return st;
  const int span = A.table ? 2 * A.buckets.reach + 1 : 0;
  const int64_t kblocks = (A.Lk + 127) / 128 * A.Hk * A.B, qblocks = (A.Lq + 127) / 128 * A.H * A.B;
  if (kblocks > kMaxGrid || qblocks > kMaxGrid) return FX_ERR_SHAPE;
  if (kblocks > 0) {
    using S = tc::DkvShape<NS, L, ST>;
    auto kern = tc::attn_dkv_kernel<T, NS, L, ST, LOAD>;
    const size_t smem = S::kTileBytes + 1024 + span * sizeof(float);
    if (raise_smem(kern, smem, S::kTileBytes + 1024 + kMaxSpan * sizeof(float))) return FX_ERR_CUDA;
    tc::TmaMaps M = rows64;
    M.m[tc::MAP_K] = rows128.m[tc::MAP_K];
    M.m[tc::MAP_V] = rows128.m[tc::MAP_V];
    kern<<<(unsigned)kblocks, S::kThreads, smem, s>>>(A, M);
    if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
  }
  if (qblocks > 0) {
    using S = tc::DqShape<NS, L, ST>;
    auto kern = tc::attn_dq_kernel<T, NS, L, ST, LOAD>;
    tc::TmaMaps M = rows64;
    M.m[tc::MAP_Q] = rows128.m[tc::MAP_Q];
    M.m[tc::MAP_DO] = rows128.m[tc::MAP_DO];
    const int nb = A.table ? A.buckets.num_buckets : 0;
    // buckets of a launch: up to kWindow, fewer where the tiles and the distances' table are large
    const DevInfo* D = dev_info();
    if (!D) return FX_ERR_DEVICE;
    const int64_t most = (int64_t)D->smem_optin - 3072;  // beside the kernel's own shared memory
    const int64_t room = (most - 1024 - S::kTileBytes - span * (int64_t)sizeof(int2)) / 1024;
    const int window = room < tc::kWindow ? (int)room : tc::kWindow;
    int w0 = 0;
    do {
      const int wn = nb - w0 < window ? nb - w0 : window;
      const size_t smem = S::kTileBytes + 1024 + (size_t)wn * 1024 + span * sizeof(int2);
      if (raise_smem(kern, smem, most)) return FX_ERR_CUDA;
      kern<<<(unsigned)qblocks, S::kThreads, smem, s>>>(A, M, w0, wn);
      if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
      w0 += window;
    } while (w0 < nb);
  }
  return FX_OK;
}

template <int LOAD>
int bwd_f32(cudaStream_t s, const AttnArgs& A) {
  return A.D <= 32 ? bwd<float, 3, Narrow, 1, LOAD>(s, A) : bwd<float, 3, Half, 1, LOAD>(s, A);
}

template <int LOAD>
int bwd_bf16(cudaStream_t s, const AttnArgs& A) {
  return A.D <= 64 ? bwd<bf16, 1, Half, 2, LOAD>(s, A) : bwd<bf16, 1, Whole, 2, LOAD>(s, A);
}

}  // namespace

int launch_attn_tc_bwd(cudaStream_t s, const AttnArgs& A, bool is_f32, bool aligned) {
  if (is_f32) return aligned ? bwd_f32<LOAD_PIECES>(s, A) : bwd_f32<LOAD_ENTRIES>(s, A);
  return aligned ? bwd_bf16<LOAD_TMA>(s, A) : bwd_bf16<LOAD_ENTRIES>(s, A);
}

int launch_attn_tc_fwd(cudaStream_t s, const AttnArgs& A, bool is_f32, bool aligned) {
  if (is_f32) return aligned ? fwd_f32<LOAD_PIECES>(s, A) : fwd_f32<LOAD_ENTRIES>(s, A);
  return aligned ? fwd_bf16<LOAD_TMA>(s, A) : fwd_bf16<LOAD_ENTRIES>(s, A);
}

// Parts that fill the device: of 128 keys at least in float32, of 512 in bfloat16 and none below 2048
// keys. Measured, us, without and with: 8 heads of 512 x 512 float32 dim 64 67 and 32; 8 of 1024 x 1024 bfloat16
// dim 64 30 and 36 in two parts; 8 heads of 128 queries on 2048 keys 44 and 28, of 64 on 16384 263 and 34.
int attn_tc_splits(const AttnArgs& A, bool is_f32, int sms) {
  const int rows = !is_f32 && A.D > 64 && A.Lq > 128 ? 256 : 128;            // of a block
  const int resident = (is_f32 ? A.D <= 64 : rows == 128) ? 2 : 1;           // blocks an SM holds
  const int64_t blocks = (A.Lq + rows - 1) / rows * A.H * A.B, fill = (int64_t)sms * resident / blocks;
  const int64_t most = is_f32 ? A.Lk / 128 : A.Lk < 2048 ? 1 : A.Lk / 512;
  const int64_t splits = fill < most ? fill : most;
  return splits < 1 ? 1 : (int)splits;
}

int attn_tc_status(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, fx::umma::fx_status_word, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(fx::umma::fx_status_word, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace fxh
