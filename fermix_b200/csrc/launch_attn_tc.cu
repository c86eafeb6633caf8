// The tcgen05 kernels of the biased attention (attn_tc.cuh): launch shapes.
#include "attn_host.cuh"
#include "attn_tc.cuh"
#include "attn_tc_grad.cuh"

namespace fxh {

namespace {

template <typename T, int NS, int QT, int BN, int DC, int ST, bool VEC>
int fwd(cudaStream_t s, const AttnArgs& A) {
  using S = tc::FwdShape<T, NS, QT, BN, DC, ST>;
  const size_t smem = S::kTileBytes + 1024 + (A.table ? (2 * A.buckets.reach + 1) * sizeof(float) : 0);
  auto kern = tc::attn_fwd_kernel<T, NS, QT, BN, DC, ST, VEC>;
  if (raise_smem(kern, smem)) return FX_ERR_CUDA;
  const int64_t blocks = (A.Lq + 128 * QT - 1) / (128 * QT) * A.H * A.B;
  if (blocks > kMaxGrid) return FX_ERR_SHAPE;
  kern<<<(unsigned)blocks, S::kThreads, smem, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <bool VEC>
int fwd_shape(cudaStream_t s, const AttnArgs& A, bool is_f32) {
  if (is_f32) return A.D <= 64 ? fwd<float, 3, 1, 64, 1, 1, VEC>(s, A) : fwd<float, 3, 1, 64, 2, 1, VEC>(s, A);
  if (A.Lq <= 128) return A.D <= 64 ? fwd<bf16, 1, 1, 64, 1, 2, VEC>(s, A) : fwd<bf16, 1, 1, 64, 2, 2, VEC>(s, A);
  return A.D <= 64 ? fwd<bf16, 1, 2, 128, 1, 2, VEC>(s, A) : fwd<bf16, 1, 2, 128, 2, 2, VEC>(s, A);
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

template <typename T, int NS, int DC, int ST, bool VEC>
int bwd(cudaStream_t s, const AttnArgs& A) {
  const int lanes = (A.D * (int)sizeof(T) + 15) / 16;
  int st = lanes <= 8 ? prep<T, 8, VEC>(s, A) : lanes <= 16 ? prep<T, 16, VEC>(s, A) : prep<T, 32, VEC>(s, A);
  if (st) return st;
  const int span = A.table ? 2 * A.buckets.reach + 1 : 0;
  const int64_t kblocks = (A.Lk + 127) / 128 * A.Hk * A.B, qblocks = (A.Lq + 127) / 128 * A.H * A.B;
  if (kblocks > kMaxGrid || qblocks > kMaxGrid) return FX_ERR_SHAPE;
  if (kblocks > 0) {
    using S = tc::DkvShape<NS, DC, ST>;
    auto kern = tc::attn_dkv_kernel<T, NS, DC, ST, VEC>;
    const size_t smem = S::kTileBytes + 1024 + span * sizeof(float);
    if (raise_smem(kern, smem)) return FX_ERR_CUDA;
    kern<<<(unsigned)kblocks, S::kThreads, smem, s>>>(A);
    if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
  }
  if (qblocks > 0) {
    using S = tc::DqShape<NS, DC, ST>;
    auto kern = tc::attn_dq_kernel<T, NS, DC, ST, VEC>;
    const int nb = A.table ? A.buckets.num_buckets : 0;
    // buckets of a launch: up to kWindow, fewer where the tiles and the distances' table are large
    const DevInfo* D = dev_info();
    if (!D) return FX_ERR_DEVICE;
    const int64_t room = ((int64_t)D->smem_optin - 4096 - S::kTileBytes - span * (int64_t)sizeof(int2)) / 1024;
    const int window = room < tc::kWindow ? (int)room : tc::kWindow;
    int w0 = 0;
    do {
      const int wn = nb - w0 < window ? nb - w0 : window;
      const size_t smem = S::kTileBytes + 1024 + (size_t)wn * 1024 + span * sizeof(int2);
      if (raise_smem(kern, smem)) return FX_ERR_CUDA;
      kern<<<(unsigned)qblocks, S::kThreads, smem, s>>>(A, w0, wn);
      if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
      w0 += window;
    } while (w0 < nb);
  }
  return FX_OK;
}

}  // namespace

int launch_attn_tc_bwd(cudaStream_t s, const AttnArgs& A, bool is_f32, bool vec) {
  if (is_f32) return vec ? bwd<float, 3, 1, 1, true>(s, A) : bwd<float, 3, 1, 1, false>(s, A);
  if (A.D <= 64) return vec ? bwd<bf16, 1, 1, 2, true>(s, A) : bwd<bf16, 1, 1, 2, false>(s, A);
  return vec ? bwd<bf16, 1, 2, 2, true>(s, A) : bwd<bf16, 1, 2, 2, false>(s, A);
}

int launch_attn_tc_fwd(cudaStream_t s, const AttnArgs& A, bool is_f32, bool vec) {
  return vec ? fwd_shape<true>(s, A, is_f32) : fwd_shape<false>(s, A, is_f32);
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
