// The tcgen05 kernels of the biased attention (attn_tc.cuh): launch shapes.
#include "attn_host.cuh"
#include "attn_tc.cuh"

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

}  // namespace

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
