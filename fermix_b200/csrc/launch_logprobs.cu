// Log probabilities of tokens (token_logprobs.cuh): checks, launch shapes, workspace.
#include "token_host.cuh"
#include "token_logprobs.cuh"

namespace {

using namespace fxh;

// Below it a difference of two logits may pass float32's range and still count, and the scale itself would be lost.
constexpr float kLeastScale = 1e-30f;

int check(const fx_logprobs_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->token_bytes != 1 && a->token_bytes != 2 && a->token_bytes != 4 && a->token_bytes != 8) return FX_ERR_DTYPE;
  if (a->rows < 0 || a->rows >= INT32_MAX || a->entries < 1 || a->entries > FX_LOGPROBS_MAX || a->top < 0 ||
      a->top > FX_TOP_MAX || !(a->scale >= kLeastScale) || a->scale > 1e30f || a->logits_stride < 0 || a->mask_stride < 0)
    return FX_ERR_SHAPE;
  return FX_OK;
}

constexpr int64_t kWarpRow = 1024;  // entries of a row that a warp takes

// Parts of a row, in 16-byte pieces: enough to give every SM eight blocks, of 4096 entries at least.
void split(const fx_logprobs_args* a, int sms, int& parts, int& per) {
  const int64_t E = a->dtype == FX_F32 ? 4 : 8, pieces = a->entries / E + 2, want = (8 * (int64_t)sms + a->rows - 1) / a->rows;
  const int64_t most = (a->entries + 4095) / 4096, n = a->entries <= kWarpRow ? 1 : want < most ? want : most;
  per = (int)(((pieces + n - 1) / n + kProbThreads - 1) / kProbThreads * kProbThreads);
  parts = (int)((pieces + per - 1) / per);
}

ProbArgs make(const fx_logprobs_args* a) {
  ProbArgs A{};
  A.tok = {a->tokens, a->token_bytes, a->has_padding != 0, a->padding};
  A.logits = a->logits;
  A.mask = a->mask;
  A.ls = a->logits_stride;
  A.ms = a->mask_stride;
  A.logp = a->logp;
  A.entropy = a->entropy;
  A.top_logp = a->top_logp;
  A.top_index = a->top_index;
  A.stats = a->stats;
  A.rows = a->rows;
  A.entries = (int)a->entries;
  A.top = a->top;
  A.scale = a->scale;
  A.glogp = a->grad_logp;
  A.gentropy = a->grad_entropy;
  A.dlogits = a->dlogits;
  return A;
}

template <typename T, bool TOP>
int run(cudaStream_t s, const ProbArgs& A) {
  if (A.entries <= kWarpRow) {
    prob_kernel<T, TOP, 1><<<(unsigned)((A.rows + kProbWarps - 1) / kProbWarps), kProbThreads, 0, s>>>(A);
  } else {
    const int64_t blocks = A.rows * A.parts;
    if (blocks > INT32_MAX) return FX_ERR_SHAPE;
    prob_kernel<T, TOP, kProbWarps><<<(unsigned)blocks, kProbThreads, 0, s>>>(A);
    if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
    if (A.parts > 1) return launch_next(prob_join_kernel<T, TOP>, (unsigned)A.rows, kProbThreads, 0, s, A);
  }
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <typename T>
int run_grad(cudaStream_t s, const ProbArgs& A) {
  if (A.entries <= kWarpRow) {
    prob_grad_kernel<T, 1><<<(unsigned)((A.rows + kProbWarps - 1) / kProbWarps), kProbThreads, 0, s>>>(A);
  } else {
    const int64_t blocks = A.rows * A.parts;
    if (blocks > INT32_MAX) return FX_ERR_SHAPE;
    prob_grad_kernel<T, kProbWarps><<<(unsigned)blocks, kProbThreads, 0, s>>>(A);
  }
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

size_t part_bytes(const fx_logprobs_args* a, int parts) {
  return parts == 1 ? 0 : align256((size_t)a->rows * parts * sizeof(float4)) +
                              align256((size_t)a->rows * parts * a->top * sizeof(int2)) + 256;
}

}  // namespace

extern "C" {

size_t fermix_token_logprobs_workspace_bytes(const fx_logprobs_args* a) {
  const DevInfo* D = dev_info();
  if (check(a) || !D || a->rows == 0) return 0;
  int parts, per;
  split(a, D->sms, parts, per);
  return part_bytes(a, parts);
}

int fermix_token_logprobs(void* stream, const fx_logprobs_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  if (a->rows == 0) return FX_OK;
  if (!a->logits || !a->tokens || !a->logp || !a->entropy || (a->top && (!a->top_logp || !a->top_index)))
    return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  ProbArgs A = make(a);
  split(a, D->sms, A.parts, A.per);
  const size_t need = part_bytes(a, A.parts);
  if (need && (!ws || wsb < need)) return FX_ERR_WORKSPACE;
  if (need) {
    A.part = reinterpret_cast<float4*>(align256(reinterpret_cast<uintptr_t>(ws)));
    A.part_top = reinterpret_cast<int2*>(reinterpret_cast<unsigned char*>(A.part) +
                                         align256((size_t)a->rows * A.parts * sizeof(float4)));
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == FX_F32) return a->top ? run<float, true>(s, A) : run<float, false>(s, A);
  return a->top ? run<bf16, true>(s, A) : run<bf16, false>(s, A);
}

int fermix_token_logprobs_grad(void* stream, const fx_logprobs_args* a) {
  const int e = check(a);
  if (e) return e;
  if (a->rows == 0) return FX_OK;
  if (!a->logits || !a->tokens || !a->entropy || !a->stats || !a->dlogits) return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  ProbArgs A = make(a);
  split(a, D->sms, A.parts, A.per);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == FX_F32 ? run_grad<float>(s, A) : run_grad<bf16>(s, A);
}

}  // extern "C"
