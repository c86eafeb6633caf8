// The bucketed position bias (position_bias.cuh): checks, launch shapes, workspace.
#include "block_host.cuh"
#include "position_bias.cuh"

namespace {

using namespace fxh;

int check(const fx_bias_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->batch < 0 || a->heads < 0 || a->q_len < 0 || a->k_len < 0) return FX_ERR_SHAPE;
  if (a->batch > INT32_MAX || a->heads > 65535 || a->q_len > (1 << 30) || a->k_len > (1 << 30)) return FX_ERR_SHAPE;
  return check_buckets(a->buckets);
}

bool empty(const fx_bias_args* a) { return a->batch == 0 || a->heads == 0 || a->q_len == 0 || a->k_len == 0; }

// Column blocks of up to 1024 (tx threads); rows a block so that there are about eight blocks
// an SM, no fewer than 16 rows a thread (a block first lays out the table of its head).
bool shape(const fx_bias_args* a, int sms, BiasArgs& A, int64_t& blocks) {
  A.tx = 1;
  while (A.tx < kBiasThreads && (int64_t)A.tx * kBiasE < a->k_len) A.tx *= 2;
  const int64_t cols = (a->k_len + A.tx * kBiasE - 1) / (A.tx * kBiasE);
  const int64_t slabs = a->batch * a->heads * cols;
  int64_t rb = (int64_t{8} * sms + slabs - 1) / slabs;
  const int64_t least = 16 * (kBiasThreads / A.tx), most = (a->q_len + least - 1) / least;
  rb = rb < most ? rb : most;
  A.rows = (int)((a->q_len + rb - 1) / rb);
  A.row_blocks = (int)((a->q_len + A.rows - 1) / A.rows);
  A.col_blocks = (int)cols;
  A.heads = (int)a->heads;
  A.batch = (int)a->batch;
  blocks = slabs * A.row_blocks;
  return blocks <= INT32_MAX;
}

BiasArgs make(const fx_bias_args* a) {
  BiasArgs A{};
  A.table = a->table;
  A.grad = a->grad;
  A.out = a->out;
  A.q_pos = a->buckets.q_pos;
  A.k_pos = a->buckets.k_pos;
  A.q_pos_stride = a->buckets.q_pos_stride;
  A.k_pos_stride = a->buckets.k_pos_stride;
  A.q_len = a->q_len;
  A.k_len = a->k_len;
  A.buckets = make_buckets(a->buckets);
  return A;
}

constexpr size_t lut_size(int reach) { return (size_t)(2 * reach + 1 + 7) / 8 * 8 * 4; }

template <typename T, int VEC>
int launch(cudaStream_t s, const BiasArgs& A, int64_t blocks, bool grad) {
  const size_t smem = lut_size(A.buckets.reach) + (grad ? (size_t)A.buckets.num_buckets * kBiasThreads * 4 : 0);
  if (grad) {
    if (raise_smem(bias_bwd_kernel<T, VEC>, smem, lut_size(FX_BUCKET_MAX_EDGE) + (size_t)FX_BUCKET_MAX * kBiasThreads * 4))
      return FX_ERR_CUDA;
    bias_bwd_kernel<T, VEC><<<(unsigned)blocks, kBiasThreads, smem, s>>>(A);
  } else {
    bias_fwd_kernel<T, VEC><<<(unsigned)blocks, kBiasThreads, smem, s>>>(A);
  }
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

// Entries of one access: the most (up to 16 bytes) that divide a row and the address.
template <typename T>
int dispatch(cudaStream_t s, const BiasArgs& A, int64_t blocks, bool grad) {
  const uintptr_t m = (uintptr_t)A.k_len * sizeof(T) | reinterpret_cast<uintptr_t>(grad ? A.grad : A.out) | 16;
  const int vec = (int)((m & (~m + 1)) / sizeof(T));
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch<T, 8>(s, A, blocks, grad);
  if (vec == 4) return launch<T, 4>(s, A, blocks, grad);
  if (vec == 2) return launch<T, 2>(s, A, blocks, grad);
  return launch<T, 1>(s, A, blocks, grad);
}

}  // namespace

extern "C" {

int fermix_position_bias(void* stream, const fx_bias_args* a) {
  const int e = check(a);
  if (e) return e;
  if (empty(a)) return FX_OK;
  if (!a->table || !a->out) return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  BiasArgs A = make(a);
  int64_t blocks;
  if (!shape(a, D->sms, A, blocks)) return FX_ERR_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == FX_F32 ? dispatch<float>(s, A, blocks, false) : dispatch<bf16>(s, A, blocks, false);
}

size_t fermix_position_bias_grad_workspace_bytes(const fx_bias_args* a) {
  const DevInfo* D = dev_info();
  if (check(a) || !D || empty(a)) return 0;
  BiasArgs A{};
  int64_t blocks;
  if (!shape(a, D->sms, A, blocks)) return 0;
  return (size_t)blocks * a->buckets.num_buckets * sizeof(float) + 256;
}

int fermix_position_bias_grad(void* stream, const fx_bias_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int nb = a->buckets.num_buckets;
  if (a->heads == 0) return FX_OK;
  if (!a->dtable) return FX_ERR_NULL;
  if (empty(a))
    return cudaMemsetAsync(a->dtable, 0, (size_t)a->heads * nb * (a->dtype == FX_F32 ? 4 : 2), s) == cudaSuccess
               ? FX_OK
               : FX_ERR_CUDA;
  if (!a->grad) return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  BiasArgs A = make(a);
  int64_t blocks;
  if (!shape(a, D->sms, A, blocks)) return FX_ERR_SHAPE;
  if (!ws || wsb < (size_t)blocks * nb * sizeof(float) + 256) return FX_ERR_WORKSPACE;
  A.part = reinterpret_cast<float*>(align256(reinterpret_cast<uintptr_t>(ws)));
  const int st = a->dtype == FX_F32 ? dispatch<float>(s, A, blocks, true) : dispatch<bf16>(s, A, blocks, true);
  if (st) return st;
  const int64_t parts = (int64_t)A.batch * A.row_blocks * A.col_blocks;
  const dim3 grid((nb + 31) / 32, (unsigned)a->heads);
  if (a->dtype == FX_F32)
    bias_finish_kernel<float><<<grid, 1024, 0, s>>>(A.part, static_cast<float*>(a->dtable), parts, nb);
  else
    bias_finish_kernel<bf16><<<grid, 1024, 0, s>>>(A.part, static_cast<bf16*>(a->dtable), parts, nb);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

}  // extern "C"
