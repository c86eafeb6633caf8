// The gated residual with its norms (residual_norm.cuh): checks, launch shapes, workspace.
#include "block_host.cuh"
#include "residual_norm.cuh"

namespace {

using namespace fxh;

int check(const fx_norm_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->groups < 0 || a->rows < 0 || a->width < 1 || a->width > FX_NORM_MAX_WIDTH || a->kind < 0 || a->kind > 1 ||
      a->gate_mode < FX_GATE_NONE || a->gate_mode > FX_GATE_GROUP)
    return FX_ERR_SHAPE;
  if (a->groups > 0 && a->rows > (int64_t{1} << 40) / a->groups) return FX_ERR_SHAPE;
  return FX_OK;
}

// Threads of a row: a 16-byte chunk each up to 512 threads (registers of the backward: five rows
// and six running sums), two or four chunks above that.
struct Shape {
  int chunks, tpr, threads, rpb;
};

Shape shape_of(const fx_norm_args* a) {
  const int64_t entries = a->dtype == FX_F32 ? 4 : 8, all = (a->width + entries - 1) / entries;
  Shape s;
  s.chunks = all <= 512 ? 1 : all <= 1024 ? 2 : 4;
  const int need = (int)((all + s.chunks - 1) / s.chunks);
  if (need <= 32) {
    s.tpr = 1;
    while (s.tpr < need) s.tpr *= 2;
    s.threads = kNormThreads;
    s.rpb = kNormThreads / s.tpr;
  } else {
    s.tpr = s.threads = (need + 31) / 32 * 32;
    s.rpb = 1;
  }
  return s;
}

// As many blocks as are resident at a time, the rows in equal contiguous parts.
void split(const fx_norm_args* a, const Shape& s, int sms, bool grad, int& grid, int64_t& per) {
  const int64_t N = a->groups * a->rows, units = (N + s.rpb - 1) / s.rpb;
  const bool f32 = a->dtype == FX_F32, one = s.chunks == 1;
  const int resident = grad ? (one ? (f32 ? kNormBwdResident<float, 1> : kNormBwdResident<bf16, 1>) : 512)
                            : (one ? (f32 ? kNormFwdResident<float, 1> : kNormFwdResident<bf16, 1>) : 512);
  const int64_t cap = (int64_t)sms * (resident / s.threads);
  const int64_t blocks = units < cap ? units : cap;
  per = (units + blocks - 1) / blocks * s.rpb;
  grid = (int)((N + per - 1) / per);
}  // per < 2^31: N <= 2^40 rows over at least 2^9 blocks where N is that large

size_t part_bytes(const fx_norm_args* a, int grid) {
  return align256((size_t)kNormSums * grid * a->width * sizeof(float));
}
size_t gpart_bytes(const fx_norm_args* a, int grid) {
  return a->gate_mode == FX_GATE_GROUP ? align256((size_t)(grid + a->groups) * a->width * sizeof(float)) : 0;
}

NormArgs make(const fx_norm_args* a, const Shape& s) {
  NormArgs A{};
  A.x = a->x;
  A.f = a->f;
  A.gate = a->gate;
  A.scale = a->scale;
  A.pw = a->post_weight;
  A.pb = a->post_bias;
  A.rw = a->pre_weight;
  A.rb = a->pre_bias;
  A.r = a->r;
  A.z = a->z;
  A.gr = a->grad_r;
  A.gz = a->grad_z;
  A.dx = a->dx;
  A.df = a->df;
  A.dgate = a->dgate;
  A.N = a->groups * a->rows;
  A.R = a->rows;
  A.eps = a->eps;
  A.W = (int)a->width;
  A.layer = a->kind;
  A.gate_mode = a->gate_mode;
  A.dgate_f32 = a->dgate_f32 != 0;
  A.tpr = s.tpr;
  return A;
}

// Whether every row and parameter is whole 16-byte chunks on 16-byte boundaries.
bool aligned(const fx_norm_args* a) {
  uintptr_t m = (uintptr_t)a->width * (a->dtype == FX_F32 ? 4 : 2);
  for (const void* p : {a->x, a->f, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->pre_bias,
                        (const void*)a->r, (const void*)a->z, a->grad_r, a->grad_z, (const void*)a->dx,
                        (const void*)a->df})
    m |= reinterpret_cast<uintptr_t>(p);
  if (a->gate_mode == FX_GATE_FULL || a->gate_mode == FX_GATE_GROUP)
    m |= reinterpret_cast<uintptr_t>(a->gate) | reinterpret_cast<uintptr_t>(a->dgate);
  return m % 16 == 0;
}

template <typename T, int NV, bool ALIGNED, bool WIDE>
int launch(cudaStream_t s, const NormArgs& A, const Shape& h, int grid, bool grad) {
  const size_t slots = grad ? NormRing<T, NV, ALIGNED, WIDE, 5>::kThreadBytes : NormRing<T, NV, ALIGNED, WIDE, 3>::kThreadBytes;
  const size_t sums = grad && !WIDE ? (size_t)(kNormThreads / 32) * sizeof(float) : 0;  // an entry of the width
  const size_t smem = h.threads * slots + A.W * sums;
  // a row of up to 512 threads, or of up to a warp's chunks in a block of kNormThreads
  const size_t most = WIDE ? 512 * slots : kNormThreads * slots + 32 * (16 / sizeof(T)) * sums;
  auto kern = !grad     ? norm_fwd_kernel<T, NV, ALIGNED, WIDE>
              : A.layer ? norm_bwd_kernel<T, NV, ALIGNED, WIDE, true>
                        : norm_bwd_kernel<T, NV, ALIGNED, WIDE, false>;
  if (raise_smem(kern, smem, most)) return FX_ERR_CUDA;
  kern<<<grid, h.threads, smem, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

// Several chunks a thread only where more than 512 threads were needed, a block to a row.
template <typename T>
int dispatch_type(cudaStream_t s, const NormArgs& A, const Shape& h, int grid, bool grad, bool al) {
  if (h.chunks == 1 && h.tpr <= 32)
    return al ? launch<T, 1, true, false>(s, A, h, grid, grad) : launch<T, 1, false, false>(s, A, h, grid, grad);
  if (h.chunks == 1)
    return al ? launch<T, 1, true, true>(s, A, h, grid, grad) : launch<T, 1, false, true>(s, A, h, grid, grad);
  if (h.chunks == 2)
    return al ? launch<T, 2, true, true>(s, A, h, grid, grad) : launch<T, 2, false, true>(s, A, h, grid, grad);
  if constexpr (sizeof(T) == 4)
    return al ? launch<T, 4, true, true>(s, A, h, grid, grad) : launch<T, 4, false, true>(s, A, h, grid, grad);
  return FX_ERR_SHAPE;
}

int dispatch(cudaStream_t s, const fx_norm_args* a, const NormArgs& A, const Shape& h, int grid, bool grad) {
  return a->dtype == FX_F32 ? dispatch_type<float>(s, A, h, grid, grad, aligned(a))
                            : dispatch_type<bf16>(s, A, h, grid, grad, aligned(a));
}

}  // namespace

extern "C" {

int fermix_residual_norm(void* stream, const fx_norm_args* a) {
  const int e = check(a);
  if (e) return e;
  const int64_t N = a->groups * a->rows;
  if (N == 0) return FX_OK;
  if (!a->x || !a->f || !a->post_weight || !a->pre_weight || !a->r || !a->z ||
      (a->gate_mode != FX_GATE_NONE && !a->gate))
    return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  const Shape h = shape_of(a);
  NormArgs A = make(a, h);
  int grid;
  split(a, h, D->sms, false, grid, A.per);
  return dispatch(static_cast<cudaStream_t>(stream), a, A, h, grid, false);
}

size_t fermix_residual_norm_grad_workspace_bytes(const fx_norm_args* a) {
  const DevInfo* D = dev_info();
  if (check(a) || !D || a->groups * a->rows == 0) return 0;
  const Shape h = shape_of(a);
  int grid;
  int64_t per;
  split(a, h, D->sms, true, grid, per);
  return part_bytes(a, grid) + gpart_bytes(a, grid) + 256;
}

int fermix_residual_norm_grad(void* stream, const fx_norm_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  const int64_t N = a->groups * a->rows;
  if (!a->dpost_weight || !a->dpre_weight || (a->post_bias && !a->dpost_bias) || (a->pre_bias && !a->dpre_bias) ||
      (a->scale && !a->dscale) || (a->gate_mode != FX_GATE_NONE && a->gate && !a->dgate))
    return FX_ERR_NULL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t size = a->dtype == FX_F32 ? 4 : 2;
  void* outs[5] = {a->dpost_weight, a->post_bias ? a->dpost_bias : nullptr, a->dpre_weight,
                   a->pre_bias ? a->dpre_bias : nullptr, a->scale ? a->dscale : nullptr};
  if (N == 0) {
    for (void* p : outs)
      if (p && cudaMemsetAsync(p, 0, (size_t)a->width * size, s) != cudaSuccess) return FX_ERR_CUDA;
    if (a->gate_mode == FX_GATE_GROUP && a->groups > 0 &&
        cudaMemsetAsync(a->dgate, 0, (size_t)(a->groups * a->width) * (a->dgate_f32 ? 4 : size), s) != cudaSuccess)
      return FX_ERR_CUDA;
    return FX_OK;
  }
  if (!a->x || !a->f || !a->post_weight || !a->pre_weight || !a->dx || !a->df ||
      (a->gate_mode != FX_GATE_NONE && !a->gate))
    return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  const Shape h = shape_of(a);
  int grid;
  int64_t per;
  split(a, h, D->sms, true, grid, per);
  if (!ws || wsb < part_bytes(a, grid) + gpart_bytes(a, grid) + 256) return FX_ERR_WORKSPACE;
  NormArgs A = make(a, h);
  A.per = per;
  A.part = reinterpret_cast<float*>(align256(reinterpret_cast<uintptr_t>(ws)));
  A.gpart = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(A.part) + part_bytes(a, grid));
  const int st = dispatch(s, a, A, h, grid, true);
  if (st) return st;
  NormFinish F{};
  F.part = A.part;
  F.gpart = A.gpart;
  F.pw = a->post_weight;
  F.pb = a->post_bias;
  F.scale = a->scale;
  F.dpw = outs[0];
  F.dpb = outs[1];
  F.drw = outs[2];
  F.drb = outs[3];
  F.dscale = outs[4];
  F.dgate = a->dgate;
  F.groups = a->gate_mode == FX_GATE_GROUP ? a->groups : 0;
  F.R = a->rows;
  F.per = per;
  F.blocks = grid;
  F.dgate_f32 = a->dgate_f32 != 0;
  F.W = (int)a->width;
  F.cols = (F.W + 31) / 32;
  const int64_t blocks = (int64_t)2 * F.cols + (F.groups * a->width + 1023) / 1024;
  if (blocks > INT32_MAX) return FX_ERR_SHAPE;
  if (a->dtype == FX_F32) norm_finish_kernel<float><<<(unsigned)blocks, 1024, 0, s>>>(F);
  else norm_finish_kernel<bf16><<<(unsigned)blocks, 1024, 0, s>>>(F);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

}  // extern "C"
