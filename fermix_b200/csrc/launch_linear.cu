// The linear map with its epilogue (linear_tc.cuh): checks, launch shapes, workspace.
#include "block_host.cuh"
#include "linear_tc.cuh"
#include "tensor_map.cuh"

namespace {

using namespace fxh;

int check(const fx_linear_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->activation < FX_ACT_NONE || a->activation > FX_ACT_TANH || a->rows < 0 || a->rows >= 1 << 30 ||
      a->inner < 1 || a->inner >= 1 << 30 || a->outer < 1 || a->outer >= 1 << 30 || a->x_stride < 0 ||
      a->weight_stride < 0 || a->residual_stride < 0 || a->dy_stride < 0)
    return FX_ERR_SHAPE;
  return FX_OK;
}

// A matrix as the tensor maps take it: (planes, rows, ld) of bfloat16.
struct Operand {
  const void* p;
  int64_t rows, cols, ld;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether a matrix of the type can be read in 16-byte pieces.
bool aligned(const void* p, int64_t stride, int64_t rows, int64_t cols, int size) {
  return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(cols * size) | (uintptr_t)(rows > 1 ? stride * size : 0)) % 16 == 0;
}
// bfloat16 rows that a tensor map can read in place (a row of zero stride is one row to it).
bool mappable(const void* p, int64_t stride, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(rows > 1 ? stride * 2 : 0)) % 16 == 0 && (rows == 1 || stride > 0) &&
         stride < (int64_t{1} << 38);
}

// How a product of rows x cols over `inner` is cut: tiles of a pair of SMs, as many whole rounds of them as there
// are, and the rest split along k so that it fills the device once. A part has four blocks of k at least, and
// after a whole round it has to save eight blocks' time (three in float32, whose blocks have six products),
// about what the join costs.
struct Cut {
  int64_t rows, cols;
  int blocks, tm, tn, whole, splits, per;
  int64_t units() const { return whole + ((int64_t)tm * tn - whole) * splits; }
  int64_t joined() const { return splits > 1 ? (int64_t)tm * tn - whole : 0; }
  size_t part_bytes() const { return (size_t)joined() * splits * (lin::kTile * lin::kTile * sizeof(float)); }
};

Cut cut_of(int64_t rows, int64_t cols, int64_t inner, bool f32, int sms) {
  Cut C;
  C.rows = rows;
  C.cols = cols;
  C.blocks = (int)ceil_div(inner, lin::kBlockK);
  C.tm = (int)ceil_div(rows, lin::kTile);
  C.tn = (int)ceil_div(cols, lin::kTile);
  const int64_t tiles = (int64_t)C.tm * C.tn, pairs = sms / 2, rest = tiles % pairs;
  C.whole = (int)tiles;
  C.splits = 1;
  C.per = C.blocks;
  int64_t splits = rest ? pairs / rest : 1;
  if (splits > C.blocks / 4) splits = C.blocks / 4;
  if (splits > 1) {
    const int64_t per = ceil_div(C.blocks, splits);
    if (tiles < pairs || C.blocks - per >= (f32 ? 3 : 8)) {
      C.whole = (int)(tiles - rest);
      C.per = (int)per;
      C.splits = (int)ceil_div(C.blocks, per);
    }
  }
  return C;
}

// The plan of a call: which operands are laid out anew, and where.
struct Space {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += align256(n);
    return at;
  }
};
int64_t ld_of(int64_t cols) { return (cols + 7) / 8 * 8; }
size_t parts_bytes(int64_t rows, int64_t cols, int planes) { return (size_t)planes * rows * ld_of(cols) * 2; }

struct LinPlan {
  bool f32;
  int planes;
  bool new_x, new_w, new_g, slope;  // laid out anew
  size_t x = 0, w = 0, g = 0, sums = 0, part = 0, bytes = 0;
  Cut y, dx, dw;
  // the pass over dy: blocks of rows, rows of a block, threads of a row
  int64_t per = 0;
  int blocks = 0, tpr = 0;
};

LinPlan plan_fwd(const fx_linear_args* a, int sms) {
  LinPlan P{};
  P.f32 = a->dtype == FX_F32;
  P.planes = P.f32 ? 3 : 1;
  P.new_x = P.f32 || !mappable(a->x, a->x_stride, a->rows);
  P.new_w = P.f32 || !mappable(a->weight, a->weight_stride, a->outer);
  P.y = cut_of(a->rows, a->outer, a->inner, P.f32, sms);
  Space S;
  if (P.new_x) P.x = S.take(parts_bytes(a->rows, a->inner, P.planes));
  if (P.new_w) P.w = S.take(parts_bytes(a->outer, a->inner, P.planes));
  P.part = S.take(P.y.part_bytes());
  P.bytes = S.bytes ? S.bytes + 256 : 0;
  return P;
}

LinPlan plan_bwd(const fx_linear_args* a, int sms) {
  LinPlan P{};
  P.f32 = a->dtype == FX_F32;
  P.planes = P.f32 ? 3 : 1;
  P.slope = a->activation != FX_ACT_NONE;
  const bool products = a->dx || a->dweight;
  P.new_x = a->dweight && (P.f32 || !mappable(a->x, a->x_stride, a->rows));
  P.new_w = a->dx && (P.f32 || !mappable(a->weight, a->weight_stride, a->outer));
  P.new_g = products && (P.f32 || P.slope || !mappable(a->dy, a->dy_stride, a->rows));
  P.tpr = 1;
  while (P.tpr < 32 && P.tpr * 8 < a->outer) P.tpr *= 2;
  const int64_t groups = 256 / P.tpr, strips = ceil_div(a->outer, P.tpr * 8);
  // eight blocks an SM, of four rows a thread at least
  int64_t blocks = ceil_div((int64_t)sms * 8, strips);
  if (blocks > ceil_div(a->rows, groups * 4)) blocks = ceil_div(a->rows, groups * 4);
  P.per = ceil_div(a->rows, blocks);
  P.blocks = (int)ceil_div(a->rows, P.per);
  P.dx = cut_of(a->rows, a->inner, a->outer, P.f32, sms);
  P.dw = cut_of(a->outer, a->inner, a->rows, P.f32, sms);
  Space S;
  if (P.new_x) P.x = S.take(parts_bytes(a->rows, a->inner, P.planes));
  if (P.new_w) P.w = S.take(parts_bytes(a->outer, a->inner, P.planes));
  if (P.new_g) P.g = S.take(parts_bytes(a->rows, a->outer, P.planes));
  if (a->dbias) P.sums = S.take((size_t)P.blocks * a->outer * sizeof(float));
  const size_t p = a->dx ? P.dx.part_bytes() : 0, q = a->dweight ? P.dw.part_bytes() : 0;
  P.part = S.take(p > q ? p : q);
  P.bytes = S.bytes ? S.bytes + 256 : 0;
  return P;
}

// The map of a matrix: boxes of 64 entries by 128 rows (K-major), 64 by 64 (MN-major).
int make_map(CUtensorMap* m, const Operand& o, int planes, bool mn) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return FX_ERR_CUDA;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)planes};
  const int64_t ld = o.rows > 1 ? o.ld : ld_of(o.cols);
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, planes > 1 ? (cuuint64_t)(o.rows * ld * 2) : (cuuint64_t)ld * 2};
  const cuuint32_t box[3] = {64, mn ? 64u : 128u, 1}, ones[3] = {1, 1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims, strides, box, ones,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? FX_OK
             : FX_ERR_CUDA;
}

// Whether y, slope, the residual and the bias are rows of whole 16-byte pieces.
bool pieces(const Epilogue& e, int64_t rows, int64_t cols, int size) {
  const uintptr_t m = reinterpret_cast<uintptr_t>(e.y) | reinterpret_cast<uintptr_t>(e.slope) |
                      reinterpret_cast<uintptr_t>(e.residual) | reinterpret_cast<uintptr_t>(e.bias) |
                      (uintptr_t)(e.residual && rows > 1 ? e.rs * size : 0) | (uintptr_t)(cols * size);
  return m % 16 == 0;
}

template <typename T, int NP, int ACT>
int launch(cudaStream_t s, const lin::Args& G, const lin::Maps& M, int64_t pairs, int64_t joined) {
  constexpr size_t smem = lin::Shape<NP>::kSmem;
  auto kern = lin::linear_tc_kernel<T, NP, ACT>;
  if (raise_smem(kern, smem, smem)) return FX_ERR_CUDA;
  kern<<<(unsigned)(2 * pairs), lin::kThreads, smem, s>>>(G, M);
  if (joined) {  // 74 tiles at most, 256 blocks each
    constexpr int N = 16 / sizeof(T);
    if (G.vec) lin::linear_join_kernel<T, ACT, N><<<(unsigned)(joined * (256 / N)), 256, 0, s>>>(G);
    else lin::linear_join_kernel<T, ACT, 1><<<(unsigned)(joined * 256), 256, 0, s>>>(G);
  }
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <typename T, int NP>
int product(cudaStream_t s, const Cut& C, const Operand& a, bool a_mn, const Operand& b, bool b_mn, const Epilogue& e,
            float* part, int sms) {
  lin::Maps M;
  int st = make_map(&M.a, a, NP, a_mn);
  if (!st) st = make_map(&M.b, b, NP, b_mn);
  if (st) return st;
  if ((int64_t)C.tm * C.tn > INT32_MAX / 2) return FX_ERR_SHAPE;
  lin::Args G{};
  G.rows = C.rows;
  G.cols = C.cols;
  G.blocks = C.blocks;
  G.tm = C.tm;
  G.tn = C.tn;
  G.whole = C.whole;
  G.splits = C.splits;
  G.per = C.per;
  G.a_mn = a_mn;
  G.b_mn = b_mn;
  G.vec = pieces(e, C.rows, C.cols, sizeof(T));
  G.polls = wait_polls();
  G.part = part;
  G.e = e;
  const int64_t pairs = C.units() < sms / 2 ? C.units() : sms / 2;
  switch (e.act) {
    case FX_ACT_RELU: return launch<T, NP, FX_ACT_RELU>(s, G, M, pairs, C.joined());
    case FX_ACT_SILU: return launch<T, NP, FX_ACT_SILU>(s, G, M, pairs, C.joined());
    case FX_ACT_GELU: return launch<T, NP, FX_ACT_GELU>(s, G, M, pairs, C.joined());
    case FX_ACT_GELU_TANH: return launch<T, NP, FX_ACT_GELU_TANH>(s, G, M, pairs, C.joined());
    case FX_ACT_TANH: return launch<T, NP, FX_ACT_TANH>(s, G, M, pairs, C.joined());
    default: return launch<T, NP, FX_ACT_NONE>(s, G, M, pairs, C.joined());
  }
}

template <typename T, int NP>
int layout(cudaStream_t s, const void* src, int64_t stride, int64_t rows, int64_t cols, void* out, int sms) {
  lin::PartsArgs A{src, stride, rows, cols, ld_of(cols), static_cast<uint16_t*>(out),
                   aligned(src, stride, rows, cols, sizeof(T))};
  const int64_t blocks = ceil_div(rows * (A.ld / 8), 256), most = (int64_t)sms * 8;
  lin::linear_parts_kernel<T, NP><<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

// The operand in place, or laid out anew at `out`.
template <typename T, int NP>
int operand(cudaStream_t s, bool anew, const void* p, int64_t stride, int64_t rows, int64_t cols, void* out, int sms,
            Operand& o) {
  o = {anew ? out : p, rows, cols, anew ? ld_of(cols) : stride};
  return anew ? layout<T, NP>(s, p, stride, rows, cols, out, sms) : FX_OK;
}

template <typename T, int NP>
int forward(cudaStream_t s, const fx_linear_args* a, const LinPlan& P, unsigned char* ws, int sms) {
  Operand x, w;
  int st = operand<T, NP>(s, P.new_x, a->x, a->x_stride, a->rows, a->inner, ws + P.x, sms, x);
  if (!st) st = operand<T, NP>(s, P.new_w, a->weight, a->weight_stride, a->outer, a->inner, ws + P.w, sms, w);
  if (st) return st;
  const Epilogue e{a->activation, a->bias, a->residual, a->residual_stride, a->y, a->slope};
  return product<T, NP>(s, P.y, x, false, w, false, e, reinterpret_cast<float*>(ws + P.part), sms);
}

template <typename T, int NP>
int backward(cudaStream_t s, const fx_linear_args* a, const LinPlan& P, unsigned char* ws, int sms) {
  Operand g{a->dy, a->rows, a->outer, a->dy_stride};
  if (P.new_g || a->dbias) {
    const void* slope = P.slope ? a->slope : nullptr;
    const int64_t ld = ld_of(a->outer);
    lin::SlopeArgs A{a->dy, slope, a->dy_stride, a->rows, a->outer, ld, P.per,
                     P.new_g ? reinterpret_cast<uint16_t*>(ws + P.g) : nullptr,
                     a->dbias ? reinterpret_cast<float*>(ws + P.sums) : nullptr, P.tpr,
                     aligned(a->dy, a->dy_stride, a->rows, a->outer, sizeof(T)) &&
                         reinterpret_cast<uintptr_t>(slope) % 16 == 0};
    const dim3 grid((unsigned)ceil_div(a->outer, P.tpr * 8), (unsigned)P.blocks);
    lin::linear_slope_kernel<T, NP><<<grid, 256, 0, s>>>(A);
    if (a->dbias) lin::linear_bias_kernel<T><<<(unsigned)ceil_div(a->outer, 32), 256, 0, s>>>(A.sums, P.blocks, a->outer, a->dbias);
    if (cudaGetLastError() != cudaSuccess) return FX_ERR_CUDA;
    if (P.new_g) g = {A.out, a->rows, a->outer, ld};
  }
  float* part = reinterpret_cast<float*>(ws + P.part);
  if (a->dx) {
    Operand w;
    int st = operand<T, NP>(s, P.new_w, a->weight, a->weight_stride, a->outer, a->inner, ws + P.w, sms, w);
    const Epilogue e{FX_ACT_NONE, nullptr, nullptr, 0, a->dx, nullptr};
    if (!st) st = product<T, NP>(s, P.dx, g, false, w, true, e, part, sms);
    if (st) return st;
  }
  if (a->dweight) {
    Operand x;
    int st = operand<T, NP>(s, P.new_x, a->x, a->x_stride, a->rows, a->inner, ws + P.x, sms, x);
    const Epilogue e{FX_ACT_NONE, nullptr, nullptr, 0, a->dweight, nullptr};
    if (!st) st = product<T, NP>(s, P.dw, g, true, x, true, e, part, sms);
    if (st) return st;
  }
  return FX_OK;
}

unsigned char* base_of(void* ws) { return reinterpret_cast<unsigned char*>(align256(reinterpret_cast<uintptr_t>(ws))); }

}  // namespace

namespace fxh {

int linear_status(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, fx::umma::fx_status_word, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int z = 0;
    if (cudaMemcpyToSymbol(fx::umma::fx_status_word, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace fxh

extern "C" {

size_t fermix_linear_workspace_bytes(const fx_linear_args* a) {
  const DevInfo* D = dev_info();
  return check(a) || !D || a->rows == 0 ? 0 : plan_fwd(a, D->sms).bytes;
}

int fermix_linear(void* stream, const fx_linear_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  if (a->rows == 0) return FX_OK;
  if (!a->x || !a->weight || !a->y) return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  const LinPlan P = plan_fwd(a, D->sms);
  if (P.bytes && (!ws || wsb < P.bytes)) return FX_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return P.f32 ? forward<float, 3>(s, a, P, base_of(ws), D->sms) : forward<bf16, 1>(s, a, P, base_of(ws), D->sms);
}

size_t fermix_linear_grad_workspace_bytes(const fx_linear_args* a) {
  const DevInfo* D = dev_info();
  return check(a) || !D || a->rows == 0 ? 0 : plan_bwd(a, D->sms).bytes;
}

int fermix_linear_grad(void* stream, const fx_linear_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t size = a->dtype == FX_F32 ? 4 : 2;
  if (a->rows == 0) {
    if (a->dweight && cudaMemsetAsync(a->dweight, 0, (size_t)(a->outer * a->inner) * size, s) != cudaSuccess)
      return FX_ERR_CUDA;
    if (a->dbias && cudaMemsetAsync(a->dbias, 0, (size_t)a->outer * size, s) != cudaSuccess) return FX_ERR_CUDA;
    return FX_OK;
  }
  if (!a->dy || (a->dx && !a->weight) || (a->dweight && !a->x) || (a->activation != FX_ACT_NONE && !a->slope))
    return FX_ERR_NULL;
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  const LinPlan P = plan_bwd(a, D->sms);
  if (P.bytes && (!ws || wsb < P.bytes)) return FX_ERR_WORKSPACE;
  return P.f32 ? backward<float, 3>(s, a, P, base_of(ws), D->sms) : backward<bf16, 1>(s, a, P, base_of(ws), D->sms);
}

}  // extern "C"
