// The linear map with its epilogue (linear_tc.cuh): checks, launch shapes, workspace.
#include "linear_rows.cuh"
#include "linear_tc.cuh"
#include "tensor_map.cuh"
#include "token_host.cuh"

namespace {

using namespace fxh;

int check(const fx_linear_args* a) {
  if (!a) return FX_ERR_NULL;
  if (a->dtype != FX_F32 && a->dtype != FX_BF16) return FX_ERR_DTYPE;
  if (a->activation < FX_ACT_NONE || a->activation > FX_ACT_TANH || a->rows < 0 || a->rows >= 1 << 30 ||
      a->inner < 1 || a->inner >= 1 << 30 || a->outer < 1 || a->outer >= 1 << 30 || a->x_stride < 0 ||
      a->weight_stride < 0 || a->residual_stride < 0 || a->dy_stride < 0)
    return FX_ERR_SHAPE;
  // the tiles of each product are counted in 32 bits
  const int64_t m = a->rows / 256 + 1, k = a->inner / 256 + 1, n = a->outer / 256 + 1, most = int64_t{1} << 28;
  return m * n > most || m * k > most || n * k > most ? FX_ERR_SHAPE : FX_OK;
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
// bfloat16 rows that a tensor map can read in place. Its rows do not share entries: those of a broadcast (stride 0) or of
// overlapping windows are laid out anew. A query of the workspace may leave the pointer out: the form that needs more.
bool mappable(const void* p, int64_t stride, int64_t rows, int64_t cols) {
  return p && (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(rows > 1 ? stride * 2 : 0)) % 16 == 0 && (rows == 1 || stride >= cols) &&
         stride < (int64_t{1} << 38);
}

// How a product of rows x cols over `inner` is cut into a launch's units.
struct Cut {
  int64_t rows, cols;
  int blocks, tm, tn, whole, splits, per;
  int tiles() const { return tm * tn; }
  int joined() const { return tiles() - whole; }
  int units() const { return whole + joined() * splits; }
  size_t part_bytes() const { return (size_t)joined() * splits * (lin::kTile * lin::kTile * sizeof(float)); }
  // the last n tiles in parts of `most` blocks of k at most
  void split(int n, int most) {
    whole = tiles() - n;
    splits = (blocks + most - 1) / most;
    per = (blocks + splits - 1) / splits;
    splits = (blocks + per - 1) / per;
    if (splits == 1) whole = tiles();
  }
};

Cut whole_of(int64_t rows, int64_t cols, int64_t inner) {
  Cut C;
  C.rows = rows;
  C.cols = cols;
  C.blocks = (int)ceil_div(inner, lin::kBlockK);
  C.tm = (int)ceil_div(rows, lin::kTile);
  C.tn = (int)ceil_div(cols, lin::kTile);
  C.whole = C.tiles();
  C.splits = 1;
  C.per = C.blocks;
  return C;
}

// How a launch's n products are cut and ordered (c[0]'s units are the long ones); `ahead` as in lin::Group.
// - Where the tiles do not fill the device once, k is split so that the parts do, four blocks at least each (two in
//   float32).
// - Of one product, the tiles after the whole rounds are split alike, if that saves the time of eight blocks (three in
//   float32, whose blocks have six products), about what the join costs.
// - Of two products, the one with the longer tiles is split where a tile takes longer than a pair's share of the work.
// Measured, us, without and with: 8192 x 8192 -> 2048 bfloat16 (256 tiles of 128 blocks on 74 pairs) 217 and 200.
int cut(Cut* c, int n, bool f32, int sms) {
  const int pairs = sms / 2, least = f32 ? 2 : 4;
  if (n == 2 && c[1].blocks > c[0].blocks) {
    const Cut t = c[0];
    c[0] = c[1];
    c[1] = t;
  }
  int64_t tiles = 0, work = 0;
  for (int i = 0; i < n; ++i) {
    tiles += c[i].tiles();
    work += (int64_t)c[i].tiles() * c[i].blocks;
  }
  // the shortest parts of the first m products with which their units fit one round
  const auto fit = [&](int m, int64_t most) {
    for (;; most += 1 + most / 32) {
      int64_t units = 0;
      for (int i = 0; i < m; ++i) units += c[i].tiles() * ceil_div(c[i].blocks, most);
      if (units <= pairs) break;
    }
    for (int i = 0; i < m; ++i) c[i].split(c[i].tiles(), (int)(most < c[i].blocks ? most : c[i].blocks));
  };
  const int64_t share = work / pairs > least ? work / pairs : least;
  if (tiles < pairs) {
    fit(n, share);
  } else if (n == 1) {
    const int rest = (int)(tiles % pairs);
    if (rest) {
      const int most = (int)ceil_div(c[0].blocks, pairs / rest);
      if (most >= least && c[0].blocks - most >= (f32 ? 3 : 8)) c[0].split(rest, most);
    }
  } else if (c[0].blocks > share && c[0].tiles() <= pairs) {
    fit(1, share);
  }
  if (n == 1) return 0;
  // the rounds of short units, beside the last of the long ones, that end the launch soonest
  const int64_t longs = c[0].units(), shorts = c[1].units(), l = c[0].per, t = c[1].per, rounds = longs / pairs,
                rest = longs % pairs;
  int best = 0;
  int64_t end = INT64_MAX;
  for (int ahead = 0; ahead <= (rest ? l / t + 1 : 0); ++ahead) {
    const int64_t left = shorts - ahead * (pairs - rest), more = left > 0 ? ceil_div(left, pairs) : 0;
    const int64_t a = rest ? (rounds + 1) * l + more * t : 0, b = rounds * l + (ahead + more) * t;
    if ((a > b ? a : b) < end) {
      end = a > b ? a : b;
      best = ahead;
    }
  }
  return best;
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
  Cut c[2];
  int products = 0, ahead = 0, dx = 0, dw = 0;  // where dx and dW are among them
  // the pass over dy: blocks of rows, rows of a block, threads of a row
  int64_t per = 0;
  int blocks = 0, tpr = 0;

  size_t part_bytes() const {
    size_t n = 0;
    for (int i = 0; i < products; ++i) n += c[i].part_bytes();
    return n;
  }
};

// Blocks of 16 outputs and eight warps while there is at most one an SM, of 32 and four warps above (float32; us: 1000 x
// 4096 x 32 23 and 41, 100000 x 264 x 32 150 and 80). Between, blocks of 32 leave SMs idle: 4096 x 8192 x 32 76.
bool few_blocks(int64_t narrow, int64_t wide, int sms) { return ceil_div(wide, 16) * ceil_div(narrow, 32) <= sms; }

// Whether the rows' kernel (linear_rows.cuh), which needs no layout, takes the call. In bfloat16 few rows, which are bound
// by the weights' bytes; measured, us, against the tiles of the tensor cores at 8192 -> 4096: 32 rows 24 and 27, 64 rows
// 52 and 26. (Rows off the 16-byte boundaries come without the ring of copies: 32 x 8191 -> 4096 76 us.)
// In float32 the tiles' launches cost about 20 us, and their layout reads and writes an operand four times as much; the
// rows' kernel costs the products of its slower instructions. Both are estimated, us, from times between 100 and 100000
// of `wide`, 4 and 512 of `narrow` and 32 and 4096 of `inner`. Measured, us, rows and tiles, wide x inner x narrow: 300 x
// 64 x 100 8 and 16, 300 x 4096 x 32 23 and 27, 129 x 5847 x 30 55 and 27, 4700 x 264 x 64 14 and 27, 4700 x 4096 x 64 61
// and 98, 10000 x 264 x 100 35 and 31, 1000 x 1024 x 256 23 and 25, 1000 x 1024 x 512 37 and 27, 100000 x 1024 x 16 96 and
// 354.
bool by_rows(const fx_linear_args* a, int sms) {
  if (a->dtype != FX_F32) return a->rows <= 32;
  const int64_t narrow = a->rows < a->outer ? a->rows : a->outer, wide = a->rows < a->outer ? a->outer : a->rows;
  const double part = narrow <= 16 ? 0.6 : 1, tiles = (a->inner < 128 ? 17 : 21) + 4.4e-6 * (double)a->inner * (double)(wide + narrow);
  // rows off the 16-byte boundaries are loaded entry by entry, and not ahead: 79 x 3158 x 1468 53 and 41
  const double k = (double)a->inner * ((a->x_stride | a->weight_stride | a->inner) % 4 ? 1.6 : 1);
  if (few_blocks(narrow, wide, sms)) return 7 + part * 0.004 * k < tiles;
  const double waves = (double)ceil_div(ceil_div(wide, 32) * ceil_div(narrow, 32), sms);
  const double one = 2.3 + 0.0085 * k, more = waves * (2.3 + 0.0055 * k);
  return 7 + part * (one > more ? one : more) < tiles;
}

template <typename T, int NP, int MT, int NT, int WARPS>
int rows_launch(cudaStream_t s, const lin::RowArgs& A, bool al) {
  const dim3 blocks((unsigned)ceil_div(A.outer, 16 * MT), (unsigned)ceil_div(A.rows, 8 * NT));
  constexpr size_t smem = lin::RowRing<T, MT, NT, WARPS>::kSmem;
  auto kern = al ? lin::linear_rows_kernel<T, NP, MT, NT, WARPS, true> : lin::linear_rows_kernel<T, NP, MT, NT, WARPS, false>;
  if (raise_smem(kern, smem, smem)) return FX_ERR_CUDA;
  kern<<<blocks, WARPS * 32, smem, s>>>(A);
  return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
}

template <typename T, int NP>
int rows_forward(cudaStream_t s, const fx_linear_args* a, int sms) {
  lin::RowArgs A{a->x, a->weight, a->x_stride, a->weight_stride, (int)a->rows, (int)a->inner, (int)a->outer, false,
                 {a->activation, a->bias, a->residual, a->residual_stride, a->y, a->slope}};
  if (NP > 1 && a->outer < a->rows) {
    A.x = a->weight;
    A.w = a->x;
    A.xs = a->weight_stride;
    A.ws = a->x_stride;
    A.rows = (int)a->outer;
    A.outer = (int)a->rows;
    A.swapped = true;
  }
  const bool al = aligned(A.x, A.xs, A.rows, A.inner, sizeof(T)) && aligned(A.w, A.ws, A.outer, A.inner, sizeof(T));
  if constexpr (NP == 1) {
    if (A.rows <= 8) return rows_launch<T, NP, 1, 1, 8>(s, A, al);
    if (A.rows <= 16) return rows_launch<T, NP, 1, 2, 8>(s, A, al);
    return rows_launch<T, NP, 2, 4, 16>(s, A, al);
  } else if (few_blocks(A.rows, A.outer, sms)) {
    if (A.rows <= 8) return rows_launch<T, NP, 1, 1, 8>(s, A, al);
    if (A.rows <= 16) return rows_launch<T, NP, 1, 2, 8>(s, A, al);
    return rows_launch<T, NP, 1, 4, 8>(s, A, al);
  } else {
    if (A.rows <= 8) return rows_launch<T, NP, 2, 1, 4>(s, A, al);
    // off the boundaries 32 outputs by 16 rows are slow (100000 x 263 x 16 117 us, of 16 outputs 74)
    if (A.rows <= 16) return al ? rows_launch<T, NP, 2, 2, 4>(s, A, al) : rows_launch<T, NP, 1, 2, 8>(s, A, al);
    return rows_launch<T, NP, 2, 4, 4>(s, A, al);
  }
}

LinPlan plan_fwd(const fx_linear_args* a, int sms) {
  LinPlan P{};
  P.f32 = a->dtype == FX_F32;
  P.planes = P.f32 ? 3 : 1;
  P.new_x = P.f32 || !mappable(a->x, a->x_stride, a->rows, a->inner);
  P.new_w = P.f32 || !mappable(a->weight, a->weight_stride, a->outer, a->inner);
  P.c[P.products++] = whole_of(a->rows, a->outer, a->inner);
  P.ahead = cut(P.c, 1, P.f32, sms);
  Space S;
  if (P.new_x) P.x = S.take(parts_bytes(a->rows, a->inner, P.planes));
  if (P.new_w) P.w = S.take(parts_bytes(a->outer, a->inner, P.planes));
  P.part = S.take(P.part_bytes());
  P.bytes = S.bytes ? S.bytes + 256 : 0;
  return P;
}

LinPlan plan_bwd(const fx_linear_args* a, int sms) {
  LinPlan P{};
  P.f32 = a->dtype == FX_F32;
  P.planes = P.f32 ? 3 : 1;
  P.slope = a->activation != FX_ACT_NONE;
  P.new_x = a->dweight && (P.f32 || !mappable(a->x, a->x_stride, a->rows, a->inner));
  P.new_w = a->dx && (P.f32 || !mappable(a->weight, a->weight_stride, a->outer, a->inner));
  P.new_g = (a->dx || a->dweight) && (P.f32 || P.slope || !mappable(a->dy, a->dy_stride, a->rows, a->outer));
  P.tpr = 1;
  while (P.tpr < 32 && P.tpr * 8 < a->outer) P.tpr *= 2;
  const int64_t groups = 256 / P.tpr, strips = ceil_div(a->outer, P.tpr * 8);
  // as many blocks as an SM holds, of four rows a thread at least
  int64_t blocks = (int64_t)sms * lin::kPrepBlocks / strips;
  if (blocks < 1) blocks = 1;
  if (blocks > ceil_div(a->rows, groups * 4)) blocks = ceil_div(a->rows, groups * 4);
  P.per = ceil_div(a->rows, blocks);
  P.blocks = (int)ceil_div(a->rows, P.per);
  if (a->dx) P.c[P.products++] = whole_of(a->rows, a->inner, a->outer);
  if (a->dweight) P.c[P.products++] = whole_of(a->outer, a->inner, a->rows);
  if (P.products) P.ahead = cut(P.c, P.products, P.f32, sms);
  if (P.products == 2) (ceil_div(a->rows, lin::kBlockK) > ceil_div(a->outer, lin::kBlockK) ? P.dx : P.dw) = 1;
  Space S;
  if (P.new_x) P.x = S.take(parts_bytes(a->rows, a->inner, P.planes));
  if (P.new_w) P.w = S.take(parts_bytes(a->outer, a->inner, P.planes));
  if (P.new_g) P.g = S.take(parts_bytes(a->rows, a->outer, P.planes));
  if (a->dbias) P.sums = S.take((size_t)P.blocks * a->outer * sizeof(float));
  P.part = S.take(P.part_bytes());
  P.bytes = S.bytes ? S.bytes + 256 : 0;
  return P;
}

// The map of a matrix: boxes of 64 entries by 128 rows (K-major), 64 by 64 (MN-major).
int make_map(CUtensorMap* m, const Operand& o, int planes, bool mn) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return FX_ERR_CUDA;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)planes};
  const int64_t ld = o.rows > 1 ? o.ld : ld_of(o.cols);
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(o.rows * ld * 2)};
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

// The products of a call, gathered for one launch.
template <typename T, int NP>
struct Products {
  const LinPlan& P;
  lin::Group G{};
  lin::Maps M;
  float* parts;

  Products(const LinPlan& P, unsigned char* ws) : P(P), parts(reinterpret_cast<float*>(ws + P.part)) {}
  int set(int n, const Operand& a, bool a_mn, const Operand& b, bool b_mn, const Epilogue& e) {
    const Cut& C = P.c[n];
    lin::Args& A = G.p[n];
    A.rows = C.rows;
    A.cols = C.cols;
    A.blocks = C.blocks;
    A.tm = C.tm;
    A.tn = C.tn;
    A.whole = C.whole;
    A.splits = C.splits;
    A.per = C.per;
    A.a_mn = a_mn;
    A.b_mn = b_mn;
    A.vec = pieces(e, C.rows, C.cols, sizeof(T));
    A.part = parts + (n ? P.c[0].part_bytes() / sizeof(float) : 0);
    A.e = e;
    int st = make_map(&M.m[2 * n], a, NP, a_mn);
    if (!st) st = make_map(&M.m[2 * n + 1], b, NP, b_mn);
    return st;
  }
  template <int ACT>
  int launch(cudaStream_t s, int sms, bool first) {
    constexpr size_t smem = lin::Shape<NP>::kSmem;
    auto kern = lin::linear_tc_kernel<T, NP, ACT>;
    if (raise_smem(kern, smem, smem)) return FX_ERR_CUDA;
    G.polls = wait_polls();
    const int units = G.p[0].units() + G.p[1].units(), pairs = units < sms / 2 ? units : sms / 2;
    G.longs = P.products == 2 ? G.p[0].units() : G.p[0].whole;
    G.shorts = units - G.longs;
    G.ahead = P.ahead;
    int st = FX_OK;
    if (!first) {
      st = launch_next(kern, 2 * pairs, lin::kThreads, smem, s, G, M);
    } else {
      kern<<<2 * pairs, lin::kThreads, smem, s>>>(G, M);
      if (cudaGetLastError() != cudaSuccess) st = FX_ERR_CUDA;
    }
    if (st) return st;
    const int joined = G.p[0].joined() + G.p[1].joined();
    if (joined) {  // tiles that are cut along k
      constexpr int N = 16 / sizeof(T);
      if (G.p[0].vec && (P.products == 1 || G.p[1].vec))
        return launch_next(lin::linear_join_kernel<T, ACT, N>, joined * (lin::kTile / N), 256, 0, s, G);
      return launch_next(lin::linear_join_kernel<T, ACT, 1>, joined * lin::kTile, 256, 0, s, G);
    }
    return FX_OK;
  }
  // `first`: nothing of this call was launched before
  int launch(cudaStream_t s, int act, int sms, bool first) {
    switch (act) {
      case FX_ACT_RELU: return launch<FX_ACT_RELU>(s, sms, first);
      case FX_ACT_SILU: return launch<FX_ACT_SILU>(s, sms, first);
      case FX_ACT_GELU: return launch<FX_ACT_GELU>(s, sms, first);
      case FX_ACT_GELU_TANH: return launch<FX_ACT_GELU_TANH>(s, sms, first);
      case FX_ACT_TANH: return launch<FX_ACT_TANH>(s, sms, first);
      default: return launch<FX_ACT_NONE>(s, sms, first);
    }
  }
};

template <typename T, int NP>
struct Prep {
  lin::PrepArgs A{};
  int n = 0, sms;

  explicit Prep(int sms) : sms(sms) {}
  // The operand in place, or laid out anew at `out`.
  Operand operand(bool anew, const void* p, int64_t stride, int64_t rows, int64_t cols, void* out) {
    if (!anew) return {p, rows, cols, stride};
    const int64_t ld = ld_of(cols), blocks = ceil_div(rows * (ld / 8), 256), most = (int64_t)sms * 8;
    A.o[n++] = {p, stride, rows, cols, ld, static_cast<uint16_t*>(out), aligned(p, stride, rows, cols, sizeof(T)),
                (int)(blocks < most ? blocks : most)};
    return {out, rows, cols, ld};
  }
  bool nothing() const { return A.g.blocks + A.o[0].blocks + A.o[1].blocks == 0; }
  int launch(cudaStream_t s) {
    if (nothing()) return FX_OK;
    const int blocks = A.g.blocks + A.o[0].blocks + A.o[1].blocks;
    lin::linear_prep_kernel<T, NP><<<blocks, 256, 0, s>>>(A);
    return cudaGetLastError() == cudaSuccess ? FX_OK : FX_ERR_CUDA;
  }
};

// A thread that has made no call yet (autograd's, on its first backward pass) has no current context, which the encoding
// of tensor maps, a driver call, needs; this runtime call brings it.
template <typename T, int NP>
int ready() {
  return raise_smem(lin::linear_tc_kernel<T, NP, FX_ACT_NONE>, lin::Shape<NP>::kSmem, lin::Shape<NP>::kSmem);
}

template <typename T, int NP>
int forward(cudaStream_t s, const fx_linear_args* a, const LinPlan& P, unsigned char* ws, int sms) {
  if (ready<T, NP>()) return FX_ERR_CUDA;
  Prep<T, NP> prep(sms);
  const Operand x = prep.operand(P.new_x, a->x, a->x_stride, a->rows, a->inner, ws + P.x);
  const Operand w = prep.operand(P.new_w, a->weight, a->weight_stride, a->outer, a->inner, ws + P.w);
  Products<T, NP> products(P, ws);
  int st = products.set(0, x, false, w, false, {a->activation, a->bias, a->residual, a->residual_stride, a->y, a->slope});
  if (!st) st = prep.launch(s);
  return st ? st : products.launch(s, a->activation, sms, prep.nothing());
}

template <typename T, int NP>
int backward(cudaStream_t s, const fx_linear_args* a, const LinPlan& P, unsigned char* ws, int sms) {
  if (ready<T, NP>()) return FX_ERR_CUDA;
  Prep<T, NP> prep(sms);
  Operand g{a->dy, a->rows, a->outer, a->dy_stride};
  if (P.new_g || a->dbias) {
    lin::PrepArgs& A = prep.A;
    A.slope = P.slope ? a->slope : nullptr;
    A.sums = a->dbias ? reinterpret_cast<float*>(ws + P.sums) : nullptr;
    A.per = P.per;
    A.tpr = P.tpr;
    const int64_t strips = ceil_div(a->outer, P.tpr * 8);
    if (strips * P.blocks > INT32_MAX / 2) return FX_ERR_SHAPE;
    A.strips = (int)strips;
    A.g = {a->dy, a->dy_stride, a->rows, a->outer, ld_of(a->outer), P.new_g ? reinterpret_cast<uint16_t*>(ws + P.g) : nullptr,
           aligned(a->dy, a->dy_stride, a->rows, a->outer, sizeof(T)) && reinterpret_cast<uintptr_t>(A.slope) % 16 == 0,
           A.strips * P.blocks};
    if (P.new_g) g = {A.g.out, a->rows, a->outer, A.g.ld};
  }
  const Epilogue none{FX_ACT_NONE, nullptr, nullptr, 0, nullptr, nullptr};
  Products<T, NP> products(P, ws);
  int st = FX_OK;
  if (a->dx) {
    const Operand w = prep.operand(P.new_w, a->weight, a->weight_stride, a->outer, a->inner, ws + P.w);
    Epilogue e = none;
    e.y = a->dx;
    st = products.set(P.dx, g, false, w, true, e);
  }
  if (!st && a->dweight) {
    const Operand x = prep.operand(P.new_x, a->x, a->x_stride, a->rows, a->inner, ws + P.x);
    Epilogue e = none;
    e.y = a->dweight;
    st = products.set(P.dw, g, true, x, true, e);
  }
  if (!st) st = prep.launch(s);
  if (st) return st;
  if (P.products) {
    products.G.sums = prep.A.sums;
    products.G.dbias = a->dbias;
    products.G.sum_blocks = P.blocks;
    products.G.sum_cols = a->outer;
    return products.launch(s, FX_ACT_NONE, sms, prep.nothing());
  }
  if (!a->dbias) return FX_OK;
  return launch_next(lin::linear_bias_kernel<T>, (unsigned)ceil_div(a->outer, 256), 256, 0, s, prep.A.sums, P.blocks, a->outer, a->dbias);
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
  return check(a) || !D || by_rows(a, D->sms) ? 0 : plan_fwd(a, D->sms).bytes;
}

int fermix_linear(void* stream, const fx_linear_args* a, void* ws, size_t wsb) {
  const int e = check(a);
  if (e) return e;
  if (a->rows == 0) return FX_OK;
  if (!a->x || !a->weight || !a->y) return FX_ERR_NULL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const DevInfo* D = dev_info();
  if (!D) return FX_ERR_DEVICE;
  if (by_rows(a, D->sms)) return a->dtype == FX_F32 ? rows_forward<float, 3>(s, a, D->sms) : rows_forward<bf16, 1>(s, a, D->sms);
  const LinPlan P = plan_fwd(a, D->sms);
  if (P.bytes && (!ws || wsb < P.bytes)) return FX_ERR_WORKSPACE;
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
