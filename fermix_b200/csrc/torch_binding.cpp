// The operators on tokens as torch functions: tensors in, C ABI arguments (include/fermix_b200_token.h), autograd nodes.
// Arguments were checked by fermix_b200/tokens.py. In Python the same took 30 to 60 us of host time a training call, more
// than the kernels of a small one, most of it with autograd's thread waiting for the interpreter lock.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "fermix_b200_token.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int status) {
  if (status) throw Failure("fermix_b200 error " + std::to_string(status) + ": " + fermix_strerror(status));
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? FX_F32 : FX_BF16; }

// fn(stream, args, workspace, bytes) on the tensor's device and its current stream.
template <typename A, typename Size, typename Fn>
void call(const Tensor& on, const A& args, Size size, Fn fn) {
  const c10::cuda::OptionalCUDAGuard guard(on.device());
  const size_t bytes = size(&args);
  Tensor ws;  // lives until the launches are queued
  if (bytes) ws = at::empty({(int64_t)bytes}, on.options().dtype(at::kByte));
  check(fn(at::cuda::getCurrentCUDAStream(on.get_device()).stream(), &args, ptr(ws), bytes));
}
template <typename A>
size_t none(const A*) {
  return 0;
}

// t as rows of `width` entries that lie next to each other, and the stride of a row.
Tensor flat(const Tensor& t, int64_t width, int64_t& stride) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  if (r.stride(1) != 1 && !(width == 1 && r.is_contiguous())) r = r.contiguous();
  stride = r.size(0) > 1 ? r.stride(0) : width;
  return r;
}

std::vector<int64_t> shape_with(const Tensor& t, int64_t drop, std::initializer_list<int64_t> more) {
  std::vector<int64_t> s(t.sizes().begin(), t.sizes().end() - drop);
  s.insert(s.end(), more);
  return s;
}

// Gradients of gradients are refused when they are asked for, as once_differentiable does.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  // undefined gradients stay; the others hang on the node that raises
  variable_list given, out = grads;
  for (auto& g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_());
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int)given.size());
  given = (*error)(std::move(given));
  size_t i = 0;
  for (auto& g : out)
    if (g.defined()) g = given[i++];
  return out;
}

// ---------------------------------------------------------------- embedding
struct Padding {
  int64_t value;
  bool given;
};

fx_embed_args embed_args(const Tensor& tokens, int dtype, int64_t rows, int64_t width, double scale, Padding pad) {
  fx_embed_args a{};
  a.dtype = dtype;
  a.token_bytes = (int)tokens.element_size();
  a.count = tokens.numel();
  a.rows = rows;
  a.width = width;
  a.padding = pad.value;
  a.has_padding = pad.given;
  a.scale = (float)scale;
  a.tokens = tokens.data_ptr();
  return a;
}

Tensor embed_forward(const Tensor& tokens, const Tensor& weight, double scale, Padding pad) {
  Tensor out = at::empty(shape_with(tokens, 0, {weight.size(1)}), weight.options());
  fx_embed_args a = embed_args(tokens, dtype_of(weight), weight.size(0), weight.size(1), scale, pad);
  a.weight = weight.data_ptr();
  a.out = out.data_ptr();
  call(weight, a, none<fx_embed_args>, [](void* s, const fx_embed_args* a, void*, size_t) { return fermix_token_embedding(s, a); });
  return out;
}

struct Embed : torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& weight, double scale, int64_t padding, bool given) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["rest"] = std::vector<int64_t>{weight.size(0), weight.size(1), padding, given};
    ctx->saved_data["scale"] = scale;
    return embed_forward(tokens, weight, scale, {padding, given});
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // one that was put elsewhere and back (saved-tensor hooks) may have other strides
    const Tensor tokens = ctx->get_saved_variables()[0].contiguous(), grad = grads[0].contiguous();
    const auto rest = ctx->saved_data["rest"].toIntVector();
    Tensor dweight = at::empty({rest[0], rest[1]}, grad.options());
    fx_embed_args a = embed_args(tokens, dtype_of(grad), rest[0], rest[1], ctx->saved_data["scale"].toDouble(), {rest[2], rest[3] != 0});
    a.grad = grad.data_ptr();
    a.dweight = dweight.data_ptr();
    call(grad, a, fermix_token_embedding_grad_workspace_bytes, fermix_token_embedding_grad);
    return once({Tensor(), dweight, Tensor(), Tensor(), Tensor()});
  }
};

Tensor token_embedding(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding, bool given) {
  const Tensor t = tokens.contiguous(), w = weight.contiguous();
  if (at::GradMode::is_enabled() && w.requires_grad()) return Embed::apply(t, w, scale, padding, given);
  return embed_forward(t, w, scale, {padding, given});
}

// ---------------------------------------------------------------- linear
// The arguments' operands, alive until the call.
struct Linear {
  fx_linear_args a{};
  Tensor x, weight, residual, dy;

  Linear(const Tensor& x_, const Tensor& weight_, int64_t activation) {
    a.dtype = dtype_of(weight_);
    a.activation = (int32_t)activation;
    a.outer = weight_.size(0);
    a.inner = weight_.size(1);
    x = flat(x_, a.inner, a.x_stride);
    weight = flat(weight_, a.inner, a.weight_stride);
    a.rows = x.size(0);
    a.x = x.data_ptr();
    a.weight = weight.data_ptr();
  }
};

std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual,
                                         int64_t activation, bool with_slope) {
  Linear l(x, weight, activation);
  Tensor y = at::empty(shape_with(x, 1, {l.a.outer}), x.options()), slope;
  if (with_slope && activation) {
    slope = at::empty({l.a.rows, l.a.outer}, x.options().dtype(l.a.dtype == FX_F32 ? at::kFloat : at::kHalf));
    l.a.slope = slope.data_ptr();
  }
  l.a.y = y.data_ptr();
  l.a.bias = ptr(bias);
  if (residual.defined()) {
    l.residual = flat(residual, l.a.outer, l.a.residual_stride);
    l.a.residual = l.residual.data_ptr();
  }
  call(x, l.a, fermix_linear_workspace_bytes, fermix_linear);
  return {y, slope};
}

struct FusedLinear : torch::autograd::Function<FusedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                        int64_t activation) {
    auto [y, slope] = linear_forward(x, weight, bias.value_or(Tensor()), residual.value_or(Tensor()), activation, true);
    ctx->save_for_backward({x, weight, slope});
    ctx->saved_data["activation"] = activation;
    // the inputs' numbers among those that are tensors
    ctx->saved_data["bias"] = bias ? 2 : -1;
    ctx->saved_data["residual"] = residual ? (bias ? 3 : 2) : -1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &dy = grads[0];
    const auto wants = [&](int64_t i) { return i >= 0 && ctx->needs_input_grad(i); };
    const bool wants_x = wants(0), wants_weight = wants(1), wants_bias = wants(ctx->saved_data["bias"].toInt());
    Tensor dx, dweight, dbias, slope;
    if (wants_x || wants_weight || wants_bias) {
      Linear l(x, weight, ctx->saved_data["activation"].toInt());
      l.dy = flat(dy, l.a.outer, l.a.dy_stride);
      l.a.dy = l.dy.data_ptr();
      if (saved[2].defined()) {
        slope = saved[2].contiguous();
        l.a.slope = slope.data_ptr();
      }
      if (wants_x) l.a.dx = (dx = at::empty(x.sizes(), x.options())).data_ptr();
      if (wants_weight) l.a.dweight = (dweight = at::empty(weight.sizes(), x.options())).data_ptr();
      if (wants_bias) l.a.dbias = (dbias = at::empty({l.a.outer}, x.options())).data_ptr();
      call(x, l.a, fermix_linear_grad_workspace_bytes, fermix_linear_grad);
    }
    return once({dx, dweight, dbias, wants(ctx->saved_data["residual"].toInt()) ? dy : Tensor(), Tensor()});
  }
};

Tensor fused_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t activation) {
  const OptTensor b = bias ? OptTensor(bias->contiguous()) : bias;
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (b && b->requires_grad()) || (residual && residual->requires_grad())))
    return FusedLinear::apply(x, weight, b, residual, activation);
  return linear_forward(x, weight, b.value_or(Tensor()), residual.value_or(Tensor()), activation, false).first;
}

// ---------------------------------------------------------------- log probabilities
struct Probs {
  fx_logprobs_args a{};
  Tensor logits, mask;

  Probs(const Tensor& logits_, const Tensor& tokens, const Tensor& mask_, double scale, Padding pad) {
    a.dtype = dtype_of(logits_);
    a.token_bytes = (int)tokens.element_size();
    a.entries = logits_.size(-1);
    logits = flat(logits_, a.entries, a.logits_stride);
    a.rows = logits.size(0);
    a.padding = pad.value;
    a.has_padding = pad.given;
    a.scale = (float)scale;
    a.logits = logits.data_ptr();
    a.tokens = tokens.data_ptr();
    if (mask_.defined()) {
      if (mask_.dim() == 1) mask = mask_.contiguous();  // one for all rows
      else mask = flat(mask_, a.entries, a.mask_stride);
      a.mask = static_cast<const uint8_t*>(mask.data_ptr());
    }
  }
};

variable_list probs_forward(const Tensor& logits, const Tensor& tokens, const Tensor& mask, double scale, Padding pad, int64_t top,
                            Tensor* stats) {
  Probs p(logits, tokens, mask, scale, pad);
  const auto real = logits.options().dtype(at::kFloat);
  variable_list out{at::empty(tokens.sizes(), real), at::empty(tokens.sizes(), real)};
  p.a.logp = out[0].data_ptr<float>();
  p.a.entropy = out[1].data_ptr<float>();
  p.a.top = (int32_t)top;
  if (top) {
    out.push_back(at::empty(shape_with(tokens, 0, {top}), real));
    out.push_back(at::empty(shape_with(tokens, 0, {top}), real.dtype(at::kLong)));
    p.a.top_logp = out[2].data_ptr<float>();
    p.a.top_index = out[3].data_ptr<int64_t>();
  }
  if (stats) p.a.stats = (*stats = at::empty({2, p.a.rows}, real)).data_ptr<float>();
  call(logits, p.a, fermix_token_logprobs_workspace_bytes, fermix_token_logprobs);
  return out;
}

struct Logprobs : torch::autograd::Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const OptTensor& given_mask, double scale,
                               int64_t padding, bool given, int64_t top) {
    const Tensor mask = given_mask.value_or(Tensor());
    Tensor stats;
    variable_list out = probs_forward(logits, tokens, mask, scale, {padding, given}, top, &stats);
    ctx->save_for_backward({logits, tokens, mask, stats, out[1]});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = std::vector<int64_t>{padding, given};
    if (top) ctx->mark_non_differentiable({out[2], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list result(7);
    if (!grads[0].defined() && !grads[1].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const auto pad = ctx->saved_data["padding"].toIntVector();
    const Tensor &logits = saved[0], tokens = saved[1].contiguous(), stats = saved[3].contiguous(), entropy = saved[4].contiguous();
    Probs p(logits, tokens, saved[2], ctx->saved_data["scale"].toDouble(), {pad[0], pad[1] != 0});
    const Tensor g = grads[0].defined() ? grads[0].contiguous() : Tensor(), e = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor dlogits = at::empty(logits.sizes(), logits.options());
    p.a.stats = stats.data_ptr<float>();
    p.a.entropy = entropy.data_ptr<float>();
    p.a.dlogits = dlogits.data_ptr();
    p.a.grad_logp = static_cast<const float*>(ptr(g));
    p.a.grad_entropy = static_cast<const float*>(ptr(e));
    call(logits, p.a, none<fx_logprobs_args>, [](void* s, const fx_logprobs_args* a, void*, size_t) { return fermix_token_logprobs_grad(s, a); });
    result[0] = dlogits;
    return once(std::move(result));
  }
};

variable_list token_logprobs(const Tensor& logits, const Tensor& tokens, const OptTensor& mask, double scale, int64_t padding, bool given,
                             int64_t top) {
  const Tensor t = tokens.contiguous();
  if (at::GradMode::is_enabled() && logits.requires_grad()) return Logprobs::apply(logits, t, mask, scale, padding, given, top);
  return probs_forward(logits, t, mask.value_or(Tensor()), scale, {padding, given}, top, nullptr);
}

}  // namespace

PYBIND11_MODULE(fermix_torch, m) {
  m.def("raise_as", [](py::object type) {  // what a failed call raises
    static py::object kept;
    kept = std::move(type);
    py::register_exception_translator([](std::exception_ptr p) {
      try {
        if (p) std::rethrow_exception(p);
      } catch (const Failure& e) {
        PyErr_SetString(kept.ptr(), e.what());
      }
    });
  });
  m.def("token_embedding", &token_embedding);
  m.def("fused_linear", &fused_linear);
  m.def("token_logprobs", &token_logprobs);
}
