"""The operators around the attention blocks of a neural wave function, on torch CUDA tensors: the
way into the network, its position-wise maps, and the way out to probabilities of sites.

* :func:`token_embedding` -- rows of a table, scaled, and the table's gradient by sorted tokens;
* :func:`fused_linear` -- the linear map with bias, activation and residual in its epilogue;
* :func:`token_logprobs` -- log probabilities of given tokens under a softmax, with entropy and
  the likeliest alternatives.

float32 and bfloat16, with the conventions of :mod:`fermix_b200.block`: sums are float32, every
result is rounded once, gradients go through torch autograd and are summed in a fixed order (two
runs give the same bits), tangents (forward mode) and ``torch.func`` transforms are refused, and there
is no CPU path and no fallback. None of this has a counterpart in the reference, whose caller
brings the network.
"""

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .block import _KIND, _call, _call_with_workspace, _ptr, _refuse_transforms, _rows, _tensor, _transformed, _wants_grad

_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8, torch.int16: 2, torch.uint8: 1}
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "tanh": 5}


def _once(fn):
    """As ``once_differentiable``, whose wrapping costs more than a small call's launches, only where a graph of the
    gradients is asked for."""
    guarded = once_differentiable(fn)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return staticmethod(backward)


# ------------------------------------------------------------------ checks
def _tokens(tokens, like, name="tokens"):
    if not isinstance(tokens, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(tokens).__name__}")
    if tokens.dtype not in _TOKEN_BYTES:
        raise TypeError(f"{name} must be an integer tensor, got {tokens.dtype}")
    if tokens.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {tokens.device}")
    return tokens.contiguous()


def _padding(padding):
    if padding is None:
        return 0, 0
    if not isinstance(padding, int) or isinstance(padding, bool) or not -(2**63) <= padding < 2**63:
        raise TypeError(f"padding must be a whole number or None, got {padding!r}")
    return padding, 1


def _flat(t, width):
    """(t as rows of `width` entries that lie next to each other, the stride of a row)."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    t = _rows(t)
    return t, (t.stride(0) if t.shape[0] > 1 else width)


# ------------------------------------------------------------------ embedding
def _embed_args(tokens, weight, scale, padding):
    a = _lib.EmbedArgs()
    a.dtype, a.token_bytes = _KIND[weight.dtype], _TOKEN_BYTES[tokens.dtype]
    a.count, (a.rows, a.width) = tokens.numel(), weight.shape
    a.padding, a.has_padding = padding
    a.scale = scale
    a.tokens = tokens.data_ptr()
    return a


def _embed_forward(tokens, weight, scale, padding):
    out = torch.empty(*tokens.shape, weight.shape[1], dtype=weight.dtype, device=weight.device)
    a = _embed_args(tokens, weight, scale, padding)
    a.weight, a.out = weight.data_ptr(), out.data_ptr()
    _call(_lib.lib().fermix_token_embedding, weight.device, ctypes.byref(a))
    return out


class _TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.table, ctx.rest = (weight.shape, weight.dtype), (scale, padding)
        return _embed_forward(tokens, weight, scale, padding)

    @_once
    def backward(ctx, grad):
        tokens = ctx.saved_tensors[0].contiguous()
        grad = grad.contiguous()
        dweight = torch.empty(ctx.table[0], dtype=ctx.table[1], device=grad.device)
        a = _embed_args(tokens, dweight, *ctx.rest)
        a.grad, a.dweight = grad.data_ptr(), dweight.data_ptr()
        L = _lib.lib()
        _call_with_workspace(L.fermix_token_embedding_grad, L.fermix_token_embedding_grad_workspace_bytes, grad.device, a)
        return None, dweight, None, None


def token_embedding(tokens, weight, *, scale=1.0, padding=None):
    """The rows of a table that the tokens name, scaled: ``scale * weight[tokens]``, (..., width).

    ``tokens`` (...) is an integer tensor, ``weight`` (rows, width), float32 or bfloat16. A token equal
    to ``padding`` (any whole number, a row of the table or not) gives zeros and has no gradient; any
    other token outside [0, rows) gives NaN and has no gradient. Differentiable in ``weight``: the rows of
    the output's gradient are summed in float32 in the tokens' order and rounded once."""
    if _transformed():
        _refuse_transforms(tokens=tokens, weight=weight)
    weight = _tensor(weight, "weight")
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= _lib.FX_EMBED_MAX_WIDTH or not 1 <= weight.shape[0] < 2**31 - 1:
        raise ValueError(f"weight must have shape (rows, width) with rows >= 1 and 1 <= width <= "
                         f"{_lib.FX_EMBED_MAX_WIDTH}, got {tuple(weight.shape)}")
    tokens = _tokens(tokens, weight)
    if tokens.numel() >= 2**31 - 1:
        raise ValueError(f"fewer than 2**31 - 1 tokens a call, got {tokens.numel()}")
    args = tokens, weight.contiguous(), float(scale), _padding(padding)
    return _TokenEmbedding.apply(*args) if _wants_grad(weight) else _embed_forward(*args)


# ------------------------------------------------------------------ linear
def _linear_args(x, weight, activation):
    """(arguments, x as rows, weight as rows): both must outlive the call."""
    a = _lib.LinearArgs()
    a.dtype, a.activation = _KIND[weight.dtype], activation
    a.outer, a.inner = weight.shape
    x, a.x_stride = _flat(x, a.inner)
    weight, a.weight_stride = _flat(weight, a.inner)
    a.rows = x.shape[0]
    a.x, a.weight = x.data_ptr(), weight.data_ptr()
    return a, x, weight


def _linear_forward(x, weight, bias, residual, activation, with_slope):
    a, rows, weight = _linear_args(x, weight, activation)
    y = torch.empty(*x.shape[:-1], a.outer, dtype=x.dtype, device=x.device)
    slope = None
    if with_slope and activation:
        slope = torch.empty(rows.shape[0], a.outer, dtype=torch.float16 if x.dtype == torch.bfloat16 else torch.float32,
                            device=x.device)
        a.slope = slope.data_ptr()
    a.y, a.bias = y.data_ptr(), _ptr(bias)
    if residual is not None:
        residual, a.residual_stride = _flat(residual, a.outer)
        a.residual = residual.data_ptr()
    L = _lib.lib()
    _call_with_workspace(L.fermix_linear, L.fermix_linear_workspace_bytes, x.device, a)
    return y, slope


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, slope = _linear_forward(x, weight, bias, residual, activation, True)
        ctx.save_for_backward(x, weight, slope)
        ctx.activation, ctx.bias = activation, bias is not None
        return y

    @_once
    def backward(ctx, dy):
        x, weight, slope = ctx.saved_tensors
        wants_x, wants_weight, wants_bias, wants_residual, _ = ctx.needs_input_grad
        dx = dweight = dbias = None
        if wants_x or wants_weight or wants_bias:
            a, rows, weight = _linear_args(x, weight, ctx.activation)
            dy_rows, a.dy_stride = _flat(dy, a.outer)
            a.dy = dy_rows.data_ptr()
            if slope is not None:
                slope = slope.contiguous()  # saved-tensor hooks may bring other strides
                a.slope = slope.data_ptr()
            if wants_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
                a.dx = dx.data_ptr()
            if wants_weight:
                dweight = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
                a.dweight = dweight.data_ptr()
            if wants_bias:
                dbias = torch.empty(a.outer, dtype=x.dtype, device=x.device)
                a.dbias = dbias.data_ptr()
            L = _lib.lib()
            _call_with_workspace(L.fermix_linear_grad, L.fermix_linear_grad_workspace_bytes, x.device, a)
        return dx, dweight, dbias, dy if wants_residual else None, None


def fused_linear(x, weight, bias=None, *, activation=None, residual=None):
    """The linear map with what follows it: ``residual + act(x @ weight.T + bias)``, (..., outer).

    ``x`` is (..., inner), ``weight`` (outer, inner), ``bias`` (outer,), ``residual`` (..., outer), float32 or
    bfloat16, all of one type; rows may be strided (a slice of a wider projection is read in place).
    ``activation`` is None, "relu", "silu", "gelu" (with the error function), "gelu_tanh" or "tanh". The
    sum, the activation and the residual are float32, rounded once. float32 has the accuracy of float32
    products; an infinity or a NaN gives NaN in the entries it reaches. Differentiable in all four; with an
    activation the derivative at each entry is kept for the backward pass (float32, or half beside
    bfloat16), under ``torch.no_grad()`` nothing is."""
    if _transformed():
        _refuse_transforms(x=x, weight=weight, bias=bias, residual=residual)
    x = _tensor(x, "x")
    if _tensor(weight, "weight", x).dim() != 2 or not weight.numel():
        raise ValueError(f"weight must have shape (outer, inner), neither zero, got {tuple(weight.shape)}")
    outer, inner = weight.shape
    if x.dim() < 1 or x.shape[-1] != inner:
        raise ValueError(f"x must have shape (..., {inner}), got {tuple(x.shape)}")
    if x.numel() >= 2**30 * inner or max(outer, inner) >= 2**30:
        raise ValueError(f"fewer than 2**30 rows and columns, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None:
        if tuple(_tensor(bias, "bias", x).shape) != (outer,):
            raise ValueError(f"bias must have shape ({outer},), got {tuple(bias.shape)}")
        bias = bias.contiguous()
    if residual is not None and _tensor(residual, "residual", x).shape != (*x.shape[:-1], outer):
        raise ValueError(f"residual must have shape {(*x.shape[:-1], outer)}, got {tuple(residual.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_ACTIVATIONS)}, got {activation!r}")
    act = _ACTIVATIONS[activation]
    if _wants_grad(x, weight, bias, residual):
        return _FusedLinear.apply(x, weight, bias, residual, act)
    return _linear_forward(x, weight, bias, residual, act, False)[0]


# ------------------------------------------------------------------ log probabilities
def _prob_args(logits, tokens, mask, scale, padding):
    """(arguments, logits as rows, mask as rows): both must outlive the call."""
    a = _lib.LogprobsArgs()
    a.dtype, a.token_bytes = _KIND[logits.dtype], _TOKEN_BYTES[tokens.dtype]
    a.entries = logits.shape[-1]
    logits, a.logits_stride = _flat(logits, a.entries)
    a.rows = logits.shape[0]
    a.padding, a.has_padding = padding
    a.scale = scale
    a.logits, a.tokens = logits.data_ptr(), tokens.data_ptr()
    if mask is not None:
        if mask.dim() == 1:
            mask = mask.contiguous()
        else:
            mask, a.mask_stride = _flat(mask, a.entries)
        a.mask = mask.data_ptr()
    return a, logits, mask


def _prob_forward(logits, tokens, mask, scale, padding, top, with_stats):
    a, rows, mask = _prob_args(logits, tokens, mask, scale, padding)
    shape, device = tokens.shape, logits.device
    logp = torch.empty(shape, dtype=torch.float32, device=device)
    entropy = torch.empty(shape, dtype=torch.float32, device=device)
    a.logp, a.entropy, a.top = logp.data_ptr(), entropy.data_ptr(), top
    out = logp, entropy
    if top:
        best = torch.empty(*shape, top, dtype=torch.float32, device=device)
        index = torch.empty(*shape, top, dtype=torch.int64, device=device)
        a.top_logp, a.top_index = best.data_ptr(), index.data_ptr()
        out += best, index
    stats = None
    if with_stats:
        stats = torch.empty(2, rows.shape[0], dtype=torch.float32, device=device)
        a.stats = stats.data_ptr()
    L = _lib.lib()
    _call_with_workspace(L.fermix_token_logprobs, L.fermix_token_logprobs_workspace_bytes, device, a)
    return out, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, scale, padding, top):
        out, stats = _prob_forward(logits, tokens, mask, scale, padding, top, True)
        ctx.save_for_backward(logits, tokens, mask, stats, out[1])
        ctx.rest = scale, padding
        ctx.mark_non_differentiable(*out[2:])
        ctx.set_materialize_grads(False)
        return out

    @_once
    def backward(ctx, grad_logp, grad_entropy, *_):
        if grad_logp is None and grad_entropy is None:
            return (None,) * 6
        logits, tokens, mask, stats, entropy = ctx.saved_tensors
        tokens, stats, entropy = tokens.contiguous(), stats.contiguous(), entropy.contiguous()
        a, rows, mask = _prob_args(logits, tokens, mask, *ctx.rest)
        grad_logp, grad_entropy = (None if g is None else g.contiguous() for g in (grad_logp, grad_entropy))
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a.stats, a.entropy, a.dlogits = stats.data_ptr(), entropy.data_ptr(), dlogits.data_ptr()
        a.grad_logp, a.grad_entropy = _ptr(grad_logp), _ptr(grad_entropy)
        _call(_lib.lib().fermix_token_logprobs_grad, logits.device, ctypes.byref(a))
        return dlogits, None, None, None, None, None


def token_logprobs(logits, tokens, *, scale=1.0, mask=None, top=0, padding=None):
    """Log probabilities of given tokens under ``softmax(scale * logits)``: ``(logp, entropy)``, or
    ``(logp, entropy, top_logp, top_index)`` with the ``top`` <= 32 likeliest entries of each row.

    ``logits`` is (..., entries), float32 or bfloat16, ``tokens`` (...) an integer tensor; ``logp``,
    ``entropy`` (in nats) and ``top_logp`` (..., top) are float32, ``top_index`` int64. ``mask`` (entries,) or
    (..., entries) bool: False leaves an entry out, whatever its logit holds. Ties among the likeliest go to
    the lowest index; behind the last entry of any probability stand -inf and index -1. A row without
    such an entry has entropy 0 and no gradient; a token that is masked, or whose logit is -inf, has
    logp -inf. A live NaN or +inf gives NaN (and indices -1) in its row. A token equal to ``padding``
    leaves its row out: logp and entropy 0, no alternatives, no gradient; any other token outside
    [0, entries) has logp NaN and no gradient through it. ``scale`` (an inverse temperature) is positive.

    Differentiable in ``logits`` through logp and entropy."""
    if _transformed():
        _refuse_transforms(logits=logits, tokens=tokens, mask=mask)
    logits = _tensor(logits, "logits")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= _lib.FX_LOGPROBS_MAX:
        raise ValueError(f"logits must have shape (..., entries) with 1 <= entries <= {_lib.FX_LOGPROBS_MAX}, got "
                         f"{tuple(logits.shape)}")
    tokens = _tokens(tokens, logits)
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must have shape {tuple(logits.shape[:-1])}, got {tuple(tokens.shape)}")
    if tokens.numel() >= 2**31 - 1:
        raise ValueError(f"fewer than 2**31 - 1 rows a call, got {tokens.numel()}")
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool:
            raise TypeError("mask must be a bool tensor (True: the entry takes part)")
        if mask.shape not in (logits.shape, logits.shape[-1:]) or mask.device != logits.device:
            raise ValueError(f"mask must have shape {tuple(logits.shape)} or {tuple(logits.shape[-1:])} on "
                             f"{logits.device}, got {tuple(mask.shape)} on {mask.device}")
    if not isinstance(top, int) or isinstance(top, bool) or not 0 <= top <= _lib.FX_TOP_MAX:
        raise ValueError(f"top must be a whole number from 0 to {_lib.FX_TOP_MAX}, got {top!r}")
    scale = float(scale)
    if not 0 < scale <= 1e30 or not math.isfinite(scale):
        raise ValueError(f"scale must be positive and at most 1e30, got {scale}")
    args = logits, tokens, mask, scale, _padding(padding), top
    if _wants_grad(logits):
        return _TokenLogprobs.apply(*args)
    return _prob_forward(*args, False)[0]
