"""The operators around the attention blocks of a neural wave function, on torch CUDA tensors: the
way into the network, its position-wise maps, and the way out to probabilities of sites.

* :func:`token_embedding` -- rows of a table, scaled, and the table's gradient by sorted tokens;
* :func:`fused_linear` -- the linear map with bias, activation and residual in its epilogue;
* :func:`token_logprobs` -- log probabilities of given tokens under a softmax, with entropy and
  the likeliest alternatives.

float32 and bfloat16, with the conventions of :mod:`fermix_b200.block`: sums are float32, every
result is rounded once (what else is rounded stands at the operator), gradients go through torch autograd and are summed in a fixed order (two
runs give the same bits), tangents (forward mode) and ``torch.func`` transforms are refused, and there
is no CPU path and no fallback. None of this has a counterpart in the reference, whose caller
brings the network.
"""

import torch

from . import _lib
from .block import _refuse_transforms, _tensor, _transformed

_TOKENS = (torch.int32, torch.int64, torch.int16, torch.uint8)
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "tanh": 5}


# ------------------------------------------------------------------ checks
def _tokens(tokens, like, name="tokens"):
    if not isinstance(tokens, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(tokens).__name__}")
    if tokens.dtype not in _TOKENS:
        raise TypeError(f"{name} must be an integer tensor, got {tokens.dtype}")
    if tokens.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {tokens.device}")
    return tokens


def _padding(padding):
    """(the token, whether there is one)."""
    if padding is None:
        return 0, False
    if not isinstance(padding, int) or isinstance(padding, bool) or not -(2**63) <= padding < 2**63:
        raise TypeError(f"padding must be a whole number or None, got {padding!r}")
    return padding, True


# ------------------------------------------------------------------ embedding
def token_embedding(tokens, weight, *, scale=1.0, padding=None):
    """The rows of a table that the tokens name, scaled: ``scale * weight[tokens]``, (..., width).

    ``tokens`` (...) is an integer tensor, ``weight`` (rows, width), float32 or bfloat16. A token equal
    to ``padding`` (any whole number, a row of the table or not) gives zeros and has no gradient; any
    other token outside [0, rows) gives NaN and has no gradient. Differentiable in ``weight``: the rows of
    the output's gradient are summed in float32 in a fixed order (by groups of a token's places) and rounded once."""
    if _transformed():
        _refuse_transforms(tokens=tokens, weight=weight)
    weight = _tensor(weight, "weight")
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= _lib.FX_EMBED_MAX_WIDTH or not 1 <= weight.shape[0] < 2**31 - 1:
        raise ValueError(f"weight must have shape (rows, width) with rows >= 1 and 1 <= width <= "
                         f"{_lib.FX_EMBED_MAX_WIDTH}, got {tuple(weight.shape)}")
    tokens = _tokens(tokens, weight)
    if tokens.numel() >= 2**31 - 1:
        raise ValueError(f"fewer than 2**31 - 1 tokens a call, got {tokens.numel()}")
    return _lib.binding().token_embedding(tokens, weight, float(scale), *_padding(padding))


# ------------------------------------------------------------------ linear
def fused_linear(x, weight, bias=None, *, activation=None, residual=None):
    """The linear map with what follows it: ``residual + act(x @ weight.T + bias)``, (..., outer).

    ``x`` is (..., inner), ``weight`` (outer, inner), ``bias`` (outer,), ``residual`` (..., outer), float32 or
    bfloat16, all of one type; rows may be strided (a slice of a wider projection is read in place).
    ``activation`` is None, "relu", "silu", "gelu" (with the error function), "gelu_tanh" or "tanh". The
    sum, the activation and the residual are float32, rounded once. float32 products have float32's accuracy,
    activations and their derivatives are good to 2^-20 of 1 + |h|; an infinity or a NaN gives NaN in the float32
    entries it reaches. Differentiable in all four; with an activation the derivative at each entry is kept for the
    backward pass (float32, or half beside bfloat16), under ``torch.no_grad()`` nothing is. In bfloat16 its product with
    the output's gradient is rounded to bfloat16 before the products of the gradients in ``x`` and ``weight``."""
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
    if residual is not None and _tensor(residual, "residual", x).shape != (*x.shape[:-1], outer):
        raise ValueError(f"residual must have shape {(*x.shape[:-1], outer)}, got {tuple(residual.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_ACTIVATIONS)}, got {activation!r}")
    return _lib.binding().fused_linear(x, weight, bias, residual, _ACTIVATIONS[activation])


# ------------------------------------------------------------------ log probabilities
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
    [0, entries) has logp NaN and no gradient through it. ``scale`` (an inverse temperature) is from 1e-30 to 1e30.

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
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"scale must be from 1e-30 to 1e30, got {scale}")
    return tuple(_lib.binding().token_logprobs(logits, tokens, mask, scale, *_padding(padding), top))
