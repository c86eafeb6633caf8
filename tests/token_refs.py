"""Plain 64-bit forms of the operators on tokens (torch, any device), differentiable by autograd;
written from the definitions."""

import math

import torch


def embedding(tokens, weight, scale=1.0, padding=None):
    t = tokens.long()
    pad = torch.zeros_like(t, dtype=torch.bool) if padding is None else t == padding
    bad = ((t < 0) | (t >= weight.shape[0])) & ~pad
    out = weight[torch.where(pad | bad, 0, t)] * scale
    out = torch.where(pad[..., None], torch.zeros_like(out), out)
    return torch.where(bad[..., None], torch.full_like(out, math.nan), out)


def activation(h, name):
    if name is None:
        return h
    if name == "relu":
        return torch.relu(h)
    if name == "silu":
        return h * torch.sigmoid(h)
    if name == "gelu":
        return h * torch.special.ndtr(h)
    if name == "gelu_tanh":
        return 0.5 * h * (1 + torch.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h**3)))
    return torch.tanh(h)


def linear(x, weight, bias=None, act=None, residual=None):
    h = x @ weight.T
    if bias is not None:
        h = h + bias
    y = activation(h, act)
    return y if residual is None else residual + y


def logprobs(logits, tokens, scale=1.0, mask=None, top=0, padding=None):
    """(logp, entropy[, top_logp, top_index]) row by row."""
    V = logits.shape[-1]
    t = tokens.long()
    pad = torch.zeros_like(t, dtype=torch.bool) if padding is None else t == padding
    x = torch.where(pad[..., None], torch.zeros_like(logits), logits)  # whatever the logits hold
    if mask is not None:
        x = torch.where(mask.expand_as(x), x, torch.full_like(x, -math.inf))
    raw = x
    dead = (raw == -math.inf)
    empty = dead.all(-1, keepdim=True)
    live = ~dead & ~empty
    x = torch.where(live, x, torch.zeros_like(x)) * scale
    m = torch.where(live, x, torch.full_like(x, -math.inf)).amax(-1, keepdim=True).detach()
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(x - m) * live
    s = e.sum(-1, keepdim=True)
    s = torch.where(empty, torch.ones_like(s), s)
    logs = x - m - torch.log(s)
    p = e / s
    entropy = -(p * torch.where(live, logs, torch.zeros_like(logs))).sum(-1)
    logs = torch.where(live, logs, torch.full_like(logs, -math.inf))
    bad = (t < 0) | (t >= V)
    logp = logs.gather(-1, torch.where(bad, 0, t)[..., None])[..., 0]
    logp = torch.where(bad, torch.full_like(logp, math.nan), logp)
    zero = torch.zeros_like(logp)
    out = torch.where(pad, zero, logp), torch.where(pad, zero, entropy)
    if top:
        order = torch.sort(raw, dim=-1, descending=True, stable=True).indices[..., :top]
        best = logs.gather(-1, order)
        gone = pad[..., None] | (best == -math.inf)
        best, order = best.masked_fill(gone, -math.inf), order.masked_fill(gone, -1)
        if top > V:
            fill = best.new_full((*best.shape[:-1], top - V), -math.inf)
            best, order = torch.cat([best, fill], -1), torch.cat([order, torch.full_like(fill, -1, dtype=order.dtype)], -1)
        out += best, order
    return out
