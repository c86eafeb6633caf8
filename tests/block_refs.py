"""Plain 64-bit forms of the attention-block operators (torch, any device), differentiable by
autograd; written from the definitions."""

import math

import torch


def edges(num_buckets, max_distance, two_sided):
    """Least distance of each bucket after the first, from real logarithms decided exactly by
    rational powers: d starts bucket exact + j when (d / exact)^m >= (max / exact)^j."""
    from fractions import Fraction

    n = num_buckets // 2 if two_sided else num_buckets
    exact = n // 2
    out = list(range(1, exact + 1))
    for j in range(1, n - exact if exact else 1):
        want = Fraction(max_distance, exact) ** j
        out.append(next(d for d in range(exact, max_distance + 1) if Fraction(d, exact) ** (n - exact) >= want))
    return out


def buckets(q_pos, k_pos, num_buckets, max_distance, two_sided):
    delta = k_pos[..., None, :].long() - q_pos[..., :, None].long()
    a = delta.abs() if two_sided else (-delta).clamp(min=0)
    b = torch.zeros_like(a)
    for e in edges(num_buckets, max_distance, two_sided):
        b += a >= e
    if two_sided:
        b += (delta > 0) * (num_buckets // 2)
    return b


def position_bias(table, q_pos, k_pos, max_distance, two_sided):
    b = buckets(q_pos, k_pos, table.shape[1], max_distance, two_sided)
    out = table[:, b]
    return out.transpose(0, 1) if b.dim() == 3 else out


def attention(q, k, v, table=None, q_pos=None, k_pos=None, key_mask=None, causal=False, scale=None, max_distance=128,
              two_sided=True):
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1], k.shape[2]
    dev = q.device
    if key_mask is not None:  # what a masked key holds must not matter
        k = torch.where(key_mask[:, None, :, None], k, torch.zeros_like(k))
        v = torch.where(key_mask[:, None, :, None], v, torch.zeros_like(v))
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    if k_pos is None:
        k_pos = torch.arange(Lk, device=dev)
    if q_pos is None:
        q_pos = torch.arange(Lk - Lq, Lk, device=dev)
    s = torch.einsum("bhid,bhjd->bhij", q, k) * (D**-0.5 if scale is None else scale)
    if table is not None:
        s = s + position_bias(table, q_pos, k_pos, max_distance, two_sided)
    allowed = torch.ones(B, 1, Lq, Lk, dtype=torch.bool, device=dev)
    if key_mask is not None:
        allowed = allowed & key_mask[:, None, None, :]
    if causal:
        later = k_pos[..., None, :] > q_pos[..., :, None]
        allowed = allowed & ~(later[:, None] if later.dim() == 3 else later)
    any_key = (allowed & (s > -math.inf)).any(-1, keepdim=True)
    s = s.masked_fill(~allowed, -math.inf).masked_fill(~any_key, 0.0)
    p = torch.softmax(s, -1) * (allowed & any_key)
    return torch.einsum("bhij,bhjd->bhid", p, v)


def norm(x, weight, bias, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return y if bias is None else y + bias


def residual_norm(x, f, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None, scale=None, kind="rms",
                  eps=1e-6):
    u = norm(f, post_weight, post_bias, kind, eps)
    if gate is not None:
        u = u * gate
    if scale is not None:
        u = u * scale
    r = x + u
    return r, norm(r, pre_weight, pre_bias, kind, eps)
