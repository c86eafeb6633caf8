"""The attention block of a neural wave function, on torch CUDA tensors: the network in front of
the determinants turns the tokens of the occupied sites into the orbitals that ``slogdet`` /
``slogpf`` take.

* :func:`biased_attention` -- softmax attention whose scores carry a learned bias of the
  distance between the tokens' positions, forward, gradient, and for a single new token;
* :func:`position_bias` -- that bias as an array, and its gradient;
* :func:`residual_norm` -- the residual between two blocks with its gate, its scale and the
  norms on both sides.

float32 and bfloat16; statistics, sums and softmax are float32, and every result is rounded
once. Gradients go through torch autograd and are summed in a fixed order (two runs give the
same bits); tangents (forward mode) and ``torch.func`` transforms are refused. There is no CPU path and, as in the rest of the package, no fallback. None of this
has a counterpart in the reference, whose caller brings the network.
"""

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_KIND = {torch.float32: _lib.FX_F32, torch.bfloat16: _lib.FX_BF16}
_INTS = (torch.int32, torch.int64, torch.int16, torch.uint8)
_GATE_NONE, _GATE_FULL, _GATE_ROW, _GATE_GROUP = range(4)


# ------------------------------------------------------------------ calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(fn, device, *args):
    """fn(stream, *args) on the device's current stream. The common case, the device being current
    already, takes no context: a small call is bound by the host."""
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _lib.check(fn(torch._C._cuda_getCurrentRawStream(index), *args))
    status = fn(torch._C._cuda_getCurrentRawStream(index), *args)
    if status:
        _lib.check(status)


def _call_with_workspace(fn, size, device, args):
    """As _call, with the workspace that size(args) asks for (kept alive until the launches are queued)."""
    ref = ctypes.byref(args)
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            nbytes = size(ref)
    else:
        nbytes = size(ref)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call(fn, device, ref, _ptr(ws), nbytes)


# ------------------------------------------------------------------ checks
def _transformed(peek=torch._C._functorch.peek_interpreter_stack):
    """Whether a forward-mode level or a torch.func transform is open."""
    return forward_ad._current_level >= 0 or peek() is not None


def _refuse_transforms(**tensors):
    """A tangent would be dropped without a word, and a transform's wrapper has no storage to read."""
    level = forward_ad._current_level
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            continue
        if torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise NotImplementedError(f"{name} is inside a torch.func transform (vmap, jvp, grad): the operators of "
                                      "fermix_b200's networks support reverse-mode autograd only")
        if level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} carries a tangent: the operators of fermix_b200's networks have no "
                                      "forward-mode derivative")


def _tensor(t, name, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if like is None:
        if t.dtype not in _KIND:
            raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
        if t.device.type != "cuda":
            raise RuntimeError(
                f"fermix_b200 runs on CUDA devices only (got a tensor on {t.device}); "
                "move it with .cuda() -- there is no CPU fallback"
            )
    else:
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must have dtype {like.dtype}, got {t.dtype}")
        if t.device != like.device:
            raise ValueError(f"{name} must be on {like.device}, got {t.device}")
    return t


@functools.lru_cache(maxsize=64, typed=True)
def _edges(num_buckets, max_distance, bidirectional):
    """The least distance of each bucket after the first, of one side: a bucket for each
    distance below half of the side's buckets, then evenly spaced in the logarithm up to
    ``max_distance`` -- bucket ``exact + j`` starts where
    log(d / exact) / log(max_distance / exact) >= j / (n - exact), in whole numbers."""
    if not isinstance(num_buckets, int) or not 1 <= num_buckets <= _lib.FX_BUCKET_MAX:
        raise ValueError(f"the table must have 1 to {_lib.FX_BUCKET_MAX} buckets, got {num_buckets}")
    if bidirectional and num_buckets % 2:
        raise ValueError(f"a bidirectional table must have an even number of buckets, got {num_buckets}")
    n = num_buckets // 2 if bidirectional else num_buckets
    exact = n // 2
    if not isinstance(max_distance, int) or not exact < max_distance <= _lib.FX_BUCKET_MAX_EDGE:
        raise ValueError(
            f"max_distance must be a whole number above {exact} (the distances with a bucket of their own) and at "
            f"most {_lib.FX_BUCKET_MAX_EDGE}, got {max_distance!r}")
    edges, d, m = list(range(1, exact + 1)), exact, n - exact
    for j in range(1, m if exact else 1):
        while d**m * exact**j < max_distance**j * exact**m:
            d += 1
        edges.append(d)
    return (ctypes.c_int32 * max(1, len(edges)))(*edges), len(edges)


def _positions(pos, length, batch, device, name):
    """pos as an int32 (length) or (batch, length) tensor with contiguous rows."""
    if not isinstance(pos, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(pos).__name__}")
    if pos.dtype not in _INTS:
        raise TypeError(f"{name} must be an integer tensor, got {pos.dtype}")
    if pos.device != device:
        raise ValueError(f"{name} must be on {device}, got {pos.device}")
    if tuple(pos.shape) not in ((length,), (batch, length)):
        raise ValueError(f"{name} must have shape ({length},) or ({batch}, {length}), got {tuple(pos.shape)}")
    return _line(pos if pos.dtype == torch.int32 else pos.to(torch.int32))


def _line(t):
    """t (positions, a mask) with the entries of a row next to each other."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _batch_stride(pos):
    return pos.stride(0) if pos is not None and pos.dim() == 2 else 0


def _set_buckets(a, num_buckets, max_distance, bidirectional, q_pos, k_pos, q_stride, k_stride):
    """a.buckets; a keeps the edges it points to, which may leave the cache before a backward pass."""
    a.edges, count = _edges(num_buckets, max_distance, bool(bidirectional))
    a.buckets = _lib.Buckets(num_buckets, int(bool(bidirectional)), count, 0, ctypes.addressof(a.edges), _ptr(q_pos),
                             _ptr(k_pos), q_stride, k_stride)


# ------------------------------------------------------------------ residual with its norms
class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, post_weight, pre_weight, post_bias, pre_bias, gate, scale, form, kind, eps):
        given = None if gate is None else gate.shape
        r, z, gate = _norm_forward(x, f, post_weight, pre_weight, post_bias, pre_bias, gate, scale, form, kind, eps)
        _, shape, gate_mode = form
        ctx.save_for_backward(x, f, post_weight, pre_weight, post_bias, pre_bias, gate, scale)
        ctx.rest, ctx.given = (shape, kind, gate_mode, eps), given
        ctx.set_materialize_grads(False)
        return r, z

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_r, grad_z):
        if grad_r is None and grad_z is None:
            return (None,) * 11
        # one that was put elsewhere and back (saved-tensor hooks) may have other strides
        saved = [None if t is None else t.contiguous() for t in ctx.saved_tensors]
        x = saved[0]
        a = _norm_args(*saved, *ctx.rest)
        grads = [None if t is None else torch.empty_like(t) for t in saved]
        shared = ctx.given is not None and ctx.given != saved[6].shape
        if shared:  # a gate expanded for the kernel: its gradient is summed in float32, rounded once
            a.dgate_f32 = 1
            grads[6] = torch.empty_like(saved[6], dtype=torch.float32)
        # every pointer's tensor stays referenced here until the launches are queued
        grad_r, grad_z = (None if g is None else g.contiguous() for g in (grad_r, grad_z))
        a.grad_r, a.grad_z = _ptr(grad_r), _ptr(grad_z)
        (a.dx, a.df, a.dpost_weight, a.dpre_weight, a.dpost_bias, a.dpre_bias, a.dgate,
         a.dscale) = (_ptr(g) for g in grads)
        L = _lib.lib()
        _call_with_workspace(L.fermix_residual_norm_grad, L.fermix_residual_norm_grad_workspace_bytes, x.device, a)
        if shared:
            grads[6] = grads[6].sum_to_size(ctx.given).to(x.dtype)
        return (*grads, None, None, None)


def _norm_args(x, f, post_weight, pre_weight, post_bias, pre_bias, gate, scale, shape, kind, gate_mode, eps):
    a = _lib.NormArgs()
    a.dtype, a.kind, a.gate_mode, a.eps = _KIND[x.dtype], kind, gate_mode, eps
    a.groups, a.rows, a.width = shape
    a.x, a.f, a.gate, a.scale = _ptr(x), _ptr(f), _ptr(gate), _ptr(scale)
    a.post_weight, a.post_bias, a.pre_weight, a.pre_bias = (_ptr(t) for t in
                                                            (post_weight, post_bias, pre_weight, pre_bias))
    return a


def _norm_forward(x, f, post_weight, pre_weight, post_bias, pre_bias, gate, scale, form, kind, eps):
    """(r, z, the gate as the kernel took it)."""
    gate_shape, shape, gate_mode = form
    if gate is not None:
        gate = gate.expand(gate_shape).contiguous()
    r, z = torch.empty_like(x), torch.empty_like(x)
    a = _norm_args(x, f, post_weight, pre_weight, post_bias, pre_bias, gate, scale, shape, kind, gate_mode, eps)
    a.r, a.z = r.data_ptr(), z.data_ptr()
    _call(_lib.lib().fermix_residual_norm, x.device, ctypes.byref(a))
    return r, z, gate


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _gate_form(gate, x):
    """(shape the kernel takes the gate in, (groups, rows, width), mode): which entries of x an entry
    of the gate is shared by. Shapes other than the kernel's four expand to the nearest one."""
    width, lead = x.shape[-1], tuple(x.shape[:-1])
    total = math.prod(lead)
    if gate is None:
        return None, (1, total, width), _GATE_NONE
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    if gate.dim() > x.dim() or any(n not in (1, m) for n, m in zip(shape, x.shape)):
        raise ValueError(f"gate must broadcast to {tuple(x.shape)}, got {tuple(gate.shape)}")
    if shape == tuple(x.shape):
        return gate.shape, (1, total, width), _GATE_FULL
    if shape[:-1] == lead:
        return gate.shape, (1, total, width), _GATE_ROW
    # the leading dimensions it has in full, then those it is shared along
    k = 0
    while shape[k] == lead[k]:
        k += 1
    if all(n == 1 for n in shape[k:-1]):
        groups = math.prod(lead[:k])
        return (gate.shape if shape[-1] == width else shape[:-1] + (width,)), (
            groups, total // groups if groups else 0, width), _GATE_GROUP
    return x.shape, (1, total, width), _GATE_FULL


def residual_norm(x, f, post_weight, pre_weight, *, post_bias=None, pre_bias=None, gate=None, scale=None, kind="rms",
                  eps=1e-6):
    """The residual between two blocks of a network with the norms on both sides of it:
    ``u = norm(f)``, ``r = x + scale * gate * u``, ``z = norm(r)``; returns ``(r, z)``.

    ``x`` is the residual stream and ``f`` the output of the block just run, (..., width), float32
    or bfloat16, width <= 8192; ``post_*`` (width,) belong to the norm of ``f``, ``pre_*`` to that
    of ``r`` (the input of the next block). ``kind="rms"`` divides by sqrt(mean square + eps);
    ``"layer"`` takes the mean off first. ``scale`` (width,) and ``gate`` (anything that broadcasts
    to ``x``: an entry each, one per row (..., 1), a vector per sample (batch, 1, width)) multiply
    the normed branch. All of one dtype; differentiable in every tensor. z is formed from the
    unrounded r."""
    if _transformed():
        _refuse_transforms(x=x, f=f, post_weight=post_weight, pre_weight=pre_weight, post_bias=post_bias,
                           pre_bias=pre_bias, gate=gate, scale=scale)
    x = _tensor(x, "x")
    if kind not in ("rms", "layer"):
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _lib.FX_NORM_MAX_WIDTH:
        raise ValueError(f"expected (..., width) with 1 <= width <= {_lib.FX_NORM_MAX_WIDTH}, got {tuple(x.shape)}")
    if _tensor(f, "f", x).shape != x.shape:
        raise ValueError(f"f must have the shape of x {tuple(x.shape)}, got {tuple(f.shape)}")
    width = x.shape[-1]
    params = []
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("post_bias", post_bias),
                    ("pre_bias", pre_bias), ("scale", scale)):
        if t is None and name not in ("post_weight", "pre_weight"):
            params.append(None)
            continue
        if tuple(_tensor(t, name, x).shape) != (width,):
            raise ValueError(f"{name} must have shape ({width},), got {tuple(t.shape)}")
        params.append(t.contiguous())
    if gate is not None:
        _tensor(gate, "gate", x)
    form = _gate_form(gate, x)
    post_weight, pre_weight, post_bias, pre_bias, scale = params
    args = (x.contiguous(), f.contiguous(), post_weight, pre_weight, post_bias, pre_bias, gate, scale)
    rest = (form, int(kind == "layer"), float(eps))
    if _wants_grad(*args):
        return _ResidualNorm.apply(*args, *rest)
    return _norm_forward(*args, *rest)[:2]


# ------------------------------------------------------------------ position bias
class _PositionBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, q_pos, k_pos, shape, max_distance, bidirectional):
        out, ctx.args = _bias_forward(table, q_pos, k_pos, shape, max_distance, bidirectional)
        ctx.save_for_backward(q_pos, k_pos)
        ctx.table = table.shape, table.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        a = _lib.BiasArgs.from_buffer_copy(ctx.args)  # the graph may be run again, from another thread too
        # alive until the launches are queued; one that was put elsewhere and back (saved-tensor hooks) may
        # have other strides
        q_pos, k_pos = ctx.saved_tensors
        q_pos, k_pos = _line(q_pos), _line(k_pos)
        grad = grad.contiguous()
        dtable = torch.empty(ctx.table[0], dtype=ctx.table[1], device=grad.device)
        a.grad, a.dtable = grad.data_ptr(), dtable.data_ptr()
        a.buckets.q_pos, a.buckets.k_pos = q_pos.data_ptr(), k_pos.data_ptr()
        a.buckets.q_pos_stride, a.buckets.k_pos_stride = _batch_stride(q_pos), _batch_stride(k_pos)
        L = _lib.lib()
        _call_with_workspace(L.fermix_position_bias_grad, L.fermix_position_bias_grad_workspace_bytes, grad.device, a)
        return dtable, None, None, None, None, None


def _bias_forward(table, q_pos, k_pos, shape, max_distance, bidirectional):
    a = _lib.BiasArgs()
    a.dtype = _KIND[table.dtype]
    a.heads, a.q_len, a.k_len = shape[-3:]
    a.batch = shape[0] if len(shape) == 4 else 1
    _set_buckets(a, table.shape[1], max_distance, bidirectional, q_pos, k_pos, _batch_stride(q_pos),
                 _batch_stride(k_pos))
    out = torch.empty(shape, dtype=table.dtype, device=table.device)
    a.table, a.out = table.data_ptr(), out.data_ptr()
    _call(_lib.lib().fermix_position_bias, table.device, ctypes.byref(a))
    return out, a


def position_bias(table, q_pos, k_pos=None, *, max_distance=128, bidirectional=True):
    """The learned bias of each pair of positions, ``table[h, bucket(k_pos - q_pos)]``: (heads,
    q_len, k_len), or (batch, heads, q_len, k_len) where a position tensor is (batch, length).

    ``table`` is (heads, num_buckets), float32 or bfloat16. A side has a bucket for each distance
    below half of its buckets, and the rest evenly spaced in the logarithm up to ``max_distance``
    (<= 2048; all longer distances share the last one); ``bidirectional`` gives half of the table to
    each sign, otherwise keys after the query share bucket 0. ``q_pos`` and ``k_pos`` (default:
    q_pos) are integer tensors within +-2**29, in any order. Differentiable in ``table``."""
    if _transformed():
        _refuse_transforms(table=table, q_pos=q_pos, k_pos=k_pos)
    table = _tensor(table, "table")
    if table.dim() != 2:
        raise ValueError(f"table must have shape (heads, num_buckets), got {tuple(table.shape)}")
    if k_pos is None:
        k_pos = q_pos
    batch = None
    for name, p in (("q_pos", q_pos), ("k_pos", k_pos)):
        if not isinstance(p, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor, got {type(p).__name__}")
        if p.dim() not in (1, 2):
            raise ValueError(f"{name} must have shape (length,) or (batch, length), got {tuple(p.shape)}")
        if p.dim() == 2:
            batch = p.shape[0]
    q = _positions(q_pos, q_pos.shape[-1], batch, table.device, "q_pos")
    k = q if k_pos is q_pos else _positions(k_pos, k_pos.shape[-1], batch, table.device, "k_pos")
    shape = (() if batch is None else (batch,)) + (table.shape[0], q.shape[-1], k.shape[-1])
    args = (table.contiguous(), q, k, shape, max_distance, bool(bidirectional))
    return _PositionBias.apply(*args) if _wants_grad(table) else _bias_forward(*args)[0]


# ------------------------------------------------------------------ attention
def _strides(t):
    return t.stride()[:3]


def _lse_parts(lse):
    """The addresses of lse[0] and lse[1] (contiguous float32)."""
    p = lse.data_ptr()
    return p, p + 2 * lse.numel()


def _attn_args(q, k, v, table, out, lse, q_pos, k_pos, key_mask, causal, scale, max_distance, bidirectional):
    a = _lib.AttnArgs()
    a.dtype, a.causal = _KIND[q.dtype], int(causal)
    a.batch, a.heads, a.q_len, a.dim = q.shape
    a.kv_heads, a.k_len = k.shape[1], k.shape[2]
    a.scale = scale
    qs, ks = _batch_stride(q_pos), _batch_stride(k_pos)
    if table is not None:
        _set_buckets(a, table.shape[1], max_distance, bidirectional, q_pos, k_pos, qs, ks)
    else:
        a.buckets.q_pos, a.buckets.k_pos, a.buckets.q_pos_stride, a.buckets.k_pos_stride = _ptr(q_pos), _ptr(
            k_pos), qs, ks
    a.q, a.k, a.v, a.table = _ptr(q), _ptr(k), _ptr(v), _ptr(table)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = _strides(q), _strides(k), _strides(v)
    if key_mask is not None:
        a.key_mask, a.mask_stride = _ptr(key_mask), key_mask.stride(0)
    a.out = _ptr(out)
    if lse is not None:
        a.lse, a.lse_low = _lse_parts(lse)
    a.out_stride[:] = _strides(out)
    return a


def _attn_forward(q, k, v, table, rest, with_lse):
    """(out, lse or None, the call's arguments)."""
    out = torch.empty_like(q)
    if out.stride(-1) != 1:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((2, *q.shape[:3]), dtype=torch.float32, device=q.device) if with_lse else None  # and lse_low
    a = _attn_args(q, k, v, table, out, lse, *rest)
    L = _lib.lib()
    _call_with_workspace(L.fermix_biased_attention, L.fermix_biased_attention_workspace_bytes, q.device, a)
    return out, lse, a


class _BiasedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, rest):
        out, lse, ctx.args = _attn_forward(q, k, v, table, rest, True)
        # the arguments hold addresses: everything they point to is saved
        ctx.save_for_backward(q, k, v, table, out, lse, *rest[:3])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, out, lse, q_pos, k_pos, key_mask = ctx.saved_tensors
        # a saved tensor may have been put elsewhere and back (saved-tensor hooks), with other strides
        q, k, v, out, lse = _rows(q), _rows(k), _rows(v), _rows(out), lse.contiguous()
        table = None if table is None else table.contiguous()
        q_pos, k_pos, key_mask = _line(q_pos), _line(k_pos), _line(key_mask)
        a = _lib.AttnArgs.from_buffer_copy(ctx.args)  # the graph may be run again, from another thread too
        a.q, a.k, a.v, a.table, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(table), out.data_ptr()
        a.lse, a.lse_low = _lse_parts(lse)
        a.q_stride[:], a.k_stride[:], a.v_stride[:], a.out_stride[:] = (_strides(q), _strides(k), _strides(v),
                                                                        _strides(out))
        a.buckets.q_pos, a.buckets.k_pos, a.key_mask = _ptr(q_pos), _ptr(k_pos), _ptr(key_mask)
        a.buckets.q_pos_stride, a.buckets.k_pos_stride = _batch_stride(q_pos), _batch_stride(k_pos)
        a.mask_stride = 0 if key_mask is None else key_mask.stride(0)
        dout = _rows(dout)
        dq, dk, dv = _rows(torch.empty_like(q)), _rows(torch.empty_like(k)), _rows(torch.empty_like(v))
        dtable = None if table is None else torch.empty_like(table)
        a.dout, a.dq, a.dk, a.dv, a.dtable = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dtable)
        a.dout_stride[:], a.dq_stride[:] = _strides(dout), _strides(dq)
        a.dk_stride[:], a.dv_stride[:] = _strides(dk), _strides(dv)
        L = _lib.lib()
        _call_with_workspace(L.fermix_biased_attention_grad, L.fermix_biased_attention_grad_workspace_bytes, q.device, a)
        return dq, dk, dv, dtable, None


def _rows(t):
    """t with the entries of a token next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 and t.is_contiguous() else t.contiguous()


def biased_attention(q, k, v, table=None, *, q_pos=None, k_pos=None, key_mask=None, causal=False, scale=None,
                     max_distance=128, bidirectional=True):
    """Attention with a learned bias of the positions' distance in its scores:
    ``softmax(scale * q k^T + table[h, bucket(k_pos - q_pos)]) v``, without the array of scores.

    ``q`` is (batch, heads, q_len, dim), ``k`` and ``v`` (batch, kv_heads, k_len, dim) with heads a
    multiple of kv_heads (head h reads key head h // (heads // kv_heads)) and dim <= 128, float32 or
    bfloat16, any strides (the head-major view of token-major storage is read in place). ``table``
    (heads, num_buckets), of the same dtype, ``max_distance`` and ``bidirectional`` are those of
    :func:`position_bias`; None: no bias. ``k_pos`` defaults to 0, 1, ..., and ``q_pos`` to the last
    q_len of them (a new token attends from the end of the cache); integer tensors (length,) or
    (batch, length), within +-2**29. ``key_mask`` (batch, k_len) bool: False leaves a key out,
    whatever its k and v hold. ``causal`` leaves out keys with k_pos > q_pos, as a table entry of -inf does
    those of its bucket; what such keys hold has to be finite (0 times NaN). A query without any
    key gives 0 and has no gradient. ``scale`` defaults to dim ** -0.5. A live infinity gives NaN in the
    rows that read it.

    Differentiable in q, k, v and table; under ``torch.no_grad()`` nothing is kept. Few queries
    (one new token) split the keys over the device and join the parts."""
    if _transformed():
        _refuse_transforms(q=q, k=k, v=v, table=table, q_pos=q_pos, k_pos=k_pos, key_mask=key_mask)
    q = _tensor(q, "q")
    for name, t in (("k", k), ("v", v)):
        _tensor(t, name, q)
    if q.dim() != 4 or k.dim() != 4 or not 1 <= q.shape[3] <= _lib.FX_ATTN_MAX_DIM:
        raise ValueError(f"q, k and v must have shape (batch, heads, length, dim) with 1 <= dim <= "
                         f"{_lib.FX_ATTN_MAX_DIM}, got {tuple(q.shape)}, {tuple(k.shape)}")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"k and v must both have shape ({q.shape[0]}, kv_heads, k_len, {q.shape[3]}), got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    batch, heads, q_len, dim = q.shape
    k_len = k.shape[2]
    if heads and (k.shape[1] == 0 or heads % k.shape[1]):
        raise ValueError(f"the {heads} heads must be a multiple of the {k.shape[1]} key heads")
    if table is not None:
        if _tensor(table, "table", q).dim() != 2 or table.shape[0] != heads:
            raise ValueError(f"table must have shape ({heads}, num_buckets), got {tuple(table.shape)}")
        table = table.contiguous()
    if q_pos is not None:
        q_pos = _positions(q_pos, q_len, batch, q.device, "q_pos")
    if k_pos is not None:
        k_pos = _positions(k_pos, k_len, batch, q.device, "k_pos")
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor) or key_mask.dtype != torch.bool:
            raise TypeError("key_mask must be a bool tensor (True: the key takes part)")
        if tuple(key_mask.shape) != (batch, k_len) or key_mask.device != q.device:
            raise ValueError(f"key_mask must have shape ({batch}, {k_len}) on {q.device}, got "
                             f"{tuple(key_mask.shape)} on {key_mask.device}")
        key_mask = _line(key_mask)
    rest = (q_pos, k_pos, key_mask, bool(causal), float(dim**-0.5 if scale is None else scale), max_distance,
            bool(bidirectional))
    q, k, v = _rows(q), _rows(k), _rows(v)
    if _wants_grad(q, k, v, table):
        return _BiasedAttention.apply(q, k, v, table, rest)
    return _attn_forward(q, k, v, table, rest, False)[0]
