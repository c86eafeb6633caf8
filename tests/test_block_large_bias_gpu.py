"""Gradients of the biased attention where a row's bias is huge beside its scores, against closed
forms in 64 bits.

A bias of -1e9 or of the type's lowest value absorbs the score that it is added to (float32 holds
-1e9 log2(e) to 128), so that a row whose keys all carry it is the plain mean of its values, and its
probabilities in the gradient are 1 / n as well. Tolerances: those of test_block_gpu.py for the largest
entry; in the norm of the difference bfloat16's four roundings (p, ds, the saved result, the
gradient) of 2^-9 each give 2^-7. At -1e4 a score is rounded to 2^-11 in base 2 (3.4e-4 of its
probability) in the forward and again in the gradient, and both enter the normaliser and the row's
delta: three times 6.8e-4, 2^-8 allows for twice that."""

import math

import pytest
import torch

import fermix_b200 as fx
from tests import block_refs as ref
from tests.test_block_gpu import FORWARD, GRADIENT, IDS, TYPES, _attention_case, _close, _grads

pytestmark = pytest.mark.gpu
NORM = {torch.float32: 2.0**-13, torch.bfloat16: 2.0**-7}

# batch, heads, key heads, q_len, k_len, dim: every forward (one token, tiles, split keys) and gradient kernel
SHAPES = [(2, 2, 1, 1, 120, 32), (2, 2, 2, 6, 300, 64), (1, 2, 1, 100, 120, 32), (2, 2, 1, 150, 400, 64),
          (1, 2, 1, 40, 90, 96), (1, 4, 2, 20, 2300, 128)]


def _formula(t, kw, cot, buckets=32, distance=128):
    """(out, dq, dk, dv, dtable) in 64 bits; entries of the table at or below -1e8 absorb the scores."""
    q, k, v, table = (t[n].double() for n in ("q", "k", "v", "table"))
    B, H, Lq, D = q.shape
    G, Lk = H // k.shape[1], k.shape[2]
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    bucket = ref.buckets(torch.arange(Lk - Lq, Lk, device="cuda"), torch.arange(Lk, device="cuda"), buckets, distance, True)
    bias = table[:, bucket][None]
    allowed = torch.ones(B, 1, 1, Lk, dtype=torch.bool, device="cuda")
    if "key_mask" in kw:
        allowed = kw["key_mask"][:, None, None, :]
    low = bias <= -1e8
    score = torch.einsum("bhid,bhjd->bhij", q, kk) / math.sqrt(D) + bias
    usual = torch.softmax(score.masked_fill(low | ~allowed, -math.inf), -1)
    mean = (allowed / allowed.sum(-1, keepdim=True)).expand(B, H, Lq, Lk)
    p = torch.where((~low & allowed).any(-1, keepdim=True), usual, mean)
    do = cot.double()
    out = p @ vv
    dv = (p.transpose(2, 3) @ do).view(B, -1, G, Lk, D).sum(2)
    dp = do @ vv.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = ds @ kk / math.sqrt(D)
    dk = (ds.transpose(2, 3) @ q).view(B, -1, G, Lk, D).sum(2) / math.sqrt(D)
    dtable = torch.zeros_like(table).index_add_(1, bucket.reshape(-1), ds.sum(0).reshape(H, -1))
    return out, (dq, dk, dv, dtable)


def _check(t, kw, cot, dtype):
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    out = fx.biased_attention(**a, **kw)
    want, exp = _formula(t, kw, cot)
    _close(out, want, FORWARD[dtype], "out")
    top = max(e.abs().max().item() for e in exp)
    for n, x, y in zip(a, _grads(out, list(a.values()), cot), exp):
        x = x.double()
        assert torch.isfinite(x).all(), n
        size = max(y.abs().max().item(), 0.01 * top)
        assert (x - y).abs().max().item() <= GRADIENT[dtype] * size, n
        assert (x - y).norm().item() <= NORM[dtype] * max(y.norm().item(), 0.01 * top * y.numel()**0.5), n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("low", ["lowest", -1e9])
@pytest.mark.parametrize("mask", [False, True])
def test_gradient_of_rows_of_one_huge_bias(shape, low, mask, dtype):
    """One head has nothing but the low value, the other its usual table."""
    t, kw, cot = _attention_case(shape, dtype, 50, mask=mask)
    t["table"][0] = torch.finfo(dtype).min if low == "lowest" else low
    if mask:
        kw["key_mask"][:, 0] = True
    _check(t, kw, cot, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gradient_where_the_low_value_excludes_earlier_keys(shape, dtype):
    """Keys at and before the query have the lowest value: the last query has nothing else."""
    t, kw, cot = _attention_case(shape, dtype, 51)
    t["table"][0, :16] = torch.finfo(dtype).min
    _check(t, kw, cot, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gradient_under_a_bias_of_minus_ten_thousand(shape, dtype):
    t, kw, cot = _attention_case(shape, dtype, 52)
    t["table"] -= 1e4
    t["table"][0] = -1e4
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    b = {n: x.detach().double().requires_grad_(True) for n, x in t.items()}
    out, want = fx.biased_attention(**a, **kw), ref.attention(**b, **kw)
    tol = max(2.0**-8, GRADIENT[dtype])
    _close(out, want, max(2.0**-9, FORWARD[dtype]), "out")
    exp = _grads(want, list(b.values()), cot.double())
    top = max(e.abs().max().item() for e in exp)
    for n, x, y in zip(a, _grads(out, list(a.values()), cot), exp):
        assert (x.double() - y).abs().max().item() <= tol * max(y.abs().max().item(), 0.01 * top), n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 96])
def test_gradient_without_the_low_part(dim, dtype, monkeypatch):
    """A caller of the C entries that passes no lse_low: an ordinary table loses nothing by it."""
    from fermix_b200 import block

    t, kw, cot = _attention_case((2, 2, 1, 70, 90, dim), dtype, 53, "sites", True)
    call = block._call_with_workspace

    def without(fn, size, device, args):
        args.lse_low = None
        call(fn, size, device, args)

    monkeypatch.setattr(block, "_call_with_workspace", without)
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    b = {n: x.detach().double().requires_grad_(True) for n, x in t.items()}
    exp = _grads(ref.attention(**b, **kw), list(b.values()), cot.double())
    for n, x, y in zip(a, _grads(fx.biased_attention(**a, **kw), list(a.values()), cot), exp):
        _close(x, y, GRADIENT[dtype], n)
