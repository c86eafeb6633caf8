"""Refusals and host-side rules of the operators on tokens (no GPU needed), and refusals on the device."""

import ctypes

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from fermix_b200.build import build

    build()
    return _lib.lib()


def test_cpu_tensors_and_types_are_refused():
    w, t = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        fx.token_embedding(t, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        fx.fused_linear(w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        fx.token_logprobs(torch.zeros(3, 8), t)
    for bad in (torch.float64, torch.float16, torch.complex64, torch.int32):
        with pytest.raises(TypeError):
            fx.token_embedding(t, w.to(bad))
        with pytest.raises(TypeError):
            fx.fused_linear(w.to(bad), w.to(bad))
        with pytest.raises(TypeError):
            fx.token_logprobs(w.to(bad), t)
    with pytest.raises(TypeError):
        fx.fused_linear([[1.0]], w)


def test_abi_argument_errors(lib):
    a = _lib.EmbedArgs()
    a.dtype, a.token_bytes, a.count, a.rows, a.width = _lib.FX_F64, 8, 1, 4, 8
    assert lib.fermix_token_embedding(None, ctypes.byref(a)) == 1
    a.dtype, a.token_bytes = _lib.FX_BF16, 3
    assert lib.fermix_token_embedding(None, ctypes.byref(a)) == 1
    a.token_bytes, a.width = 8, _lib.FX_EMBED_MAX_WIDTH + 1
    assert lib.fermix_token_embedding(None, ctypes.byref(a)) == 2
    a.width, a.rows = 8, 0
    assert lib.fermix_token_embedding(None, ctypes.byref(a)) == 2
    a.rows = 4
    assert lib.fermix_token_embedding(None, ctypes.byref(a)) == 5
    assert lib.fermix_token_embedding_grad(None, ctypes.byref(a), None, 0) == 5
    assert lib.fermix_token_embedding(None, None) == 5
    a.count = 0
    assert lib.fermix_token_embedding(None, ctypes.byref(a)) == 0

    b = _lib.LinearArgs()
    b.dtype, b.rows, b.inner, b.outer = _lib.FX_C64, 1, 8, 8
    assert lib.fermix_linear(None, ctypes.byref(b), None, 0) == 1
    b.dtype, b.activation = _lib.FX_F32, 6
    assert lib.fermix_linear(None, ctypes.byref(b), None, 0) == 2
    b.activation, b.inner = 2, 0
    assert lib.fermix_linear(None, ctypes.byref(b), None, 0) == 2
    b.inner, b.x_stride = 8, -8
    assert lib.fermix_linear(None, ctypes.byref(b), None, 0) == 2
    b.x_stride = 8
    assert lib.fermix_linear(None, ctypes.byref(b), None, 0) == 5
    assert lib.fermix_linear_grad(None, ctypes.byref(b), None, 0) == 5
    assert lib.fermix_linear(None, None, None, 0) == 5
    b.rows = 0
    assert lib.fermix_linear(None, ctypes.byref(b), None, 0) == 0
    assert lib.fermix_linear_grad(None, ctypes.byref(b), None, 0) == 0

    c = _lib.LogprobsArgs()
    c.dtype, c.token_bytes, c.rows, c.entries, c.scale = _lib.FX_C128, 4, 1, 8, 1.0
    assert lib.fermix_token_logprobs(None, ctypes.byref(c), None, 0) == 1
    c.dtype, c.top = _lib.FX_F32, _lib.FX_TOP_MAX + 1
    assert lib.fermix_token_logprobs(None, ctypes.byref(c), None, 0) == 2
    c.top = 0
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        c.scale = scale
        assert lib.fermix_token_logprobs(None, ctypes.byref(c), None, 0) == 2
    c.scale, c.entries = 1.0, 0
    assert lib.fermix_token_logprobs(None, ctypes.byref(c), None, 0) == 2
    c.entries = 8
    assert lib.fermix_token_logprobs(None, ctypes.byref(c), None, 0) == 5
    assert lib.fermix_token_logprobs_grad(None, ctypes.byref(c)) == 5
    c.rows = 0
    assert lib.fermix_token_logprobs(None, ctypes.byref(c), None, 0) == 0
    assert lib.fermix_token_logprobs_grad(None, ctypes.byref(c)) == 0


@pytest.mark.gpu
def test_argument_refusals_on_the_device():
    w = torch.zeros(6, 8, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    x = torch.zeros(3, 8, device="cuda")
    embed, linear, probs = fx.token_embedding, fx.fused_linear, fx.token_logprobs
    for err, call in (
        (TypeError, lambda: embed([1], w)),
        (TypeError, lambda: embed(t.float(), w)),
        (TypeError, lambda: embed(t.bool(), w)),
        (ValueError, lambda: embed(t.cpu(), w)),
        (ValueError, lambda: embed(t, w[0])),
        (ValueError, lambda: embed(t, w[:0])),
        (ValueError, lambda: embed(t, w[:, :0])),
        (TypeError, lambda: embed(t, w, padding=1.0)),
        (TypeError, lambda: embed(t, w, padding=2**63)),
        (ValueError, lambda: linear(x[:, :7], w)),
        (ValueError, lambda: linear(x, w[0])),
        (ValueError, lambda: linear(x, w[:0])),
        (ValueError, lambda: linear(x[:, :0], w[:, :0])),
        (TypeError, lambda: linear(x, w.bfloat16())),
        (ValueError, lambda: linear(x, w.cpu())),
        (ValueError, lambda: linear(x, w, w[0])),
        (ValueError, lambda: linear(x, w, residual=x)),
        (TypeError, lambda: linear(x, w, residual=torch.zeros(3, 6, device="cuda", dtype=torch.bfloat16))),
        (ValueError, lambda: linear(x, w, activation="swish")),
        (ValueError, lambda: probs(x, t[:2])),
        (TypeError, lambda: probs(x, t.float())),
        (ValueError, lambda: probs(x[:, :0], t)),
        (ValueError, lambda: probs(x, t, top=33)),
        (ValueError, lambda: probs(x, t, top=-1)),
        (ValueError, lambda: probs(x, t, scale=0.0)),
        (ValueError, lambda: probs(x, t, scale=float("inf"))),
        (ValueError, lambda: probs(x, t, scale=float("nan"))),
        (TypeError, lambda: probs(x, t, mask=x)),
        (ValueError, lambda: probs(x, t, mask=torch.ones(3, 7, dtype=torch.bool, device="cuda"))),
        (ValueError, lambda: probs(x, t, mask=torch.ones(3, 8, dtype=torch.bool))),
    ):
        with pytest.raises(err):
            call()
