"""Refusals and host-side rules of the attention-block operators (no GPU needed)."""

import ctypes

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib, block
from tests import block_refs as ref


@pytest.fixture(scope="module")
def lib():
    from fermix_b200.build import build

    build()
    return _lib.lib()


@pytest.mark.parametrize("two_sided", [True, False])
@pytest.mark.parametrize("buckets,distance", [(1, 1), (2, 2), (2, 8), (3, 5), (4, 40), (16, 64), (32, 128), (64, 512),
                                              (256, 2048)])
def test_bucket_edges_are_exact(buckets, distance, two_sided):
    if two_sided and buckets % 2:
        with pytest.raises(ValueError):
            block._edges(buckets, distance, two_sided)
        return
    got, n = block._edges(buckets, distance, two_sided)
    assert list(got)[:n] == ref.edges(buckets, distance, two_sided)
    assert n < (buckets // 2 if two_sided else buckets) or n == 0


@pytest.mark.parametrize("buckets,distance", [(0, 8), (257, 2048), (32, 8), (32, 2049), (32, 128.0), (8, 0)])
def test_bucket_refusals(buckets, distance):
    with pytest.raises(ValueError):
        block._edges(buckets, distance, False if buckets == 257 else True)


def test_cpu_tensors_and_types_are_refused():
    x = torch.zeros(2, 4, 8, 16)
    w = torch.ones(16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fx.biased_attention(x, x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        fx.residual_norm(x, x, w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        fx.position_bias(torch.zeros(4, 32), torch.arange(4))
    for bad in (torch.float64, torch.float16, torch.complex64, torch.int32):
        with pytest.raises(TypeError):
            fx.biased_attention(x.to(bad), x.to(bad), x.to(bad))
        with pytest.raises(TypeError):
            fx.residual_norm(x.to(bad), x.to(bad), w.to(bad), w.to(bad))
        with pytest.raises(TypeError):
            fx.position_bias(torch.zeros(4, 32).to(bad), torch.arange(4))
    with pytest.raises(TypeError):
        fx.biased_attention([[1.0]], x, x)


def test_abi_argument_errors(lib):
    a = _lib.NormArgs()
    a.dtype, a.groups, a.rows, a.width = _lib.FX_F64, 1, 1, 8
    assert lib.fermix_residual_norm(None, ctypes.byref(a)) == 1
    a.dtype, a.width = _lib.FX_F32, _lib.FX_NORM_MAX_WIDTH + 1
    assert lib.fermix_residual_norm(None, ctypes.byref(a)) == 2
    a.width, a.rows = 8, 0
    assert lib.fermix_residual_norm(None, ctypes.byref(a)) == 0  # nothing to do
    a.rows, a.gate_mode = 1, 4
    assert lib.fermix_residual_norm(None, ctypes.byref(a)) == 2
    a.gate_mode = 0
    assert lib.fermix_residual_norm(None, ctypes.byref(a)) == 5  # pointers missing
    assert lib.fermix_residual_norm(None, None) == 5

    edges = (ctypes.c_int32 * 3)(1, 2, 1)
    b = _lib.BiasArgs()
    b.dtype, b.batch, b.heads, b.q_len, b.k_len = _lib.FX_BF16, 1, 1, 4, 4
    b.buckets.num_buckets, b.buckets.num_edges, b.buckets.edges = 8, 3, ctypes.addressof(edges)
    assert lib.fermix_position_bias(None, ctypes.byref(b)) == 2  # descending edges
    edges[2] = _lib.FX_BUCKET_MAX_EDGE + 1
    assert lib.fermix_position_bias(None, ctypes.byref(b)) == 2
    edges[2] = 5
    assert lib.fermix_position_bias(None, ctypes.byref(b)) == 5
    b.buckets.two_sided, b.buckets.num_buckets = 1, 6
    assert lib.fermix_position_bias(None, ctypes.byref(b)) == 2  # three edges need four buckets a side
    b.buckets.two_sided, b.buckets.edges = 0, None
    assert lib.fermix_position_bias(None, ctypes.byref(b)) == 5
    b.q_len, b.buckets.num_edges = 0, 0
    assert lib.fermix_position_bias(None, ctypes.byref(b)) == 0

    c = _lib.AttnArgs()
    c.dtype, c.batch, c.heads, c.kv_heads, c.q_len, c.k_len, c.dim = _lib.FX_C64, 1, 4, 2, 1, 1, 64
    assert lib.fermix_biased_attention(None, ctypes.byref(c), None, 0) == 1
    c.dtype, c.dim = _lib.FX_F32, 129
    assert lib.fermix_biased_attention(None, ctypes.byref(c), None, 0) == 2
    c.dim, c.kv_heads = 64, 3
    assert lib.fermix_biased_attention(None, ctypes.byref(c), None, 0) == 2
    c.kv_heads = 2
    assert lib.fermix_biased_attention(None, ctypes.byref(c), None, 0) == 5
    assert lib.fermix_biased_attention_grad(None, ctypes.byref(c), None, 0) == 5
    c.batch = 0
    assert lib.fermix_biased_attention(None, ctypes.byref(c), None, 0) == 0
    assert lib.fermix_biased_attention_grad(None, ctypes.byref(c), None, 0) == 0


@pytest.mark.gpu
def test_argument_refusals_on_the_device():
    x = torch.zeros(2, 4, 8, 16, device="cuda")
    t = torch.zeros(4, 32, device="cuda")
    w = torch.ones(16, device="cuda")
    attn = fx.biased_attention
    for err, call in (
        (ValueError, lambda: attn(x[0], x, x)),
        (ValueError, lambda: attn(x, x[:, :3], x[:, :3])),
        (ValueError, lambda: attn(x, x, x[:, :, :4])),
        (ValueError, lambda: attn(x, x[:1], x[:1])),
        (ValueError, lambda: attn(x, x[..., :8], x[..., :8])),
        (ValueError, lambda: attn(*(torch.zeros(1, 1, 2, 129, device="cuda"),) * 3)),
        (TypeError, lambda: attn(x, x.bfloat16(), x)),
        (TypeError, lambda: attn(x, x, x, t.bfloat16())),
        (ValueError, lambda: attn(x, x, x, t[:2])),
        (ValueError, lambda: attn(x, x, x, t, max_distance=8)),
        (ValueError, lambda: attn(x, x, x, t[:, :31])),
        (TypeError, lambda: attn(x, x, x, t, q_pos=torch.zeros(8, device="cuda"))),
        (ValueError, lambda: attn(x, x, x, t, q_pos=torch.zeros(7, device="cuda", dtype=torch.int32))),
        (ValueError, lambda: attn(x, x, x, t, k_pos=torch.zeros(8, dtype=torch.int32))),
        (TypeError, lambda: attn(x, x, x, key_mask=torch.zeros(2, 8, device="cuda"))),
        (ValueError, lambda: attn(x, x, x, key_mask=torch.zeros(2, 7, device="cuda", dtype=torch.bool))),
        (ValueError, lambda: attn(x, x, x.cpu())),
        (ValueError, lambda: fx.position_bias(t[0], torch.arange(3, device="cuda"))),
        (ValueError, lambda: fx.position_bias(t, torch.zeros(1, 1, 1, device="cuda", dtype=torch.int32))),
        (TypeError, lambda: fx.position_bias(t, [1, 2])),
        (TypeError, lambda: fx.position_bias(t, torch.zeros(3, device="cuda"))),
        (ValueError, lambda: fx.position_bias(t, torch.zeros(2, 3, device="cuda", dtype=torch.int32),
                                              torch.zeros(3, 3, device="cuda", dtype=torch.int32))),
        (ValueError, lambda: fx.residual_norm(x, x[..., :8], w, w)),
        (ValueError, lambda: fx.residual_norm(x, x, w[:8], w)),
        (TypeError, lambda: fx.residual_norm(x, x, w, w.bfloat16())),
        (ValueError, lambda: fx.residual_norm(x, x, w, w, kind="mean")),
        (ValueError, lambda: fx.residual_norm(x, x, w, w, gate=torch.ones(3, 1, device="cuda"))),
        (ValueError, lambda: fx.residual_norm(x, x, w, w, gate=torch.ones(1, 2, 4, 8, 16, device="cuda"))),
        (ValueError, lambda: fx.residual_norm(*(torch.zeros(1, 8193, device="cuda"),) * 2,
                                              *(torch.zeros(8193, device="cuda"),) * 2)),
        (TypeError, lambda: fx.residual_norm(x, x, None, w)),
    ):
        with pytest.raises(err):
            call()
