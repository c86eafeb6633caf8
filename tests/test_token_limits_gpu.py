"""The operators on tokens at the ends of what they accept."""

import ctypes

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib

pytestmark = pytest.mark.gpu


# one pass of the sort, and two
@pytest.mark.parametrize("kind,rows", [(torch.uint8, 3), (torch.int16, 3000)], ids=["u8", "i16"])
def test_embedding_gradient_of_the_most_tokens(kind, rows):
    """2^31 - 2 tokens: the last window of the sorted list ends, and the places of the last block of the sort lie, behind
    2^31 - 1. Whole numbers, exact."""
    count = 2**31 - 2
    tokens = torch.zeros(count, dtype=kind, device="cuda")
    tokens[-150:] = 1
    tokens[-3:] = rows - 1
    weight = torch.tensor([3.0, 5.0, 7.0], device="cuda", dtype=torch.bfloat16).repeat(rows // 3)[:, None].requires_grad_()
    out = fx.token_embedding(tokens, weight)
    assert out.shape == (count, 1)
    assert out[-151:, 0].tolist() == [3.0] + [5.0] * 147 + [7.0] * 3 and out[:2, 0].tolist() == [3.0, 3.0]
    cot = torch.zeros_like(out)
    cot[-200:] = 1
    cot[:5] = 2
    (grad,) = torch.autograd.grad(out, weight, cot)
    assert grad[0] == 50 + 10 and grad[1] == 147 and grad[rows - 1] == 3
    assert int((grad != 0).sum()) == 3
    del out, cot, tokens
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [7, 70, 400, 2100])
def test_linear_of_overlapping_windows(rows, dtype):
    """Rows that share entries (windows of a sequence, 8 and 3 entries apart): the numbers of their copies."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    line = torch.randn(8 * rows + 1200, generator=gen, device="cuda").to(dtype)
    for hop in (8, 3):
        x, w = line.unfold(0, 72, hop)[:rows], line[5:].unfold(0, 72, hop)[:130]
        dy = line[16:].unfold(0, 130, hop)[:rows]
        assert x.stride() == (hop, 1) and dy.stride() == (hop, 1)
        results = []
        for copy in (lambda t: t, lambda t: t.contiguous()):
            leaves = [copy(t).detach().requires_grad_() for t in (x, w)]
            y = fx.fused_linear(*leaves, activation="silu")
            plain = fx.fused_linear(*leaves)
            results.append((y, plain, *torch.autograd.grad(y, leaves, copy(dy)), *torch.autograd.grad(plain, leaves, copy(dy))))
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("kind", [_lib.FX_F32, _lib.FX_BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,inner,outer", [(700, 136, 264), (2400, 136, 1208)])
def test_linear_workspace_asked_for_without_pointers(rows, inner, outer, kind):
    """A query without operands covers operands anywhere: what the call itself needs is never more, and it runs."""
    L, dtype = _lib.lib(), {_lib.FX_F32: torch.float32, _lib.FX_BF16: torch.bfloat16}[kind]
    stream = torch.cuda.current_stream().cuda_stream
    made = [torch.randn(n + 1, device="cuda").to(dtype) for n in (rows * inner, outer * inner, rows * outer)]
    outs = [torch.empty(n, dtype=dtype, device="cuda") for n in (rows * outer, rows * inner, outer * inner, outer)]
    a = _lib.LinearArgs()
    a.dtype, a.rows, a.inner, a.outer = kind, rows, inner, outer
    a.x_stride, a.weight_stride, a.dy_stride = inner, inner, outer
    asked = L.fermix_linear_workspace_bytes(ctypes.byref(a))
    a.dx, a.dweight, a.dbias = (t.data_ptr() for t in outs[1:])
    asked_grad = L.fermix_linear_grad_workspace_bytes(ctypes.byref(a))
    assert asked_grad > 0
    assert asked > 0 or (kind == _lib.FX_F32 and rows == 700)  # a small float32 map needs none
    for off in (0, 1):
        a.x, a.weight, a.dy = (t[off:].data_ptr() for t in made)
        a.y = outs[0].data_ptr()
        assert L.fermix_linear_workspace_bytes(ctypes.byref(a)) <= asked
        assert L.fermix_linear_grad_workspace_bytes(ctypes.byref(a)) <= asked_grad
        ws = torch.empty(max(asked, asked_grad), dtype=torch.uint8, device="cuda")
        assert L.fermix_linear(stream, ctypes.byref(a), ws.data_ptr(), asked) == 0
        assert L.fermix_linear_grad(stream, ctypes.byref(a), ws.data_ptr(), asked_grad) == 0
        x, w, dy = (t[off:off + n].view(-1, c) for t, n, c in zip(made, (rows * inner, outer * inner, rows * outer),
                                                                   (inner, inner, outer)))
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        y = fx.fused_linear(*leaves, bias := torch.zeros(outer, dtype=dtype, device="cuda", requires_grad=True))
        want = (y, *torch.autograd.grad(y, (*leaves, bias), dy.clone()))
        assert all(torch.equal(got, w.reshape(-1)) for got, w in zip(outs, want))
