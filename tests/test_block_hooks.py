"""Saved tensors that come back from their hooks with other strides than they went with: sliced
positions and masks under torch.autograd.graph.save_on_cpu."""

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib, block


@pytest.mark.parametrize("n", [1, 5])
def test_position_bias_gradient_takes_the_strides_of_what_comes_back(n, monkeypatch):
    """The arguments of the gradient's call, without a device: (batch, length) positions that were rows of
    a wider array and come back contiguous."""
    sites = torch.arange(24, dtype=torch.int32).view(3, 8)
    args = _lib.BiasArgs()
    args.dtype, args.batch, args.heads, args.q_len, args.k_len = _lib.FX_F32, 3, 1, n, n
    block._set_buckets(args, 8, 16, True, sites[:, :n], sites[:, :n], 8, 8)

    class Ctx:
        pass

    ctx = Ctx()
    ctx.args, ctx.table = args, ((1, 8), torch.float32)
    ctx.saved_tensors = sites[:, :n].clone(), torch.empty(2 * n, 3, dtype=torch.int32).t()[:, ::2]
    seen = []
    monkeypatch.setattr(block, "_call_with_workspace", lambda fn, size, device, a: seen.append(a))
    block._PositionBias.backward(ctx, torch.ones(3, 1, n, n))
    b = seen[0].buckets
    assert b.q_pos_stride == n
    assert b.k_pos_stride in (n, 1) and (n == 1 or b.k_pos_stride == n)  # not contiguous along the row: copied
    assert b.q_pos == ctx.saved_tensors[0].data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [32, 96])
def test_gradients_with_saved_tensors_on_the_host(dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(71)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    B, L = 5, 37
    sites = torch.randint(-300, 300, (B, 2 * L), generator=g, device="cuda", dtype=torch.int32)
    mask = torch.rand(B, 2 * L, generator=g, device="cuda") < 0.7
    q, k, v = (randn(B, L, 4, dim).transpose(1, 2).requires_grad_(True) for _ in range(3))
    table = randn(4, 32).requires_grad_(True)
    x, f, w = randn(B, L, 40).requires_grad_(True), randn(B, L, 40).requires_grad_(True), randn(40).requires_grad_(True)
    gate = randn(B, 1, 40).requires_grad_(True)
    cot = randn(B, 4, L, dim), randn(B, 4, L, L), randn(B, L, 40)

    def run():
        a = fx.biased_attention(q, k, v, table, q_pos=sites[:, :L], k_pos=sites[:, L:], key_mask=mask[:, 3:3 + L])
        b = fx.position_bias(table, sites[:, :L], sites[:, L:])
        r, z = fx.residual_norm(x, f, w, w, gate=gate)
        leaves = [q, k, v, table, x, f, w, gate]
        first = torch.autograd.grad([a, b, r, z], leaves, [*cot, cot[2]], retain_graph=True)
        again = torch.autograd.grad([a, b, r, z], leaves, [*cot, cot[2]])  # one graph, run twice
        assert all(torch.equal(i, j) for i, j in zip(first, again))
        return first

    def reversed_strides(t):
        return t.permute(*range(t.dim() - 1, -1, -1)).clone(memory_format=torch.contiguous_format).permute(
            *range(t.dim() - 1, -1, -1))

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    assert all(torch.equal(i, j) for i, j in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, reversed_strides):
        got = run()
    assert all(torch.equal(i, j) for i, j in zip(got, want))
