"""The operators on tokens at the ends of what they accept."""

import pytest
import torch

import fermix_b200 as fx

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
