"""token_logprobs on rows that leave nothing without a mask, and ties of signed zeros."""

import math

import pytest
import torch

import fermix_b200 as fx

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("entries", [1, 5, 70, 1024, 1500, 30000])
@pytest.mark.parametrize("masked", [False, True])
def test_a_row_without_entries_has_no_gradient(entries, masked, dtype):
    """Rows of -inf, and rows whose mask leaves only entries of -inf: the same as rows that the mask leaves nothing of."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(6, entries, generator=gen, device="cuda").to(dtype)
    tokens = torch.randint(0, entries, (6,), generator=gen, device="cuda")
    empty = [0, 3, 5]
    logits[empty] = -math.inf
    mask = None
    if masked:
        mask = torch.ones(6, entries, dtype=torch.bool, device="cuda")
        logits[5, ::2] = 1.0
        mask[5, ::2] = False  # what is left is -inf, or nothing
        tokens[5] = entries - 1
    logits.requires_grad_()
    lp, ent = fx.token_logprobs(logits, tokens, scale=1.3, mask=mask)
    assert (lp[empty] == -math.inf).all() and (ent[empty] == 0).all()
    for cots in ((torch.ones(6, device="cuda"), None), (torch.full((6,), -2.5, device="cuda"), torch.ones(6, device="cuda"))):
        outs, given = ((lp,), cots[:1]) if cots[1] is None else ((lp, ent), cots)
        (grad,) = torch.autograd.grad(outs, logits, given, retain_graph=True)
        assert (grad[empty] == 0).all()
        if entries > 1:
            assert all((grad[r] != 0).any() for r in (1, 2, 4))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("entries", [9, 40, 700, 1030, 9000, 70001])
def test_ties_of_signed_zeros_go_to_the_lowest_index(entries, masked, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.full((4, entries), -1.0, device="cuda")
    x[0, 0], x[0, 8] = -0.0, 0.0  # the later one is the positive zero, in another lane
    x[1, entries - 1], x[1, entries // 2] = 0.0, -0.0
    zeros = torch.rand(2, entries, generator=gen, device="cuda")
    x[2:] = torch.where(zeros < 0.5, -0.0, 0.0)
    x[3, ::3] = -1.0
    x = x.to(dtype)
    mask = torch.rand(4, entries, generator=gen, device="cuda") < 0.9 if masked else None
    live = x if mask is None else x.masked_fill(~mask, -math.inf)
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    for top in (1, 2, 9, 32):
        got = fx.token_logprobs(x, tokens, mask=mask, top=top)[3][:, :entries]
        want = torch.sort(live + 0.0, dim=-1, descending=True, stable=True)  # -0 + 0 is +0
        assert torch.equal(got, want.indices.masked_fill(want.values == -math.inf, -1)[:, :top])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_scales_at_their_ends(dtype):
    """Logits over the whole range of the type at the least and the largest scale; scales outside are refused by name."""
    x = torch.tensor([[-3e38, 3e38, 0.0, 1e30, -math.inf], [1.0, 1.0 + 2.0**-7, 0.0, -1.0, 1.0]], device="cuda").to(dtype)
    t = torch.tensor([1, 1], device="cuda")
    for scale in (1e-30, 1e30):
        lp, ent, best, index = fx.token_logprobs(x, t, scale=scale, top=2)
        assert lp[0] == 0 and ent[0] == 0 and best[0].tolist()[0] == 0 and index[0].tolist() == [1, 3]
        if scale > 1:
            assert lp[1] == 0 and ent[1] == 0 and index[1].tolist() == [1, 0]
        else:  # even odds
            assert (lp[1] + math.log(5)).abs() <= 2.0**-20 and (ent[1] - math.log(5)).abs() <= 2.0**-20
    for scale in (9e-31, 1e-44, 1e-60, 1.1e30):
        with pytest.raises(ValueError, match="scale"):
            fx.token_logprobs(x, t, scale=scale)
