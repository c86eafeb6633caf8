"""The example's network on the operators on tokens: the proposed moves' probabilities and their gradient against the
same formula in 64 bits."""

import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_proposals_of_the_example(dtype):
    import neural_orbitals as ex

    torch.manual_seed(1)
    model = ex.NeuralOrbitals(40, 12).cuda().to(dtype)
    occ = torch.rand(9, 40, device="cuda").topk(12).indices.sort().values.to(torch.int32)
    z = model.tokens(occ).detach().requires_grad_()
    free = torch.ones(9, 40, dtype=torch.bool, device="cuda").scatter_(1, occ.long(), False)
    site = free.float().argmax(1).to(torch.int32)
    site[0] = occ[0, 3]  # staying is a move
    site[1] = occ[1, 5]  # another electron's site is not
    logp, entropy, best, index = ex.proposal(model, z, occ, 3, site, top=4)
    free.scatter_(1, occ[:, 3:4].long(), True)
    x = z.detach().double().requires_grad_()
    logits = (x[:, 3] @ model.embed.weight.detach().double().T).to(dtype).double() if dtype == torch.bfloat16 else (
        x[:, 3] @ model.embed.weight.detach().double().T)
    want = torch.log_softmax((logits / 8).masked_fill(~free, -math.inf), -1)
    # logits of 64 terms up to about 20, rounded to the type (2^-8 of them, 2^-18 in float32), divided by 8
    tol = 2.0**-6 if dtype == torch.bfloat16 else 2.0**-15
    given = want.gather(1, site[:, None].long())[:, 0]
    assert logp[1] == -math.inf and given[1] == -math.inf
    fine = torch.isfinite(given)
    assert (logp.double() - given)[fine].abs().max() <= tol
    assert (entropy.double() + (want.exp() * want.masked_fill(~free, 0)).sum(1)).abs().max() <= 4 * tol
    assert (best.double() - want.topk(4).values).abs().max() <= tol
    assert free.gather(1, index).all()
    (grad,) = torch.autograd.grad(logp[fine].sum(), z)
    (wgrad,) = torch.autograd.grad(given[fine].sum(), x)
    assert (grad.double() - wgrad).norm() <= 2 * tol * wgrad.norm()
    assert (grad[:, :3] == 0).all()
