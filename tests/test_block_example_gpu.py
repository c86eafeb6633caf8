"""The example of the attention-block operators with slogdet: its log|psi| and gradient against the
same network in 64 bits, a training step, and the moved electron's token."""

import math
import os
import sys

import pytest
import torch

from tests import block_refs as ref

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _plain(model, occ):
    """The example's forward in 64 bits from the plain forms."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in model.named_parameters()}
    x = z = p["embed.weight"][occ.long()]
    filling = torch.full((occ.shape[0], 1), occ.shape[1] / model.sites, dtype=torch.float64, device="cuda")
    for i, blk in enumerate(model.blocks):
        w = {n[len(f"blocks.{i}."):]: t for n, t in p.items() if n.startswith(f"blocks.{i}.")}
        b, n, width = x.shape
        y = (z @ w["qkv.weight"].T).view(b, n, blk.heads + 2 * blk.kv_heads, blk.dim).transpose(1, 2)
        q, k, v = y.split([blk.heads, blk.kv_heads, blk.kv_heads], 1)
        a = ref.attention(q, k, v, w["table"], q_pos=occ, k_pos=occ, max_distance=64)
        gate = torch.sigmoid(filling @ w["gate.weight"].T + w["gate.bias"])[:, None, :]
        x, z = ref.residual_norm(x, a.transpose(1, 2).reshape(b, n, width) @ w["out.weight"].T, w["post1"], w["pre1"],
                                 gate=gate, scale=w["scale1"])
        f = torch.nn.functional.silu(z @ w["up.weight"].T) @ w["down.weight"].T
        x, z = ref.residual_norm(x, f, w["post2"], w["pre2"], scale=w["scale2"])
    phi = z @ p["orbitals.weight"].T
    return torch.linalg.slogdet(phi / math.sqrt(phi.shape[-1]))[1], p


def test_example_matches_64_bits_and_trains(capsys):
    import neural_orbitals as ex

    model, occ, _ = ex.main(["--samples", "8", "--electrons", "12", "--sites", "40", "--steps", "2"])
    assert "step 1" in capsys.readouterr().out
    _, logabs = model(occ)
    want, p = _plain(model, occ)
    # log|det| of 12 x 12 float32 matrices, condition numbers up to 1e5
    assert (logabs.double() - want).abs().max() < 2e-2
    model.zero_grad()  # the training step left its own
    logabs.sum().backward()
    want.sum().backward()
    for n, t in model.named_parameters():
        g, h = t.grad.double(), p[n].grad
        assert torch.isfinite(g).all(), n
        assert (g - h).norm() <= 2e-2 * max(h.norm().item(), 1e-3), n


def test_example_bfloat16_runs_and_moved_token_matches(capsys):
    import neural_orbitals as ex

    model, occ, logabs = ex.main(["--samples", "4", "--electrons", "6", "--sites", "20", "--steps", "1", "--dtype",
                                  "bfloat16"])
    assert torch.isfinite(logabs).all()
    model = model.float()
    blk, z = model.blocks[0], model.embed(occ.long()).detach()
    site = (occ[:, 2] + 3).to(torch.int32)
    got = ex.moved_token(blk, z, occ, 2, site)
    q, k, v = (t.double() for t in blk.heads_of(z))
    keep = torch.ones_like(occ, dtype=torch.bool)
    keep[:, 2] = False
    want = ref.attention(q[:, :, 2:3], k, v, blk.table.double(), q_pos=site[:, None], k_pos=occ, key_mask=keep,
                         max_distance=64)
    assert (got.double() - want).abs().max() <= 2.0**-15 * want.abs().max()
