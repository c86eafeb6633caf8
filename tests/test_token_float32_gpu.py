"""The float32 products of fused_linear hold 24 bits: all three parts of an operand take part, and long sums are not left to
accumulators that cut off. Each case for the kernel of few or small rows and for the tiles, whole and split along k."""

import pytest
import torch

import fermix_b200 as fx

pytestmark = pytest.mark.gpu


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


# rows, inner: the rows' kernel, and tiles (whole and split)
@pytest.mark.parametrize("rows,inner", [(5, 512), (33, 300), (700, 64), (3000, 1000), (700, 2048), (20000, 512)])
def test_single_products(rows, inner):
    """A diagonal matrix leaves one product an entry. Of its value the terms left out (second by third part, twice, and
    third by third) are 2^-8 2^-16 each at most: 2^-23 together. Of the six that are added, each cut off below the sum's last
    bit (2^-23 of it at most), only those of the first parts are as large as the sum: 2^-23, and 2^-23 for the others; the
    result's rounding 2^-24. Below 2^-21 in all; without a third part it would be up to 2^-17."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x, d = _normal(gen, rows, inner), _normal(gen, inner)
    for w in (torch.ones_like(d), d):
        want = x.double() * w.double()
        assert ((fx.fused_linear(x, torch.diag(w)).double() - want).abs() <= 2.0**-21 * want.abs()).all()
        own = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(fx.fused_linear(own, torch.diag(w)), own, x)
        assert ((dx.double() - want).abs() <= 2.0**-21 * want.abs()).all()
    # one row of g, one of x: dW is their outer product
    w = torch.zeros(inner, inner, device="cuda", requires_grad=True)
    g, one = torch.zeros(rows, inner, device="cuda"), torch.zeros(rows, inner, device="cuda")
    g[rows // 2], one[rows // 2] = x[0], d
    (dw,) = torch.autograd.grad(fx.fused_linear(one, w), w, g)
    want = x[0].double()[:, None] * d.double()
    assert ((dw.double() - want).abs() <= 2.0**-21 * want.abs()).all()


# rows, outer: few rows, the rows' kernel; tiles split along k; tiles whole
@pytest.mark.parametrize("rows,outer", [(16, 1000), (150, 300), (600, 700), (2600, 2100)])
@pytest.mark.parametrize("inner", [2048, 8192])
def test_long_sums_are_not_cut_off(rows, outer, inner):
    """Of positive terms a sum that stays in an accumulator loses half a last bit (2^-23 of it at most) with every
    addition, always downwards, and is half of the whole in the mean: 2^-25 of the whole an addition. There are 24 for each 64
    entries, so with all of k in one accumulator 768 2^-25 = 2^-15.4 at 2048 entries; of sums that end after 128 entries at
    most, 48 2^-25 = 12 2^-23. The additions between those are rounded to nearest: no sign, and 2^-24 sqrt(64) or less in the
    mean square. The mean is held to 16 2^-23 = 2^-19, the largest to twice that.
    With random signs the sums grow as the root of k: what a sum of 128 entries loses, 12 2^-23 of its size, adds up over
    them as their sizes do, and the roundings between them, 2^-24 sqrt(64) / 2 or less, stay below 16 2^-23 together with it."""
    gen = torch.Generator(device="cuda").manual_seed(inner)
    x = torch.rand(rows, inner, generator=gen, device="cuda") + 0.5
    w = torch.rand(outer, inner, generator=gen, device="cuda") + 0.5
    want = x.double() @ w.double().T
    off = (fx.fused_linear(x, w).double() - want) / want
    assert off.mean().abs() <= 2.0**-19 and off.abs().max() <= 2.0**-18
    x, w = _normal(gen, rows, inner), _normal(gen, outer, inner)
    size = ((x.double()**2) @ (w.double()**2).T).sqrt()
    off = (fx.fused_linear(x, w).double() - x.double() @ w.double().T) / size
    assert off.square().mean().sqrt() <= 2.0**-19
