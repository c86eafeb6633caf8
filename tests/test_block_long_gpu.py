"""Output and gradients of long sequences in the norm of the difference, which a dropped row or tile
shows in: the largest entry of 4096 rows does not.

Tolerances, of the 64-bit result's norm: bfloat16 rounds the probabilities and the output once each
(2^-8 for the output), and for a gradient p or ds, the saved output in delta, and the result, each
2^-9 at most: 2^-7. A missing tile of 128 of 1100 keys is 2^-3, one row of 1023 2^-5. float32: those of
test_block_gpu.py."""

import pytest
import torch

import fermix_b200 as fx
from tests import block_refs as ref
from tests.test_block_gpu import FORWARD, GRADIENT, IDS, TYPES, _attention_case, _grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(2, 4, 2, 1023, 1100, 64), (1, 2, 1, 2047, 2049, 64), (1, 4, 1, 700, 1500, 128),
                                   (3, 2, 2, 513, 511, 40), (1, 2, 2, 1100, 900, 33)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("form", ["plain", "sites", "causal", "prefix"])
def test_norm_of_the_difference(shape, form, dtype):
    t, kw, cot = _attention_case(shape, dtype, 90, "sites" if form == "sites" else "end", form == "sites")
    more = {}
    if form == "causal":
        more["causal"] = True
    if form == "prefix":  # lengths of their own, as of padded samples
        n = torch.tensor([shape[4] // 3, shape[4], shape[4] - 1], device="cuda")[: shape[0]]
        kw["key_mask"] = torch.arange(shape[4], device="cuda") < n[:, None]
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    b = {n: x.detach().double().requires_grad_(True) for n, x in t.items()}
    out, want = fx.biased_attention(**a, **kw, **more), ref.attention(**b, **kw, **more)
    tol = 2.0**-8 if dtype == torch.bfloat16 else FORWARD[dtype]
    assert ((out.double() - want).norm() / want.norm()).item() <= tol
    tol = 2.0**-7 if dtype == torch.bfloat16 else GRADIENT[dtype]
    got, exp = _grads(out, list(a.values()), cot), _grads(want, list(b.values()), cot.double())
    top = max(y.abs().max().item() for y in exp)
    for n, x, y in zip(a, got, exp):
        # keys that all share one bucket give the table no gradient: held to a hundredth of the others' entries
        size = max(y.norm().item(), 0.01 * top * y.numel() ** 0.5)
        assert (x.double() - y).norm().item() <= tol * size, n
