"""residual_norm with an eps of zero, or one that float32 does not hold, at row counts that leave part
of a block without rows, against the plain 64-bit form. Tolerances as in test_block_gpu.py."""

import pytest
import torch

import fermix_b200 as fx
from tests import block_refs as ref
from tests.test_block_gpu import FORWARD, GRADIENT, IDS, TYPES, _close, _gen, _grads, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "full", "row", "group"])
@pytest.mark.parametrize("shape", [(1, 16), (3, 7, 16), (5, 3, 33), (1001, 128), (7, 143, 128), (3, 11, 250), (2, 3, 1000)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("eps", [0.0, 1e-60])
def test_gradient_without_eps(shape, kind, gate, eps, dtype):
    g = _gen(60)
    W = shape[-1]
    t = {"x": _randn(g, *shape, dtype=dtype), "f": _randn(g, *shape, dtype=dtype, scale=3.0),
         "post_weight": (1 + _randn(g, W, scale=0.2)).to(dtype), "pre_weight": (1 + _randn(g, W, scale=0.2)).to(dtype),
         "post_bias": _randn(g, W, dtype=dtype), "pre_bias": _randn(g, W, dtype=dtype), "scale": _randn(g, W, dtype=dtype)}
    if gate != "none":
        form = {"full": shape, "row": shape[:-1] + (1,), "group": (shape[0],) + (1,) * (len(shape) - 2) + (W,)}[gate]
        t["gate"] = _randn(g, *form, dtype=dtype)
    a = {n: x.requires_grad_(True) for n, x in t.items()}
    b = {n: x.detach().double().requires_grad_(True) for n, x in t.items()}
    got, want = fx.residual_norm(**a, kind=kind, eps=eps), ref.residual_norm(**b, kind=kind, eps=0.0)
    for n, x, y in zip("rz", got, want):
        _close(x, y, FORWARD[dtype], n)
    cot = [_randn(g, *shape, dtype=dtype) for _ in range(2)]
    exp = _grads(want, list(b.values()), [c.double() for c in cot])
    for n, x, y in zip(a, _grads(got, list(a.values()), cot), exp):
        _close(x, y, GRADIENT[dtype], n)
