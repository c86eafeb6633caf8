"""Waits that run out in the attention kernels, forward and gradient: with no polls allowed every wait
gives up at once, the call returns with nothing under way, the status says so, what depends on it is
NaN, and the next call is right again."""

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib
from tests.test_block_gpu import IDS, TYPES, _attention_case, _grads

pytestmark = pytest.mark.gpu

# fewer, as many and more tiles than are under way at a time; one and two query tiles a block
SHAPES = [(1, 2, 2, 100, 60, 64), (2, 2, 1, 256, 256, 32), (1, 2, 1, 300, 1000, 64), (1, 2, 2, 300, 700, 128)]


def _case(shape, dtype, mask):
    t, kw, cot = _attention_case(shape, dtype, 80, "sites", mask)
    return {n: x.detach().requires_grad_(True) for n, x in t.items()}, kw, cot


class _NoPolls:
    def __enter__(self):
        self.before = _lib.lib().fermix_set_wait_polls(0)

    def __exit__(self, *_):
        _lib.lib().fermix_set_wait_polls(self.before)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("mask", [False, True])
def test_forward(shape, mask, dtype):
    a, kw, _ = _case(shape, dtype, mask)
    with torch.no_grad():
        want = fx.biased_attention(**a, **kw)
        assert _lib.device_status(clear=True) == 0
        with _NoPolls():
            out = fx.biased_attention(**a, **kw)
            assert _lib.device_status(clear=True) == _lib.FX_ERR_TIMEOUT
        assert torch.isnan(out).all()
        assert torch.equal(fx.biased_attention(**a, **kw), want)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("mask", [False, True])
def test_gradient(shape, mask, dtype):
    if dtype == torch.float32 and shape[-1] > 64:
        pytest.skip("no waits on this path")
    a, kw, cot = _case(shape, dtype, mask)
    out = fx.biased_attention(**a, **kw)
    leaves = list(a.values())
    want = torch.autograd.grad(out, leaves, cot, retain_graph=True)
    assert _lib.device_status(clear=True) == 0
    with _NoPolls():
        got = torch.autograd.grad(out, leaves, cot, retain_graph=True)
        assert _lib.device_status(clear=True) == _lib.FX_ERR_TIMEOUT
    if not mask:
        for n, x in zip(a, got):
            assert torch.isnan(x).all(), n
    for x, y in zip(_grads(out, leaves, cot), want):
        assert torch.equal(x, y)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_of_rows_without_a_sum(shape, dtype):
    """Scores that never came leave a row's sum at zero as a row without keys has it: NaN all the same."""
    a, kw, _ = _case(shape, dtype, False)
    a["table"] = torch.full_like(a["table"], -float("inf"))
    with torch.no_grad(), _NoPolls():
        out = fx.biased_attention(**a, **kw)
        assert _lib.device_status(clear=True) == _lib.FX_ERR_TIMEOUT
    assert torch.isnan(out).all()
    with torch.no_grad():
        assert (fx.biased_attention(**a, **kw) == 0).all()
