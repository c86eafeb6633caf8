"""What the refusals of the operators on tokens say (no GPU needed)."""

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from fermix_b200.build import build

    build()
    return _lib.lib()


def test_refused_transforms_name_no_other_operator():
    t = torch.zeros(3, dtype=torch.int64)
    for call in (lambda w: fx.token_embedding(t, w), lambda w: fx.fused_linear(w, w), lambda w: fx.token_logprobs(w, t)[0]):
        with pytest.raises(NotImplementedError, match="torch.func") as error:
            torch.func.grad(lambda w: call(w).sum())(torch.zeros(3, 8))
        assert "attention" not in str(error.value)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(torch.zeros(3, 8), torch.ones(3, 8))
            with pytest.raises(NotImplementedError, match="tangent") as error:
                call(dual)
            assert "attention" not in str(error.value)


def test_a_bad_shape_names_the_limits_of_all_operators(lib):
    text = lib.fermix_strerror(2).decode()
    assert "fermix_b200_block.h" in text and "fermix_b200_token.h" in text
