"""Tangents and function transforms, which the attention-block operators do not have, are refused by
name rather than dropped."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import fermix_b200 as fx

pytestmark = pytest.mark.gpu


def _calls():
    x, w = torch.randn(2, 4, 8, 16, device="cuda"), torch.ones(16, device="cuda")
    pos = torch.arange(8, device="cuda")
    table = torch.randn(4, 32, device="cuda")
    attn = {"q": x, "k": x + 1, "v": x + 2, "table": table}
    norm = {"x": x, "f": x + 1, "post_weight": w, "pre_weight": w + 1, "post_bias": w + 2, "pre_bias": w + 3,
            "gate": x + 2, "scale": w + 4}
    return [(fx.biased_attention, attn, {}), (fx.position_bias, {"table": table}, {"q_pos": pos}),
            (fx.residual_norm, norm, {})]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(3))
def test_a_tangent_is_refused_by_name(which, grad):
    fn, tensors, rest = _calls()[which]
    for name in tensors:
        with forward_ad.dual_level():
            args = {n: t.detach().requires_grad_(grad) for n, t in tensors.items()}
            fn(**args, **rest)  # a level alone changes nothing
            args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
            with pytest.raises(NotImplementedError, match=f"{name} carries a tangent"):
                fn(**args, **rest)


@pytest.mark.parametrize("which", range(3))
def test_function_transforms_are_refused_by_name(which):
    fn, tensors, rest = _calls()[which]
    for name, t in tensors.items():
        def of(x):
            out = fn(**{**tensors, name: x}, **rest)
            return out[0].sum() if isinstance(out, tuple) else out.sum()

        for transform in (lambda: torch.func.jvp(of, (t,), (t,)), lambda: torch.func.grad(of)(t),
                          lambda: torch.func.vmap(of)(t[None])):
            with pytest.raises(NotImplementedError, match=name):
                transform()
    if which < 2:
        pos = torch.arange(8, device="cuda")[None]
        with pytest.raises(NotImplementedError, match="q_pos"):
            torch.func.vmap(lambda p: fn(**tensors, q_pos=p))(pos)
    if which == 0:
        with pytest.raises(NotImplementedError, match="key_mask"):
            torch.func.vmap(lambda m: fn(**tensors, key_mask=m))(torch.ones(1, 2, 8, dtype=torch.bool, device="cuda"))
