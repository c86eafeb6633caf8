"""The operators on tokens (token_embedding, fused_linear, token_logprobs) against plain 64-bit forms
on the same inputs.

Tolerances, with u the unit roundoff of the type (half a step: 2^-24, 2^-8; half 2^-11), each bound written where it
is used: a result rounded once is off by u of itself; a float32 sum of n terms by at most
n 2^-24 of the sum of their magnitudes, which bounds every product and table gradient here."""

import math

import pytest
import torch

import fermix_b200 as fx
from tests import token_refs as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "tanh"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _within(got, want, bound, name):
    """|got - want| <= bound, entry by entry, and the same entries finite."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, name
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), name
    assert torch.equal(torch.isnan(want), torch.isnan(got)), name
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), name
    err = torch.where(fine, (got - want).abs(), torch.zeros_like(want))
    over = (err - bound).max().item() if err.numel() else 0.0
    assert over <= 0, f"{name}: {err.max().item():.3g}, {over:.3g} above the bound"


# ------------------------------------------------------------------ embedding
# tokens' shape, rows, width
TABLES = [
    ((1,), 1, 1),
    ((3, 5), 7, 33),
    ((2048,), 64, 64),
    ((64, 32), 64, 64),
    ((4097,), 300, 40),
    ((5000,), 2047, 24),
    ((5000,), 2048, 24),
    ((3001,), 50001, 100),
    ((9, 1000), 513, 1000),
    ((2,), 20000, 2056),
    ((70000,), 3, 16),
    ((20000,), 1, 520),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape,rows,width", TABLES)
def test_embedding(shape, rows, width, dtype):
    gen = _gen(1)
    weight = _randn(gen, rows, width, dtype=dtype).requires_grad_()
    tokens = (torch.rand(shape, generator=gen, device="cuda").square() * rows).long().clamp(max=rows - 1)
    out = fx.token_embedding(tokens, weight, scale=1.7)
    w = weight.detach().double().requires_grad_()
    want = ref.embedding(tokens, w, 1.7)
    # the scale is float32 (2^-24), one product, one rounding
    _within(out, want, want.detach().abs() * (U[dtype] + 2.0**-22), "out")
    cot = _randn(gen, *shape, width, dtype=dtype)
    (grad,) = torch.autograd.grad(out, weight, cot)
    (wgrad,) = torch.autograd.grad(want, w, cot.double(), retain_graph=True)
    # sums of up to n terms, in float32: n 2^-24 of the magnitudes' sum
    (size,) = torch.autograd.grad(want, w, cot.double().abs())
    n = torch.bincount(tokens.reshape(-1), minlength=rows)[:, None]
    _within(grad, wgrad, wgrad.abs() * U[dtype] + size * (n + 4) * 2.0**-24, "grad")
    assert (grad[n[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("kind", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_embedding_token_types_and_layouts(kind):
    gen = _gen(2)
    weight = _randn(gen, 100, 48)
    tokens = torch.randint(0, 100, (17, 30), generator=gen, device="cuda").to(kind)
    want = weight[tokens.long()]
    assert torch.equal(fx.token_embedding(tokens, weight), want)
    assert torch.equal(fx.token_embedding(tokens.T, weight), want.transpose(0, 1))
    assert torch.equal(fx.token_embedding(tokens, weight.T.contiguous().T), want)
    wide = torch.cat([weight, weight], 1)
    assert torch.equal(fx.token_embedding(tokens, wide[:, 1:48]), want[..., 1:])  # off the 16-byte boundary


@pytest.mark.parametrize("count", [50, 9000])
def test_embedding_padding_and_tokens_outside(count):
    gen = _gen(3)
    weight = _randn(gen, 40, 16).requires_grad_()
    tokens = torch.randint(0, 40, (count,), generator=gen, device="cuda")
    tokens[::3] = -1
    tokens[1], tokens[4], tokens[7] = 40, -2, 2**40
    out = fx.token_embedding(tokens, weight, padding=-1)
    want = ref.embedding(tokens, weight.detach(), padding=-1)
    assert torch.equal(torch.nan_to_num(out, 7.0), torch.nan_to_num(want, 7.0))
    (grad,) = torch.autograd.grad(out, weight, torch.ones_like(out))
    n = torch.bincount(tokens[(tokens >= 0) & (tokens < 40)], minlength=40)
    assert torch.equal(grad, n[:, None].float().expand_as(grad))
    # a row of the table as the padding: zeros, and no gradient
    tokens = tokens.clamp(0, 39)
    out = fx.token_embedding(tokens, weight, padding=0)
    assert (out[tokens == 0] == 0).all() and torch.equal(out[tokens != 0], weight.detach()[tokens[tokens != 0]])
    (grad,) = torch.autograd.grad(out, weight, torch.ones_like(out))
    assert (grad[0] == 0).all() and torch.equal(grad[1:, 0], torch.bincount(tokens, minlength=40)[1:].float())


def test_embedding_gradient_of_one_frequent_token():
    # one token almost everywhere: its run crosses hundreds of windows
    for width in (16, 600, 2048):
        tokens = torch.full((40000,), 5, device="cuda")
        tokens[123] = 2
        weight = torch.zeros(70000, width, device="cuda", requires_grad=True)
        cot = torch.randint(-3, 4, (40000, width), device="cuda", generator=_gen(4)).float()
        (grad,) = torch.autograd.grad(fx.token_embedding(tokens, weight), weight, cot)
        assert torch.equal(grad[2], cot[123])
        assert torch.equal(grad[5], cot.double().sum(0).sub(cot[123]).float())  # whole numbers below 2^24: exact
        assert int((grad != 0).any(1).sum()) <= 2


def test_embedding_without_tokens():
    weight = torch.ones(5, 8, device="cuda", requires_grad=True)
    out = fx.token_embedding(torch.zeros(0, 3, dtype=torch.int64, device="cuda"), weight)
    assert out.shape == (0, 3, 8)
    (grad,) = torch.autograd.grad(out, weight, torch.zeros_like(out))
    assert (grad == 0).all()


# ------------------------------------------------------------------ linear
# rows, inner, outer
MAPS = [
    (1, 1, 1),
    (1, 1024, 512),
    (2, 33, 65),
    (5, 520, 129),
    (16, 256, 96),
    (17, 264, 300),
    (33, 1000, 77),
    (64, 64, 2048),
    (100, 72, 256),
    (129, 200, 1),
    (255, 31, 130),
    (512, 64, 128),
    (1000, 320, 200),
    (1, 8192, 40),
    (300, 2056, 264),
    (4100, 16, 24),
]


def _bounds(x, weight, bias, act, residual, cot, dtype):
    """64-bit values and bounds of the errors. A product's sum is off by at most e = (inner + 8) 2^-24 of
    the magnitudes' sum in float32; half of that many 2^-24 in the mean, so this bound is not near.
    The activations' slopes are at most 1.2 and their second derivatives at most 1.1, so act(h) moves by
    1.2 e, the slope by 1.1 e; their own evaluation is good to 2^-20 of 1 + |h|. In bfloat16 the factor
    g of the two products is rounded to 2^-8 and the slope kept to 2^-11."""
    u, slack = U[dtype], 2.0**-20
    t = [None if v is None else v.detach().double().requires_grad_() for v in (x, weight, bias, residual)]
    out = ref.linear(t[0], t[1], t[2], act, t[3])
    leaves = [v for v in t if v is not None]
    wants = torch.autograd.grad(out, leaves, cot.double())
    a, b = x.detach().double().abs(), weight.detach().double().abs()
    h = a @ b.T + (0 if bias is None else bias.detach().double().abs())
    k = x.shape[-1]
    e = (k + 8) * 2.0**-24 * h
    own = slack * (1 + h) if act else 0
    err_y = out.detach().abs() * u + 1.2 * e + own
    if residual is not None:
        err_y = err_y + residual.detach().double().abs() * 2.0**-23
    # g = dy act'(h)
    c = cot.double().abs()
    gerr = c * (1.1 * e * bool(act) + (slack if act else 0))
    gmax = c * (1.2 if act else 1.0)
    round_g = 0.0 if dtype == torch.float32 or act is None else 2.0**-8 + 2.0**-11
    rows, outer = cot.shape
    gerr = gerr + round_g * gmax + (2.0**-23 * gmax if act else 0)
    errs = [gerr @ b + (outer + 8) * 2.0**-24 * (gmax @ b), gerr.T @ a + (rows + 8) * 2.0**-24 * (gmax.T @ a)]
    if bias is not None:
        errs.append(gerr.sum(0) + (rows + 8) * 2.0**-24 * gmax.sum(0))
    if residual is not None:
        errs.append(torch.zeros_like(c))
    errs = [er + w.abs() * u for er, w in zip(errs, wants)]
    return out, wants, err_y, errs


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,inner,outer", MAPS)
def test_linear(rows, inner, outer, dtype):
    for i, act in enumerate(ACTS):
        gen = _gen(10 + i)
        x = _randn(gen, rows, inner, dtype=dtype).requires_grad_()
        weight = _randn(gen, outer, inner, dtype=dtype, scale=1.5 * inner**-0.5).requires_grad_()
        bias = _randn(gen, outer, dtype=dtype).requires_grad_() if i % 2 else None
        residual = _randn(gen, rows, outer, dtype=dtype).requires_grad_() if i % 3 == 1 else None
        cot = _randn(gen, rows, outer, dtype=dtype)
        want, wgrads, err, errs = _bounds(x, weight, bias, act, residual, cot, dtype)
        out = fx.fused_linear(x, weight, bias, activation=act, residual=residual)
        with torch.no_grad():
            assert torch.equal(out, fx.fused_linear(x, weight, bias, activation=act, residual=residual))
        _within(out, want, err, f"out, {act}")
        leaves = [t for t in (x, weight, bias, residual) if t is not None]
        grads = torch.autograd.grad(out, leaves, cot)
        names = [n for n, t in zip(("x", "weight", "bias", "residual"), (x, weight, bias, residual)) if t is not None]
        for n, g, w, e in zip(names, grads, wgrads, errs):
            _within(g, w, e, f"d_{n}, {act}")


# float32 on both sides of the sizes where its kernels take turns: groups of 64 of the lesser side, either side the
# longer one, rows off the 16-byte boundaries; long sums; and tiles cut along them
@pytest.mark.parametrize("rows,inner,outer", [
    (65, 40, 65), (130, 263, 300), (300, 264, 129), (1000, 64, 150), (97, 700, 770), (200, 1600, 66), (66, 2049, 70),
    (70, 2100, 90), (4000, 64, 65), (33, 4097, 2050), (2050, 100, 40), (5000, 60, 33), (4801, 24, 257), (16500, 100, 20)])
def test_linear_float32_between_kernels(rows, inner, outer):
    gen = _gen(rows)
    for act, withbias in ((None, True), ("gelu", False), ("silu", True)):
        x = _randn(gen, rows, inner).requires_grad_()
        weight = _randn(gen, outer, inner, scale=1.5 * inner**-0.5).requires_grad_()
        bias = _randn(gen, outer).requires_grad_() if withbias else None
        residual = _randn(gen, rows, outer).requires_grad_() if act else None
        cot = _randn(gen, rows, outer)
        want, wgrads, err, errs = _bounds(x, weight, bias, act, residual, cot, torch.float32)
        out = fx.fused_linear(x, weight, bias, activation=act, residual=residual)
        _within(out, want, err, f"out, {act}")
        leaves = [t for t in (x, weight, bias, residual) if t is not None]
        for g, w, e in zip(torch.autograd.grad(out, leaves, cot), wgrads, errs):
            _within(g, w, e, f"gradient, {act}")
        wide = _randn(gen, rows, inner + 5)[:, 3:inner + 3]  # another stride, off the boundaries
        with torch.no_grad():
            assert torch.equal(fx.fused_linear(wide, weight, bias), fx.fused_linear(wide.contiguous(), weight, bias))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows", [3, 70, 400])
def test_linear_strided_rows_and_leading_dimensions(rows, dtype):
    gen = _gen(30)
    wide, weights = _randn(gen, rows, 200, dtype=dtype), _randn(gen, 150, 96, dtype=dtype, scale=0.1)
    res = _randn(gen, rows, 99, dtype=dtype)
    for x, w in ((wide[:, 8:72], weights[3:40, 16:80]), (wide[:, 3:67], weights[:37, 1:65]),
                 (wide[:, :128:2], weights[:74:2, :64]), (wide[:64].T[:, :min(64, rows)], weights[:37, :min(64, rows)])):
        r = res[:1, 5:5 + w.shape[0]].expand(x.shape[0], -1)
        got = fx.fused_linear(x, w, activation="tanh", residual=r)
        assert torch.equal(got, fx.fused_linear(x.contiguous(), w.contiguous(), activation="tanh", residual=r.contiguous()))
    x = _randn(gen, 2, rows, 3, 64, dtype=dtype)
    w = weights[:37, :64]
    flat = fx.fused_linear(x.view(-1, 64), w)
    assert torch.equal(fx.fused_linear(x, w), flat.view(2, rows, 3, 37))
    assert fx.fused_linear(x[0, 0, 0], w).shape == (37,)
    t = x.transpose(1, 2)
    assert torch.equal(fx.fused_linear(t, w), fx.fused_linear(t.contiguous(), w))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_gradients_one_at_a_time_and_of_strided_cotangents(dtype):
    gen = _gen(31)
    tensors = [_randn(gen, 90, 72, dtype=dtype), _randn(gen, 56, 72, dtype=dtype, scale=0.1), _randn(gen, 56, dtype=dtype),
               _randn(gen, 90, 56, dtype=dtype)]
    cot = _randn(gen, 56, 90, dtype=dtype).T
    every = [t.clone().requires_grad_() for t in tensors]
    out = fx.fused_linear(every[0], every[1], every[2], activation="silu", residual=every[3])
    want = torch.autograd.grad(out, every, cot)
    for i in range(4):
        one = [t.clone().requires_grad_(i == j) for j, t in enumerate(tensors)]
        out = fx.fused_linear(one[0], one[1], one[2], activation="silu", residual=one[3])
        (got,) = torch.autograd.grad(out, one[i], cot)
        assert torch.equal(got, want[i]), i
    # a broadcast residual: its gradient is summed by what expanded it
    row = tensors[3][:1].clone().requires_grad_()
    out = fx.fused_linear(tensors[0], tensors[1], activation="relu", residual=row.expand(90, 56))
    (got,) = torch.autograd.grad(out, row, cot)
    # sums by torch in the type
    assert (got.double() - cot.double().sum(0, keepdim=True)).abs().max() <= 90 * U[dtype] * cot.double().abs().sum(0).max()


@pytest.mark.parametrize("act", ACTS[1:])
def test_linear_activations_at_their_ends(act):
    h = torch.tensor([-1e38, -1e4, -100.0, -89.0, -30.0, -14.5, -10.0, -6.0, -1.0, -1e-3, -1e-30, 0.0, 1e-30, 1e-3, 0.5, 3.0, 9.0,
                      15.0, 40.0, 100.0, 1e4, 1e38], device="cuda")
    x = h[:, None].clone().requires_grad_()
    one = torch.ones(1, 1, device="cuda")
    y = fx.fused_linear(x, one, activation=act)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    d = h.double()[:, None].clone().requires_grad_()
    want = ref.activation(d, act)
    (wg,) = torch.autograd.grad(want, d, torch.ones_like(want))
    if act == "gelu_tanh":  # 64-bit autograd multiplies infinities by zero at the ends
        wg = torch.where(d.detach().abs() > 1e3, (d.detach() > 0).double(), wg)
    assert torch.isfinite(y).all() and torch.isfinite(g).all()
    # the function to 2^-20 of 1 + |h|, absolute where it is small
    assert ((y.double() - want).abs() <= 2.0**-20 * (want.abs() + 1.0).clamp(max=1e38)).all()
    assert ((g.double() - wg).abs() <= 2.0**-18).all()


def test_linear_infinities_and_nan_stay_in_their_rows():
    gen = _gen(33)
    for dtype in TYPES:
        for rows in (4, 40, 300):
            x = _randn(gen, rows, 136, dtype=dtype)
            w = _randn(gen, 72, 136, dtype=dtype)
            want = fx.fused_linear(x, w)
            bad = x.clone()
            bad[1, 5], bad[3, 100] = math.nan, math.inf
            got = fx.fused_linear(bad, w)
            assert torch.isnan(got[1]).all() and not torch.isfinite(got[3]).any()
            keep = [i for i in range(rows) if i not in (1, 3)]
            assert torch.equal(got[keep], want[keep])


def test_linear_large_values_in_float32():
    x = torch.full((70, 64), 3.0e38, device="cuda")
    w = torch.full((40, 64), 2.0**-8, device="cuda")
    # 64 products of 1.17e36; float32 holds the sum
    got = fx.fused_linear(x, w)
    assert torch.allclose(got, torch.full_like(got, 3.0e38 * 2.0**-2), rtol=1e-6)
    tiny = torch.full((70, 64), 2.0**-120, device="cuda")
    got = fx.fused_linear(tiny, torch.ones(40, 64, device="cuda"))
    assert torch.allclose(got, torch.full_like(got, 2.0**-114), rtol=1e-6, atol=0)


def test_linear_without_rows():
    w = torch.ones(5, 8, device="cuda", requires_grad=True)
    b = torch.ones(5, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, 8, device="cuda", requires_grad=True)
    out = fx.fused_linear(x, w, b, activation="silu")
    assert out.shape == (0, 3, 5)
    grads = torch.autograd.grad(out, (x, w, b), torch.zeros_like(out))
    assert grads[0].shape == x.shape and (grads[1] == 0).all() and (grads[2] == 0).all()


# ------------------------------------------------------------------ log probabilities
# rows, entries
ROWS = [(1, 1), (3, 2), (5, 31), (64, 64), (7, 255), (64, 512), (33, 1000), (2, 2048), (9, 4099), (3, 20000), (2, 131071),
        (1, 65536), (300, 24), (4, 1024), (5, 1032)]


def _prob_bound(logits, scale, entries, want):
    """x - m is off by 2^-24 of itself, its exponential by 2^-22 and by 2^-23 |scale (x - m)|; the sum of
    `entries` terms, in parts, by 2^-20 of it at most; the subtraction rounds to 2^-23 of the value."""
    return 2.0**-19 + 2.0**-22 * want.detach().abs()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,entries", ROWS)
@pytest.mark.parametrize("masked", [False, True])
def test_logprobs(rows, entries, masked, dtype):
    gen = _gen(40)
    logits = _randn(gen, rows, entries, dtype=dtype, scale=3.0).requires_grad_()
    tokens = torch.randint(0, entries, (rows,), generator=gen, device="cuda")
    mask = torch.rand(rows, entries, generator=gen, device="cuda") < 0.5 if masked else None
    top = min(9, entries)
    d = logits.detach().double().requires_grad_()
    want = ref.logprobs(d, tokens, 0.8, mask, top)
    got = fx.token_logprobs(logits, tokens, scale=0.8, mask=mask, top=top)
    for n, a, b in zip(("logp", "entropy", "top_logp"), got, want):
        fine = torch.where(torch.isfinite(b), b, torch.zeros_like(b))
        _within(a, b, _prob_bound(logits, 0.8, entries, fine), n)
    assert torch.equal(got[3], want[3])  # bfloat16 has ties: the lowest index first
    with torch.no_grad():
        again = fx.token_logprobs(logits, tokens, scale=0.8, mask=mask)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    g, e = _randn(gen, rows), _randn(gen, rows)
    (grad,) = torch.autograd.grad(got[:2], logits, (g, e))
    # the formula in 64 bits; a row that nothing is left of has p = 0
    keep = torch.ones_like(d, dtype=torch.bool) if mask is None else mask
    logs = torch.log_softmax((d.detach() * 0.8).masked_fill(~keep, -math.inf), -1)
    logs = torch.where(keep, logs, torch.zeros_like(logs))
    p = torch.exp(logs) * keep
    hit = torch.nn.functional.one_hot(tokens, entries).double()
    ent = -(p * logs).sum(-1, keepdim=True)
    gd, ed = g.double()[:, None], e.double()[:, None]
    wgrad = torch.where(keep, 0.8 * (gd * (hit - p) - ed * p * (logs + ent)), torch.zeros_like(p))
    # p is off by 2^-19 of itself: 2^-22 from the exponential, 2^-23 of its argument (up to 2^6 / 4) and
    # the sum's; log p and the entropy by 2^-19 of 1 + their size
    bound = wgrad.abs() * U[dtype] + 2.0**-18 * p * (gd.abs() + ed.abs() * (logs.abs() + ent + 1)) + 2.0**-22 * gd.abs() * hit
    _within(grad, wgrad, bound, "d_logits")
    if masked:
        assert (grad[~mask] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("entries", [5, 70, 1500, 30000])
def test_logprobs_rows_that_leave_nothing_and_live_infinities(entries, dtype):
    gen = _gen(41)
    low = torch.finfo(dtype).min
    logits = _randn(gen, 12, entries, dtype=dtype)
    mask = torch.ones(12, entries, dtype=torch.bool, device="cuda")
    logits[0] = -math.inf
    mask[1] = False
    logits[1, :3] = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype)
    logits[2] = low  # all at the lowest value: even odds
    logits[3, 1:] = -math.inf
    mask[4, 2] = False
    logits[4, 2] = math.nan
    logits[5, 2] = math.nan
    logits[6, 2] = math.inf
    logits[7, 1:] = low
    logits[8, 1::2] = low
    logits[9] = 0
    logits[10, 2] = -math.inf
    tokens = torch.full((12,), 2, device="cuda")
    tokens[11] = entries
    x = logits.requires_grad_()
    lp, ent, best, index = fx.token_logprobs(x, tokens, mask=mask, top=4)
    (grad,) = torch.autograd.grad((lp, ent), x, (torch.ones_like(lp), torch.ones_like(ent)))
    n = math.log(entries)
    for r in (0, 1):
        assert lp[r] == -math.inf and ent[r] == 0 and (index[r] == -1).all() and (best[r] == -math.inf).all()
        assert (grad[r] == 0).all() or r == 0
    assert (grad[1] == 0).all()
    for r in (2, 9):
        assert abs(lp[r].item() + n) <= 2.0**-20 * (1 + n) and abs(ent[r].item() - n) <= 2.0**-20 * (1 + n)
        assert index[r].tolist() == [0, 1, 2, 3]
    for r in (3, 7):
        assert ent[r] == 0 and index[r, 0] == 0 and best[r, 0] == 0
    assert lp[3] == -math.inf and index[3, 1:].tolist() == [-1] * 3
    assert lp[4] == -math.inf and torch.isfinite(ent[4]) and not (index[4] == 2).any() and grad[4, 2] == 0
    for r in (5, 6):
        assert torch.isnan(lp[r]) and torch.isnan(ent[r]) and torch.isnan(best[r]).all() and (index[r] == -1).all()
        assert torch.isnan(grad[r]).any()
    assert torch.isfinite(ent[8]) and torch.isfinite(lp[8])
    assert lp[10] == -math.inf and torch.isfinite(ent[10])
    assert torch.isnan(lp[11]) and torch.isfinite(ent[11]) and torch.isfinite(grad[11]).all()
    assert torch.isfinite(grad[[2, 3, 4, 7, 8, 9]]).all()


@pytest.mark.parametrize("entries", [40, 3000, 40000])
def test_logprobs_padding_strides_and_shared_masks(entries):
    gen = _gen(42)
    wide = _randn(gen, 6, 10, entries + 8)
    logits = wide[:, :, 3:entries + 3]
    tokens = torch.randint(0, entries, (6, 10), generator=gen, device="cuda", dtype=torch.int32)
    tokens[:, 7:] = -100
    wide[:, 8] = math.nan
    mask = torch.rand(entries, generator=gen, device="cuda") < 0.7
    x = logits.detach().requires_grad_()
    lp, ent, best, index = fx.token_logprobs(x, tokens, mask=mask, top=3, padding=-100)
    clean = torch.nan_to_num(logits.contiguous())
    full = mask.expand(6, 10, entries)
    want = fx.token_logprobs(clean, tokens, mask=full, top=3, padding=-100)
    for a, b in zip((lp, ent, best), want):
        assert torch.allclose(a, b, rtol=2.0**-20, atol=2.0**-19)
    assert torch.equal(index, want[3])
    assert (lp[:, 7:] == 0).all() and (ent[:, 7:] == 0).all() and (index[:, 7:] == -1).all()
    (grad,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert (grad[:, 7:] == 0).all() and torch.isfinite(grad).all()
    (only,) = torch.autograd.grad(fx.token_logprobs(x, tokens, mask=mask, padding=-100)[1].sum(), x)
    assert (only[:, 7:] == 0).all() and torch.isfinite(only).all()


def test_logprobs_more_alternatives_than_entries_and_all_equal():
    lp, ent, best, index = fx.token_logprobs(torch.zeros(3, 5, device="cuda"), torch.tensor([0, 4, 2], device="cuda"), top=32)
    assert index[0].tolist() == [0, 1, 2, 3, 4] + [-1] * 27
    for entries in (700, 9000, 70000):
        x = torch.zeros(2, entries, device="cuda", dtype=torch.bfloat16)
        x[1, 11::13] = 1
        index = fx.token_logprobs(x, torch.zeros(2, dtype=torch.int64, device="cuda"), top=32)[3]
        assert index[0].tolist() == list(range(32)) and index[1].tolist() == list(range(11, 11 + 13 * 32, 13))
        ramp = torch.arange(entries, device="cuda").float()[None]  # every entry passes the last of the list
        index = fx.token_logprobs(ramp, torch.zeros(1, dtype=torch.int64, device="cuda"), top=32, scale=1e-3)[3]
        assert index[0].tolist() == list(range(entries - 1, entries - 33, -1))


def test_logprobs_gradient_against_differences():
    gen = _gen(43)
    x = _randn(gen, 2, 37).requires_grad_()
    t = torch.tensor([3, 30], device="cuda")
    f = lambda y: (lambda o: 1.3 * o[0].double().sum() - 0.7 * o[1].double().sum())(fx.token_logprobs(y, t, scale=1.2))
    (grad,) = torch.autograd.grad(f(x), x)
    step = 2.0**-5
    for i, j in ((0, 3), (0, 0), (1, 30), (1, 36)):
        up, down = x.detach().clone(), x.detach().clone()
        up[i, j] += step
        down[i, j] -= step
        slope = (f(up) - f(down)).item() / (up[i, j] - down[i, j]).item()
        # the third derivative, at most 10 or so, times step^2 / 6; rounding 2^-20 of 10 over the step
        assert abs(slope - grad[i, j].item()) <= 10 * step**2 / 6 + 2.0**-16 / step


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_model_of_all_three(dtype):
    """Padded sequences through embedding, two maps with a residual, tied logits and a loss, against 64 bits."""
    gen = _gen(50)
    V, W = 200, 64
    params = [_randn(gen, V, W, dtype=dtype), _randn(gen, 2 * W, W, dtype=dtype, scale=0.1), _randn(gen, 2 * W, dtype=dtype),
              _randn(gen, W, 2 * W, dtype=dtype, scale=0.1)]
    tokens = torch.randint(0, V, (7, 33), generator=gen, device="cuda")
    tokens[2, 20:] = -1
    target = torch.where(tokens < 0, -1, (tokens * 7 + 1) % V)

    def model(embed, linear, logprobs, table, up, bias, down):
        x = embed(tokens, table)
        x = linear(linear(x, up, bias, "gelu", None), down, None, None, x)
        lp, ent = logprobs(linear(x, table, None, None, None), target)
        return -lp.sum() - 0.1 * ent.sum()

    own = [p.clone().requires_grad_() for p in params]
    loss = model(lambda t, w: fx.token_embedding(t, w, scale=0.5, padding=-1),
                 lambda x, w, b, a, r: fx.fused_linear(x, w, b, activation=a, residual=r),
                 lambda x, t: fx.token_logprobs(x, t, padding=-1), *own)
    grads = torch.autograd.grad(loss, own)
    plain = [p.double().requires_grad_() for p in params]
    want = model(lambda t, w: ref.embedding(t, w, 0.5, -1), ref.linear, lambda x, t: ref.logprobs(x, t, padding=-1), *plain)
    wgrads = torch.autograd.grad(want, plain)
    # four roundings on the way in bfloat16, each of up to 2^-8 of its values: 2^-6 of a gradient's norm; float32's sums of up to 200 terms, 2^-15
    tol = 2.0**-6 if dtype == torch.bfloat16 else 2.0**-15
    assert abs(loss.item() - want.item()) <= tol * abs(want.item())
    for g, w in zip(grads, wgrads):
        assert (g.double() - w).norm() <= tol * w.norm()


def test_second_derivatives_are_refused():
    w = torch.randn(9, 8, device="cuda", requires_grad=True)
    t = torch.randint(0, 9, (5,), device="cuda")
    x = torch.randn(5, 8, device="cuda", requires_grad=True)
    for out, leaf in ((fx.token_embedding(t, w), w), (fx.fused_linear(x, w, activation="silu"), x),
                      (fx.token_logprobs(x, t.clamp(max=7))[0], x)):
        (g,) = torch.autograd.grad((out * out).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
