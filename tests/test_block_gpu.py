"""The attention-block operators (biased_attention, position_bias, residual_norm) against plain
64-bit forms on the same inputs.

Tolerances, as a part of the largest magnitude of the 64-bit result, with u the unit roundoff
of the type (2^-24, 2^-9). Forward: in bfloat16 the probabilities and the result are each
rounded once and the products are exact in float32, 8 u covers these two with the sums' spread;
in float32 the scores' dot products (up to 128 terms) and the exponential of scores up to about
20 carry some 2^8 u, 2^9 u allows for both. Gradients: three more rounded quantities (the score
gradients, the saved result in its row products, the result), four times the forward's.
Channel and table gradients are sums over many rows, whose rounding errors have no common sign:
the same bound."""

import pytest
import torch

import fermix_b200 as fx
from tests import block_refs as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
FORWARD = {torch.float32: 2.0**-15, torch.bfloat16: 2.0**-6}
GRADIENT = {torch.float32: 2.0**-13, torch.bfloat16: 2.0**-4}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _close(got, want, tol, name):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), name
    if want.numel():
        err, top = (got - want).abs().max().item(), want.abs().max().item()
        assert err <= tol * max(top, 1e-30), f"{name}: {err:.3g} of {top:.3g}"


def _grads(out, leaves, cot):
    return torch.autograd.grad(out, leaves, cot, allow_unused=True)


# ------------------------------------------------------------------ attention
# batch, heads, key heads, q_len, k_len, dim
SHAPES = [
    (1, 1, 1, 1, 1, 1),
    (2, 2, 1, 3, 5, 7),
    (1, 4, 2, 17, 33, 16),
    (2, 2, 2, 64, 64, 32),
    (3, 2, 1, 129, 257, 64),
    (2, 4, 1, 1, 300, 40),
    (1, 2, 2, 200, 130, 128),
    (1, 2, 2, 65, 63, 96),
    (1, 8, 2, 1, 1025, 64),
    (1, 3, 3, 255, 255, 33),
    (2, 6, 2, 5, 700, 128),
    (1, 1, 1, 513, 511, 8),
]


def _attention_case(shape, dtype, seed, positions="end", mask=False, buckets=32):
    B, H, Hk, Lq, Lk, D = shape
    g = _gen(seed)
    t = {
        "q": _randn(g, B, Lq, H, D, dtype=dtype).transpose(1, 2),
        "k": _randn(g, B, Lk, Hk, D, dtype=dtype).transpose(1, 2),
        "v": _randn(g, B, Lk, Hk, D, dtype=dtype).transpose(1, 2),
        "table": _randn(g, H, buckets, dtype=dtype),
    }
    kw = {}
    if positions == "sites":  # unsorted, of both signs, another set for each sample
        kw["q_pos"] = torch.randint(-400, 400, (B, Lq), generator=g, device="cuda")
        kw["k_pos"] = torch.randint(-400, 400, (B, Lk), generator=g, device="cuda", dtype=torch.int32)
    if mask:
        kw["key_mask"] = torch.rand(B, Lk, generator=g, device="cuda") < 0.6
    return t, kw, _randn(g, B, H, Lq, D, dtype=dtype)


def _check_attention(t, kw, cot, dtype, max_distance=128, two_sided=True, **more):
    leaves = [n for n in ("q", "k", "v", "table") if t.get(n) is not None]
    a = {n: t[n].detach().requires_grad_(True) for n in leaves}
    b = {n: t[n].detach().double().requires_grad_(True) for n in leaves}
    out = fx.biased_attention(**a, **kw, **more, max_distance=max_distance, bidirectional=two_sided)
    want = ref.attention(**b, **kw, **more, max_distance=max_distance, two_sided=two_sided)
    assert out.dtype == dtype
    _close(out, want, FORWARD[dtype], "out")
    with torch.no_grad():
        _close(fx.biased_attention(**a, **kw, **more, max_distance=max_distance, bidirectional=two_sided), want,
               FORWARD[dtype], "out without gradient")
    got = _grads(out, [a[n] for n in leaves], cot)
    exp = _grads(want, [b[n] for n in leaves], cot.double())
    top = max(e.abs().max().item() for e in exp if e.numel())
    for n, x, y in zip(leaves, got, exp):
        # a gradient that cancels to little beside the others is held to a hundredth of theirs
        x, y = x.double(), y.double()
        assert torch.isfinite(x).all(), n
        if y.numel():
            assert (x - y).abs().max().item() <= GRADIENT[dtype] * max(y.abs().max().item(), 0.01 * top), n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_default_positions(shape, dtype):
    _check_attention(*_attention_case(shape, dtype, 1), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_sites_and_mask(shape, dtype):
    _check_attention(*_attention_case(shape, dtype, 2, "sites", True, 16), dtype, max_distance=300)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_causal_one_sided(shape, dtype):
    _check_attention(*_attention_case(shape, dtype, 3), dtype, two_sided=False, causal=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [SHAPES[2], SHAPES[4], SHAPES[8]], ids=lambda s: "x".join(map(str, s)))
def test_attention_causal_by_sites(shape, dtype):
    # a query whose position is before every key's has no key
    _check_attention(*_attention_case(shape, dtype, 4, "sites", True), dtype, causal=True, scale=0.3)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [SHAPES[3], SHAPES[5], SHAPES[6]], ids=lambda s: "x".join(map(str, s)))
def test_attention_without_table(shape, dtype):
    t, kw, cot = _attention_case(shape, dtype, 5, mask=True)
    t.pop("table")
    _check_attention(t, kw, cot, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("buckets,distance,two_sided", [(1, 4, False), (2, 8, True), (2, 8, False), (256, 2048, True),
                                                        (255, 2048, False)])
def test_attention_bucket_counts(buckets, distance, two_sided, dtype):
    t, kw, cot = _attention_case((1, 2, 1, 130, 190, 32), dtype, 6, "sites", buckets=buckets)
    kw = {n: p * 7 for n, p in kw.items()}
    _check_attention(t, kw, cot, dtype, max_distance=distance, two_sided=two_sided)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len,k_len", [(0, 5), (4, 0), (0, 0)])
def test_attention_of_length_zero(q_len, k_len, dtype):
    t, kw, cot = _attention_case((2, 2, 1, q_len, k_len, 16), dtype, 7)
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    out = fx.biased_attention(**a)
    assert out.shape == (2, 2, q_len, 16) and (out == 0).all()
    for n, g in zip(a, _grads(out, list(a.values()), cot)):
        assert g.shape == a[n].shape and (g == 0).all(), n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len,k_len,dim", [(1, 40, 64), (1, 1000, 64), (70, 200, 64), (150, 150, 32)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_masked_keys_may_hold_anything(q_len, k_len, dim, poison, dtype):
    """NaN and infinities in masked keys, one sample without any key: zero rows, zero gradients."""
    t, kw, cot = _attention_case((3, 2, 1, q_len, k_len, dim), dtype, 8, mask=True)
    kw["key_mask"][1] = False
    kw["key_mask"][2, :] = False
    kw["key_mask"][2, k_len // 2] = True
    dead = ~kw["key_mask"][:, None, :, None]
    clean = {n: x.clone() for n, x in t.items()}
    t["k"] = t["k"].masked_fill(dead, poison)
    t["v"] = t["v"].masked_fill(dead, poison)
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    out = fx.biased_attention(**a, **kw)
    grads = _grads(out, list(a.values()), cot)
    c = {n: x.detach().requires_grad_(True) for n, x in clean.items()}
    out2 = fx.biased_attention(**c, **kw)
    assert torch.equal(out, out2)
    for n, x, y in zip(a, grads, _grads(out2, list(c.values()), cot)):
        assert torch.equal(x, y), n
    assert (out[1] == 0).all() and (grads[0][1] == 0).all() and (grads[1][1] == 0).all() and (grads[2][1] == 0).all()
    assert (grads[1].masked_select(dead) == 0).all() and (grads[2].masked_select(dead) == 0).all()
    _check_attention(clean, kw, cot, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len", [1, 100])
def test_bucket_of_minus_infinity_and_of_the_lowest_value(q_len, dtype):
    """A table entry of -inf leaves its pairs out; one of the type's lowest value does so where any
    other is there, and a row of nothing else is the plain mean."""
    t, kw, cot = _attention_case((1, 2, 2, q_len, 120, 32), dtype, 9, buckets=8)
    t["table"][0, :4] = -float("inf")  # keys at and before the query
    t["table"][1, :] = torch.finfo(dtype).min
    out = fx.biased_attention(**t)
    b = {n: x.double() for n, x in t.items()}
    _close(out, ref.attention(**b), FORWARD[dtype], "out")
    assert (out[0, 0, -1] == 0).all()  # the last query has no key left
    _close(out[0, 1], t["v"][0, 1].double().mean(0).expand(q_len, -1), FORWARD[dtype], "mean")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len", [1, 150])
def test_nan_in_a_live_place_reaches_its_rows_only(q_len, dtype):
    t, kw, cot = _attention_case((2, 2, 2, q_len, 150, 64), dtype, 10)
    t["q"][0, 1, q_len // 2, 3] = float("nan")
    out = fx.biased_attention(**t)
    bad = torch.isnan(out).any(-1)
    assert bad[0, 1, q_len // 2] and bad.sum() == 1
    t, kw, cot = _attention_case((2, 2, 2, q_len, 150, 64), dtype, 10)
    t["k"][1, 0, 100, 0] = float("nan")
    bad = torch.isnan(fx.biased_attention(**t)).any(-1)
    assert bad[1, 0].all() and bad.sum() == q_len


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len", [1, 140])
def test_attention_strides_and_broadcast(q_len, dtype):
    """Head-major, token-major, sliced (unaligned), reversed-order and expanded inputs give the bits of
    contiguous ones; an expanded input's gradient is the sum over its copies."""
    g = _gen(11)
    big = {n: _randn(g, 2, 4, L, 72, dtype=dtype) for n, L in (("q", q_len), ("k", 150), ("v", 150))}
    table = _randn(g, 4, 32, dtype=dtype)
    for cut in (slice(0, 64), slice(1, 65), slice(8, 72)):
        x = {n: y[..., cut] for n, y in big.items()}
        whole = fx.biased_attention(*(y.contiguous() for y in x.values()), table)
        assert torch.equal(fx.biased_attention(**x, table=table), whole)
        token = {n: y.transpose(1, 2).contiguous().transpose(1, 2) for n, y in x.items()}
        assert torch.equal(fx.biased_attention(**token, table=table), whole)
        inner = {n: y.transpose(2, 3).contiguous().transpose(2, 3) for n, y in x.items()}
        assert torch.equal(fx.biased_attention(**inner, table=table), whole)
    q = big["q"][..., :64].detach().requires_grad_(True)
    k1, v1 = (big[n][:1, :1, :, :64].detach().requires_grad_(True) for n in ("k", "v"))
    out = fx.biased_attention(q, k1.expand(2, 4, -1, -1), v1.expand(2, 4, -1, -1), table)
    cot = _randn(g, *out.shape, dtype=dtype)
    d = [t.detach().double().requires_grad_(True) for t in (q, k1, v1)]
    want = ref.attention(d[0], d[1].expand(2, 4, -1, -1), d[2].expand(2, 4, -1, -1), table.double())
    _close(out, want, FORWARD[dtype], "out")
    for n, x, y in zip("qkv", _grads(out, [q, k1, v1], cot), _grads(want, d, cot.double())):
        _close(x, y, GRADIENT[dtype], n)
    # a cotangent of one value, expanded
    kv = (k1.expand(2, 4, -1, -1), v1.expand(2, 4, -1, -1))
    (x,) = _grads(fx.biased_attention(q, *kv, table).sum(), [q], None)
    (y,) = _grads(fx.biased_attention(q, *kv, table), [q], torch.ones(q.shape, dtype=dtype, device="cuda"))
    assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_gradient_against_differences(dtype):
    """The directional derivative along the gradient itself, from central differences of the
    64-bit form at the same inputs: step 2^-10 of the inputs' norm, truncation about its square."""
    t, kw, cot = _attention_case((2, 4, 2, 70, 90, 48), dtype, 12, "sites", True)
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    grads = _grads(fx.biased_attention(**leaves, **kw), list(leaves.values()), cot)
    for (n, x), g in zip(t.items(), grads):
        d = g.double() / g.double().norm()
        h = 2.0**-10 * x.double().norm()

        def value(sign):
            b = {m: y.double() for m, y in t.items()}
            b[n] = b[n] + sign * h * d
            return (ref.attention(**b, **kw) * cot.double()).sum()

        slope = (value(1) - value(-1)) / (2 * h)
        assert abs(slope / g.double().norm() - 1) < GRADIENT[dtype] + 1e-3, n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_repeats_bit_for_bit_and_on_other_streams(dtype):
    t, kw, cot = _attention_case((4, 8, 2, 300, 333, 64), dtype, 13, "sites", True)

    def run():
        a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
        out = fx.biased_attention(**a, **kw)
        return [out.detach(), *_grads(out, list(a.values()), cot)]

    first = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = run()
    s.synchronize()
    for x, y in zip(first, second):
        assert torch.equal(x, y)


def test_attention_offsets_past_32_bits():
    """A cache whose last tokens start more than 2^32 elements into their storage."""
    big = torch.empty(1, 1, 70_000, 65_536, dtype=torch.bfloat16, device="cuda")  # 9.2 GB
    g = _gen(14)
    k = big[..., :64]
    k.copy_(_randn(g, 1, 1, 70_000, 64, dtype=torch.bfloat16))
    for q_len in (1, 130):
        q = _randn(g, 1, 1, q_len, 64, dtype=torch.bfloat16, scale=3.0)
        want = ref.attention(q.double(), k.double(), k.double())
        _close(fx.biased_attention(q, k, k), want, FORWARD[torch.bfloat16], "out")


# ------------------------------------------------------------------ position bias
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("batch,heads,q_len,k_len", [(0, 1, 1, 1), (0, 3, 5, 7), (2, 1, 1, 33), (3, 2, 130, 255),
                                                     (0, 2, 257, 1032), (0, 5, 64, 2049), (1, 2, 0, 4), (0, 2, 4, 0)])
@pytest.mark.parametrize("buckets,distance,two_sided", [(32, 128, True), (16, 40, False), (1, 4, False), (2, 4, True),
                                                        (256, 2048, True)])
def test_position_bias(batch, heads, q_len, k_len, buckets, distance, two_sided, dtype):
    g = _gen(20)
    lead = (batch,) if batch else ()
    q_pos = torch.randint(-1500, 1500, (*lead, q_len), generator=g, device="cuda")
    k_pos = torch.arange(-k_len // 2, k_len - k_len // 2, device="cuda", dtype=torch.int32)
    if batch:
        k_pos = torch.randint(-1500, 1500, (batch, k_len), generator=g, device="cuda", dtype=torch.int32)
    table = _randn(g, heads, buckets, dtype=dtype).requires_grad_(True)
    out = fx.position_bias(table, q_pos, k_pos, max_distance=distance, bidirectional=two_sided)
    t64 = table.detach().double().requires_grad_(True)
    want = ref.position_bias(t64, q_pos, k_pos, distance, two_sided)
    assert out.dtype == dtype and torch.equal(out.double(), want)
    cot = _randn(g, *out.shape, dtype=dtype)
    (x,), (y,) = _grads(out, [table], cot), _grads(want, [t64], cot.double())
    _close(x, y, FORWARD[dtype], "table")
    (z,) = _grads(fx.position_bias(table, q_pos, k_pos, max_distance=distance, bidirectional=two_sided), [table], cot)
    assert torch.equal(x, z)


def test_position_bias_far_positions_and_gradient_differences():
    g = _gen(21)
    pos = torch.tensor([-(2**30), -5, 0, 3, 2**30 - 1], device="cuda")
    table = _randn(g, 2, 32).requires_grad_(True)
    out = fx.position_bias(table, pos)
    assert torch.equal(out, ref.position_bias(table, pos, pos, 128, True))
    # linear in the table: differences are exact up to rounding
    cot = _randn(g, 2, 5, 5)
    (grad,) = _grads(out, [table], cot)
    step = _randn(g, 2, 32)
    with torch.no_grad():
        change = ((fx.position_bias(table + step, pos) - fx.position_bias(table - step, pos)) * cot).double().sum() / 2
    assert abs(change - (grad * step).double().sum()) < 1e-5 * (grad * step).double().abs().sum()


def test_position_bias_agrees_with_the_attention():
    """The attention's own bias is the materialised one: softmax(bias) v."""
    g = _gen(22)
    table, v = _randn(g, 4, 32), _randn(g, 2, 4, 99, 32)
    pos = torch.randint(0, 300, (2, 99), generator=g, device="cuda", dtype=torch.int32)
    out = fx.biased_attention(torch.zeros_like(v), v, v, table, q_pos=pos, k_pos=pos)
    want = torch.softmax(fx.position_bias(table, pos).double(), -1) @ v.double()
    _close(out, want, FORWARD[torch.float32], "out")


# ------------------------------------------------------------------ residual norm
NORM_SHAPES = [(1, 1), (3, 5), (2, 7, 16), (5, 33), (4, 3, 128), (2, 61, 255), (9, 256), (3, 17, 500), (7, 1000),
               (2, 3, 1001), (5, 2048), (3, 4096), (2, 4100), (2, 8192), (1, 8191), (0, 64), (2, 0, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("gate", ["none", "full", "row", "group", "middle"])
def test_residual_norm(shape, kind, gate, dtype):
    g = _gen(30)
    W = shape[-1]
    t = {"x": _randn(g, *shape, dtype=dtype), "f": _randn(g, *shape, dtype=dtype, scale=3.0),
         "post_weight": (1 + _randn(g, W, scale=0.2)).to(dtype), "pre_weight": (1 + _randn(g, W, scale=0.2)).to(dtype)}
    if kind == "layer" or gate == "row":
        t["post_bias"], t["pre_bias"] = _randn(g, W, dtype=dtype), _randn(g, W, dtype=dtype)
    if gate != "none":
        t["scale"] = _randn(g, W, dtype=dtype)
        lead = len(shape) - 1
        form = {"full": shape, "row": shape[:-1] + (1,), "group": (shape[0],) + (1,) * (lead - 1) + (W,),
                "middle": (1,) * lead + (1,)}[gate]
        t["gate"] = _randn(g, *form, dtype=dtype)
    a = {n: x.requires_grad_(True) for n, x in t.items()}
    b = {n: x.detach().double().requires_grad_(True) for n, x in t.items()}
    r, z = fx.residual_norm(**a, kind=kind, eps=1e-5)
    r64, z64 = ref.residual_norm(**b, kind=kind, eps=1e-5)
    assert r.dtype == z.dtype == dtype
    _close(r, r64, FORWARD[dtype], "r")
    _close(z, z64, FORWARD[dtype], "z")
    cr, cz = _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)
    for outs, cots in (((0, 1), (0, 1)), ((0,), (0,)), ((1,), (1,))):
        got = _grads([(r, z)[i] for i in outs], list(a.values()), [(cr, cz)[i] for i in cots]) if len(outs) == 2 else \
            _grads((fx.residual_norm(**a, kind=kind, eps=1e-5))[outs[0]], list(a.values()), (cr, cz)[cots[0]])
        exp = torch.autograd.grad([(r64, z64)[i] for i in outs], list(b.values()),
                                  [(cr, cz)[i].double() for i in cots], allow_unused=True, retain_graph=True)
        for n, x, y in zip(a, got, exp):
            y = torch.zeros_like(b[n]) if y is None else y
            x = torch.zeros_like(a[n]) if x is None else x
            # a width of 1 or 2 makes the norm's own gradient cancel exactly or nearly
            floor = 1.0 if W < 8 else 1e-30
            assert torch.isfinite(x).all(), n
            if y.numel():
                err, top = (x.double() - y).abs().max().item(), max(y.abs().max().item(), floor)
                assert err <= GRADIENT[dtype] * top, f"{n} {outs}: {err:.3g} of {top:.3g}"


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_residual_norm_strides_offsets_and_streams(dtype):
    g = _gen(31)
    big = _randn(g, 6, 40, 130, dtype=dtype)
    w = _randn(g, 131, dtype=dtype)
    x, f = big[:3, :, 1:129], big[3:, :, 2:130]
    want = fx.residual_norm(x.contiguous(), f.contiguous(), w[:128].clone(), w[2:130].clone())
    for got in (fx.residual_norm(x, f, w[:128], w[2:130]),
                fx.residual_norm(x.transpose(0, 1).contiguous().transpose(0, 1), f, w[:128], w[2:130])):
        for u, v in zip(got, want):
            assert torch.equal(u, v)
    # unaligned storage (one entry off a 16-byte boundary)
    flat = torch.empty(3 * 40 * 128 + 1, dtype=dtype, device="cuda")
    y = flat[1:].view(3, 40, 128)
    y.copy_(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fx.residual_norm(y, f, w[:128], w[2:130])
    s.synchronize()
    for u, v in zip(got, want):
        assert torch.equal(u, v)


def test_residual_norm_rows_of_zero_and_of_large_values():
    w = torch.ones(64, device="cuda")
    x = torch.zeros(4, 64, device="cuda", requires_grad=True)
    f = torch.zeros(4, 64, device="cuda", requires_grad=True)
    r, z = fx.residual_norm(x, f, w, w)
    (dx, df) = _grads(z.sum(), [x, f], None)
    assert (r == 0).all() and (z == 0).all() and torch.isfinite(dx).all() and torch.isfinite(df).all()
    # a large mean: the centred squares are taken after it is off
    g = _gen(32)
    f = _randn(g, 8, 256) + 1e4
    r, z = fx.residual_norm(torch.zeros_like(f), f, torch.ones(256, device="cuda"), torch.ones(256, device="cuda"),
                            kind="layer")
    r64, _ = ref.residual_norm(torch.zeros_like(f).double(), f.double(), torch.ones(256, device="cuda").double(),
                               torch.ones(256, device="cuda").double(), kind="layer")
    # the mean itself is known to 1e4 u = 6e-4
    assert (r.double() - r64).abs().max() < 2e-3


def test_residual_norm_gradient_against_differences():
    g = _gen(33)
    t = {"x": _randn(g, 6, 5, 96), "f": _randn(g, 6, 5, 96), "post_weight": 1 + _randn(g, 96, scale=0.1),
         "pre_weight": 1 + _randn(g, 96, scale=0.1), "gate": _randn(g, 6, 1, 96), "scale": _randn(g, 96)}
    cot = _randn(g, 6, 5, 96), _randn(g, 6, 5, 96)
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    grads = _grads(fx.residual_norm(**leaves, kind="layer"), list(leaves.values()), cot)
    for (n, x), gr in zip(t.items(), grads):
        d = gr.double() / gr.double().norm()
        h = 2.0**-12 * x.double().norm()

        def value(sign):
            b = {m: y.double() for m, y in t.items()}
            b[n] = b[n] + sign * h * d
            out = ref.residual_norm(**b, kind="layer")
            return sum((o * c.double()).sum() for o, c in zip(out, cot))

        slope = (value(1) - value(-1)) / (2 * h)
        assert abs(slope / gr.double().norm() - 1) < 1e-3, n
