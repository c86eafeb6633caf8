"""Edges of the attention kernels' schemes, against the plain 64-bit form: references that have to
move, caches longer than a warp's record of live keys, several queries of a group in one block,
tables that take several launches, misaligned masks, keys that are all far or all near.

Tolerances as in test_block_gpu.py; where scores are large, a score's own rounding, |s| 2^-23 in
float32, is a relative error of the probabilities: 2^9 times that for scores to 600, so 2^-9."""

import pytest
import torch

import fermix_b200 as fx
from tests import block_refs as ref
from tests.test_block_gpu import FORWARD, GRADIENT, IDS, TYPES, _attention_case, _check_attention, _close, _gen, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("q_len,k_len,dim", [(1, 700, 64), (100, 700, 64), (300, 520, 128), (40, 300, 32)])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_far_above_and_below_the_first_keys(q_len, k_len, dim, rising, dtype):
    """Scores that grow (or fall) by hundreds along the keys, so that a row's reference moves in later
    tiles and part-way through one."""
    g = _gen(40)
    q = _randn(g, 2, 2, q_len, dim, dtype=dtype)
    q[..., 0] = 1.0
    k = _randn(g, 2, 2, k_len, dim, dtype=dtype)
    ramp = torch.linspace(0, 600 * dim**0.5, k_len, device="cuda")
    k[..., 0] = (ramp if rising else ramp.flip(0)).to(dtype)
    v = _randn(g, 2, 2, k_len, dim, dtype=dtype)
    want = ref.attention(q.double(), k.double(), v.double())
    tol = 2.0**-9 if dtype == torch.float32 else FORWARD[dtype]
    _close(fx.biased_attention(q, k, v), want, tol, "out")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    cot = _randn(g, 2, 2, q_len, dim, dtype=dtype)
    out = fx.biased_attention(*leaves)
    _close(out, want, tol, "out with gradient")
    b = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    exp = torch.autograd.grad(ref.attention(*b), b, cot.double())
    top = exp[2].abs().max().item()
    for n, x, y in zip("qkv", torch.autograd.grad(out, leaves, cot), exp):
        assert torch.isfinite(x).all(), n
        # the ramp itself enters dq (times k, up to 600 sqrt(dim)) and the row sums cancel
        bound = max(y.abs().max().item(), top * (k.abs().max().item() if n == "q" else 1.0))
        assert (x.double() - y).abs().max().item() <= max(4 * tol, GRADIENT[dtype]) * bound, n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,q_len", [(1, 1, 1), (8, 1, 2), (16, 1, 1), (4, 4, 7), (12, 3, 4)])
def test_few_queries_over_a_long_masked_cache(heads, kv_heads, q_len, dtype):
    g = _gen(41)
    B, L, D = 2, 20011, 64
    q = _randn(g, B, heads, q_len, D, dtype=dtype)
    k, v = (_randn(g, B, L, kv_heads, D, dtype=dtype).transpose(1, 2) for _ in range(2))
    table = _randn(g, heads, 32, dtype=dtype)
    mask = torch.rand(B, L + 3, generator=g, device="cuda") < 0.5
    mask[0, 9000:] = False
    mask[1, :15000] = False
    for m in (None, mask[:, :L], mask[:, 3:]):  # the last two off a 16-byte boundary by the odd length
        want = ref.attention(q.double(), k.double(), v.double(), table.double(), key_mask=m)
        _close(fx.biased_attention(q, k, v, table, key_mask=m), want, FORWARD[dtype], "out")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 72, 128])
def test_tables_of_several_launches_and_far_reach(dim, dtype):
    t, kw, cot = _attention_case((1, 2, 1, 150, 260, dim), dtype, 42, "sites", True, buckets=200)
    kw = {n: p * 5 if p.dtype != torch.bool else p for n, p in kw.items()}
    _check_attention(t, kw, cot, dtype, max_distance=2048)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("offset", [0, 50, 400, -400])
def test_all_keys_on_one_side(offset, dtype):
    """Every pair beyond the reach on one side, across it, and equal positions."""
    t, kw, cot = _attention_case((2, 2, 2, 130, 140, 32), dtype, 43, buckets=16)
    g = _gen(44)
    kw["q_pos"] = torch.randint(0, 8, (2, 130), generator=g, device="cuda", dtype=torch.int32)
    kw["k_pos"] = torch.randint(0, 8, (2, 140), generator=g, device="cuda", dtype=torch.int32) + offset
    _check_attention(t, kw, cot, dtype)
    kw["k_pos"] = torch.full_like(kw["k_pos"], 7)
    _check_attention(t, kw, cot, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_timeouts_are_reported_and_give_nan(dtype):
    """With no polls allowed every wait gives up: the call returns, the status says so, the outputs
    that depend on it are NaN, and the next call is right again."""
    from fermix_b200 import _lib

    t, kw, cot = _attention_case((1, 2, 2, 256, 256, 64), dtype, 45)
    lib = _lib.lib()
    assert _lib.device_status(clear=True) == 0
    before = lib.fermix_set_wait_polls(0)
    try:
        out = fx.biased_attention(**t)
        assert _lib.device_status(clear=True) == _lib.FX_ERR_TIMEOUT
        assert torch.isnan(out).all()
    finally:
        lib.fermix_set_wait_polls(before)
    _close(fx.biased_attention(**t), ref.attention(**{n: x.double() for n, x in t.items()}), FORWARD[dtype], "out")
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [33, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_len,k_len", [(4, 1, 20, 5003), (2, 2, 130, 2500), (3, 3, 300, 2048)])
@pytest.mark.parametrize("causal", [False, True])
def test_tiles_of_queries_over_split_keys(heads, kv_heads, q_len, k_len, causal, dim, dtype):
    """Few blocks of queries: the keys are split; some parts are masked whole, and a batch has no key."""
    g = _gen(45)
    q = _randn(g, 3, heads, q_len, dim, dtype=dtype)
    k, v = (_randn(g, 3, kv_heads, k_len, dim, dtype=dtype) for _ in range(2))
    table = _randn(g, heads, 32, dtype=dtype)
    mask = torch.rand(3, k_len, generator=g, device="cuda") < 0.5
    mask[0, 700:] = False
    mask[1] = False
    want = ref.attention(q.double(), k.double(), v.double(), table.double(), key_mask=mask, causal=causal)
    out = fx.biased_attention(q, k, v, table, key_mask=mask, causal=causal)
    _close(out, want, FORWARD[dtype], "out")
    assert not out[1].any()


@pytest.mark.parametrize("dim", [32, 40, 64])
def test_long_float32_sums(dim):
    """2048 queries and keys, two query heads a key head. An accumulator cuts off up to 2^-23 of itself
    96 times before its sum is moved on, half of that on average and while it grows from zero: 3e-6;
    the scores' own products add as much again at most."""
    t, kw, cot = _attention_case((1, 2, 1, 2048, 2048, dim), torch.float32, 46, "sites", True)
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    b = {n: x.detach().double().requires_grad_(True) for n, x in t.items()}
    out, want = fx.biased_attention(**a, **kw), ref.attention(**b, **kw)
    got = torch.autograd.grad(out, list(a.values()), cot)
    exp = torch.autograd.grad(want, list(b.values()), cot.double())
    for n, x, y in [("out", out, want), *zip(a, got, exp)]:
        assert ((x.double() - y).norm() / y.norm()).item() <= 6e-6, n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_bucket_edges_outlive_their_cache(dtype):
    """The buckets of a forward pass are those of its backward pass, whatever was asked for in between."""
    import gc

    from fermix_b200 import block

    t, kw, cot = _attention_case((1, 2, 2, 40, 50, 16), dtype, 47)
    a = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    pos = torch.arange(50, device="cuda")
    want = torch.autograd.grad(fx.biased_attention(**a, **kw), list(a.values()), cot)
    bias_want = torch.autograd.grad(fx.position_bias(a["table"], pos).sum(), a["table"])
    out, bias = fx.biased_attention(**a, **kw), fx.position_bias(a["table"], pos)
    block._edges.cache_clear()
    gc.collect()
    others = [block._edges(32, 200 + n, True) for n in range(40)]  # the freed arrays' sizes
    got = torch.autograd.grad(out, list(a.values()), cot)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(torch.autograd.grad(bias.sum(), a["table"])[0], bias_want[0])
    assert len(others) == 40
