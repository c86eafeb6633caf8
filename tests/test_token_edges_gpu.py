"""The operators on tokens away from the default stream and thread: streams, graphs, saved-tensor hooks, transforms,
bounded waits, large offsets, repeated calls."""

import ctypes
import threading

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib
from tests import token_refs as ref

pytestmark = pytest.mark.gpu


def _case(dtype, rows=300, inner=136, outer=264, entries=2100, seed=0):
    """(leaves, a function of them that runs all three operators and returns their outputs)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device="cuda") * scale).to(dtype)
    tokens = torch.randint(0, 70, (rows,), generator=gen, device="cuda")
    target = torch.randint(0, entries, (rows,), generator=gen, device="cuda")
    leaves = [r(70, inner), r(outer, inner, scale=0.1), r(outer), r(entries, outer, scale=0.1)]

    def run(table, weight, bias, head):
        x = fx.token_embedding(tokens, table, scale=2.0)
        y = fx.fused_linear(x, weight, bias, activation="gelu")
        return fx.token_logprobs(fx.fused_linear(y, head), target, top=3)

    return leaves, run


def _grads(leaves, run):
    own = [t.detach().requires_grad_() for t in leaves]
    out = run(*own)
    return (*out, *torch.autograd.grad((out[0].sum(), out[1].mean()), own))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_same_bits_again_on_another_stream_and_in_threads(dtype):
    leaves, run = _case(dtype)
    want = _grads(leaves, run)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _grads(leaves, run)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                results[i] = _grads(leaves, run)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(want, r))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [5, 300])
def test_captured_and_replayed_with_other_values(dtype, rows):
    leaves, run = _case(dtype, rows=rows)
    held = [t.clone().requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = run(*held)
            torch.autograd.grad((out[0].sum(), out[1].mean()), held)
            del out
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held)
        grads = torch.autograd.grad((out[0].sum(), out[1].mean()), held)
    others = _case(dtype, rows=rows, seed=7)[0]
    for values in (leaves, others):
        with torch.no_grad():
            for h, v in zip(held, values):
                h.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = _grads(values, run)
        assert all(torch.equal(a, b) for a, b in zip((*out, *grads), want))


def test_saved_tensors_put_elsewhere_and_back():
    leaves, run = _case(torch.float32)
    want = _grads(leaves, run)

    def pack(t):
        return t.cpu()

    def unpack(t):
        if t.dim() == 2:  # back with other strides
            return t.T.contiguous().T.cuda()
        return t.cuda()

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        own = [t.detach().requires_grad_() for t in leaves]
        out = run(*own)
    got = torch.autograd.grad((out[0].sum(), out[1].mean()), own)
    # a transposed operand is laid out anew, the numbers are the same
    assert all(torch.equal(a, b) for a, b in zip(want[4:], got))


def test_a_graph_used_twice_and_gradients_of_one_output():
    leaves, run = _case(torch.float32)
    own = [t.detach().requires_grad_() for t in leaves]
    out = run(*own)
    first = torch.autograd.grad(out[0].sum(), own, retain_graph=True)
    again = torch.autograd.grad(out[0].sum(), own, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    both = torch.autograd.grad((out[0].sum(), out[1].sum()), own, retain_graph=True)
    other = torch.autograd.grad(out[1].sum(), own)
    for a, b, c in zip(first, other, both):
        assert (a + b - c).norm() <= 2.0**-18 * (a.norm() + b.norm())
    assert not out[2].requires_grad and not out[3].requires_grad


def test_no_grad_keeps_nothing():
    leaves, run = _case(torch.bfloat16)
    own = [t.detach().requires_grad_() for t in leaves]
    with torch.no_grad():
        out = run(*own)
    assert not any(t.requires_grad for t in out)
    with torch.inference_mode():
        again = run(*own)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_transforms_and_tangents_are_refused():
    w, t = torch.randn(9, 8, device="cuda"), torch.randint(0, 8, (4,), device="cuda")
    x = torch.randn(4, 8, device="cuda")
    calls = (lambda v: fx.token_embedding(t, v).sum(), lambda v: fx.fused_linear(x, v).sum(),
             lambda v: fx.token_logprobs(v[:4], t)[0].sum())
    for call in calls:
        with pytest.raises(NotImplementedError, match="torch.func"):
            torch.func.grad(call)(w)
        with pytest.raises(NotImplementedError, match="torch.func"):
            torch.func.vmap(lambda s: call(w * s))(torch.ones(3, device="cuda"))
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
            with pytest.raises(NotImplementedError, match="tangent"):
                call(dual)


def test_a_wait_that_runs_out_is_reported_and_leaves_nan():
    x, w = torch.randn(300, 256, device="cuda"), torch.randn(300, 256, device="cuda")
    L = _lib.lib()
    want = fx.fused_linear(x, w, activation="relu")
    assert _lib.device_status() == 0
    old = L.fermix_set_wait_polls(0)
    try:
        # a float32 map of this size has no wait that could run out: its kernel keeps its sums in registers
        assert torch.equal(fx.fused_linear(x, w, activation="relu"), want)
        assert _lib.device_status() == 0
        for a, b in ((x.bfloat16(), w.bfloat16()), (x.repeat(8, 1), w.repeat(4, 1))):
            got = fx.fused_linear(a, b, activation="relu")
            assert torch.isnan(got).any()
            assert _lib.device_status() == _lib.FX_ERR_TIMEOUT
            _lib.device_status(clear=True)
        fx.fused_linear(x.bfloat16(), w.bfloat16())
        assert _lib.device_status(clear=True) == _lib.FX_ERR_TIMEOUT
    finally:
        L.fermix_set_wait_polls(old)
    assert torch.equal(fx.fused_linear(x, w, activation="relu"), want)
    assert _lib.device_status() == 0


def test_offsets_beyond_32_bits():
    rows, width = 2**21 + 9, 1024 + 8
    table = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")  # 2.2e9 entries
    picks = torch.tensor([0, rows - 1, 2**21, 5], device="cuda")
    table[picks] = torch.arange(4, device="cuda", dtype=torch.bfloat16)[:, None].expand(4, width)
    out = fx.token_embedding(picks, table)
    assert torch.equal(out[:, 0].float(), torch.arange(4, device="cuda").float()) and torch.equal(out, table[picks])
    # rows of logits far apart, and of x
    lines = table[:: 2**21 + 8]  # the first and the last row
    lp, ent = fx.token_logprobs(lines, torch.tensor([1, 2], device="cuda"))
    assert (lp + torch.log(torch.tensor(float(width)))).abs().max() < 1e-5
    y = fx.fused_linear(lines, torch.ones(3, width, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(y.float(), torch.tensor([[0.0], [width]], device="cuda").expand(2, 3))
    x = table[:: 2**15][:65].clone().fill_(1)  # more rows than the small kernel takes
    far = torch.empty(65, 2**25 + 8, dtype=torch.bfloat16, device="cuda")[:, :width]
    far.copy_(x)
    w = torch.full((40, width), 0.5, dtype=torch.bfloat16, device="cuda")
    assert (fx.fused_linear(far, w) == width / 2).all()
    del far, table


def test_workspace_too_small_is_an_error():
    L = _lib.lib()
    x, w, y = torch.zeros(300, 64, device="cuda"), torch.zeros(300, 64, device="cuda"), torch.zeros(300, 300, device="cuda")
    a = _lib.LinearArgs()
    a.dtype, a.rows, a.inner, a.outer, a.x_stride, a.weight_stride = _lib.FX_F32, 300, 64, 300, 64, 64
    a.x, a.weight, a.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    # a small map needs none
    assert L.fermix_linear_workspace_bytes(ctypes.byref(a)) == 0
    assert L.fermix_linear(stream, ctypes.byref(a), None, 0) == 0
    x, w, y = torch.zeros(2400, 64, device="cuda"), torch.zeros(1200, 64, device="cuda"), torch.zeros(2400, 1200, device="cuda")
    a.rows, a.outer, a.x, a.weight, a.y = 2400, 1200, x.data_ptr(), w.data_ptr(), y.data_ptr()
    need = L.fermix_linear_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert need > 0
    assert L.fermix_linear(stream, ctypes.byref(a), ws.data_ptr(), need - 1) == 4
    assert L.fermix_linear(stream, ctypes.byref(a), None, 0) == 4
    assert L.fermix_linear(stream, ctypes.byref(a), ws.data_ptr(), need) == 0
    e = _lib.EmbedArgs()
    e.dtype, e.token_bytes, e.count, e.rows, e.width, e.scale = _lib.FX_F32, 8, 20000, 30000, 64, 1.0
    t, g, d = torch.zeros(20000, dtype=torch.int64, device="cuda"), torch.zeros(20000, 64, device="cuda"), torch.zeros(30000, 64, device="cuda")
    e.tokens, e.grad, e.dweight = t.data_ptr(), g.data_ptr(), d.data_ptr()
    need = L.fermix_token_embedding_grad_workspace_bytes(ctypes.byref(e))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert L.fermix_token_embedding_grad(stream, ctypes.byref(e), ws.data_ptr(), need - 1) == 4
    assert L.fermix_token_embedding_grad(stream, ctypes.byref(e), ws.data_ptr(), need) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("count", [100, 5000, 30000])
def test_embedding_against_plain_sums_of_tokens_in_any_order(count):
    """Sorted, reversed, equal and random tokens take the same places: whole numbers, exact."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randint(0, 3000, (count,), generator=gen, device="cuda", dtype=torch.int32)
    cot = torch.randint(-4, 5, (count, 24), generator=gen, device="cuda").float()
    for tokens in (base, base.sort().values, base.sort(descending=True).values, torch.full_like(base, 2999), base % 2 * 2999):
        w = torch.zeros(3000, 24, device="cuda", requires_grad=True)
        (grad,) = torch.autograd.grad(fx.token_embedding(tokens, w), w, cot)
        want = torch.zeros(3000, 24, dtype=torch.float64, device="cuda").index_add_(0, tokens.long(), cot.double())
        assert torch.equal(grad.double(), want)


def test_linear_shapes_around_every_switch():
    """Whole numbers, exact in both types: rows, widths and depths on both sides of each kernel's limits."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        for rows in (1, 8, 9, 16, 17, 32, 33, 64, 65, 256, 257):
            for inner, outer in ((1, 3), (31, 32), (64, 33), (72, 64), (264, 65), (1000, 257)):
                x = torch.randint(-2, 3, (rows, inner), generator=gen, device="cuda").to(dtype)
                w = (torch.randint(-1, 2, (outer, inner), generator=gen, device="cuda") * (torch.rand(
                    outer, inner, generator=gen, device="cuda") < 30.0 / inner)).to(dtype)  # sums below 2^8
                want = ref.linear(x.double(), w.double())
                got = fx.fused_linear(x, w)
                assert torch.equal(got.double(), want.to(dtype).double()), (dtype, rows, inner, outer)
