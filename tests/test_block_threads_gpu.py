"""Calls of one kernel from two threads, with tables and widths that ask for different amounts of shared
memory: a launch must not find the limit lowered by the other thread's call."""

import ctypes
import threading

import pytest
import torch

import fermix_b200 as fx
from fermix_b200 import _lib, block

pytestmark = pytest.mark.gpu


def _attention(reach, dtype, dim, q_len):
    g = torch.Generator(device="cuda").manual_seed(70)
    q = torch.randn(1, 1, q_len, dim, generator=g, device="cuda").to(dtype)
    table = torch.randn(1, 32, generator=g, device="cuda").to(dtype)
    return lambda: fx.biased_attention(q, q, q, table, max_distance=reach)


def _bias(reach, dtype):
    table = torch.ones(1, 128 if reach < 200 else 256, dtype=dtype, device="cuda", requires_grad=True)
    pos = torch.arange(4, device="cuda", dtype=torch.int32)
    return lambda: torch.autograd.grad(fx.position_bias(table, pos, max_distance=reach).sum(), table)[0]


def _norm(width, dtype):
    x, w = torch.ones(1, width, dtype=dtype, device="cuda"), torch.ones(width, dtype=dtype, device="cuda")
    return lambda: fx.residual_norm(x, x, w, w)[1]


PAIRS = {
    "tiles": lambda t: [_attention(r, t, 64, 40) for r in (17, 2048)],
    "rows": lambda t: [_attention(r, t, 64, 1) for r in (200, 2000)],
    "bias": lambda t: [_bias(r, t) for r in (80, 2048)],
    "norm": lambda t: [_norm(w, t) for w in (4096 if t == torch.float32 else 8192, 2052 if t == torch.float32 else 4104)],
}


def _entries(call, monkeypatch):
    """The last C entry that a call makes, with its arguments and what they point to."""
    made = []

    def record(fn, device, *args):
        made.append((fn, args))
        _lib.check(fn(torch.cuda.current_stream(device).cuda_stream, *args))

    def record_with_workspace(fn, size, device, args):
        ws = torch.empty(size(ctypes.byref(args)), dtype=torch.uint8, device=device)
        record(fn, device, ctypes.byref(args), ws.data_ptr(), ws.numel())
        made.append((fn, made.pop()[1], ws))

    with monkeypatch.context() as m:
        m.setattr(block, "_call", record)
        m.setattr(block, "_call_with_workspace", record_with_workspace)
        out = call()
    return (*made[-1], out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("pair", PAIRS)
def test_two_threads_of_different_sizes(pair, dtype, monkeypatch):
    calls = PAIRS[pair](dtype)
    want = [c() for c in calls]
    entries = [_entries(c, monkeypatch) for c in calls]
    torch.cuda.synchronize()
    failed, streams = [0, 0], [torch.cuda.Stream() for _ in calls]

    def work(n):
        fn, args, stream = *entries[n][:2], streams[n].cuda_stream
        for _ in range(20000):
            failed[n] += fn(stream, *args) != 0

    threads = [threading.Thread(target=work, args=(n,)) for n in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert failed == [0, 0]
    assert all(torch.equal(c(), w) for c, w in zip(calls, want))
