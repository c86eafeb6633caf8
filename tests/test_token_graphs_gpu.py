"""Captured calls of the operators on tokens whose launches are several: sorted tokens, tiles cut along k, rows in parts.
Replayed with other values, and two graphs at once on two streams."""

import pytest
import torch

import fermix_b200 as fx

pytestmark = pytest.mark.gpu


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


# each: (its inputs for a seed, its outputs and gradients)
def _embedding(count, rows, width):
    def make(gen):
        return [torch.randint(0, rows, (count,), generator=gen, device="cuda"), _normal(gen, rows, width), _normal(gen, count, width)]

    def run(tokens, table, cot):
        out = fx.token_embedding(tokens, table)
        return out, *torch.autograd.grad(out, table, cot)

    return make, run, (1,)


def _linear(rows, inner, outer, dtype):
    def make(gen):
        return [_normal(gen, rows, inner).to(dtype), _normal(gen, outer, inner, scale=inner**-0.5).to(dtype),
                _normal(gen, outer).to(dtype), _normal(gen, rows, outer).to(dtype)]

    def run(x, weight, bias, cot):
        out = fx.fused_linear(x, weight, bias, activation="gelu")
        return out, *torch.autograd.grad(out, (x, weight, bias), cot)

    return make, run, (0, 1, 2)


def _logprobs(rows, entries, dtype):
    def make(gen):
        return [_normal(gen, rows, entries).to(dtype), torch.randint(0, entries, (rows,), generator=gen, device="cuda"),
                _normal(gen, rows)]

    def run(logits, tokens, cot):
        out = fx.token_logprobs(logits, tokens, top=4)
        return *out, *torch.autograd.grad(out[:2], logits, (cot, cot))

    return make, run, (0,)


CASES = {
    "sorted by a block": _embedding(6000, 3000, 48),
    "sorted, one pass": _embedding(30000, 500, 72),
    "sorted, two passes": _embedding(30000, 5000, 33),
    "tiles along k, f32": _linear(300, 4000, 520, torch.float32),
    "tiles along k, bf16": _linear(300, 4000, 520, torch.bfloat16),
    "tiles, last round cut": _linear(5200, 1100, 1100, torch.bfloat16),
    "rows in parts": _logprobs(3, 90001, torch.float32),
}


def _capture(make, run, leaves, seed):
    """(graph, its inputs, its outputs)."""
    held = make(torch.Generator(device="cuda").manual_seed(seed))
    for i in leaves:
        held[i].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = run(*held)
        del out
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held)
    return graph, held, out


@pytest.mark.parametrize("case", CASES)
def test_replayed_with_other_values(case):
    make, run, leaves = CASES[case]
    graph, held, out = _capture(make, run, leaves, 1)
    for seed in (1, 2, 3):
        values = make(torch.Generator(device="cuda").manual_seed(seed))
        with torch.no_grad():
            for h, v in zip(held, values):
                h.copy_(v)
        for t in out:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i in leaves:
            values[i].requires_grad_()
        assert all(torch.equal(a, b) for a, b in zip(out, run(*values)))


@pytest.mark.parametrize("case", CASES)
def test_two_graphs_at_once(case):
    make, run, leaves = CASES[case]
    both = [_capture(make, run, leaves, seed) for seed in (4, 5)]
    want = [[t.detach().clone() for t in run(*held)] for _, held, _ in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, (graph, _, _) in zip(streams, both):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, _, out), w in zip(both, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))
