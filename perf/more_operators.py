"""What is measured of the operators around the attention blocks: the tokens' embedding with its
gradient, the linear map with bias, activation and residual, and the log probabilities of given
tokens with entropy and top alternatives.

``own`` is False: ``run`` computes the operators in their plain form, elementary torch
operations in 32 bits, rounded once at the end. ``own`` is True: ``run`` makes the calls a user
makes (``fermix_b200.token_embedding``, ``fused_linear``, ``token_logprobs``).
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh", "tanh"]


# ------------------------------------------------------------------ cases
def _embed(name, mode, dtype, batch, length, rows, width, tokens, scale):
    return {"name": name, "op": "embed", "mode": mode, "dtype": dtype, "batch": batch, "length": length, "rows": rows,
            "width": width, "tokens": tokens, "scale": scale}


def _linear(name, mode, dtype, rows, inner, outer, activation, bias, residual):
    return {"name": name, "op": "linear", "mode": mode, "dtype": dtype, "rows": rows, "inner": inner, "outer": outer,
            "activation": activation, "bias": bias, "residual": residual}


def _logp(name, mode, dtype, rows, entries, masked, top, scale):
    return {"name": name, "op": "logp", "mode": mode, "dtype": dtype, "rows": rows, "entries": entries,
            "masked": masked, "top": top, "scale": scale}


def listed():
    return [
        # the first step of a small wave function, trained (64 samples of 32 electrons on 64 sites): latency
        _embed("embed-small-f32", "train", "f32", 64, 32, 64, 64, "occupied", 1.0),
        # 4096 walkers of 128 electrons on 512 sites, trained: every row of the table sums many tokens
        _embed("embed-electrons-f32", "train", "f32", 4096, 128, 512, 128, "occupied", 8.0),
        # padded sequences over a large table, some tokens far more frequent than others, an odd width
        _embed("embed-words-bf16", "train", "bf16", 64, 1025, 50001, 1000, "frequent", 31.0),
        # one moved electron's token through a map with its activation: latency
        _linear("linear-one-bf16", "infer", "bf16", 1, 1024, 4096, "gelu", True, False),
        # one token for each of 32 walkers through the map back onto the residual stream: the weights' bytes
        _linear("linear-walkers-bf16", "infer", "bf16", 32, 8192, 4096, "none", True, True),
        # the position-wise map of a small wave function, trained (64 samples of 32 electrons): latency
        _linear("linear-small-f32", "train", "f32", 2048, 64, 128, "silu", False, False),
        # the training step over 512 walkers of 128 electrons, in the precision of the determinants
        _linear("linear-electrons-f32", "train", "f32", 65536, 256, 512, "silu", True, False),
        # the training step over odd sizes (rows, widths off every tile), the residual added
        _linear("linear-odd-bf16", "train", "bf16", 4001, 1000, 777, "tanh", True, True),
        # the widening map of a large block, trained
        _linear("linear-wide-bf16", "train", "bf16", 8192, 2048, 8192, "gelu", True, False),
        # the site each of 64 walkers' next electron moves to, occupied sites left out: latency
        _logp("logp-sites-f32", "infer", "f32", 64, 512, True, 8, 1.0),
        # few rows over many alternatives, an odd number of them
        _logp("logp-long-bf16", "infer", "bf16", 16, 131071, False, 16, 0.7),
        # the training step of an ordered wave function's conditionals
        _logp("logp-chain-bf16", "train", "bf16", 8191, 32000, False, 0, 1.0),
    ]


def _log(rng, low, high):
    """A whole number, its logarithm uniform in [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embed", "linear", "linear", "logp"])
    dtype = rng.choice(["f32", "bf16"])
    mode = rng.choice(["train", "train", "infer"])
    if op == "embed":
        width = _log(rng, 16, 4096)
        batch = _log(rng, 1, min(4096, (1 << 26) // width))
        length = _log(rng, 1, max(1, min(2048, (1 << 26) // width // batch)))
        rows = _log(rng, 2, min(131072, (1 << 26) // width))
        tokens = rng.choice(["uniform", "frequent"] + (["occupied"] if rows >= 2 * length else []))
        return _embed("", mode, dtype, batch, length, rows, width, tokens, rng.choice([1.0, math.sqrt(width)]))
    if op == "linear":
        inner, outer = _log(rng, 16, 8192), _log(rng, 16, 8192)
        few = rng.random() < 0.3
        most = (1 << 33 if dtype == "f32" else 1 << 36) // (inner * outer)
        rows = _log(rng, 1, 128) if few else _log(rng, 129, max(129, min(65536, most)))
        return _linear("", "infer" if few else mode, dtype, rows, inner, outer, rng.choice(ACTIVATIONS),
                       rng.random() < 0.6, rng.random() < 0.4)
    entries = _log(rng, 2, 200000)
    rows = _log(rng, 1, min(65536, max(1, (1 << 27) // entries)))
    train = mode == "train"
    return _logp("", mode, dtype, rows, entries, rng.random() < 0.4,
                 0 if train else min(entries, rng.choice([0, 1, 4, 16, 32])), rng.choice([1.0, 0.7, 1.6]))


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    state = {"case": case, "leaves": []}
    if case["op"] == "embed":
        B, L, V, W = case["batch"], case["length"], case["rows"], case["width"]
        state["weight"] = normal(V, W)
        state["padding"] = None
        if case["tokens"] == "occupied":  # the sorted sites of each sample
            n = 2 * L if V >= 2 * L else V
            first = torch.randint(0, V - n + 1, (B, 1), generator=gen, device="cuda")
            state["tokens"] = (uniform(B, n).topk(L, dim=1).indices.sort(dim=1).values + first).to(torch.int32)
        else:
            u = uniform(B, L).double()
            if case["tokens"] == "frequent":  # token v about as often as 1 / (v + 1), the tails padded
                tokens = torch.exp(u * math.log(V + 1)).sub_(1)
                state["padding"] = -1
            else:
                tokens = u * V
            tokens = tokens.long().clamp_(0, V - 1)
            if state["padding"] is not None:
                live = torch.randint((L + 1) // 2, L + 1, (B, 1), generator=gen, device="cuda")
                tokens[torch.arange(L, device="cuda")[None, :] >= live] = -1
            state["tokens"] = tokens
        if train:
            state["grads"] = (normal(B, L, W),)
            state["leaves"] = ["weight"]
    elif case["op"] == "linear":
        M, K, N = case["rows"], case["inner"], case["outer"]
        state["x"] = normal(M, K)
        state["weight"] = normal(N, K, scale=K**-0.5)
        state["bias"] = normal(N, scale=0.1) if case["bias"] else None
        state["residual"] = normal(M, N) if case["residual"] else None
        if train:
            state["grads"] = (normal(M, N),)
            state["leaves"] = [n for n in ("x", "weight", "bias", "residual") if state[n] is not None]
    else:
        R, V = case["rows"], case["entries"]
        state["logits"] = normal(R, V, scale=2.0)
        state["mask"] = None
        state["tokens"] = (uniform(R).double() * V).long().clamp_(0, V - 1)
        if case["masked"]:  # the given token stays
            state["mask"] = uniform(R, V) < 0.75
            state["mask"].scatter_(1, state["tokens"][:, None], True)
        if train:
            state["grads"] = (torch.randn(R, generator=gen, device="cuda"),
                              torch.randn(R, generator=gen, device="cuda") * 0.01)
            state["leaves"] = ["logits"]
    for n in state["leaves"]:
        state[n].requires_grad_(True)
    return state


# ------------------------------------------------------------------ plain forms
def _plain_embed(state):
    case, weight, tokens = state["case"], state["weight"].detach(), state["tokens"].reshape(-1).long()
    live = tokens >= 0
    at = tokens.clamp(min=0)
    out = (weight[at].float() * case["scale"] * live[:, None]).to(weight.dtype).view(*state["tokens"].shape, -1)
    if case["mode"] != "train":
        return {"out": out}
    rows = state["grads"][0].reshape(-1, case["width"]).float() * live[:, None]
    sums = torch.zeros(weight.shape, dtype=torch.float32, device="cuda").index_add_(0, at, rows)
    return {"out": out, "d_weight": (sums * case["scale"]).to(weight.dtype)}


def _plain_linear(state):
    h = torch.matmul(state["x"].float(), state["weight"].float().T)
    if state["bias"] is not None:
        h = h + state["bias"].float()
    activation = state["case"]["activation"]
    if activation == "relu":
        h = h.clamp(min=0)
    elif activation == "silu":
        h = h / (1 + torch.exp(-h))
    elif activation == "gelu":
        h = 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
    elif activation == "gelu_tanh":
        h = 0.5 * h * (1 + torch.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h * h * h)))
    elif activation == "tanh":
        h = torch.tanh(h)
    if state["residual"] is not None:
        h = state["residual"].float() + h
    return (h.to(state["x"].dtype),)


def _plain_logp(state):
    case = state["case"]
    x = state["logits"].float()
    if state["mask"] is not None:
        x = x.masked_fill(~state["mask"], -math.inf)
    c = (x - x.amax(-1, keepdim=True).detach()) * case["scale"]
    logs = c - torch.log(torch.exp(c).sum(-1, keepdim=True))
    p = torch.exp(logs)
    entropy = -(p * logs.masked_fill(logs == -math.inf, 0.0)).sum(-1)
    out = (torch.gather(logs, -1, state["tokens"][:, None])[:, 0], entropy)
    if case["top"]:
        index = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        best = torch.gather(logs, -1, index)
        out += (best, index.masked_fill(best == -math.inf, -1))
    return out


# ------------------------------------------------------------------ one pass
def _own(state):
    import fermix_b200 as fx

    case = state["case"]
    if case["op"] == "embed":
        return (fx.token_embedding(state["tokens"], state["weight"], scale=case["scale"], padding=state["padding"]),)
    if case["op"] == "linear":
        return (fx.fused_linear(state["x"], state["weight"], state["bias"],
                                activation=None if case["activation"] == "none" else case["activation"],
                                residual=state["residual"]),)
    return fx.token_logprobs(state["logits"], state["tokens"], scale=case["scale"], mask=state["mask"], top=case["top"])


NAMES = {"embed": ("out",), "linear": ("out",), "logp": ("logp", "entropy", "top_logp", "top_index")}


def run(state):
    case = state["case"]
    if not own and case["op"] == "embed":
        return _plain_embed(state)
    form = _own if own else {"linear": _plain_linear, "logp": _plain_logp}[case["op"]]
    if case["mode"] != "train":
        with torch.no_grad():
            return dict(zip(NAMES[case["op"]], form(state)))
    out = form(state)
    grads = torch.autograd.grad(out, [state[n] for n in state["leaves"]], state["grads"])
    outputs = {n: t.detach() for n, t in zip(NAMES[case["op"]], out)}
    outputs.update(("d_" + n, g) for n, g in zip(state["leaves"], grads))
    return outputs


# ------------------------------------------------------------------ floors
def work(case):
    size = BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "embed":
        N, V, W = case["batch"] * case["length"], case["rows"], case["width"]
        entries = min(N, V) * W + N * W + (N * W + V * W if train else 0)
        return {"bytes": size * entries + N * (4 if case["tokens"] == "occupied" else 8),
                "flops": N * W * (3 if train else 1)}
    if case["op"] == "linear":
        M, K, N = case["rows"], case["inner"], case["outer"]
        entries = M * K + N * K + M * N + (N if case["bias"] else 0) + (M * N if case["residual"] else 0)
        if train:
            entries = 2 * entries  # the gradient of each input, and of the output
        return {"bytes": size * entries, "flops": 2 * M * N * K * (3 if train else 1)}
    n = case["rows"] * case["entries"]
    return {"bytes": size * n * (2 if train else 1) + (n if case["masked"] else 0) + case["rows"] * (16 + 12 * case["top"]),
            "flops": n * (16 if train else 8)}


# ------------------------------------------------------------------ 64 bits
def _exact_embed(state):
    case = state["case"]
    weight = state["weight"].detach().double() * case["scale"]
    B, L, W = case["batch"], case["length"], case["width"]
    # a row of zeros behind the table stands for the padding
    table = torch.cat([weight, weight.new_zeros(1, W)])
    tokens = torch.where(state["tokens"] < 0, case["rows"], state["tokens"].long())
    out = {"out": torch.nn.functional.embedding(tokens, table)}
    if case["mode"] == "train":
        order = torch.argsort(tokens.reshape(-1))
        count = torch.bincount(tokens.reshape(-1), minlength=case["rows"] + 1)
        d = torch.zeros_like(table)
        for part in range(0, W, 256):  # sums of the sorted rows, some columns at a time
            rows = state["grads"][0].reshape(B * L, W)[:, part:part + 256].double()[order]
            d[:, part:part + 256] = torch.segment_reduce(rows, "sum", lengths=count, unsafe=True, initial=0)
        out["d_weight"] = d[:-1] * case["scale"]
    return out


def _exact_linear(state):
    case = state["case"]
    d = {n: state[n].detach().double() for n in ("x", "weight", "bias", "residual") if state[n] is not None}
    h = d["x"] @ d["weight"].T + d.get("bias", 0.0)
    activation = case["activation"]
    one = torch.ones_like(h)
    if activation == "none":
        y, slope = h, one
    elif activation == "relu":
        y, slope = torch.where(h > 0, h, 0.0 * one), (h > 0).double()
    elif activation == "silu":
        s = torch.sigmoid(h)
        y, slope = h * s, s * (1 + h * (1 - s))
    elif activation == "gelu":
        cdf = torch.special.ndtr(h)
        y, slope = h * cdf, cdf + h * torch.exp(-h.square() / 2) / math.sqrt(2 * math.pi)
    elif activation == "gelu_tanh":
        # 1/2 (1 + tanh(u)) is the sigmoid of 2 u
        u = 2 * math.sqrt(2 / math.pi) * (h + 0.044715 * h**3)
        s = torch.sigmoid(u)
        y, slope = h * s, s + h * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * h.square())
    else:
        y = torch.tanh(h)
        slope = 1 - y.square()
    out = {"out": y + d.get("residual", 0.0)}
    if case["mode"] == "train":
        dy = state["grads"][0].double()
        g = dy * slope
        grads = {"x": g @ d["weight"], "weight": g.T @ d["x"], "bias": g.sum(0), "residual": dy}
        out.update(("d_" + n, grads[n]) for n in state["leaves"])
    return out


def _exact_logp(state):
    case = state["case"]
    names, parts = NAMES["logp"], []
    step = max(1, (1 << 25) // case["entries"])  # rows at a time
    for r in range(0, case["rows"], step):
        rows = slice(r, r + step)
        x = state["logits"][rows].detach().double() * case["scale"]
        if state["mask"] is not None:
            x = torch.where(state["mask"][rows], x, -math.inf)
        logs = torch.log_softmax(x, -1)
        p = logs.exp()
        entropy = torch.special.entr(p).sum(-1)
        token = state["tokens"][rows, None]
        part = {"logp": logs.gather(1, token)[:, 0], "entropy": entropy}
        if case["top"]:
            part["top_logp"] = logs.topk(case["top"], -1).values
        if case["mode"] == "train":
            g, e = (t[rows, None].double() for t in state["grads"])
            hit = torch.zeros_like(p).scatter_(1, token, 1.0)
            part["d_logits"] = case["scale"] * (g * (hit - p) - e * (p * entropy[:, None] - torch.special.entr(p)))
        parts.append(part)
    out = {n: torch.cat([part[n] for part in parts]) for n in parts[0]}
    if case["top"]:
        out["top_index"] = None  # ties among equal logits: no computed number
    return {n: out[n] for n in (*names, "d_logits") if n in out}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "linear": _exact_linear, "logp": _exact_logp}[case["op"]](state)
