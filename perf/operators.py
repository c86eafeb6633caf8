"""What is measured of the attention-block operators in front of the determinants: the biased
attention over occupied sites, the bucketed position bias and the gated residual with its norms.

``own`` is False: ``run`` computes the operators in their plain form, elementary torch
operations in 32 bits, rounded once at the end. ``own`` is True: ``run`` makes the calls a user
makes (``fermix_b200.biased_attention``, ``position_bias``, ``residual_norm``).
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------ cases
def _attention(name, mode, dtype, batch, heads, kv_heads, q_len, k_len, dim, positions, masked, causal, buckets,
               max_distance):
    return {"name": name, "op": "attention", "mode": mode, "dtype": dtype, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "q_len": q_len, "k_len": k_len, "dim": dim, "positions": positions,
            "masked": masked, "causal": causal, "buckets": buckets, "max_distance": max_distance}


def _bias(name, mode, dtype, batch, heads, q_len, k_len, positions, buckets, max_distance):
    return {"name": name, "op": "bias", "mode": mode, "dtype": dtype, "batch": batch, "heads": heads,
            "q_len": q_len, "k_len": k_len, "positions": positions, "buckets": buckets,
            "max_distance": max_distance}


def _norm(name, mode, dtype, groups, rows, width, kind, gate, scale):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "groups": groups, "rows": rows,
            "width": width, "kind": kind, "gate": gate, "scale": scale}


def listed():
    return [
        # one moved electron's token against the sites of a small lattice: latency
        _attention("attn-one-short", "infer", "bf16", 1, 8, 8, 1, 512, 64, "end", False, False, 32, 128),
        # one new token per walker over long caches of different lengths, heads sharing keys
        _attention("attn-one-long", "infer", "bf16", 32, 8, 2, 1, 65536, 64, "end", True, False, 32, 128),
        # the training step of a wave function of 128 electrons on 512 sites, in the precision of the determinants
        _attention("attn-electrons-f32", "train", "f32", 512, 4, 4, 128, 128, 32, "occupied", False, False, 32, 128),
        # the training step over 512 sites, lattices of several sizes padded to one length
        _attention("attn-sites-bf16", "train", "bf16", 64, 8, 8, 512, 512, 64, "end", True, False, 32, 128),
        # the training step of an ordered (causal) wave function over a long chain, an odd length
        _attention("attn-chain-bf16", "train", "bf16", 1, 8, 8, 4095, 4095, 64, "end", False, True, 32, 128),
        # evaluation over a 64 x 64 lattice with wide heads, four of them sharing a key head
        _attention("attn-lattice-bf16", "infer", "bf16", 2, 16, 4, 4096, 4096, 128, "end", False, False, 64, 512),
        # the bias of a small lattice, trained: latency
        _bias("bias-small-f32", "train", "f32", 1, 4, 128, 128, "end", 32, 128),
        # the bias of a 64 x 64 lattice, trained
        _bias("bias-lattice-bf16", "train", "bf16", 1, 8, 4096, 4096, "end", 32, 128),
        # a bias for each sample's own occupied sites
        _bias("bias-occupied-f32", "train", "f32", 128, 8, 255, 255, "occupied", 32, 128),
        # one token between two blocks: latency
        _norm("norm-one-bf16", "infer", "bf16", 1, 1, 256, "rms", "none", True),
        # the training step of 4096 walkers of 128 electrons, a gate for each entry
        _norm("norm-electrons-f32", "train", "f32", 4096, 128, 128, "rms", "full", True),
        # odd rows and width, centred norms, a gate vector for each sample
        _norm("norm-samples-bf16", "train", "bf16", 61, 513, 1000, "layer", "group", True),
    ]


def _log(rng, low, high):
    """A whole number, its logarithm uniform in [low, high]."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = max(low, min(high, n))
    return n - 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["attention", "attention", "bias", "norm"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4])
        heads = kv_heads * rng.choice([1, 2, 4])
        dim = rng.choice([16, 32, 40, 64, 64, 96, 128])
        buckets, distance = rng.choice([(32, 128), (16, 64), (64, 512)])
        masked = rng.random() < 0.4
        shape = rng.choice(["one", "train", "train", "infer"])
        if shape == "one":
            k_len = _log(rng, 16, 65536)
            batch = _log(rng, 1, max(1, min(64, (1 << 28) // (k_len * kv_heads * dim * 4))))
            return _attention("", "infer", dtype, batch, heads, kv_heads, 1, k_len, dim, "end", masked, False,
                              buckets, distance)
        causal = rng.random() < 0.3
        positions = rng.choice(["end", "occupied"]) if not causal else "end"
        length = _log(rng, 17, 2048)
        cost = 64 * 8 * 512 * 512 // (length * length * heads)
        batch = _log(rng, 1, max(1, min(512, cost // (2 if dtype == "f32" else 1) * 64 // max(64, dim))))
        q_len = length if positions == "occupied" or rng.random() < 0.7 else _log(rng, 2, length)
        return _attention("", shape, dtype, batch, heads, kv_heads, q_len, length, dim, positions, masked, causal,
                          buckets, distance)
    if op == "bias":
        heads = rng.choice([1, 2, 4, 8, 12])
        buckets, distance = rng.choice([(32, 128), (16, 64), (64, 512)])
        length = _log(rng, 17, 2048)
        if rng.random() < 0.5:
            batch = _log(rng, 1, max(1, min(256, (1 << 25) // (length * length * heads))))
            return _bias("", "train", dtype, batch, heads, length, length, "occupied", buckets, distance)
        return _bias("", "train", dtype, 1, heads, _log(rng, 1, length), length, "end", buckets, distance)
    width = _log(rng, 16, 4096)
    total = max(1, (1 << 25) // width)
    groups = _log(rng, 1, min(4096, total))
    rows = _log(rng, 1, min(2048, max(1, total // groups)))
    return _norm("", rng.choice(["train", "train", "infer"]), dtype, groups, rows, width,
                 rng.choice(["rms", "layer"]), rng.choice(["none", "full", "row", "group"]), rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _sites(gen, batch, n):
    """Sorted occupied sites of each sample: n of 2 n."""
    return torch.rand(batch, 2 * n, generator=gen, device="cuda").topk(n, dim=1).indices.sort(dim=1).values.to(torch.int32)


def _lengths(gen, batch, low, high):
    return torch.randint(max(1, low), high + 1, (batch,), generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    state = {"case": case}
    if case["op"] == "attention":
        B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        Lq, Lk = case["q_len"], case["k_len"]
        # token-major storage, as a projection leaves it; the operators take the head-major view
        state["q"] = normal(B, Lq, H, D).transpose(1, 2)
        state["k"] = normal(B, Lk, Hk, D).transpose(1, 2)
        state["v"] = normal(B, Lk, Hk, D).transpose(1, 2)
        state["table"] = normal(H, case["buckets"])
        state["q_pos"] = state["k_pos"] = state["key_mask"] = None
        if case["positions"] == "occupied":
            state["q_pos"] = state["k_pos"] = _sites(gen, B, Lk)
        if case["masked"]:
            n = _lengths(gen, B, (Lk + 1) // 2, Lk)
            state["key_mask"] = torch.arange(Lk, device="cuda")[None, :] < n[:, None]
            if Lq == 1:  # the new token is the last live one
                state["q_pos"] = (n - 1).to(torch.int32)[:, None]
        if train:
            state["grad"] = normal(B, Lq, H, D).transpose(1, 2)
            leaves = ["q", "k", "v", "table"]
    elif case["op"] == "bias":
        B, H, Lq, Lk = case["batch"], case["heads"], case["q_len"], case["k_len"]
        state["table"] = normal(H, case["buckets"])
        state["q_pos"] = state["k_pos"] = None
        if case["positions"] == "occupied":
            state["q_pos"] = state["k_pos"] = _sites(gen, B, Lk)
            state["grad"] = normal(B, H, Lq, Lk)
        else:
            state["q_pos"] = torch.arange(Lk - Lq, Lk, device="cuda", dtype=torch.int32)
            state["k_pos"] = torch.arange(Lk, device="cuda", dtype=torch.int32)
            state["grad"] = normal(H, Lq, Lk)
        leaves = ["table"]
    else:
        G, R, W = case["groups"], case["rows"], case["width"]
        state["x"] = normal(G, R, W)
        state["f"] = normal(G, R, W, scale=2.0)
        gate = {"none": None, "full": (G, R, W), "row": (G, R, 1), "group": (G, 1, W)}[case["gate"]]
        state["gate"] = None if gate is None else normal(*gate)
        state["scale"] = normal(W, scale=0.1) if case["scale"] else None
        state["post_weight"] = (1 + normal(W, scale=0.1, kind=torch.float32)).to(dtype)
        state["pre_weight"] = (1 + normal(W, scale=0.1, kind=torch.float32)).to(dtype)
        layer = case["kind"] == "layer"
        state["post_bias"] = normal(W, scale=0.1) if layer else None
        state["pre_bias"] = normal(W, scale=0.1) if layer else None
        if train:
            state["grad_r"] = normal(G, R, W)
            state["grad_z"] = normal(G, R, W)
            leaves = ["x", "f", "post_weight", "pre_weight", "gate", "scale", "post_bias", "pre_bias"]
    if train:
        state["leaves"] = [n for n in leaves if state[n] is not None]
        for n in state["leaves"]:
            state[n].requires_grad_(True)
    return state


# ------------------------------------------------------------------ plain forms
def _edges(buckets, max_distance, bidirectional):
    """Bucket j >= 1 of a distance holds d >= edges[j - 1]: one bucket a distance below half of
    them, then buckets evenly spaced in the logarithm up to max_distance; whole numbers exactly."""
    n = buckets // 2 if bidirectional else buckets
    exact = n // 2
    edges = list(range(1, exact + 1))
    m = n - exact
    d = exact
    for j in range(1, m):
        # the least d with log(d / exact) / log(max_distance / exact) >= j / m
        while d ** m * exact ** j < max_distance ** j * exact ** m:
            d += 1
        edges.append(d)
    return edges


def _buckets(q_pos, k_pos, case, bidirectional):
    """(..., Lq, Lk) bucket of every pair."""
    delta = k_pos[..., None, :].long() - q_pos[..., :, None].long()
    edges = torch.tensor(_edges(case["buckets"], case["max_distance"], bidirectional), device="cuda")
    if bidirectional:
        return torch.bucketize(delta.abs(), edges, right=True) + (delta > 0) * (case["buckets"] // 2)
    return torch.bucketize((-delta).clamp(min=0), edges, right=True)


def _positions(state):
    case, q, k = state["case"], state["q_pos"], state["k_pos"]
    if k is None:
        k = torch.arange(case["k_len"], device="cuda")
    if q is None:
        q = torch.arange(case["k_len"] - case["q_len"], case["k_len"], device="cuda")
    return q, k


def _spread(table, bucket):
    """table[h, bucket], (H, Lq, Lk) or (B, H, Lq, Lk): gathered from a copy of the table for each
    query, so that the gradient's additions are spread over the queries."""
    index = bucket if bucket.dim() == 2 else bucket[:, None]
    shape = bucket.shape[:-2] + table.shape[:1] + bucket.shape[-2:]
    rows = table.float()[:, None, :].expand(shape[:-1] + table.shape[1:])
    return torch.gather(rows, -1, index.expand(shape))


def _plain_attention(state):
    case = state["case"]
    B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    Lq, Lk = case["q_len"], case["k_len"]
    q = state["q"].float().reshape(B, Hk, H // Hk * Lq, D)
    k, v = state["k"].float(), state["v"].float()
    q_pos, k_pos = _positions(state)
    bucket = _buckets(q_pos, k_pos, case, not case["causal"])
    bias = _spread(state["table"], bucket)
    s = torch.matmul(q, k.transpose(-1, -2)).view(B, H, Lq, Lk) * (D ** -0.5) + bias
    if state["key_mask"] is not None:
        s = s.masked_fill(~state["key_mask"][:, None, None, :], -math.inf)
    if case["causal"]:
        s = s.masked_fill(k_pos[..., None, :] > q_pos[..., :, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).detach())
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p.view(B, Hk, H // Hk * Lq, Lk), v).view(B, H, Lq, D).to(state["q"].dtype)


def _plain_bias(state):
    bucket = _buckets(state["q_pos"], state["k_pos"], state["case"], True)
    return _spread(state["table"], bucket).to(state["table"].dtype)


def _plain_normed(x, weight, bias, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    return y if bias is None else y + bias.float()


def _plain_norm(state):
    kind, dtype = state["case"]["kind"], state["x"].dtype
    u = _plain_normed(state["f"].float(), state["post_weight"], state["post_bias"], kind)
    if state["gate"] is not None:
        u = u * state["gate"].float()
    if state["scale"] is not None:
        u = u * state["scale"].float()
    r = state["x"].float() + u
    z = _plain_normed(r, state["pre_weight"], state["pre_bias"], kind)
    return r.to(dtype), z.to(dtype)


# ------------------------------------------------------------------ one pass
def _own(state):
    import fermix_b200 as fx

    case = state["case"]
    if case["op"] == "attention":
        return fx.biased_attention(state["q"], state["k"], state["v"], state["table"], q_pos=state["q_pos"],
                                   k_pos=state["k_pos"], key_mask=state["key_mask"], causal=case["causal"],
                                   max_distance=case["max_distance"], bidirectional=not case["causal"])
    if case["op"] == "bias":
        return fx.position_bias(state["table"], state["q_pos"], state["k_pos"], max_distance=case["max_distance"])
    return fx.residual_norm(state["x"], state["f"], state["post_weight"], state["pre_weight"],
                            post_bias=state["post_bias"], pre_bias=state["pre_bias"], gate=state["gate"],
                            scale=state["scale"], kind=case["kind"])


def run(state):
    case = state["case"]
    form = _own if own else {"attention": _plain_attention, "bias": _plain_bias, "norm": _plain_norm}[case["op"]]
    if case["mode"] != "train":
        with torch.no_grad():
            out = form(state)
        return dict(zip(("r", "z"), out)) if case["op"] == "norm" else {"out": out}
    out = form(state)
    leaves = [state[n] for n in state["leaves"]]
    if case["op"] == "norm":
        grads = torch.autograd.grad(out, leaves, (state["grad_r"], state["grad_z"]))
        outputs = {"r": out[0].detach(), "z": out[1].detach()}
    else:
        grads = torch.autograd.grad(out, leaves, state["grad"])
        outputs = {"out": out.detach()}
    outputs.update(("d_" + n, g) for n, g in zip(state["leaves"], grads))
    return outputs


# ------------------------------------------------------------------ floors
def work(case):
    size = BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "attention":
        B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        Lq, Lk = case["q_len"], case["k_len"]
        live = 0.75 * Lk if case["masked"] else Lk  # the lengths are uniform in the upper half
        pairs = B * H * (Lq * live if not case["causal"] else Lq * (Lk - (Lq - 1) / 2))
        io = 2 * B * H * Lq * D + 2 * B * Hk * live * D
        return {"bytes": int(size * (2 * io if train else io) + (B * Lk if case["masked"] else 0)),
                "flops": int(pairs * D * (12 if train else 4))}
    if case["op"] == "bias":
        n = case["batch"] * case["heads"] * case["q_len"] * case["k_len"]
        return {"bytes": 2 * size * n, "flops": n}
    n = case["groups"] * case["rows"] * case["width"]
    gate = {"none": 0, "full": n, "row": case["groups"] * case["rows"],
            "group": case["groups"] * case["width"]}[case["gate"]]
    tensors = 9 * n + 2 * gate if train else 4 * n + gate
    return {"bytes": size * tensors, "flops": n * (40 if train else 12)}


# ------------------------------------------------------------------ 64 bits
def _exact_attention(state):
    case = state["case"]
    B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    Lq, Lk, G = case["q_len"], case["k_len"], case["heads"] // case["kv_heads"]
    out, dq = (torch.empty(B, H, Lq, D, dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.empty(B, Hk, Lk, D, dtype=torch.float64, device="cuda") for _ in range(2))
    dtable = torch.zeros(H, case["buckets"], dtype=torch.float64, device="cuda")
    q_pos, k_pos = _positions(state)
    one_way = case["causal"]
    for b in range(B):
        qp = (q_pos[b] if q_pos.dim() == 2 else q_pos).double()
        kp = (k_pos[b] if k_pos.dim() == 2 else k_pos).double()
        delta = kp[None, :] - qp[:, None]
        n = case["buckets"] if one_way else case["buckets"] // 2
        far = torch.clamp(-delta, min=0) if one_way else delta.abs()
        bucket = torch.zeros_like(far, dtype=torch.long)
        for edge in _edges(case["buckets"], case["max_distance"], not one_way):
            bucket += far >= edge
        if not one_way:
            bucket += n * (delta > 0)
        allowed = torch.ones(Lq, Lk, dtype=torch.bool, device="cuda")
        if state["key_mask"] is not None:
            allowed &= state["key_mask"][b][None, :]
        if one_way:
            allowed &= delta <= 0
        for g in range(Hk):
            heads = slice(g * G, (g + 1) * G)
            q, k, v = state["q"][b, heads].double(), state["k"][b, g].double(), state["v"][b, g].double()
            s = q @ k.T / math.sqrt(D) + state["table"][heads].double()[:, bucket]
            p = torch.softmax(s.masked_fill(~allowed, -math.inf), -1)
            out[b, heads] = p @ v
            if case["mode"] == "train":
                do = state["grad"][b, heads].double()
                dv[b, g] = (p.transpose(1, 2) @ do).sum(0)
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dq[b, heads] = ds @ k / math.sqrt(D)
                dk[b, g] = (ds.transpose(1, 2) @ q).sum(0) / math.sqrt(D)
                dtable[heads].index_add_(1, bucket.reshape(-1), ds.reshape(G, -1))
    if case["mode"] != "train":
        return {"out": out}
    return {"out": out, "d_q": dq, "d_k": dk, "d_v": dv, "d_table": dtable}


def _exact_bias(state):
    case = state["case"]
    delta = state["k_pos"][..., None, :].double() - state["q_pos"][..., :, None].double()
    bucket = (case["buckets"] // 2) * (delta > 0).long()
    for edge in _edges(case["buckets"], case["max_distance"], True):
        bucket += delta.abs() >= edge
    table, grad = state["table"].double(), state["grad"].double()
    d_table = torch.zeros_like(table)
    if bucket.dim() == 2:
        out = torch.stack([row[bucket] for row in table])
        d_table.index_add_(1, bucket.reshape(-1), grad.reshape(case["heads"], -1))
    else:
        out = torch.stack([row[bucket] for row in table], 1)
        d_table.index_add_(1, bucket.reshape(-1), grad.transpose(0, 1).reshape(case["heads"], -1))
    return {"out": out, "d_table": d_table}


def _exact_normed(x, weight, bias, layer):
    c = x - x.mean(-1, keepdim=True) if layer else x
    inv = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6)
    n = c * inv
    return n, inv, n * weight + (0 if bias is None else bias)


def _exact_back(dn, n, inv, layer):
    """Through a norm without weights: n = c inv."""
    dx = inv * (dn - n * (dn * n).mean(-1, keepdim=True))
    return dx - dx.mean(-1, keepdim=True) if layer else dx


def _exact_norm(state):
    case = state["case"]
    layer = case["kind"] == "layer"
    d = {n: t.detach().double() for n, t in state.items() if isinstance(t, torch.Tensor)}
    gate, scale = d.get("gate", 1.0), d.get("scale", 1.0)
    nf, inv_f, u = _exact_normed(d["f"], d["post_weight"], d.get("post_bias"), layer)
    r = d["x"] + scale * gate * u
    nr, inv_r, z = _exact_normed(r, d["pre_weight"], d.get("pre_bias"), layer)
    if case["mode"] != "train":
        return {"r": r, "z": z}
    dz = d["grad_z"]
    dr = d["grad_r"] + _exact_back(dz * d["pre_weight"], nr, inv_r, layer)
    du = dr * scale * gate
    g = {"x": dr, "f": _exact_back(du * d["post_weight"], nf, inv_f, layer), "post_weight": (du * nf).sum((0, 1)),
         "pre_weight": (dz * nr).sum((0, 1)), "post_bias": du.sum((0, 1)), "pre_bias": dz.sum((0, 1))}
    if "gate" in d:
        g["gate"] = (dr * scale * u).sum_to_size(d["gate"].shape)
    if "scale" in d:
        g["scale"] = (dr * gate * u).sum((0, 1))
    return {"r": r, "z": z, **{"d_" + n: g[n] for n in state["leaves"]}}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "bias": _exact_bias, "norm": _exact_norm}[case["op"]](state)
