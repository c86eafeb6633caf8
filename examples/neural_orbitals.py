"""A small neural wave function on the operators of its network and slogdet: occupied sites ->
tokens -> attention blocks -> orbitals -> log|psi| = log|det|, one training step of it, the
evaluation of one electron's token against the others, and the probability of the site that a
move proposes.

    python -m examples.neural_orbitals [--samples 64] [--electrons 32] [--sites 64] [--dtype float32]

psi(occ) = det of the (electrons x electrons) matrix whose row i is a linear map of electron i's
token after the blocks. The tokens of one sample attend to each other with a learned bias of
their sites' distance; the determinant is float32 whatever the blocks' type.
"""

import argparse
import math

import torch

import fermix_b200 as fx


class Table(torch.nn.Embedding):
    """Sites -> tokens."""

    def forward(self, sites):
        return fx.token_embedding(sites, self.weight)


class Map(torch.nn.Linear):
    """residual + activation(linear map)."""

    def forward(self, x, activation=None, residual=None):
        return fx.fused_linear(x, self.weight, self.bias, activation=activation, residual=residual)


class Block(torch.nn.Module):
    """Attention over the electrons, then a position-wise map; between them, and after, the residual
    with its norms (``residual_norm`` returns the stream and the next part's normed input)."""

    def __init__(self, width, heads, kv_heads, buckets=16):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.qkv = Map(width, (heads + 2 * kv_heads) * self.dim, bias=False)
        self.out = Map(width, width, bias=False)
        self.up = Map(width, 2 * width, bias=False)
        self.down = Map(2 * width, width, bias=False)
        self.table = torch.nn.Parameter(torch.zeros(heads, buckets))
        for i in (1, 2):
            self.register_parameter(f"post{i}", torch.nn.Parameter(torch.ones(width)))
            self.register_parameter(f"pre{i}", torch.nn.Parameter(torch.ones(width)))
            self.register_parameter(f"scale{i}", torch.nn.Parameter(torch.full((width,), 0.1)))
        self.gate = Map(1, width)

    def heads_of(self, z):
        """(q, k, v), head-major views of the token-major projection."""
        b, n, _ = z.shape
        y = self.qkv(z).view(b, n, self.heads + 2 * self.kv_heads, self.dim).transpose(1, 2)
        return y.split([self.heads, self.kv_heads, self.kv_heads], dim=1)

    def forward(self, x, z, occ, filling):
        b, n, width = x.shape
        q, k, v = self.heads_of(z)
        a = fx.biased_attention(q, k, v, self.table, q_pos=occ, k_pos=occ, max_distance=64)
        gate = torch.sigmoid(self.gate(filling))[:, None, :]  # one vector per sample
        x, z = fx.residual_norm(x, self.out(a.transpose(1, 2).reshape(b, n, width)), self.post1, self.pre1, gate=gate,
                                scale=self.scale1)
        f = self.down(self.up(z, activation="silu"))
        return fx.residual_norm(x, f, self.post2, self.pre2, scale=self.scale2)


class NeuralOrbitals(torch.nn.Module):
    def __init__(self, sites, electrons, width=64, heads=4, kv_heads=2, blocks=2):
        super().__init__()
        self.embed = Table(sites, width)
        self.blocks = torch.nn.ModuleList(Block(width, heads, kv_heads) for _ in range(blocks))
        self.orbitals = Map(width, electrons, bias=False)
        self.sites = sites

    def tokens(self, occ):
        x = z = self.embed(occ)
        filling = torch.full((occ.shape[0], 1), occ.shape[1] / self.sites, dtype=x.dtype, device=x.device)
        for block in self.blocks:
            x, z = block(x, z, occ, filling)
        return z

    def forward(self, occ):
        """(sign, log|psi|) of each sample."""
        phi = self.orbitals(self.tokens(occ)).float()
        return fx.slogdet(phi / math.sqrt(phi.shape[-1]))


def moved_token(block, z, occ, electron, site):
    """The attention output of one electron at another site, against the other electrons' keys: one
    query a sample, the moved electron itself left out by the mask."""
    q, k, v = block.heads_of(z)
    rows = torch.arange(z.shape[0], device=z.device)
    keep = torch.ones(occ.shape, dtype=torch.bool, device=z.device)
    keep[rows, electron] = False
    with torch.no_grad():
        return fx.biased_attention(q[rows, :, electron][:, :, None, :], k, v, block.table, q_pos=site[:, None],
                                   k_pos=occ, key_mask=keep, max_distance=64)


def proposal(model, z, occ, electron, site, top=0):
    """log-probability of one electron's move to a site, under a softmax over the sites that are free (its own among
    them) of its token against the sites' table; the entropy, and the likeliest sites."""
    rows = torch.arange(z.shape[0], device=z.device)
    free = torch.ones(z.shape[0], model.sites, dtype=torch.bool, device=z.device).scatter_(1, occ.long(), False)
    free[rows, occ[:, electron].long()] = True
    logits = fx.fused_linear(z[rows, electron], model.embed.weight)
    return fx.token_logprobs(logits, site, scale=z.shape[-1] ** -0.5, mask=free, top=top)


def step(model, optimiser, occ, energy):
    """One step of the variational gradient 2 <(E - <E>) grad log|psi|>; returns log|psi|."""
    _, logabs = model(occ)
    loss = 2 * ((energy - energy.mean()) * logabs).mean()
    optimiser.zero_grad(set_to_none=True)
    loss.backward()
    optimiser.step()
    return logabs.detach()


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--samples", type=int, default=64)
    p.add_argument("--electrons", type=int, default=32)
    p.add_argument("--sites", type=int, default=64)
    p.add_argument("--steps", type=int, default=5)
    p.add_argument("--dtype", choices=["float32", "bfloat16"], default="float32")
    a = p.parse_args(argv)
    torch.manual_seed(0)
    dtype = getattr(torch, a.dtype)
    model = NeuralOrbitals(a.sites, a.electrons).cuda().to(dtype)
    optimiser = torch.optim.SGD(model.parameters(), lr=1e-2)
    occ = torch.rand(a.samples, a.sites, device="cuda").topk(a.electrons).indices.sort().values.to(torch.int32)
    # a diagonal stand-in for the local energy: neighbouring pairs
    energy = (occ[:, 1:] - occ[:, :-1] == 1).sum(1).float()
    for n in range(a.steps):
        logabs = step(model, optimiser, occ, energy)
        print(f"step {n}: <log|psi|> = {logabs.mean().item():.4f}")
    block = model.blocks[0]
    bias = fx.position_bias(block.table.detach(), occ[0], max_distance=64)
    site = (occ[:, 0] + 1).remainder(a.sites).to(torch.int32)
    out = moved_token(block, model.embed(occ).detach(), occ, 0, site)
    print(f"bias of the first sample: {tuple(bias.shape)}, moved electron's token: {tuple(out.shape)}")
    with torch.no_grad():
        logp, entropy, _, likeliest = proposal(model, model.tokens(occ), occ, 0, site, top=3)
    print(f"first sample's move to site {site[0].item()}: log p = {logp[0].item():.3f} (entropy {entropy[0].item():.3f}), "
          f"likeliest sites {likeliest[0].tolist()}")
    return model, occ, logabs


if __name__ == "__main__":
    main()
