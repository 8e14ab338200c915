"""A small fermionic wave function on a chain, and an autoregressive sampler of configurations, from
the operators of fermix_amd.network:

* ``Pairing``: electrons at sites x_1 .. x_n attend to each other with a bias by their distance, and
  log|psi| is the Pfaffian of a pairing matrix made of their features and of a learned function of
  their distance (attention, residual_norm, relative_bias, slogpf);
* ``Sampler``: a causal network over the chain's sites that draws occupations one site at a time
  from a paged cache (attention_step) and is trained over whole configurations (attention).

    python examples/network.py            trains both for a few steps on one GPU
"""

import math
import os
import sys

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fermix_amd as fx


class Block(nn.Module):
    """Attention and a two-layer map, each between norms with a gate and a residual scale. ``z`` is
    the normed residual stream, which the block before has formed already."""

    def __init__(self, dim, heads, buckets):
        super().__init__()
        self.heads = heads
        self.qkv = nn.Linear(dim, 3 * dim, bias=False)
        self.out = nn.Linear(dim, dim, bias=False)
        self.mlp = nn.Sequential(nn.Linear(dim, 2 * dim), nn.GELU(), nn.Linear(2 * dim, dim))
        self.table = nn.Parameter(torch.zeros(buckets, heads))
        self.gate = nn.Linear(dim, dim)
        self.scale = nn.ParameterList([nn.Parameter(torch.full((dim,), 0.3)) for _ in range(2)])
        self.post = nn.ParameterList([nn.Parameter(torch.ones(dim)) for _ in range(2)])
        self.pre = nn.ParameterList([nn.Parameter(torch.ones(dim)) for _ in range(2)])

    def join(self, i, x, h, gate=None):
        return fx.residual_norm(x, h, post_weight=self.post[i], gate=gate, scale=self.scale[i], pre_weight=self.pre[i])

    def forward(self, x, z, attend):
        """attend(q, k, v, table): (.., heads, d) each."""
        q, k, v = self.qkv(z).unflatten(-1, (3, self.heads, -1)).unbind(-3)
        h = attend(q, k, v, self.table).flatten(-2)
        x, z = self.join(0, x, self.out(h), torch.sigmoid(self.gate(z)))
        return self.join(1, x, self.mlp(z))


class Pairing(nn.Module):
    def __init__(self, sites, dim=64, heads=4, blocks=2, distance=16):
        super().__init__()
        self.embed = nn.Embedding(sites, dim)
        self.register_buffer("buckets", fx.distance_buckets(16, distance))
        self.blocks = nn.ModuleList(Block(dim, heads, 16) for _ in range(blocks))
        self.pair = nn.Linear(dim, dim, bias=False)
        self.by_distance = nn.Parameter(0.1 * torch.randn(16, 1))

    def forward(self, sites):
        """sign, log|psi| of configurations (B, n) of an even number of electrons."""
        x = self.embed(sites)
        z = x
        pos = sites.to(torch.int32)
        for block in self.blocks:
            x, z = block(x, z, lambda q, k, v, t: fx.attention(q, k, v, table=t, buckets=self.buckets, q_pos=pos, k_pos=pos))
        a = self.pair(z) @ z.transpose(1, 2) / math.sqrt(z.shape[-1])
        a = a + fx.relative_bias(self.by_distance, self.buckets, pos, pos)[:, 0]
        return fx.slogpf(a)  # of (a - a^T) / 2


class Sampler(nn.Module):
    """Occupation 0 / 1 of each site given those before it."""

    def __init__(self, sites, dim=64, heads=4, blocks=2):
        super().__init__()
        self.sites, self.heads, self.dim = sites, heads, dim
        self.embed = nn.Embedding(3, dim)  # 2: nothing yet
        self.register_buffer("buckets", fx.distance_buckets(16, 32, bidirectional=False))
        self.blocks = nn.ModuleList(Block(dim, heads, 16) for _ in range(blocks))
        self.head = nn.Linear(dim, 2)

    def forward(self, occupied):
        """log p of configurations (B, sites) of 0 and 1."""
        start = torch.full_like(occupied[:, :1], 2)
        x = self.embed(torch.cat([start, occupied[:, :-1]], 1))
        z = x
        for block in self.blocks:
            x, z = block(x, z, lambda q, k, v, t: fx.attention(q, k, v, table=t, buckets=self.buckets, causal=True))
        logp = F.log_softmax(self.head(z).float(), -1)
        return logp.gather(-1, occupied[..., None])[..., 0].sum(-1)

    @torch.no_grad()
    def sample(self, batch, page=16):
        """configurations (batch, sites) and their log p, one site at a time."""
        dev, dtype = self.head.weight.device, self.embed.weight.dtype
        pages = -(-self.sites // page)
        shape = (len(self.blocks), 2, batch * pages, page, self.heads, self.dim // self.heads)
        cache = torch.empty(shape, device=dev, dtype=dtype)
        table = torch.arange(batch * pages, device=dev, dtype=torch.int32).view(batch, pages)
        token = torch.full((batch,), 2, device=dev)
        total, drawn = torch.zeros(batch, device=dev), []
        for site in range(self.sites):
            lengths = torch.full((batch,), site, device=dev, dtype=torch.int32)
            x = self.embed(token)
            z = x
            for block, (k_cache, v_cache) in zip(self.blocks, cache):
                x, z = block(x, z, lambda q, k, v, t: fx.attention_step(
                    q, k_cache, v_cache, table, lengths, k=k, v=v, table=t, buckets=self.buckets))
            logp = F.log_softmax(self.head(z).float(), -1)
            token = torch.multinomial(logp.exp(), 1)[:, 0]
            total += logp.gather(-1, token[:, None])[:, 0]
            drawn.append(token)
        return torch.stack(drawn, 1), total


def train(model, loss_of, steps, lr=5e-3):
    opt = torch.optim.Adam(model.parameters(), lr)
    losses = []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        loss = loss_of(model)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


def misfit(model, where):
    """Mean square distance of log|psi|, up to a constant, from a target that falls with the electrons' spread."""
    target = -0.05 * (where - where.float().mean(1, keepdim=True)).abs().sum(1)
    off = model(where)[1] - target
    return (off - off.mean()).square().mean()


def main(sites=32, electrons=16, batch=256, steps=60, seed=0):
    torch.manual_seed(seed)
    dev = "cuda"
    where = torch.rand(batch, sites, device=dev).argsort(1)[:, :electrons].sort(1).values
    pairing = Pairing(sites).to(dev)
    fit = train(pairing, lambda m: misfit(m, where), steps)
    print("pairing function: mean square misfit of log|psi| %.4f -> %.4f" % (fit[0], fit[-1]), flush=True)

    occupied = torch.zeros(batch, sites, dtype=torch.long, device=dev).scatter_(1, where, 1)
    sampler = Sampler(sites).to(dev)
    nll = train(sampler, lambda m: -m(occupied).mean(), steps)
    print("sampler: -log p of the configurations %.3f -> %.3f" % (nll[0], nll[-1]), flush=True)
    drawn, logp = sampler.sample(batch)
    with torch.no_grad():
        whole = sampler(drawn)
    off = (logp - whole).abs().max().item()
    print("sampled %d configurations, %.1f electrons each; log p by steps and as a whole differ by %.1e" % (
        batch, drawn.float().sum(1).mean().item(), off), flush=True)
    return fit, nll, off


if __name__ == "__main__":
    main()
