"""Local attention with a learned position bias, trained and then decoded.

A small model of two halves, on synthetic sequences (a random motif, repeated,
some tokens replaced):

* the source half reads the whole sequence with the trunk's two tracks side by
  side: local attention in both directions (``flash_window_attn``), and a
  Sinkhorn transport whose cost is biased by relative position
  (``relative_position_bias`` + ``sinkhorn_solve`` + ``compute_transport_output``);
* the answering half is causal: ``flash_window_attn`` over all positions in
  training, ``window_attn_decode`` over a cache for one token at a time.

Every weight is trained, the bias weights of all three included.  The script
prints the loss, generates, and compares the cached steps with one pass over the
whole generated sequence.

    python examples/window_attention.py [--steps 200] [--tokens 96]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepfold-linear_b200"))

from deepfold.model.kernels.flash_window_attn import flash_window_attn, window_attn_decode  # noqa: E402
from deepfold.model.position_encoding import RelativeBuckets, relative_position_bias  # noqa: E402
from deepfold.model.sinkhorn import compute_transport_output, sinkhorn_solve  # noqa: E402

VOCAB, PERIOD = 16, 5


class LocalAttention(nn.Module):
    """Windowed attention with sinks; query heads share key heads."""

    def __init__(self, dim, heads, kv_heads, head_dim, window, sinks, causal, dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        self.options = dict(window=window, sinks=sinks)
        self.causal = causal
        self.buckets = RelativeBuckets.log(16, 32, bidirectional=not causal)
        self.norm = nn.LayerNorm(dim)
        self.qkv = nn.Linear(dim, (heads + 2 * kv_heads) * head_dim, bias=False)
        self.out = nn.Linear(heads * head_dim, dim, bias=False)
        self.pos_weight = nn.Parameter(torch.zeros(heads, self.buckets.num_buckets))

    def project(self, x):
        """x (B,n,dim) as Q (B,H,n,d), K and V (B,H_kv,n,d): views of one projection."""
        h = self.qkv(self.norm(x)).to(self.dtype).unflatten(-1, (-1, self.head_dim)).transpose(1, 2)
        return h.split([self.heads, self.kv_heads, self.kv_heads], dim=1)

    def forward(self, x, mask=None):
        q, k, v = self.project(x)
        o = flash_window_attn(q, k, v, causal=self.causal, pos_weight=self.pos_weight, buckets=self.buckets,
                              mask=mask, **self.options)
        return x + self.out(o.transpose(1, 2).flatten(2).to(x.dtype))

    def new_cache(self, batch, n_max, device):
        return [torch.empty(batch, self.kv_heads, n_max, self.head_dim, dtype=self.dtype, device=device)
                for _ in range(2)]

    def fill(self, x, cache):
        """The keys and values of positions 0 .. n-1, and the forward's output."""
        _, k, v = self.project(x)
        for store, new in zip(cache, (k, v)):
            store[:, :, :x.shape[1]] = new
        return self(x)

    def step(self, x, cache, lengths):
        """One token a sequence: x (B,dim) at position lengths[b]."""
        q, k, v = (t[:, :, 0] for t in self.project(x[:, None]))
        rows = torch.arange(x.shape[0], device=x.device)
        for store, new in zip(cache, (k, v)):
            store[rows, :, lengths] = new
        o = window_attn_decode(q, *cache, lengths + 1, pos_weight=self.pos_weight, buckets=self.buckets,
                               **self.options)
        return x + self.out(o.flatten(1).to(x.dtype))


class BiasedTransport(nn.Module):
    """Sinkhorn transport between the tokens; the cost takes a learned bias by relative position."""

    def __init__(self, dim, heads, head_dim, iterations=4):
        super().__init__()
        self.heads, self.head_dim, self.iterations = heads, head_dim, iterations
        self.buckets = RelativeBuckets.log(16, 32, bidirectional=True)
        self.norm = nn.LayerNorm(dim)
        self.qkvg = nn.Linear(dim, 4 * heads * head_dim, bias=False)
        self.out = nn.Linear(heads * head_dim, dim, bias=False)
        self.pos_weight = nn.Parameter(torch.zeros(heads, self.buckets.num_buckets))
        self.register_buffer("eps", torch.full((heads,), 0.5))

    def forward(self, x):
        B, n, _ = x.shape
        h = self.qkvg(self.norm(x)).unflatten(-1, (4, self.heads, self.head_dim)).permute(2, 0, 3, 1, 4)
        q, k, v, g = (t.contiguous() for t in h)
        cost = -q @ k.mT * self.head_dim ** -0.5 - relative_position_bias(self.pos_weight, self.buckets, n, n)
        marginal = torch.full((B, self.heads, n), 1.0 / n, device=x.device).log()
        log_u, log_v = sinkhorn_solve(cost, marginal, marginal, self.eps, K=self.iterations)
        o, _, _ = compute_transport_output(v, g, log_u, log_v, cost, self.eps)
        return x + self.out(o)


class Model(nn.Module):
    def __init__(self, dim=64, heads=4, kv_heads=2, head_dim=16, window=24, sinks=2):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, dim)
        self.source = LocalAttention(dim, heads, heads, head_dim, window, sinks, causal=False)
        self.transport = BiasedTransport(dim, heads, head_dim)
        self.answer = LocalAttention(dim, heads, kv_heads, head_dim, window, sinks, causal=True)
        self.logits = nn.Sequential(nn.LayerNorm(dim), nn.Linear(dim, VOCAB))

    def context(self, source, mask=None):
        """What the source half says of a sequence, (B,1,dim)."""
        x = self.transport(self.source(self.embed(source), mask))
        return x.mean(1, keepdim=True)

    def forward(self, tokens, source):
        return self.logits(self.answer(self.embed(tokens) + self.context(source)))

    @torch.no_grad()
    def generate(self, prompt, source, n_new):
        """Greedy: (tokens (B, n + n_new), the logits of every generated step)."""
        B, n = prompt.shape
        ctx = self.context(source)
        cache = self.answer.new_cache(B, n + n_new, prompt.device)
        logits = [self.logits(self.answer.fill(self.embed(prompt) + ctx, cache)[:, -1])]
        tokens = [prompt, logits[0].argmax(-1, keepdim=True)]
        lengths = torch.full((B,), n, dtype=torch.int64, device=prompt.device)
        while len(logits) < n_new:
            x = self.embed(tokens[-1][:, 0]) + ctx[:, 0]
            logits.append(self.logits(self.answer.step(x, cache, lengths)))
            tokens.append(logits[-1].argmax(-1, keepdim=True))
            lengths += 1
        return torch.cat(tokens, 1), torch.stack(logits, 1)


def batch(B, n, generator, device):
    """(tokens, source): a random motif of PERIOD tokens repeated, and the same with a tenth of them replaced."""
    motif = torch.randint(VOCAB, (B, PERIOD), generator=generator)
    tokens = motif.repeat(1, n // PERIOD + 1)[:, :n]
    noise = torch.randint(VOCAB, (B, n), generator=generator)
    source = torch.where(torch.rand(B, n, generator=generator) < 0.1, noise, tokens)
    return tokens.to(device), source.to(device)


def run(steps=200, n=96, B=16, n_new=32, seed=0, device="cuda", log=print):
    """Train, generate, compare; returns (first loss, last loss, share of right tokens, largest difference of the
    cached steps' logits from one pass over the generated sequence)."""
    torch.manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    model = Model().to(device)
    optimizer = torch.optim.AdamW(model.parameters(), lr=5e-3)
    losses = []
    for i in range(steps):
        tokens, source = batch(B, n, g, device)
        loss = F.cross_entropy(model(tokens[:, :-1], source).flatten(0, 1), tokens[:, 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if log and (i % 20 == 0 or i == steps - 1):
            log(f"step {i:3d}  loss {float(losses[-1]):.3f}")
    tokens, source = batch(B, n + n_new, g, device)
    out, logits = model.generate(tokens[:, :n], source[:, :n], n_new)
    right = float((out[:, n:] == tokens[:, n:]).float().mean())
    with torch.no_grad():
        again = model.logits(model.answer(model.embed(out[:, :-1]) + model.context(source[:, :n])))[:, n - 1:]
    apart = float((again - logits).abs().max())
    if log:
        log(f"generated {n_new} tokens a sequence, {100 * right:.1f} % as the motif has them; "
            f"cached steps within {apart:.4f} of one pass (logits)")
    return float(losses[0]), float(losses[-1]), right, apart


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--tokens", type=int, default=96)
    args = parser.parse_args()
    run(args.steps, args.tokens)
