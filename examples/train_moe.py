#!/usr/bin/env python3
"""Trains a small mixture-of-experts language model on one GPU with the operators of muon_amd next to each other:

    route_topk        the experts of each token, their weights, and the losses that keep the experts balanced
    residual_norm     the norm after each block, its gate and residual scale, and the norm before the next block
    clip_coefficient, AdamW(state_bits=8)     embedding, head, router, norms, gates and scales, clipped on the way
    clip_grad_norm_, SingleDeviceMuon         every matrix of the experts and of the token mixing (3-D: a batch of matrices)

The data is a seeded random Markov chain over a small vocabulary, so nothing has to be downloaded.

    python examples/train_moe.py [--steps 200] [--width 256] [--layers 4] [--experts 8] [--top-k 2] [--state-bits 8]
"""
import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import muon_amd  # noqa: E402

VOCAB, LENGTH, BATCH = 128, 64, 16


class Block(nn.Module):
    """Mixes each token with the ones before it, then sends it through its experts."""

    def __init__(self, width, experts, top_k):
        super().__init__()
        self.top_k = top_k
        self.mix = nn.Parameter(torch.randn(2 * width, width) * (2 * width) ** -0.5)
        self.router = nn.Parameter(torch.randn(width, experts) * width ** -0.5)
        self.up = nn.Parameter(torch.randn(experts, width, 2 * width) * width ** -0.5)
        self.down = nn.Parameter(torch.randn(experts, 2 * width, width) * (2 * width) ** -0.5)
        self.gate = nn.Parameter(torch.zeros(width, 1))
        self.post_weight = nn.Parameter(torch.ones(width))
        self.pre_weight = nn.Parameter(torch.ones(width))            # of the norm before the block that follows
        self.scale = nn.Parameter(torch.full((width,), 0.5))

    def forward(self, stream, y):
        """stream: the residual stream, fp32; y: its norm, bf16.  -> both after this block, and the router's losses."""
        before = torch.cat([torch.zeros_like(y[:, :1]), y[:, :-1]], 1)
        tokens = torch.cat([y, before], -1).flatten(0, 1) @ self.mix.bfloat16()
        routing = muon_amd.route_topk(tokens @ self.router.bfloat16(), self.top_k)
        out = torch.zeros_like(tokens)
        for e in range(self.up.size(0)):
            token, choice = torch.where(routing.indices == e)
            hidden = torch.relu(tokens[token] @ self.up[e].bfloat16()).square()
            out = out.index_add(0, token, (hidden @ self.down[e].bfloat16()) * routing.weights[token, choice, None].bfloat16())
        out = out.view_as(y)
        stream, y = muon_amd.residual_norm(stream, out, self.post_weight, self.pre_weight, gate=out @ self.gate.bfloat16(), scale=self.scale)
        return stream, y, routing.balance_loss, routing.z_loss


class Model(nn.Module):
    def __init__(self, width, layers, experts, top_k):
        super().__init__()
        self.embedding = nn.Parameter(torch.randn(VOCAB, width))
        self.head = nn.Parameter(torch.zeros(width, VOCAB))
        self.blocks = nn.ModuleList(Block(width, experts, top_k) for _ in range(layers))

    def forward(self, ids):
        stream = self.embedding[ids]
        y = (stream * torch.rsqrt(stream.square().mean(-1, keepdim=True) + 1e-6)).bfloat16()
        balance = z = 0.0
        for block in self.blocks:
            stream, y, b, lse = block(stream, y)
            balance, z = balance + b, z + lse
        return (y @ self.head.bfloat16()).float(), balance / len(self.blocks), z / len(self.blocks)


def batches(device, seed=0):
    """Batches of sequences in which each token's successor is one of four, by fixed chances."""
    gen = torch.Generator().manual_seed(seed)
    successors = torch.randint(VOCAB, (VOCAB, 4), generator=gen)
    while True:
        ids = torch.randint(VOCAB, (BATCH, 1), generator=gen)
        for _ in range(LENGTH):
            pick = torch.multinomial(torch.tensor([0.55, 0.25, 0.15, 0.05]), BATCH, replacement=True, generator=gen)
            ids = torch.cat([ids, successors[ids[:, -1], pick][:, None]], 1)
        yield ids.to(device)


def train(steps=200, width=256, layers=4, experts=8, top_k=2, state_bits=8, seed=0, report=None):
    """-> the losses of all steps (next-token cross entropy in nats)."""
    torch.manual_seed(seed)
    device = torch.device("cuda", torch.cuda.current_device())
    model = Model(width, layers, experts, top_k).to(device)
    matrices = [p for b in model.blocks for p in (b.mix, b.up, b.down)]
    ids_of_matrices = {id(p) for p in matrices}
    others = [p for p in model.parameters() if id(p) not in ids_of_matrices]
    muon = muon_amd.SingleDeviceMuon(matrices, lr=0.02, weight_decay=0.01)
    adamw = muon_amd.AdamW(others, lr=3e-3, betas=(0.9, 0.95), weight_decay=0.01, state_bits=state_bits)
    losses = []
    for step, ids in zip(range(steps), batches(device, seed)):
        logits, balance, z = model(ids[:, :-1])
        loss = nn.functional.cross_entropy(logits.flatten(0, 1), ids[:, 1:].flatten())
        (loss + 0.01 * balance + 0.001 * z).backward()
        muon_amd.clip_grad_norm_(matrices, 1.0)
        norm, coefficient = muon_amd.clip_coefficient(others, 1.0)
        muon.step()
        adamw.step(grad_scale=coefficient)
        muon.zero_grad()
        adamw.zero_grad()
        losses.append(loss.detach())
        balance = balance.detach()
        if report and (step % report == 0 or step == steps - 1):
            print(f"step {step:4d}  loss {float(losses[-1]):.4f}  balance {float(balance):.3f}  gradient norm {float(norm):.3f}", flush=True)
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--top-k", type=int, default=2)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    train(a.steps, a.width, a.layers, a.experts, a.top_k, a.state_bits, report=20)
