"""Train a small encoder through the alignment: one block of rotary self-attention, one with a learned relative
position bias, residual dropout after each, then soft Smith-Waterman of the two sequences' embeddings.

Pairs of sequences of uneven lengths share a planted segment, written in other letters in the second (a fixed
exchange, which the encoder has to learn); the loss asks the alignment to prefer the true partner over another
sequence of the batch.  Run it from the repository's root (needs a B200):

    python examples/encode_align.py --steps 60
"""
import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import d2p_b200 as d2p


class Block(nn.Module):
    """x + dropout(attention(...) Wo): rotary with head norms, or with a bias by relative position."""

    def __init__(self, width, heads, key_heads, rotary, p):
        super().__init__()
        self.heads, self.key_heads, self.size, self.rotary, self.p = heads, key_heads, width // heads, rotary, p
        self.norm = nn.LayerNorm(width)
        self.qkv = nn.Linear(width, (heads + 2 * key_heads) * self.size, bias=False)
        self.out = nn.Linear(heads * self.size, width, bias=False)
        if rotary:
            self.q_weight, self.k_weight = (nn.Parameter(torch.ones(self.size)) for _ in range(2))
        else:
            self.bias = nn.Parameter(torch.zeros(32, heads))

    def forward(self, x, lengths, cos, sin, seed, offset):
        B, L, _ = x.shape
        qkv = self.qkv(self.norm(x)).view(B, L, self.heads + 2 * self.key_heads, self.size)
        q, k, v = qkv.split([self.heads, self.key_heads, self.key_heads], 2)
        if self.rotary:
            q, k = d2p.qk_norm_rope(q, k, self.q_weight, self.k_weight, cos, sin)
            y = d2p.attention(q, k, v, lengths=lengths)
        else:
            y = d2p.attention(q, k, v, bias=self.bias, lengths=lengths)
        return d2p.dropout_add(self.out(y.flatten(2)), x, self.p if self.training else 0.0, seed, offset)


class Encoder(nn.Module):
    def __init__(self, letters=25, width=128, heads=4, key_heads=2, blocks=2, p=0.1, longest=1024):
        super().__init__()
        self.embed = nn.Embedding(letters, width)
        self.blocks = nn.ModuleList(Block(width, heads, key_heads, i % 2 == 0, p) for i in range(blocks))
        half = width // heads // 2
        angle = torch.arange(longest)[:, None] * 10000.0 ** (-torch.arange(half) / half)
        self.register_buffer("cos", angle.cos())
        self.register_buffer("sin", angle.sin())
        self.scale = width ** -0.25

    def forward(self, tokens, length, seed=0, step=0):
        lengths = torch.stack([length, length], 1).to(torch.int32)
        x = self.embed(tokens)
        for i, block in enumerate(self.blocks):
            x = block(x, lengths, self.cos, self.sin, seed, step * len(self.blocks) + i)
        return x * self.scale


def pairs(batch, longest, letters, generator):
    """Two sets of sequences of uneven lengths; x's partner in y has a segment of x in exchanged letters."""
    other = torch.randperm(letters, generator=torch.Generator().manual_seed(1))
    lx, ly = (torch.randint(longest * 2 // 3, longest + 1, (batch,), generator=generator) for _ in range(2))
    x, y = (torch.randint(0, letters, (batch, longest), generator=generator) for _ in range(2))
    n = longest // 2
    for b in range(batch):
        i, j = (int(torch.randint(0, int(l) - n + 1, (1,), generator=generator)) for l in (lx[b], ly[b]))
        y[b, j:j + n] = other[x[b, i:i + n]]
    return x, y, lx, ly


def train(steps, batch=16, longest=192, seed=0, report=print):
    generator = torch.Generator().manual_seed(seed)
    torch.manual_seed(seed)
    model = Encoder().cuda()
    # matrices in bf16 for the tensor cores, norms and the bias by position in fp32; attention takes either bias
    for module in model.modules():
        if isinstance(module, (nn.Linear, nn.LayerNorm, nn.Embedding)):
            module.to(torch.bfloat16)
    optimizer = torch.optim.AdamW(model.parameters(), lr=5e-3)
    losses = []
    for step in range(steps):
        x, y, lx, ly = (t.cuda() for t in pairs(batch, longest, 25, generator))
        ex = model(x, lx, seed, 2 * step)
        ey = model(y, ly, seed, 2 * step + 1)
        lengths = torch.stack([lx, ly], 1).to(torch.int32)
        other = torch.stack([lx, ly.roll(1)], 1).to(torch.int32)
        true = d2p.soft_sw_embed(ex, ey, gap=-1.0, temperature=1.0, lengths=lengths).value
        false = d2p.soft_sw_embed(ex, ey.roll(1, 0), gap=-1.0, temperature=1.0, lengths=other).value
        loss = torch.nn.functional.softplus((false - true) / 10.0).mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if report and (step % 10 == 0 or step + 1 == steps):
            report(f"step {step:3d}  loss {losses[-1]:.4f}  true pairs ahead {float((true > false).float().mean()):.2f}")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=60)
    train(parser.parse_args().steps)
