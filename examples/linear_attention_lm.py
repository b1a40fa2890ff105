"""A small language model on convolved linear attention, or (--layer delta) on the gated delta rule: trained, then
continued token by token.

    python examples/linear_attention_lm.py [--steps 200] [--generate 24] [--layer delta]

Each training sequence repeats a short random word over and over, so a model that has learned
to look back a word's length predicts everything after the first repetition.  Training
runs the layers on whole sequences (grouped dynamic convolution, chunked linear attention) and the
loss on the hidden states and the vocabulary's weight; generating runs a prompt once and
then one token at a time on the layers' caches.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from dynamic_conv1d_b200 import ConvolvedGatedDelta, ConvolvedLinearAttention, ResidualRMSNorm, linear_cross_entropy  # noqa: E402


class Block(nn.Module):
    def __init__(self, d_model: int, n_heads: int):
        super().__init__()
        self.norm1, self.norm2 = nn.RMSNorm(d_model), nn.RMSNorm(d_model)
        self.attn = ConvolvedLinearAttention(d_model, n_heads)
        self.mlp = nn.Sequential(nn.Linear(d_model, 4 * d_model, bias=False), nn.SiLU(), nn.Linear(4 * d_model, d_model, bias=False))

    def forward(self, x):
        x = x + self.attn(self.norm1(x))
        return x + self.mlp(self.norm2(x))

    def prompt(self, x):
        y, cache = self.attn.prompt(self.norm1(x))
        x = x + y
        return x + self.mlp(self.norm2(x)), cache

    def step(self, x, cache):
        x = x + self.attn.step(self.norm1(x), cache)
        return x + self.mlp(self.norm2(x))


class DeltaBlock(nn.Module):
    """The same on the gated delta rule, the second norm fused with the residual stream before it."""

    def __init__(self, d_model: int, n_heads: int):
        super().__init__()
        self.norm1, self.norm2 = nn.RMSNorm(d_model), ResidualRMSNorm(d_model)
        self.attn = ConvolvedGatedDelta(d_model, n_heads)
        self.mlp = nn.Sequential(nn.Linear(d_model, 4 * d_model, bias=False), nn.SiLU(), nn.Linear(4 * d_model, d_model, bias=False))

    def _rest(self, y, x):
        y, x = self.norm2(y, x)
        return x + self.mlp(y)

    def forward(self, x):
        return self._rest(self.attn(self.norm1(x)), x)

    def prompt(self, x):
        y, cache = self.attn.prompt(self.norm1(x))
        return self._rest(y, x), cache

    def step(self, x, cache):
        return self._rest(self.attn.step(self.norm1(x), cache), x)


class LanguageModel(nn.Module):
    def __init__(self, vocab: int, d_model: int = 256, n_heads: int = 4, n_layers: int = 2, layer: str = "linear"):
        super().__init__()
        self.embed = nn.Embedding(vocab, d_model)
        nn.init.normal_(self.embed.weight, std=d_model**-0.5)
        block = DeltaBlock if layer == "delta" else Block
        self.blocks = nn.ModuleList(block(d_model, n_heads) for _ in range(n_layers))
        self.norm = nn.RMSNorm(d_model)
        self.scale = d_model**0.5

    def hidden(self, tokens):
        x = self.embed(tokens) * self.scale
        for b in self.blocks:
            x = b(x)
        return self.norm(x)

    def loss(self, tokens):
        """Mean cross entropy of every next token (the vocabulary's weight is the embedding's)."""
        h = self.hidden(tokens[:, :-1])
        return linear_cross_entropy(h.contiguous(), self.embed.weight, tokens[:, 1:].contiguous())

    @torch.no_grad()
    def generate(self, prompt, n: int):
        x = self.embed(prompt) * self.scale
        caches = []
        for b in self.blocks:
            x, c = b.prompt(x)
            caches.append(c)
        h = self.norm(x[:, -1])
        out = []
        for _ in range(n):
            token = (h @ self.embed.weight.T).argmax(-1)
            out.append(token)
            x = self.embed(token) * self.scale
            for b, c in zip(self.blocks, caches):
                x = b.step(x, c)
            h = self.norm(x)
        return torch.stack(out, 1)


def repeating_words(batch: int, length: int, word: int, vocab: int, g: torch.Generator):
    w = torch.randint(0, vocab, (batch, word), device=g.device, generator=g)
    return w.repeat(1, -(-length // word))[:, :length]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--vocab", type=int, default=500)
    ap.add_argument("--generate", type=int, default=24)
    ap.add_argument("--layer", choices=("linear", "delta"), default="linear")
    a = ap.parse_args(argv)
    device = torch.device("cuda")
    torch.manual_seed(0)
    g = torch.Generator(device=device).manual_seed(1)
    model = LanguageModel(a.vocab, layer=a.layer).to(device, torch.bfloat16)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3, weight_decay=0.0)
    first = last = None
    for i in range(a.steps):
        loss = model.loss(repeating_words(32, 129, 6, a.vocab, g))
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if i % 20 == 0 or i == a.steps - 1:
            last = loss.item()
            first = last if first is None else first
            print(f"step {i}: loss {last:.3f}")
    text = repeating_words(8, 40 + a.generate, 6, a.vocab, g)
    right = (model.generate(text[:, :40], a.generate) == text[:, 40:]).float().mean().item() if a.generate else 0.0
    print(f"{100 * right:.0f}% of the generated tokens continue their word")
    return first, last, right


if __name__ == "__main__":
    main()
