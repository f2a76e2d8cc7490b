"""One attention layer serving prompts with an image inside, from an 8-bit cache that is kept within a budget.

    python examples/kv8_session.py [--batch 4] [--text 200] [--image 24x32] [--new 64] [--budget 512] [--e4m3]

What a server does with the package, step by step:
  1. the prompt: one projection gives q, k and v; rope_axes rotates q and k by (time, height, width); kv8_append
     stores k and v in 8 bits; kv8_attention attends the cache and accumulates each token's attention weight;
  2. kv8_evict cuts every head's cache to the budget: the tokens that got most weight, and the last ones;
  3. each new token: project, rotate, append, attend (accumulating on), project out;
     when a sequence's cache is full again, evict again.
It prints the bytes the cache takes, and how far the layer's outputs are from the same layer's over 16-bit keys and
values of all tokens. (Weights and inputs are random, so attention is spread evenly over the tokens: the worst case
for an eviction, which in a trained model drops tokens that hardly anything attends to.)
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gguf_train_b200 import (KV8Cache, functional as F, kv8_append, kv8_attention, kv8_evict, rope_axes,  # noqa: E402
                             scaled_dot_product_attention)

SECTIONS = (16, 24, 24)  # pairs of dimensions for time, height, width: head size 128


def image_positions(batch: int, text: int, rows: int, cols: int, new: int) -> torch.Tensor:
    """(3, batch, text + rows * cols + new) positions: half the text, the image on its grid, the rest of the text."""
    head = text // 2
    before = torch.arange(head).expand(3, -1)
    cell = torch.arange(rows * cols)
    image = torch.stack((torch.full_like(cell, head), head + cell // cols, head + cell % cols))
    start = head + max(rows, cols)
    after = torch.arange(start, start + text - head + new).expand(3, -1)
    return torch.cat((before, image, after), dim=1)[:, None].expand(3, batch, -1).to("cuda", torch.int32).contiguous()


class Layer:
    """Grouped-query attention with random weights, in bf16."""

    def __init__(self, embed: int, heads: int, kv_heads: int, head_dim: int = 128, seed: int = 0) -> None:
        g = torch.Generator("cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        mk = lambda n, m: (torch.randn((n, m), device="cuda", generator=g) * m ** -0.5).to(torch.bfloat16)  # noqa: E731
        self.w_qkv, self.w_out = mk((heads + 2 * kv_heads) * head_dim, embed), mk(embed, heads * head_dim)

    def project(self, x: torch.Tensor, positions: torch.Tensor):
        """x (B, n, E) -> rotated q (B, H, n, D) and k, and v as a view of the projection."""
        qkv = F.linear(x, self.w_qkv).unflatten(-1, (-1, self.head_dim)).transpose(1, 2)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        q, k = rope_axes(q, positions, SECTIONS, k=k)
        return q, k, v

    def out(self, y: torch.Tensor) -> torch.Tensor:
        return F.linear(y.transpose(1, 2).flatten(2), self.w_out)


def run(batch=4, text=200, rows=24, cols=32, new=64, budget=512, recent=64, capacity=640, e4m3=False, embed=1024, heads=16,
        kv_heads=4, quiet=False) -> float:
    """The session; returns the relative error of the new tokens' outputs against 16-bit attention over all tokens."""
    dtype = torch.float8_e4m3fn if e4m3 else torch.int8
    say = (lambda *a: None) if quiet else print
    layer = Layer(embed, heads, kv_heads)
    n = text + rows * cols
    positions = image_positions(batch, text, rows, cols, new)
    x = torch.randn((batch, n + new, embed), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)

    # the prompt
    q, k, v = layer.project(x[:, :n], positions[:, :, :n])
    full_k, full_v = [k], [v]  # for the comparison only
    prompt = KV8Cache.empty(batch, kv_heads, n, layer.head_dim, dtype=dtype)
    score = torch.zeros((batch, kv_heads, n), device="cuda")
    kv8_append(prompt, k, v)
    y = kv8_attention(q, prompt, score=score)
    want = scaled_dot_product_attention(q, k, v, is_causal=True)
    say(f"prompt of {n} tokens: cache {prompt.nbytes() / 2**20:.1f} MB, in 16 bits {2 * k.numel() * 2 / 2**20:.1f} MB; "
        f"outputs off by {rel(layer.out(y), layer.out(want)):.4f}")

    # decoding from a cache that holds `capacity` tokens, cut to `budget` whenever it is full
    cache = KV8Cache.empty(batch, kv_heads, capacity, layer.head_dim, dtype=dtype)
    spare = KV8Cache.empty(batch, kv_heads, capacity, layer.head_dim, dtype=dtype)
    cache, score, _ = kv8_evict(prompt, score, min(budget, n), recent=min(recent, budget, n), out=cache)
    held, err = min(budget, n), []
    del prompt
    for t in range(n, n + new):
        if held == capacity:
            spare, score, _ = kv8_evict(cache, score, budget, recent=recent, out=spare)
            cache, spare, held = spare, cache, budget
        q, k, v = layer.project(x[:, t:t + 1], positions[:, :, t:t + 1].contiguous())
        kv8_append(cache, k, v)
        held += 1
        y = kv8_attention(q, cache, score=score)
        full_k.append(k)
        full_v.append(v)
        want = scaled_dot_product_attention(q, torch.cat(full_k, 2), torch.cat(full_v, 2))
        err.append(rel(layer.out(y), layer.out(want)))
    mean = sum(err) / max(1, len(err))
    say(f"{new} new tokens from at most {capacity} cached: cache {cache.nbytes() / 2**20:.1f} MB; outputs off by {mean:.3f} "
        f"on average ({budget} of {n} prompt tokens kept)")
    return mean


def rel(got: torch.Tensor, want: torch.Tensor) -> float:
    return ((got.float() - want.float()).norm() / want.float().norm()).item()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--text", type=int, default=200)
    ap.add_argument("--image", default="24x32", help="rows x columns of the image's tokens")
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--budget", type=int, default=512)
    ap.add_argument("--capacity", type=int, default=640)
    ap.add_argument("--e4m3", action="store_true", help="codes in e4m3 instead of int8")
    a = ap.parse_args()
    rows, cols = (int(n) for n in a.image.split("x"))
    run(a.batch, a.text, rows, cols, a.new, a.budget, recent=min(64, a.budget), capacity=max(a.capacity, a.budget + 1), e4m3=a.e4m3)


if __name__ == "__main__":
    main()
