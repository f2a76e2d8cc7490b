"""One latent attention layer serving prompts behind a system prompt that all of them share.

    python examples/latent_session.py [--batch 8] [--system 2000] [--text 300] [--new 32]

What a server does with the package, step by step:
  1. the system prompt, once: its latents and rotated rotary keys go into a LatentCache of one sequence (latent_append);
  2. each prompt: keys and values expanded from the latents by the layer's up-projections, latent_sdpa over them for the
     prompt alone (here for the comparison); latent_append stores what follows the system prompt;
  3. each new token: project, take the query through the keys' up-projection, rotate, append, latent_attention over the
     shared prefix and the sequence's own rows (its prompt as one chunk first), and back through the values' up-projection.
It prints what the caches take, and how far the outputs are from expanded attention over all tokens in f32.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gguf_train_b200 import LatentCache, functional as F, latent_append, latent_attention, latent_sdpa, rope_axes  # noqa: E402


class Layer:
    """Latent attention with random weights, in bf16: keys of Dn values a head and Dr rotary ones, values of Dn."""

    def __init__(self, embed=1024, heads=16, latent=256, Dn=64, Dr=32, seed=0) -> None:
        g = torch.Generator("cuda").manual_seed(seed)
        mk = lambda *s: (torch.randn(s, device="cuda", generator=g) * s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
        self.heads, self.latent, self.Dn, self.Dr = heads, latent, Dn, Dr
        self.scale = 1.0 / math.sqrt(Dn + Dr)
        self.w_q, self.w_down = mk(heads * (Dn + Dr), embed), mk(latent + Dr, embed)
        self.w_k, self.w_v = mk(heads, Dn, latent), mk(heads, Dn, latent)

    def down(self, x):
        """x (B, n, E) -> latents (B, n, R) and rotary keys (B, n, Dr), not rotated yet."""
        return F.linear(x, self.w_down).split((self.latent, self.Dr), dim=-1)

    def query(self, x, first):
        """The heads' queries (B, H, n, Dn + Dr), the rotary part rotated for positions first, first + 1, .."""
        q = F.linear(x, self.w_q).unflatten(-1, (self.heads, -1)).transpose(1, 2)
        pos = torch.arange(first, first + x.shape[1], device="cuda", dtype=torch.int32)[None]
        return torch.cat((q[..., :self.Dn], rope_axes(q[..., self.Dn:], pos, [self.Dr // 2])), dim=-1)

    def absorb(self, q):
        """q with its first part taken through the keys' up-projection: what latent_attention takes."""
        return torch.cat((torch.einsum("bhnd,hdr->bhnr", q[..., :self.Dn], self.w_k), q[..., self.Dn:]), dim=-1)

    def values(self, y):
        return torch.einsum("bhnr,hdr->bhnd", y, self.w_v)

    def expand(self, latent, k_rope, first):
        """Keys and values (B, H, n, Dn) of latents, and their rotary keys rotated for positions first, .."""
        pos = torch.arange(first, first + latent.shape[1], device="cuda", dtype=torch.int32)[None]
        k, v = (torch.einsum("bnr,hdr->bhnd", latent, w) for w in (self.w_k, self.w_v))
        return k, rope_axes(k_rope[:, None], pos, [self.Dr // 2])[:, 0], v


def rel(got: torch.Tensor, want: torch.Tensor) -> float:
    return ((got.float() - want.float()).norm() / want.float().norm()).item()


def run(batch=8, system=2000, text=300, new=32, quiet=False, **sizes):
    """The session; returns the relative errors (expanded prompt, absorbed prompt, new tokens' mean)."""
    say = (lambda *a: None) if quiet else print
    layer = Layer(**sizes)
    E = layer.w_q.shape[1]
    g = torch.Generator("cuda").manual_seed(1)
    x_sys = torch.randn((1, system, E), device="cuda", generator=g).to(torch.bfloat16)
    x = torch.randn((batch, text + new, E), device="cuda", generator=g).to(torch.bfloat16)
    rope = dict(mode=2)

    prefix = LatentCache.empty(1, system, layer.latent, layer.Dr)
    latent_append(prefix, *layer.down(x_sys), rope=rope)
    cache = LatentCache.empty(batch, text + new, layer.latent, layer.Dr)

    # all of it once more in f32, for the comparison
    both = torch.cat((x_sys.expand(batch, -1, -1), x), dim=1)
    k, kr, v = layer.expand(*layer.down(both), 0)
    keys = torch.cat((k, kr[:, None].expand(-1, layer.heads, -1, -1)), dim=-1).float()

    def exact(q, first):
        s = torch.einsum("bhnd,bhsd->bhns", q.float(), keys[:, :, :first + q.shape[2]]) * layer.scale
        i = first + torch.arange(q.shape[2], device="cuda")
        s = s.masked_fill(torch.arange(s.shape[-1], device="cuda") > i[:, None], float("-inf"))
        return torch.softmax(s, -1) @ v[:, :, :first + q.shape[2]].float()

    # the prompts: expanded (system prompt and text in one), and as one chunk over the caches
    q_all = layer.query(both[:, :system + text], 0)
    expanded = latent_sdpa(q_all, k[:, :, :system + text], kr[:, :system + text], v[:, :, :system + text], is_causal=True,
                           scale=layer.scale)[:, :, system:]
    q = q_all[:, :, system:]
    latent_append(cache, *layer.down(x[:, :text]), rope=rope, prefix=prefix)
    y = layer.values(latent_attention(layer.absorb(q), cache, layer.scale, prefix=prefix))
    want = exact(q, system)
    errs = [rel(expanded, want), rel(y, want)]
    say(f"{batch} prompts of {text} tokens behind {system}: caches {(prefix.nbytes() + cache.nbytes()) / 2**20:.1f} MB, expanded keys "
        f"and values {2 * k.numel() * 2 / 2**20:.1f} MB; outputs off by {errs[0]:.4f} expanded, {errs[1]:.4f} absorbed")

    steps = []
    for t in range(text, text + new):
        q = layer.query(x[:, t:t + 1], system + t)
        latent_append(cache, *layer.down(x[:, t:t + 1]), rope=rope, prefix=prefix)
        y = layer.values(latent_attention(layer.absorb(q), cache, layer.scale, prefix=prefix))
        steps.append(rel(y, exact(q, system + t)))
    errs.append(sum(steps) / max(1, len(steps)))
    say(f"{new} new tokens each: outputs off by {errs[2]:.4f} on average")
    return errs


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, n in (("batch", 8), ("system", 2000), ("text", 300), ("new", 32)):
        ap.add_argument(f"--{name}", type=int, default=n)
    run(**vars(ap.parse_args()))


if __name__ == "__main__":
    main()
