"""Offsets that rise along the keys, by far more than the 2^8 that a row's scores may stay above its offset, in a segment's first, middle and
last tiles; and segments of a single tile. What the softmax warps hand to one another (maxima, factors, sums) is written
over from tile to tile, so each call is repeated to the same bits.

The scores climb by one dimension, in which every query has 8 and a row the height of its place; the tolerances are those of
test_gpu_latent.py, in which the height enters by the scores' magnitudes."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_latent import TYPES, _cache, _check

pytestmark = pytest.mark.gpu


def _heights(kind, n, lens, gen):
    """(B, n): a row's height in steps of 9, each some 6 in a score."""
    i = torch.arange(n, device="cuda")
    if kind == "steps":  # every tile of 64 rows above the one before
        return (9.0 * (i // 64)).expand(len(lens), n)
    if kind == "last":  # the newest tokens far above everything before
        return torch.where(i[None] >= torch.tensor(lens, device="cuda")[:, None] - 2, 90.0, 0.0)
    return 9.0 * torch.randint(0, 10, (len(lens), n), device="cuda", generator=gen).float()


def _run(B, H, Lq, R, lens, cap, P, kind, dt, times):
    from gguf_train_b200 import _C, latent_attention

    gen = torch.Generator(device="cuda").manual_seed(B + H + R)
    cache = _cache(B, cap, R, 32, lens, dt, gen)
    held = torch.arange(cap, device="cuda")[None] < cache.lens[:, None]
    cache.rows[..., -1] = torch.where(held, _heights(kind, cap, lens, gen).to(dt), cache.rows[..., -1])
    prefix = _cache(1, P + 5, R, 32, [P], dt, gen) if P else None
    if P:
        prefix.rows[0, :P, -1] = _heights("steps" if kind == "last" else kind, P, [P], gen)[0].to(dt)
    q = torch.randn((B, H, Lq, R + 32), device="cuda", generator=gen).to(dt)
    q[..., -1] = 8.0
    scale = 1.0 / math.sqrt(96)
    out, lse = latent_attention(q, cache, scale, prefix=prefix, need_lse=True)
    assert _C.device_status() == 0
    _check(q, cache, scale, None, prefix, out, lse)
    for _ in range(times):
        again, l2 = latent_attention(q, cache, scale, prefix=prefix, need_lse=True)
        assert torch.equal(again, out) and torch.equal(l2, lse)


@pytest.mark.parametrize("kind", ["steps", "last", "mixed"])
@pytest.mark.parametrize("H,Lq", [(1, 1), (16, 1), (7, 9), (20, 3)])
@pytest.mark.parametrize("R", [64, 128, 192, 320, 512])
def test_offsets_that_rise(R, H, Lq, kind):
    """Several tiles a segment: 40 sequences of up to 1500 rows."""
    lens = [Lq + (1500 - Lq) * b // 39 for b in range(40)]
    _run(40, H, Lq, R, lens, 1500, 0, kind, TYPES["bf16" if R != 192 else "f16"], 20)


@pytest.mark.parametrize("kind", ["steps", "last", "mixed"])
@pytest.mark.parametrize("B,H,Lq,P", [(24, 16, 1, 5000), (9, 5, 3, 3001), (3, 40, 2, 900)])
@pytest.mark.parametrize("R", [128, 320, 512])
def test_offsets_that_rise_behind_a_prefix(R, B, H, Lq, P, kind):
    _run(B, H, Lq, R, [Lq + 400 * b // B for b in range(B)], 400, P, kind, torch.bfloat16, 20)


@pytest.mark.parametrize("R,H,Lq", [(64, 3, 1), (128, 16, 1), (320, 7, 5), (512, 16, 1), (512, 64, 1)])
def test_segments_of_one_tile(R, H, Lq):
    """Many sequences of at most one tile each, several a CTA."""
    _run(500, H, Lq, R, [Lq + b % (65 - Lq) for b in range(500)], 64, 0, "mixed", torch.bfloat16, 300)
