"""Expanded latent attention where a thread block has more than one piece of work, where offsets rise tile after tile, and past 32 bits.

The forward's blocks claim (batch, head, pair of query tiles) items, one block a multiprocessor: the cases here have several items a block, of one
key tile and of many, with and without sequences that have nothing to attend. Tolerances as in test_gpu_latent_sdpa.py."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_latent_sdpa import TYPES, _exact, _inputs

pytestmark = pytest.mark.gpu


def _run(leaves, g, causal, scale, lens, times):
    from gguf_train_b200 import _C, latent_sdpa

    def step():
        out = latent_sdpa(*leaves, is_causal=causal, scale=scale, seq_lens=lens)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    got = step()
    assert _C.device_status() == 0
    for name, x, (want, tol) in zip(("out", "dq", "dk", "dk_rope", "dv"), got, _exact(*leaves, g, causal, scale, lens)):
        far = float(((x.double() - want).abs() / tol).max())
        assert far <= 1.0, f"{name}: {far:.3g} of the tolerance"
    for _ in range(times):
        assert all(torch.equal(a, b) for a, b in zip(step(), got))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,H,Hkv,L,S,Dn,Dr,lens", [
    (3, 24, 8, 1100, 1100, 128, 64, None),
    (3, 24, 24, 1100, 1100, 64, 32, [1100, 0, 613]),
    (3, 24, 8, 700, 700, 128, 48, [1, 700, 130]),
    (64, 16, 4, 70, 70, 128, 64, None),
    (64, 16, 16, 70, 70, 64, 32, [(37 * b) % 71 for b in range(64)]),
    (30, 8, 8, 300, 300, 64, 64, [0, 300, 128, 129, 64, 65] * 5),
    (2, 40, 20, 1500, 300, 64, 16, None),
    (4, 50, 10, 200, 900, 128, 32, None),
])
def test_more_items_than_multiprocessors(B, H, Hkv, L, S, Dn, Dr, lens, causal, dtype):
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    leaves, g = _inputs(B, H, Hkv, L, S, Dn, Dr, Dn, TYPES[dtype], L + H, n)
    _run(leaves, g, causal, 1.0 / math.sqrt(Dn + Dr), n, 10)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("kind", ["steps", "last", "mixed"])
@pytest.mark.parametrize("B,H,Hkv,L,Dn,Dr", [(2, 3, 3, 700, 128, 64), (3, 2, 1, 520, 64, 32), (2, 40, 40, 390, 64, 64)])
def test_offsets_that_rise(B, H, Hkv, L, Dn, Dr, kind, padded, causal, dtype):
    """One rotary dimension holds 8 in every query and a height in every key: 12 steps of it are some 10 or 14 powers of 2 in a score, more
    than the 8 that a row's scores may stay above its offset."""
    lens = torch.tensor([L - L // 5, L // 3, L][:B], dtype=torch.int32, device="cuda") if padded else None
    leaves, g = _inputs(B, H, Hkv, L, L, Dn, Dr, Dn, TYPES[dtype], L, lens)
    held = torch.ones((B, L), dtype=torch.bool, device="cuda") if lens is None else torch.arange(L, device="cuda") < lens[:, None]
    i = torch.arange(L, device="cuda")
    n = torch.full((B,), L, device="cuda") if lens is None else lens
    if kind == "steps":    # every key tile above the one before
        height = (12.0 * (i // 128)).expand(B, L)
    elif kind == "last":   # the newest tokens far above everything before
        height = torch.where(i[None] >= n[:, None] - 3, 90.0, 0.0)
    else:
        height = 12.0 * torch.randint(0, 8, (B, L), device="cuda", generator=torch.Generator(device="cuda").manual_seed(L)).float()
    with torch.no_grad():
        q, kr = leaves[0], leaves[2]
        kr[..., -1] = torch.where(held, height.to(kr.dtype), kr[..., -1])
        q[..., -1] = torch.where(held[:, None], torch.full_like(q[..., -1], 8.0), q[..., -1])
    _run(leaves, g, causal, 1.0 / math.sqrt(Dn + Dr), lens, 10)


def test_offsets_past_32_bits():
    """q and dq of 2.4e9 values, and 4.7 GB of the rotary gradient's shares: the last sequence starts beyond 2^31 values and 2^32 bytes.
    Sequences of length 0 keep the work small."""
    from gguf_train_b200 import _C, latent_sdpa

    B, H, L, Dn, Dr = 16, 128, 9000, 64, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    shapes = ((B, H, L, Dn + Dr), (B, H, L, Dn), (B, L, Dr), (B, H, L, Dn), (B, H, L, Dn))
    xs = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in shapes]
    lens = torch.tensor([3] + [0] * (B - 2) + [400], dtype=torch.int32, device="cuda")
    for x in xs:
        for b in (0, B - 1):
            x[b].copy_(torch.randn(x.shape[1:], device="cuda", generator=gen, dtype=torch.bfloat16))

    def step(ts, n):
        leaves = [t.detach().requires_grad_() for t in ts[:4]]
        out = latent_sdpa(*leaves, is_causal=True, seq_lens=n)
        return [out.detach(), *torch.autograd.grad(out, leaves, ts[4])]

    got = step(xs, lens)
    assert _C.device_status() == 0
    for b in (0, B - 1):
        one = step([x[b:b + 1].clone() for x in xs], lens[b:b + 1].clone())
        assert all(torch.equal(a[b], c[0]) for a, c in zip(got, one))
        assert all(bool(c.any()) for c in one)
    for a in got:
        assert not any(bool(a[b].any()) for b in range(1, B - 1))
    del xs, got, one
    torch.cuda.empty_cache()
