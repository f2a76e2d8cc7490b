"""The latent cache and absorbed attention over it against the formulas in 64 bits.

Tolerances, with u = eps / 2 of the stored type: a weight enters its product rounded once (u of itself, in f16 at least 2^-25 of
the row's largest) and the output is rounded once more; scores are sums of D f32 products and D f32 additions, each off by at
most 2^-23 of the sum of magnitudes (the tensor cores' additions cut off, which is a whole step), and an error e of a
score is one of e in each weight's logarithm, twice that after the division by their sum. So
    |out - exact| <= u |exact| + (u + 2 e) sum w |c| + 2^-25 sum |c| / sum(w / max w),  e = D 2^-22 scale max(|q| . |k|)
and the log-sum-exp is off by e, the weights' own u does not enter it, and a few roundings of itself.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _cache(B, cap, R, Dr, lens, dt, gen, past=float("nan")):
    from gguf_train_b200 import LatentCache

    rows = torch.randn((B, cap, R + Dr), device="cuda", generator=gen).to(dt)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if past is not None:  # rows behind the lengths hold anything
        rows.masked_fill_((torch.arange(cap, device="cuda")[None] >= lens[:, None])[..., None], past)
    return LatentCache(rows, lens, R)


def _check(q, cache, scale, counts, prefix, out, lse):
    B, H, Lq, D = q.shape
    R, u = cache.latent_dim, torch.finfo(q.dtype).eps / 2
    for b in range(B):
        n = max(0, min(int(cache.lens[b]), cache.capacity))
        m = Lq if counts is None else max(0, min(int(counts[b]), Lq))
        keys = cache.rows[b, :n].double()
        P = 0
        if prefix is not None:
            P = int(prefix.lens[0])
            keys = torch.cat((prefix.rows[0, :P].double(), keys))
        qb = q[b].double()
        x = torch.einsum("hid,sd->his", qb, keys) * scale
        i = torch.arange(Lq, device="cuda")
        last = torch.where(i < m, torch.full_like(i, P) + (n - m + i).clamp(min=-1), torch.full_like(i, -1))
        x = x.masked_fill(torch.arange(keys.shape[0], device="cuda")[None] > last[:, None], float("-inf"))
        z = torch.logsumexp(x, -1) if keys.shape[0] else torch.full((H, Lq), float("-inf"), device="cuda", dtype=torch.float64)
        dead = torch.isinf(z)
        w = torch.exp(x - torch.where(dead, torch.zeros_like(z), z)[..., None]).masked_fill(dead[..., None], 0.0)
        want = w @ keys[:, :R]
        mags = w @ keys[:, :R].abs()
        e = D * 2.0 ** -22 * scale * float(torch.einsum("hid,sd->his", qb.abs(), keys.abs()).max()) if keys.shape[0] else 0.0
        spread = torch.where(dead, torch.ones_like(z), 1.0 / w.amax(-1)) if keys.shape[0] else torch.ones_like(z)  # sum of w / max w
        low = 2.0 ** -25 * keys[:, :R].abs().sum(0) / spread[..., None] if q.dtype == torch.float16 else 0.0
        tol = u * want.abs() + (u + 2 * e) * mags + low + 1e-30
        got = out[b].double()
        assert torch.isfinite(got).all(), f"sequence {b}: not finite"
        far = (got - want).abs() / tol
        assert float(far.max()) <= 1.0, f"sequence {b}: {float(far.max()):.3g} of the tolerance"
        assert torch.equal(dead, torch.isinf(lse[b])) and bool((got[dead] == 0).all())
        if not bool(dead.all()):
            off = (lse[b].double() - z)[~dead].abs()
            assert float((off / (e + 1e-6 + 2.0 ** -21 * z[~dead].abs())).max()) <= 1.0


CASES = [
    # B, H, Lq, R, Dr, capacity, lens, prefix rows
    (1, 1, 1, 64, 16, 40, [1], 0),
    (3, 1, 1, 128, 32, 300, [0, 64, 65], 0),
    (2, 16, 1, 512, 64, 1000, [1000, 63], 0),
    (5, 16, 1, 512, 64, 700, [129, 0, 700, 1, 640], 0),
    (2, 20, 1, 192, 48, 257, [257, 128], 0),
    (2, 72, 1, 256, 64, 300, [300, 17], 0),
    (1, 130, 2, 64, 64, 200, [199], 0),
    (3, 7, 5, 320, 32, 400, [5, 63, 400], 0),
    (2, 16, 4, 512, 64, 512, [130, 511], 0),
    (2, 64, 3, 448, 16, 200, [3, 190], 0),
    (2, 4, 33, 384, 64, 300, [33, 300], 0),
    (1, 32, 70, 512, 64, 400, [333], 0),
    (2, 3, 150, 128, 48, 200, [150, 190], 0),
    (40, 2, 1, 64, 16, 90, [(7 * b) % 91 for b in range(40)], 0),
    # behind a prefix
    (1, 1, 1, 64, 16, 40, [1], 1),
    (6, 16, 1, 512, 64, 100, [1, 0, 100, 64, 37, 5], 200),
    (9, 4, 1, 256, 32, 70, [b * 8 for b in range(9)], 64),
    (5, 12, 3, 256, 48, 90, [3, 50, 90, 64, 4], 333),
    (3, 72, 1, 128, 32, 64, [1, 30, 64], 129),
    (2, 16, 9, 512, 64, 70, [9, 70], 190),
    (7, 40, 1, 512, 64, 40, [1, 2, 3, 4, 5, 6, 7], 65),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])) + f"+{c[7]}")
@pytest.mark.parametrize("ragged", [False, True])
def test_attention(case, dtype, ragged):
    from gguf_train_b200 import _C, latent_attention

    B, H, Lq, R, Dr, cap, lens, P = case
    gen = torch.Generator(device="cuda").manual_seed(B * 1000 + H)
    dt = TYPES[dtype]
    cache = _cache(B, cap, R, Dr, lens, dt, gen)
    prefix = _cache(1, P + 5, R, Dr, [P], dt, gen) if P else None
    q = torch.randn((B, Lq, H, R + Dr), device="cuda", generator=gen).to(dt).transpose(1, 2)
    counts = torch.randint(0, Lq + 1, (B,), device="cuda", generator=gen).to(torch.int32) if ragged else None
    scale = 1.0 / math.sqrt(64 + Dr)
    out, lse = latent_attention(q, cache, scale, counts=counts, prefix=prefix, need_lse=True)
    assert _C.device_status() == 0
    _check(q, cache, scale, counts, prefix, out, lse)
    again = latent_attention(q, cache, scale, counts=counts, prefix=prefix)
    assert torch.equal(again, out)  # the same bits on every run


@pytest.mark.parametrize("B,H,Lq,R,cap,P", [
    (3, 5, 1, 192, 40, 300), (5, 3, 2, 512, 70, 5000), (60, 6, 1, 256, 70, 700), (90, 1, 3, 128, 130, 129), (41, 9, 3, 448, 65, 64),
    (200, 2, 1, 64, 200, 0), (300, 7, 1, 320, 90, 65)])
def test_rows_that_are_no_multiple_of_four(B, H, Lq, R, cap, P):
    """Several sequences' rows in an item over the prefix, where a sequence's do not begin at a multiple of four rows; more items than
    multiprocessors."""
    from gguf_train_b200 import _C, latent_attention

    gen = torch.Generator(device="cuda").manual_seed(B + H)
    lens = [(37 * b) % (cap + 1) for b in range(B)]
    cache = _cache(B, cap, R, 32, lens, torch.bfloat16, gen)
    prefix = _cache(1, P + 5, R, 32, [P], torch.bfloat16, gen) if P else None
    q = torch.randn((B, H, Lq, R + 32), device="cuda", generator=gen).to(torch.bfloat16)
    counts = torch.randint(0, Lq + 1, (B,), device="cuda", generator=gen).to(torch.int32)
    for c in (None, counts):
        out, lse = latent_attention(q, cache, 0.1, counts=c, prefix=prefix, need_lse=True)
        assert _C.device_status() == 0
        _check(q, cache, 0.1, c, prefix, out, lse)


@pytest.mark.parametrize("mode", [None, 0, 2])
@pytest.mark.parametrize("dtype,source", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("B,n,R,Dr,cap,lens,far", [
    (1, 1, 64, 16, 4, [0], 0), (3, 5, 512, 64, 40, [0, 7, 35], 0), (2, 130, 192, 48, 300, [100, 3], 1000000),
    (70, 1, 128, 32, 9, [b % 9 for b in range(70)], 7),
])
def test_append(mode, dtype, source, B, n, R, Dr, cap, lens, far):
    from gguf_train_b200 import LatentCache, _C, latent_append

    gen = torch.Generator(device="cuda").manual_seed(n)
    src = {"f32": torch.float32, **TYPES}[source]
    x = torch.randn((B, n, R + Dr), device="cuda", generator=gen).to(src)
    cache = _cache(B, cap, R, Dr, lens, TYPES[dtype], gen, past=None)
    before = cache.rows.clone()
    prefix = None
    if far:  # positions behind a prefix, which need not hold its rows here
        prefix = LatentCache(cache.rows.new_zeros((1, 0, R + Dr)), torch.tensor([far], dtype=torch.int32, device="cuda"), R)
    counts = None if n == 1 else torch.randint(0, n + 1, (B,), device="cuda", generator=gen).to(torch.int32)
    rope = None if mode is None else dict(mode=mode, freq_base=5000.0, freq_scale=0.5)
    latent_append(cache, x[..., :R], x[..., R:], counts=counts, rope=rope, prefix=prefix)
    assert _C.device_status() == 0
    want, size = before.double(), before.double().abs()
    for b in range(B):
        m = n if counts is None else int(counts[b])
        new = x[b, :m].double()
        size[b, lens[b]:lens[b] + m] = new.abs()
        if mode is not None:
            pos = far + lens[b] + torch.arange(m, device="cuda", dtype=torch.float64)
            half = Dr // 2
            a = 0.5 * pos[:, None] * 5000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            i0, i1 = (slice(R, None, 2), slice(R + 1, None, 2)) if mode == 0 else (slice(R, R + half), slice(R + half, None))
            x0, x1 = new[:, i0].clone(), new[:, i1].clone()
            new[:, i0], new[:, i1] = x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos()
            for s in (i0, i1):
                size[b, lens[b]:lens[b] + m, s] = x0.abs() + x1.abs()
        want[b, lens[b]:lens[b] + m] = new
        assert int(cache.lens[b]) == lens[b] + m
    # one rounding to the stored type, and in f32 the angle's (2^-26 of a turn), the sine's and cosine's, two products and a sum
    tol = torch.finfo(TYPES[dtype]).eps / 2 * want.abs() + (2.0 ** -26 * 6.3 + 6 * 2.0 ** -23) * size + 2.0 ** -25
    assert bool(((cache.rows.double() - want).abs() <= tol).all())


def test_rows_past_the_capacity_are_dropped():
    from gguf_train_b200 import _C, latent_append

    gen = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn((4, 8, 96), device="cuda", generator=gen).to(torch.bfloat16)
    from gguf_train_b200 import LatentCache

    keep = big.clone()
    cache = LatentCache(big[1:3], torch.tensor([6, 8], dtype=torch.int32, device="cuda"), 64)
    x = torch.randn((2, 5, 96), device="cuda", generator=gen)
    latent_append(cache, x[..., :64], x[..., 64:])
    assert _C.device_status() == 62 and _C.device_status() == 0
    assert cache.lens.tolist() == [8, 8]
    keep[1, 6:] = x[0, :2].to(torch.bfloat16)
    assert torch.equal(big, keep)


def test_refusals():
    from gguf_train_b200 import LatentCache, latent_append, latent_attention

    bf = torch.bfloat16
    cache = LatentCache.empty(2, 10, 64, 32)
    q = torch.zeros((2, 4, 1, 96), dtype=bf, device="cuda")
    x = torch.zeros((2, 3, 96), dtype=bf, device="cuda")
    for bad, match in [(lambda: LatentCache.empty(2, 10, 96, 32), "multiple of 64"),
                       (lambda: LatentCache.empty(2, 10, 64, 8), "multiple of 16"),
                       (lambda: LatentCache.empty(2, 10, 64, 32, dtype=torch.float32), "bfloat16 or torch.float16"),
                       (lambda: LatentCache(cache.rows[:, ::2], cache.lens, 64), "contiguous"),
                       (lambda: LatentCache(cache.rows, cache.lens.long(), 64), "int32"),
                       (lambda: setattr(cache, "lens", cache.lens[:1]), "only be replaced"),
                       (lambda: latent_attention(q.half(), cache, 0.1), "cache's type"),
                       (lambda: latent_attention(q[..., :64], cache, 0.1), "q must be"),
                       (lambda: latent_attention(q[:1], cache, 0.1), "q must be"),
                       (lambda: latent_attention(q, cache, 0.0), "scale"),
                       (lambda: latent_attention(q, cache, 0.1, counts=cache.lens.long()), "counts"),
                       (lambda: latent_attention(q, cache, 0.1, prefix=cache), "prefix"),
                       (lambda: latent_attention(q.cpu(), cache, 0.1), "CUDA tensors only"),
                       (lambda: latent_append(cache, x[..., :64], x[:, :2, 64:]), "latent must be"),
                       (lambda: latent_append(cache, x[..., :64], x[..., 64:].float()), "one type"),
                       (lambda: latent_append(cache, x[..., :64], x[..., 64:], rope=dict(mode=1)), "mode must be"),
                       (lambda: latent_append(cache, x[..., :64], x[..., 64:], rope=dict(n_dims=32)), "rope takes")]:
        with pytest.raises(RuntimeError, match=match):
            bad()


def test_strides_and_alignment():
    """Views whose rows do not start on 16 bytes, broadcast heads, odd layouts: the same as contiguous copies."""
    from gguf_train_b200 import _C, latent_append, latent_attention

    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = _cache(2, 100, 64, 32, [100, 30], torch.bfloat16, gen)
    big = torch.randn((2, 5, 3, 103), device="cuda", generator=gen).to(torch.bfloat16)
    for q in (big[..., 3:99], big[..., 3:99].transpose(1, 2), big[:, :1, :, :96].expand(2, 5, 3, 96),
              torch.randn((2, 4, 96, 2), device="cuda", generator=gen).to(torch.bfloat16).transpose(2, 3)):
        assert torch.equal(latent_attention(q, cache, 0.1), latent_attention(q.contiguous(), cache, 0.1))
    x = torch.randn((2, 4, 101), device="cuda", generator=gen)
    a, b = _cache(2, 9, 64, 32, [0, 4], torch.float16, gen, past=0.0), _cache(2, 9, 64, 32, [0, 4], torch.float16, gen, past=0.0)
    b.rows = a.rows.clone()
    latent_append(a, x[..., 5:69], x[..., 69:], rope=dict(mode=2))
    latent_append(b, x[..., 5:69].contiguous(), x[..., 69:].contiguous(), rope=dict(mode=2))
    assert torch.equal(a.rows, b.rows) and _C.device_status() == 0


def test_empty_calls():
    from gguf_train_b200 import LatentCache, latent_append, latent_attention

    bf = torch.bfloat16
    q = torch.ones((2, 4, 3, 96), dtype=bf, device="cuda")
    none = LatentCache.empty(2, 0, 64, 32)
    out, lse = latent_attention(q, none, 0.1, need_lse=True)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
    out, lse = latent_attention(q, none, 0.1, prefix=LatentCache.empty(1, 0, 64, 32), need_lse=True)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
    shared = LatentCache(torch.ones((1, 2, 96), dtype=bf, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"), 64)
    out = latent_attention(q, none, 0.1, prefix=shared)
    assert bool((out == 1).all())
    assert latent_attention(q[:, :, :0], none, 0.1).shape == (2, 4, 0, 64)
    assert latent_attention(q[:, :0], none, 0.1).shape == (2, 0, 3, 64)
    assert latent_attention(q[:0], LatentCache.empty(0, 4, 64, 32), 0.1).shape == (0, 4, 3, 64)
    x = torch.ones((2, 0, 96), dtype=bf, device="cuda")
    latent_append(none, x[..., :64], x[..., 64:])
