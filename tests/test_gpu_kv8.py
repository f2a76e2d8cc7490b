"""The block-scaled 8-bit cache on the GPU: append, read, attention, eviction, and their refusals, against plain
implementations in 64 bits (and, where codes have to agree to the bit, in the same f32 steps).

Tolerances:
* a code stands for its value to half a step: int8 0.5 scale, e4m3 2^-4 of the value (or 2^-10 scale when
  subnormal), each with 1e-5 relative for the f32 steps;
* attention: scores are f32 sums of D products, |error| <= ds = (D + 8) 2^-23 sum|q||k| * scale + |score| 2^-22; a
  weight is then off by a factor e^(2 ds), by 2^-10.5 where it is rounded to f16 for the product (16-bit q; f32 q
  splits it in two: 2^-20) and by 2^-25 of the row's largest weight in all (f16's smallest step, weights scaled by
  2^15); the sum over n keys adds n 2^-24; the result is rounded once.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FMTS = [torch.int8, torch.float8_e4m3fn]
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def quantise(x, s, fmt):
    """The codes of f32 x at f32 scales s, as f32 numbers, in the operator's own steps."""
    y = torch.where(s > 0, x / s, torch.zeros_like(x))
    y = torch.where(y.isnan(), torch.zeros_like(y), y).clamp(-TOP[fmt], TOP[fmt])
    return y.round() if fmt == torch.int8 else y.to(fmt).float()


def scale_of(amax, fmt):
    return amax * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32, device="cuda")


def values(cache, upto=None):
    """(k, v) of the cache in float64."""
    cap = cache.capacity if upto is None else upto
    return tuple((c[:, :, :cap].float() * s.repeat_interleave(cache.block, 2)[:, :, :cap, None]).double()
                 for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))


def random_cache(B, Hkv, cap, D, block, fmt, lens, seed, dirty=True):
    """A filled cache; with `dirty` the rows past the lengths, and the scales of blocks that hold none, are NaN."""
    from gguf_train_b200 import KV8Cache

    g = gen(seed)
    cache = KV8Cache.empty(B, Hkv, cap, D, block, fmt)
    cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    n = cache.lens.clamp(0, cap)[:, None]
    past = (torch.arange(cap, device="cuda")[None] >= n)[:, None, :, None]
    blocks_past = (torch.arange(cache.k_scale.shape[2], device="cuda")[None] * block >= n)[:, None]
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.randn(c.shape, device="cuda", generator=g) * (TOP[fmt] / 4)
        x = x.clamp(-TOP[fmt], TOP[fmt])
        c.copy_(x.round().to(torch.int8) if fmt == torch.int8 else x.to(fmt))
        s.copy_((0.5 + torch.rand(s.shape, device="cuda", generator=g)) * (4 / TOP[fmt]))
        if dirty:
            c.view(torch.uint8).masked_fill_(past, 0xFF if fmt != torch.int8 else 0x80)
            s.masked_fill_(blocks_past, float("nan"))
    return cache


# ------------------------------------------------------------------ append

def append_reference(state, x, lens, counts, block, fmt):
    """One append in plain steps on (codes f32, scales) of shape (B, Hkv, cap, D) / (B, Hkv, nb)."""
    codes, scales = state
    B, Hkv, cap, _ = codes.shape
    for b in range(B):
        p, end = lens[b], min(lens[b] + counts[b], cap)
        for j in range(p // block, -(-end // block)):
            r0, r1 = max(j * block, p), min((j + 1) * block, end)
            if r0 >= r1:
                continue
            new = x[b, :, r0 - p:r1 - p].float()
            fin = torch.where(new.isfinite(), new.abs(), torch.zeros_like(new))
            old = scales[b, :, j] if j * block < p else torch.zeros(Hkv, device="cuda")
            s = torch.maximum(old, scale_of(fin.amax((1, 2)), fmt))
            held = codes[b, :, j * block:r0]
            again = quantise(held * old[:, None, None], s[:, None, None].expand_as(held), fmt)
            codes[b, :, j * block:r0] = torch.where((s > old)[:, None, None], again, held)
            codes[b, :, r0:r1] = quantise(new, s[:, None, None].expand_as(new), fmt)
            scales[b, :, j] = s


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("B,Hkv,cap,D,block,dt,steps", [
    (2, 2, 100, 64, 16, torch.float32, (1, 1, 1, 14, 1, 30)),
    (3, 1, 300, 128, 64, torch.bfloat16, (70, 1, 1, 100)),
    (1, 3, 70, 16, 128, torch.float16, (5, 64, 1)),
    (2, 2, 130, 256, 32, torch.bfloat16, (33, 1, 95)),
    (4, 2, 64, 80, 16, torch.float16, (0, 17, 2)),
])
def test_append_matches_the_steps(fmt, B, Hkv, cap, D, block, dt, steps):
    from gguf_train_b200 import KV8Cache, _C, kv8_append, kv8_read

    g = gen(1)
    cache = KV8Cache.empty(B, Hkv, cap, D, block, fmt)
    cache.k.view(torch.uint8).fill_(0x7F)  # whatever an earlier user of the memory left
    cache.v.view(torch.uint8).fill_(0x7F)
    cache.k_scale.fill_(float("nan"))
    cache.v_scale.fill_(float("nan"))
    ref = [(torch.zeros((B, Hkv, cap, D), device="cuda"), torch.zeros_like(cache.k_scale)) for _ in range(2)]
    lens = [0] * B
    for t, n in enumerate(steps):
        # later rows are larger now and then, so that scales grow over rows already held
        x = [(torch.randn((B, n, Hkv, D), device="cuda", generator=g) * (1 + t % 3)).to(dt).transpose(1, 2) for _ in range(2)]
        cnt = torch.randint(0, n + 1, (B,), generator=torch.Generator().manual_seed(t)) if t % 2 else torch.full((B,), n)
        kv8_append(cache, *x, counts=cnt.to("cuda", torch.int32) if t % 2 else None)
        for r, xx in zip(ref, x):
            append_reference(r, xx, lens, cnt.tolist(), block, fmt)
        lens = [min(a + b, cap) for a, b in zip(lens, cnt.tolist())]
    assert cache.lens.tolist() == lens
    rk, rv = kv8_read(cache, None, cap)
    for c, s, r, back in ((cache.k, cache.k_scale, ref[0], rk), (cache.v, cache.v_scale, ref[1], rv)):
        for b, n in enumerate(lens):
            nb = -(-n // block)
            assert torch.equal(c[b, :, :n].float(), r[0][b, :, :n])
            assert torch.equal(s[b, :, :nb], r[1][b, :, :nb])
            want = r[0][b, :, :n] * r[1][b, :, :nb].repeat_interleave(block, 1)[:, :n, None]
            assert torch.equal(back[b, :, :n], want)
    assert _C.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
def test_append_error_against_64_bits(fmt):
    """Values of one append are within half a step of what was appended."""
    from gguf_train_b200 import KV8Cache, kv8_append, kv8_read

    x = torch.randn((2, 3, 95, 64), device="cuda", generator=gen(2)) * torch.logspace(-3, 3, 95, device="cuda")[:, None]
    cache = kv8_append(KV8Cache.empty(2, 3, 95, 64, 32, fmt), x, -x)
    k, v = kv8_read(cache, None, 95)
    s = cache.k_scale.double().repeat_interleave(32, 2)[:, :, :95, None]
    half = 0.5 * s if fmt == torch.int8 else torch.maximum(x.double().abs() * 2.0 ** -4, s * 2.0 ** -10)
    assert ((k.double() - x.double()).abs() <= half * (1 + 1e-5)).all()
    assert torch.equal(v, -k)


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
def test_append_of_values_that_are_not_finite_and_of_zeros(fmt):
    from gguf_train_b200 import KV8Cache, kv8_append, kv8_read

    x = torch.zeros((1, 1, 40, 32), device="cuda")
    x[0, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), float("-inf"), 2.0])
    x[0, 0, 16:20] = 1e-42  # subnormal scale or none
    x[0, 0, 35, 7] = float("inf")  # a block with no finite nonzero value: scale 0
    cache = kv8_append(KV8Cache.empty(1, 1, 40, 32, 16, fmt), x, x)
    k, _ = kv8_read(cache, None, 40)
    assert k.isfinite().all()
    assert torch.allclose(k[0, 0, 0, :4], torch.tensor([0.0, 2.0, -2.0, 2.0], device="cuda"), rtol=1e-6)
    assert (k[0, 0, 1:16] == 0).all() and (k[0, 0, 20:32] == 0).all() and (k[0, 0, 32:] == 0).all()
    assert (k[0, 0, 16:20] - 1e-42).abs().max() <= 1e-42


def test_append_drops_rows_past_the_capacity_and_says_so():
    from gguf_train_b200 import KV8Cache, _C, kv8_append

    cache = KV8Cache.empty(2, 1, 20, 16, 16)
    guard = cache.k.clone()
    x = torch.ones((2, 1, 18, 16), device="cuda")
    kv8_append(cache, x, x)
    assert _C.device_status() == 0
    kv8_append(cache, x[:, :, :5], x[:, :, :5], counts=torch.tensor([2, 5], dtype=torch.int32, device="cuda"))
    assert _C.device_status() == 61
    assert cache.lens.tolist() == [20, 20] and guard.shape == cache.k.shape
    kv8_append(cache, x[:, :, :1], x[:, :, :1], advance=False)
    assert _C.device_status() == 61 and (cache.k == 127).all()


def test_read_starts_anywhere():
    from gguf_train_b200 import kv8_read

    cache = random_cache(3, 2, 50, 48, 16, torch.int8, [50, 50, 50], 3, dirty=False)
    start = torch.tensor([0, 13, -4], dtype=torch.int32, device="cuda")
    k, v = kv8_read(cache, start, 45, dtype=torch.bfloat16)
    for b, s in enumerate(start.tolist()):
        for got, want in zip((k, v), values(cache)):
            for t in (0, 3, 4, 5, 36, 37, 44):
                row = want[b, :, s + t].to(torch.bfloat16) if 0 <= s + t < 50 else torch.zeros((2, 48), dtype=torch.bfloat16, device="cuda")
                assert torch.equal(got[b, :, t], row), (b, t)


# ------------------------------------------------------------------ attention

def attention_reference(q, cache, counts=None, scale=None):
    """(out, lse, weight, per-element error bound without the output rounding, score bound) in float64."""
    B, H, Lq, D = q.shape
    Hkv, cap = cache.k.shape[1:3]
    G, sc = H // Hkv, 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((B, H, Lq, D), dtype=torch.float64, device="cuda")
    bound, lse = torch.zeros_like(out), torch.full((B, H, Lq), -math.inf, dtype=torch.float64, device="cuda")
    lse_bound = torch.zeros_like(lse)
    weight, wbound = (torch.zeros((B, Hkv, cap), dtype=torch.float64, device="cuda") for _ in range(2))
    K, V = values(cache)
    wide = q.dtype == torch.float32
    for b in range(B):
        n = min(max(int(cache.lens[b]), 0), cap)
        c = Lq if counts is None else min(max(counts[b], 0), Lq)
        if n == 0 or c == 0:
            continue
        k, v = K[b, :, None, :n], V[b, :, None, :n]
        qq = q[b].double().view(Hkv, G, Lq, D)[:, :, :c]
        ends = n - c + 1 + torch.arange(c, device="cuda")
        hidden = torch.arange(n, device="cuda")[None] >= ends[:, None]
        s = (qq @ k.transpose(-1, -2) * sc).masked_fill(hidden, -math.inf)
        z = torch.logsumexp(s, -1)
        p = torch.where(z[..., None].isinf(), torch.zeros_like(s), torch.exp(s - z[..., None]))
        ds = (D + 8) * 2.0 ** -23 * (qq.abs() @ k.abs().transpose(-1, -2)).amax(-1, keepdim=True) * sc
        ds = ds + s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True) * 2.0 ** -22 + 2.0 ** -21
        f = 2 * ds + (2.0 ** -20 if wide else 2.0 ** -10.5) + n * 2.0 ** -24
        av = p @ v.abs()
        top = p.amax(-1, keepdim=True)
        tiny = 2.0 ** (-38 if wide else -25) * top * v.abs().sum(-2, keepdim=True)
        out[b].view(Hkv, G, Lq, D)[:, :, :c] = p @ v
        bound[b].view(Hkv, G, Lq, D)[:, :, :c] = f * av + tiny
        lse[b].view(Hkv, G, Lq)[:, :, :c] = z
        lse_bound[b].view(Hkv, G, Lq)[:, :, :c] = ds[..., 0] + (n + 4) * 2.0 ** -24 + z.masked_fill(z.isinf(), 0).abs() * 2.0 ** -22
        weight[b, :, :n] = p.sum((1, 2))
        wbound[b, :, :n] = (p * (2 * ds + (n + G * c + 8) * 2.0 ** -24)).sum((1, 2))
    return out, lse, weight, bound, lse_bound, wbound


def check_attention(q, cache, counts=None, scale=None, score=True):
    from gguf_train_b200 import _C, kv8_attention

    B, H, Lq, D = q.shape
    ct = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    want, wlse, weight, bound, lbound, wbound = attention_reference(q, cache, counts, scale)
    kw = {}
    if score:
        base = torch.rand((B, cache.k.shape[1], cache.capacity), device="cuda", generator=gen(99))
        kw = {"score": base.clone()}
    out, lse = kv8_attention(q, cache, scale=scale, counts=ct, need_lse=True, **kw)
    tol = bound + ULP[q.dtype] * (want.abs() + bound) + 1e-7 * (q.dtype == torch.float16) + 1e-30
    err = (out.double() - want).abs()
    assert out.isfinite().all() and (err <= tol).all(), f"out: {(err / tol).max().item():.2f} of the tolerance"
    assert torch.equal(lse.isinf(), wlse.isinf())
    live = ~wlse.isinf()
    assert ((lse.double() - wlse).abs()[live] <= lbound[live]).all()
    if score:
        got = kw["score"]
        below = torch.arange(cache.capacity, device="cuda")[None] < cache.lens.clamp(0, cache.capacity)[:, None]
        below = below[:, None].expand_as(got)
        assert torch.equal(got[~below], base[~below])
        e = (got.double() - base.double() - weight).abs()
        assert (e <= wbound + (base.double() + weight) * 2.0 ** -24)[below].all()
        # into another tensor, without the log-sum-exp, the same bits
        other = torch.full_like(base, -7.0)
        out2 = kv8_attention(q, cache, scale=scale, counts=ct, score=base, score_out=other)
        assert torch.equal(out2, out) and torch.equal(other[below], got[below]) and (other[~below] == -7.0).all()
    assert _C.device_status() == 0
    return out


SHAPES = [
    # B, H, Hkv, Lq, D, cap, block, lens
    (1, 1, 1, 1, 16, 1, 16, [1]),
    (1, 8, 8, 1, 64, 512, 16, [333]),
    (3, 4, 2, 1, 128, 700, 64, [700, 0, 17]),
    (2, 32, 8, 1, 128, 2500, 32, [2500, 1]),
    (5, 5, 1, 1, 80, 300, 128, [300, 16, 15, 129, 128]),
    (1, 16, 1, 1, 256, 1000, 64, [999]),
    (2, 24, 1, 1, 96, 200, 16, [200, 64]),
    (2, 8, 2, 4, 128, 400, 64, [400, 3]),          # fewer rows cached than queries: the first see nothing
    (2, 6, 3, 7, 64, 150, 32, [150, 77]),
    (2, 4, 1, 33, 128, 513, 64, [513, 40]),
    (1, 8, 2, 130, 128, 1111, 128, [1111]),
    (2, 4, 4, 257, 64, 300, 16, [300, 280]),
    (1, 3, 1, 200, 48, 260, 32, [231]),
    (1, 2, 2, 64, 256, 190, 64, [190]),
    (2, 4, 1, 70, 256, 300, 32, [300, 71]),
    (6, 8, 2, 5, 128, 400, 64, [0, 1, 127, 128, 129, 400]),
    (3, 4, 1, 16, 64, 1000, 16, [1000, 15, 640]),
    (2, 4, 2, 9, 48, 260, 32, [260, 131]),
    (2, 20, 1, 3, 112, 5000, 128, [5000, 3]),
    (1, 8, 1, 90, 64, 700, 128, [700]),
    # caches of more than 2048 rows: the keys of a head are split over the SMs and joined
    (1, 4, 1, 1, 128, 4100, 64, [4099]),
    (2, 8, 8, 1, 64, 3000, 16, [3000, 5]),
    (1, 10, 1, 1, 128, 2300, 32, [2222]),
    (2, 4, 1, 5, 128, 2600, 128, [2600, 2049]),
    (1, 8, 1, 4, 64, 2100, 32, [2100]),
    (1, 2, 1, 30, 80, 2200, 16, [2195]),
    (1, 1, 1, 3, 256, 2500, 64, [2500]),
    (1, 3, 1, 5, 240, 2100, 32, [2100]),
]


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:7])))
def test_attention_matches_64_bits(fmt, dt, shape):
    B, H, Hkv, Lq, D, cap, block, lens = shape
    cache = random_cache(B, Hkv, cap, D, block, fmt, lens, 4)
    q = (torch.randn((B, Lq, H, D), device="cuda", generator=gen(5)) * 1.2).to(dt).transpose(1, 2)
    check_attention(q, cache)


@pytest.mark.parametrize("Lq", [1, 5, 40, 140])
def test_attention_with_counts(Lq):
    cache = random_cache(5, 2, 400, 128, 64, torch.float8_e4m3fn, [400, 3, 0, 129, 250], 6)
    q = torch.randn((5, 8, Lq, 128), device="cuda", generator=gen(7)).to(torch.bfloat16)
    check_attention(q, cache, counts=[Lq, Lq, Lq, 0, max(1, Lq // 2)])


# where the kernels change over, in long caches: full tiles of rows with weights, the first rows past a tile, many
# rows in so few items that each is cut into parts (some of them past a sequence's end)
EDGES = [
    (1, 8, 1, 4, 128, 2600, 64, [2600]),
    (2, 12, 1, 2, 64, 4200, 16, [4200, 31]),
    (1, 3, 1, 11, 128, 2100, 32, [2099]),
    (1, 32, 2, 1, 256, 1500, 128, [1500]),
    (1, 17, 1, 1, 256, 1200, 16, [1200]),
    (3, 4, 1, 33, 128, 8192, 64, [8192, 5, 0]),
    (2, 8, 2, 40, 64, 5000, 128, [3000, 5000]),
    (1, 1, 1, 300, 96, 9000, 16, [8999]),
    (5, 4, 2, 129, 64, 1600, 32, [1600, 1100, 129, 70, 513]),
]


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", EDGES, ids=lambda s: "x".join(map(str, s[:7])))
def test_attention_where_kernels_change_over(fmt, dt, shape):
    B, H, Hkv, Lq, D, cap, block, lens = shape
    cache = random_cache(B, Hkv, cap, D, block, fmt, lens, 31)
    q = (torch.randn((B, Lq, H, D), device="cuda", generator=gen(32)) * 1.2).to(dt).transpose(1, 2)
    check_attention(q, cache)
    check_attention(q, cache, counts=[max(0, Lq - 3 * b) for b in range(B)])


def test_attention_over_many_short_sequences_and_one_long():
    lens = [(37 * i) % 90 for i in range(300)] + [6000]
    cache = random_cache(301, 1, 6000, 64, 32, torch.int8, lens, 8)
    q = torch.randn((301, 2, 1, 64), device="cuda", generator=gen(9)).to(torch.float16)
    check_attention(q, cache)


def test_attention_lengths_outside_the_cache_are_clamped():
    cache = random_cache(3, 1, 64, 32, 16, torch.int8, [64, 64, 64], 10)
    q = torch.randn((3, 2, 2, 32), device="cuda", generator=gen(11)).to(torch.bfloat16)
    want = check_attention(q, cache, score=False)
    cache.lens.copy_(torch.tensor([70, -3, 64], dtype=torch.int32))
    from gguf_train_b200 import kv8_attention

    out = kv8_attention(q, cache)
    assert torch.equal(out[0], want[0]) and (out[1] == 0).all() and torch.equal(out[2], want[2])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_attention_scales_far_apart(dt):
    """Blocks whose values differ by many orders, a block of zeros (scale 0), and queries from tiny to huge."""
    for block in (16, 64):
        cache = random_cache(2, 1, 256, 64, block, torch.int8, [256, 250], 12)
        nb = cache.k_scale.shape[2]
        cache.v_scale.copy_(torch.logspace(-6, 4, nb, device="cuda").expand(2, 1, nb))
        cache.k_scale.copy_((0.02 * torch.logspace(0, -5, nb, device="cuda")).expand(2, 1, nb))
        cache.k_scale[:, :, 1] = 0
        cache.v_scale[:, :, 1] = 0
        cache.k[:, :, block:2 * block] = 0
        cache.v[:, :, block:2 * block] = 0
        for size in (1e-6, 1.0, 30.0):
            q = (torch.randn((2, 2, 3, 64), device="cuda", generator=gen(13)) * size).to(dt)
            check_attention(q, cache)


def test_attention_large_scores():
    """Softmax dominated by one key, and scores far above what exp() holds."""
    cache = random_cache(1, 1, 300, 128, 64, torch.int8, [300], 14)
    q = (torch.randn((1, 4, 2, 128), device="cuda", generator=gen(15)) * 60).to(torch.bfloat16)
    check_attention(q, cache, scale=1.0)


def test_attention_row_of_nan_stays_in_its_row():
    from gguf_train_b200 import kv8_attention

    cache = random_cache(2, 2, 200, 64, 32, torch.int8, [200, 150], 16)
    for Lq in (1, 3, 150):
        q = torch.randn((2, 4, Lq, 64), device="cuda", generator=gen(17)).to(torch.bfloat16)
        want = kv8_attention(q, cache)
        bad = q.clone()
        bad[0, 1, Lq // 2, 5] = float("nan")
        bad[1, 2, 0, 3] = float("inf")
        out = kv8_attention(bad, cache)
        touched = torch.zeros((2, 4, Lq), dtype=torch.bool, device="cuda")
        touched[0, 1, Lq // 2] = touched[1, 2, 0] = True
        assert out[touched].isnan().any(-1).all()
        assert torch.equal(out[~touched], want[~touched])


def test_attention_strides_and_streams():
    """q as a view of a wider projection, at an odd element offset too; a call on a side stream; the same bits twice."""
    from gguf_train_b200 import kv8_attention

    cache = random_cache(2, 2, 500, 64, 64, torch.float8_e4m3fn, [500, 321], 18)
    buf = torch.randn((2, 6, 4 * 64 * 3 + 1), device="cuda", generator=gen(19)).to(torch.bfloat16)
    for off in (0, 1):
        q = buf[..., off:off + 4 * 64 * 3].unflatten(-1, (12, 64))[:, :, 2:10:2].transpose(1, 2)
        assert not q.is_contiguous()
        want = kv8_attention(q.contiguous(), cache)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = kv8_attention(q, cache)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want)
        check_attention(q, cache)


def test_attention_without_queries_or_rows():
    from gguf_train_b200 import KV8Cache, kv8_attention

    cache = random_cache(2, 1, 40, 32, 16, torch.int8, [40, 9], 20)
    assert kv8_attention(torch.empty((2, 2, 0, 32), device="cuda"), cache).shape == (2, 2, 0, 32)
    score, other = torch.rand((2, 1, 40), device="cuda"), torch.zeros((2, 1, 40), device="cuda")
    kv8_attention(torch.empty((2, 2, 0, 32), device="cuda"), cache, score=score, score_out=other)
    assert torch.equal(other[0], score[0]) and torch.equal(other[1, :, :9], score[1, :, :9]) and (other[1, :, 9:] == 0).all()
    none = KV8Cache.empty(2, 1, 0, 32)
    out, lse = kv8_attention(torch.ones((2, 2, 3, 32), device="cuda"), none, need_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


# ------------------------------------------------------------------ eviction

def evict_reference(cache, score, budget, recent, out_block):
    """Per (b, hk): kept rows, and the codes (f32) and scales of the new cache in the operator's steps."""
    fmt, T = cache.k.dtype, cache.block
    B, Hkv = cache.k.shape[:2]
    res = {}
    for b in range(B):
        n = min(max(int(cache.lens[b]), 0), cache.capacity)
        for h in range(Hkv):
            if n <= budget:
                idx = list(range(n))
            else:
                s = [(-math.inf if math.isnan(x) else x) for x in score[b, h, :n - recent].tolist()]
                first = sorted(range(n - recent), key=lambda i: (-s[i], i))[:budget - recent]
                idx = sorted(first) + list(range(n - recent, n))
            rows = torch.tensor(idx, dtype=torch.long, device="cuda")
            new = []
            for c, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                x = c[b, h].float()[rows] * sc[b, h, rows // T][:, None]
                scales, codes = [], []
                for j in range(0, len(idx), out_block):
                    s = scale_of(x[j:j + out_block].abs().amax(), fmt)
                    scales.append(s)
                    codes.append(quantise(x[j:j + out_block], s.expand_as(x[j:j + out_block]), fmt))
                new.append((torch.cat(codes) if codes else x, torch.stack(scales) if scales else x.new_zeros(0)))
            res[b, h] = (idx, new)
    return res


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("B,Hkv,cap,D,block,out_block,budget,recent,lens", [
    (2, 2, 200, 64, 16, 16, 50, 10, [200, 49]),
    (3, 1, 700, 128, 64, 32, 130, 0, [700, 130, 131]),
    (2, 3, 90, 16, 32, 128, 40, 40, [90, 0]),        # recent only
    (1, 2, 5000, 48, 128, 64, 1111, 1, [4999]),
    (2, 1, 60, 256, 16, 64, 59, 30, [60, 60]),
    (1, 1, 30, 32, 16, 16, 1, 0, [30]),
    (1, 1, 1500, 32, 16, 16, 1200, 1100, [1500]),
])
def test_evict_keeps_the_heaviest_rows(fmt, B, Hkv, cap, D, block, out_block, budget, recent, lens):
    from gguf_train_b200 import KV8Cache, _C, kv8_evict

    cache = random_cache(B, Hkv, cap, D, block, fmt, lens, 21)
    score = torch.rand((B, Hkv, cap), device="cuda", generator=gen(22))
    score = (score * 37).floor() / 37  # many ties
    score[:, :, 3::17] = float("nan")
    score[:, :, 5::19] = float("inf")
    score[:, :, 7::23] = float("-inf")
    score[:, :, 8::29] = -0.0
    out = KV8Cache.empty(B, Hkv, budget + 3, D, out_block, fmt)
    out2, score_out, kept = kv8_evict(cache, score, budget, recent, out=out)
    assert out2 is out
    for (b, h), (idx, new) in evict_reference(cache, score, budget, recent, out_block).items():
        m = len(idx)
        assert out.lens[b] == m
        assert kept[b, h, :m].tolist() == idx and (kept[b, h, m:] == -1).all()
        assert torch.equal(score_out[b, h, :m].nan_to_num(-5.0), score[b, h, idx].nan_to_num(-5.0))
        assert (score_out[b, h, m:] == 0).all()
        for (c, s), (rc, rs) in zip(((out.k, out.k_scale), (out.v, out.v_scale)), new):
            assert torch.equal(c[b, h, :m].float(), rc)
            assert torch.equal(s[b, h, :len(rs)], rs)
    assert _C.device_status() == 0


def test_evict_of_equal_scores_and_negative_ones():
    from gguf_train_b200 import kv8_evict

    cache = random_cache(1, 1, 300, 32, 16, torch.int8, [300], 23)
    _, _, kept = kv8_evict(cache, torch.zeros((1, 1, 300), device="cuda"), 100, 20)
    assert kept[0, 0].tolist() == list(range(80)) + list(range(280, 300))
    score = -torch.arange(300, device="cuda", dtype=torch.float32)[None, None]
    _, _, kept = kv8_evict(cache, score.contiguous(), 10)
    assert kept[0, 0].tolist() == list(range(10))


# ------------------------------------------------------------------ together

def test_a_session_of_append_attend_evict_stays_near_16_bit_attention():
    """A prompt, an eviction and decode steps: the outputs follow full-precision attention over the same kept tokens
    within what 8-bit keys and values cost (int8 of N(0,1): steps of 4.5/127, scores off by about
    sqrt(D) 0.01 / sqrt(D), values by 0.01)."""
    from gguf_train_b200 import KV8Cache, kv8_append, kv8_attention, kv8_evict

    g = gen(24)
    B, H, Hkv, D, n = 2, 8, 2, 64, 300
    k, v = (torch.randn((B, Hkv, n + 20, D), device="cuda", generator=g) for _ in range(2))
    cache = KV8Cache.empty(B, Hkv, n + 20, D, 64)
    score = torch.zeros((B, Hkv, n + 20), device="cuda")
    kv8_append(cache, k[:, :, :n], v[:, :, :n])
    q = torch.randn((B, H, n, D), device="cuda", generator=g).to(torch.bfloat16)
    kv8_attention(q, cache, score=score)
    small = KV8Cache.empty(B, Hkv, 128, D, 64)
    small, sscore, kept = kv8_evict(cache, score, 100, recent=30, out=small)
    rows = [kept.long()]
    for t in range(n, n + 20):
        kv8_append(small, k[:, :, t:t + 1], v[:, :, t:t + 1])
        q = torch.randn((B, H, 1, D), device="cuda", generator=g).to(torch.bfloat16)
        out = kv8_attention(q, small, score=sscore)
        rows.append(torch.full((B, Hkv, 1), t, device="cuda"))
        at = torch.cat(rows, -1)[..., None].expand(-1, -1, -1, D)
        kk, vv = (torch.gather(x, 2, at).repeat_interleave(H // Hkv, 1).double() for x in (k, v))
        want = torch.softmax(q.double() @ kk.transpose(-1, -2) / math.sqrt(D), -1) @ vv
        assert (out.double() - want).abs().max() < 0.08
    assert small.lens.tolist() == [120, 120]


def test_refusals():
    from gguf_train_b200 import KV8Cache, _C, kv8_append, kv8_attention, kv8_evict, kv8_read
    from gguf_train_b200.kv8 import _t4
    import ctypes

    cache = random_cache(2, 2, 40, 32, 16, torch.int8, [40, 9], 25)
    x = torch.zeros((2, 2, 3, 32), device="cuda")
    with pytest.raises(RuntimeError, match="must be \\(2, 2, n, 32\\)"):
        kv8_append(cache, x[..., :16], x[..., :16])
    with pytest.raises(RuntimeError, match="f32, f16 or bf16"):
        kv8_append(cache, x.double(), x.double())
    with pytest.raises(RuntimeError, match="counts must be"):
        kv8_append(cache, x, x, counts=torch.ones(2, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv8_append(cache, x.cpu(), x.cpu())
    with pytest.raises(RuntimeError, match="q must be"):
        kv8_attention(x[:1], cache)
    with pytest.raises(RuntimeError, match="divisible"):
        kv8_attention(torch.zeros((2, 3, 1, 32), device="cuda"), cache)
    with pytest.raises(RuntimeError, match="score must be"):
        kv8_attention(x, cache, score=torch.zeros((2, 2, 39), device="cuda"))
    with pytest.raises(RuntimeError, match="score_out needs score"):
        kv8_attention(x, cache, score_out=torch.zeros((2, 2, 40), device="cuda"))
    with pytest.raises(RuntimeError, match="scale must be finite"):
        kv8_attention(x, cache, scale=float("nan"))
    with pytest.raises(RuntimeError, match="not be negative"):
        kv8_read(cache, None, -1)
    score = torch.zeros((2, 2, 40), device="cuda")
    for budget, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(RuntimeError, match="budget must be"):
            kv8_evict(cache, score, budget, recent)
    with pytest.raises(RuntimeError, match="fewer than the budget"):
        kv8_evict(cache, score, 8, out=KV8Cache.empty(2, 2, 7, 32, 16))
    with pytest.raises(RuntimeError, match="must agree"):
        kv8_evict(cache, score, 8, out=KV8Cache.empty(2, 2, 8, 32, 16, torch.float8_e4m3fn))
    with pytest.raises(RuntimeError, match="share no memory"):
        kv8_evict(cache, score, 8, out=cache)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        KV8Cache.empty(1, 1, 8, 40)
    with pytest.raises(RuntimeError, match="block must be"):
        KV8Cache.empty(1, 1, 8, 32, block=48)
    with pytest.raises(RuntimeError, match="int8 or"):
        KV8Cache.empty(1, 1, 8, 32, dtype=torch.uint8)
    # the C entry checks for itself
    bad = _C.KV8.from_buffer_copy(cache._native)
    bad.block = 20
    t = _t4(x)
    assert _C.lib.gtb_kv8_append(ctypes.byref(bad), t, t, None, 0, None) == -1
    assert b"16, 32, 64 or 128" in _C.lib.gtb_last_error()
    bad = _C.KV8.from_buffer_copy(cache._native)
    bad.k = bad.k + 1
    assert _C.lib.gtb_kv8_append(ctypes.byref(bad), t, t, None, 0, None) == -1
    host = torch.zeros((2, 2, 3, 32))
    assert _C.lib.gtb_kv8_append(ctypes.byref(cache._native), _t4(host), t, None, 0, None) == -1
    assert b"no CPU path" in _C.lib.gtb_last_error()
