"""The latent attention calls used together: the example session (examples/latent_session.py), a step replayed from a CUDA graph,
streams, and what inputs that are not finite do.

The session in bf16: queries taken through the keys' up-projection are rounded once more than expanded ones (2^-9 / sqrt(3) of a
value each, which in a score of unit spread is as much), outputs and their up-projections are rounded twice; each of the
steps is off by at most 2^-8 of its size, and there are six of them on the way: q, the absorbed q, the weights, the
output, the latents' products with w_v, and the expanded keys and values of the comparison."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "latent_session.py")


def _session():
    spec = importlib.util.spec_from_file_location("latent_session", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("sizes", [dict(), dict(heads=8, latent=512, Dn=128, Dr=64, batch=3, system=130, text=65, new=5),
                                   dict(heads=40, latent=128, Dn=64, Dr=16, batch=2, system=1, text=3, new=3)], ids=str)
def test_session(sizes):
    from gguf_train_b200 import _C

    errs = _session().run(quiet=True, **{**dict(batch=4, system=300, text=70, new=6), **sizes})
    assert _C.device_status() == 0
    assert all(e <= 6 * 2.0 ** -8 for e in errs), errs


@pytest.mark.parametrize("Lq,H,P", [(1, 16, 0), (1, 16, 200), (3, 20, 200), (70, 16, 90), (1, 4, 700)])
def test_a_step_replayed_from_a_graph(Lq, H, P):
    """Replayed over changed inputs and a growing cache: the bits of the same calls made one by one."""
    from gguf_train_b200 import LatentCache, _C, latent_append, latent_attention

    B, R, Dr, cap, steps = 3, 256, 32, 400, 3
    gen = torch.Generator(device="cuda").manual_seed(7)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    rows, lens = r(B, cap, R + Dr), torch.tensor([cap - steps * Lq, 63, 0], dtype=torch.int32, device="cuda")
    prefix = LatentCache(r(1, P, R + Dr), torch.tensor([P], dtype=torch.int32, device="cuda"), R) if P else None
    xs = [(r(B, H, Lq, R + Dr), r(B, Lq, R), r(B, Lq, Dr)) for _ in range(steps)]

    def step(q, c, k, cache):
        latent_append(cache, c, k, rope=dict(mode=2), prefix=prefix)
        return latent_attention(q, cache, 0.07, prefix=prefix, need_lse=True)

    cache = LatentCache(rows.clone(), lens.clone(), R)
    want = [[t.clone() for t in (*step(*x, cache), cache.rows, cache.lens)] for x in xs]
    cache = LatentCache(rows.clone(), lens.clone(), R)
    buf = [t.clone() for t in xs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        res = step(*buf, cache)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for x, w in zip(xs, want):
        for a, b in zip(buf, x):
            a.copy_(b)
        graph.replay()
        for got, exp in zip((*res, cache.rows, cache.lens), w):
            assert torch.equal(got, exp)
    torch.cuda.synchronize()
    del graph
    assert _C.device_status() == 0


@pytest.mark.parametrize("padded", [False, True])
def test_a_training_step_replayed_from_a_graph(padded):
    from gguf_train_b200 import _C, latent_sdpa

    B, H, L, Dn, Dr = 2, 3, 200, 64, 32
    gen = torch.Generator(device="cuda").manual_seed(8)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    sets = [[r(B, H, L, Dn + Dr), r(B, H, L, Dn), r(B, L, Dr), r(B, H, L, Dn), r(B, H, L, Dn)] for _ in range(3)]
    lens = [torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([200, 7], [0, 129], [64, 200])]

    def step(q, k, kr, v, g, n):
        leaves = [t.detach().requires_grad_() for t in (q, k, kr, v)]
        out = latent_sdpa(*leaves, is_causal=True, seq_lens=n if padded else None)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    want = [[t.clone() for t in step(*s, n)] for s, n in zip(sets, lens)]
    buf, nb = [t.clone() for t in sets[0]], lens[0].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(*buf, nb)
        graph.capture_begin()
        res = step(*buf, nb)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for s, n, w in zip(sets, lens, want):
        for a, b in zip(buf, s):
            a.copy_(b)
        nb.copy_(n)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(res, w))
    torch.cuda.synchronize()
    del graph
    assert _C.device_status() == 0


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing: the bits of the same calls one after the other."""
    from gguf_train_b200 import LatentCache, _C, latent_attention, latent_sdpa

    gen = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    caches = [LatentCache(r(4, 3000, 576), torch.tensor(n, dtype=torch.int32, device="cuda"), 512) for n in ([3000, 1, 77, 900], [5, 2999, 0, 640])]
    qs = [r(4, 16, 1, 576) for _ in range(2)]
    xs = [(r(2, 4, 500, 192), r(2, 4, 500, 128), r(2, 500, 64), r(2, 4, 500, 128)) for _ in range(2)]
    calls = [lambda i=i: (latent_attention(qs[i], caches[i], 0.07), latent_sdpa(*xs[i], is_causal=True)) for i in range(2)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
    assert _C.device_status() == 0


def test_lengths_out_of_range_are_read_as_the_nearest():
    from gguf_train_b200 import LatentCache, _C, latent_attention, latent_sdpa

    gen = torch.Generator(device="cuda").manual_seed(10)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    rows, q = r(2, 100, 96), r(2, 4, 2, 96)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    a = latent_attention(q, LatentCache(rows, i32(-5, 1000000), 64), 0.1, counts=i32(-1, 7))
    b = latent_attention(q, LatentCache(rows, i32(0, 100), 64), 0.1, counts=i32(0, 2))
    assert torch.equal(a, b)
    x = (r(2, 2, 70, 96), r(2, 2, 70, 64), r(2, 70, 32), r(2, 2, 70, 64))
    assert torch.equal(latent_sdpa(*x, seq_lens=i32(-3, 900)), latent_sdpa(*x, seq_lens=i32(0, 70)))
    # more new tokens than rows: those whose own row is missing attend what there is, the first ones nothing
    out, lse = latent_attention(q, LatentCache(rows, i32(1, 1), 64), 0.1, need_lse=True)
    assert bool((out[:, :, 0] == 0).all()) and bool(torch.isneginf(lse[:, :, 0]).all())
    assert torch.allclose(out[:, :, 1].float(), rows[:, None, 0, :64].float().expand(2, 4, 64), rtol=2.0 ** -7)
    assert _C.device_status() == 0


def test_values_that_are_not_finite_stay_in_their_rows():
    """A query that is NaN gives NaN, alone; scores far below any mask value still weigh; an infinite score gives NaN."""
    from gguf_train_b200 import LatentCache, latent_attention, latent_sdpa

    gen = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    cache = LatentCache(r(2, 700, 160), torch.tensor([700, 650], dtype=torch.int32, device="cuda"), 128)
    q = r(2, 5, 3, 160)
    want, wl = latent_attention(q, cache, 0.1, need_lse=True)
    bad = q.clone()
    bad[1, 2, 1] = float("nan")
    got, gl = latent_attention(bad, cache, 0.1, need_lse=True)
    assert bool(torch.isnan(got[1, 2, 1]).all()) and bool(torch.isnan(gl[1, 2, 1]))
    got[1, 2, 1], gl[1, 2, 1] = want[1, 2, 1], wl[1, 2, 1]
    assert torch.equal(got, want) and torch.equal(gl, wl)
    # scores of about -1e32: a constant far below any masking value, which the softmax does not see
    rows = r(1, 70, 160)
    rows[..., 159] = -1.0
    low = LatentCache(rows, torch.tensor([70], dtype=torch.int32, device="cuda"), 128)
    q = torch.zeros((1, 1, 1, 160), dtype=torch.bfloat16, device="cuda")
    q[..., 159] = 1e32
    out, lse = latent_attention(q, low, 1.0, need_lse=True)
    mean = rows[0, :, :128].double().mean(0)
    assert bool(((out[0, 0, 0].double() - mean).abs() <= 2.0 ** -8 * (mean.abs() + rows[0, :, :128].double().abs().mean(0))).all())
    assert abs(float(lse) / -float(q[0, 0, 0, 159]) - 1.0) < 1e-6
    x = [r(1, 2, 150, 96), r(1, 2, 150, 64), r(1, 150, 32), r(1, 2, 150, 64)]
    want = latent_sdpa(*x, is_causal=True)
    x[0][0, 1, 77] = float("nan")
    got = latent_sdpa(*x, is_causal=True)
    assert bool(torch.isnan(got[0, 1, 77]).all())
    got[0, 1, 77] = want[0, 1, 77]
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    """A cache whose last sequence starts beyond 2^32 bytes and 2^31 values."""
    from gguf_train_b200 import LatentCache, _C, latent_append, latent_attention

    cap, D = 1 << 21, 576
    rows = torch.zeros((2, cap, D), dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([3, cap - 70], dtype=torch.int32, device="cuda")
    cache = LatentCache(rows, lens, 512)
    gen = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn((2, 70, D), device="cuda", generator=gen).to(torch.bfloat16)
    latent_append(cache, x[..., :512], x[..., 512:])
    assert torch.equal(rows[1, cap - 70:], x[1]) and torch.equal(rows[0, 3:73], x[0])
    q = torch.randn((2, 2, 1, D), device="cuda", generator=gen).to(torch.bfloat16)
    out, lse = latent_attention(q, cache, 0.2, need_lse=True)
    n = torch.tensor([73, cap], device="cuda").double()
    for b in range(2):  # rows of zeros have score 0
        s = torch.einsum("hd,sd->hs", q[b, :, 0].double(), x[b].double()) * 0.2
        total = s.exp().sum(-1) + (n[b] - 70)
        want = s.exp() @ x[b, :, :512].double() / total[:, None]
        mags = s.exp() @ x[b, :, :512].double().abs() / total[:, None]
        e = D * 2.0 ** -22 * 0.2 * float((q[b, :, 0].double().abs() @ x[b].double().abs().t()).max())
        assert bool(((out[b, :, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * e) * mags + 1e-30).all())
        assert bool(((lse[b, :, 0].double() - total.log()).abs() <= e + 2.0 ** -20 * total.log()).all())
    assert _C.device_status() == 0
