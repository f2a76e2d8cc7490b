"""rope_axes (several position axes) on the GPU against the rotation in 64 bits: layouts of pairs and axes,
types, strides, long and negative positions, the gradient against the formula and against differences,
and the call's refusals.

Tolerance: the angle is exact to 2^-33 of a turn and then rounded to f32 (relative 2^-24 of half a turn at most:
2e-7 rad), sine and cosine carry a few ulp: |error| <= 6e-7 (|x0| + |x1|), plus one rounding to the output type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(x, pos, sections, mode=2, base=10000.0, scale=1.0, interleaved=False, per_axis=False, sign=1.0):
    """(y, |x0| + |x1| per element) in float64; pos (A, B, S)."""
    x = x.detach().double().cpu().numpy()
    pos = pos.cpu().numpy().astype(np.float64)
    P, A = sum(sections), len(sections)
    y, mag = x.copy(), np.abs(x)
    used = [0] * A
    left = [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(P):
        a = (i % A if i < A * sections[i % A] else 0) if interleaved else left[i]
        f = scale * base ** (-(used[a] / sections[a] if per_axis else i / P))
        used[a] += 1
        c0, c1 = (2 * i, 2 * i + 1) if mode == 0 else (i, i + P)
        ang = (pos[a] * f)[:, None]
        c, s = np.cos(ang), sign * np.sin(ang)
        y[..., c0] = x[..., c0] * c - x[..., c1] * s
        y[..., c1] = x[..., c0] * s + x[..., c1] * c
        mag[..., c0] = mag[..., c1] = np.abs(x[..., c0]) + np.abs(x[..., c1])
    return y, mag


def check(got, want, mag, dtype):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    tol = 6e-7 * mag + ULP[dtype] * np.abs(want) + (6e-8 if dtype == torch.float16 else 1e-38)
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / tol):.2f} of the tolerance"


def positions(A, B, S, hi, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-hi if hi > 10 ** 6 else 0, hi, (A, B, S), generator=g).to("cuda", torch.int32)


CASES = [
    # B, H, Hkv, S, D, sections, mode, interleaved, per_axis, dtype, largest position
    (1, 1, 1, 1, 16, (3, 2, 2), 2, False, False, torch.float32, 100),
    (2, 4, 1, 7, 128, (16, 24, 24), 2, False, False, torch.bfloat16, 32768),
    (2, 3, 1, 33, 128, (16, 24, 24), 0, False, False, torch.float16, 1000),
    (3, 5, 2, 65, 128, (24, 20, 20), 2, True, False, torch.bfloat16, 100000),
    (1, 2, 2, 17, 64, (12, 10, 10), 0, True, False, torch.float32, 2 ** 31 - 1),
    (2, 2, 2, 130, 80, (20, 20), 2, False, True, torch.float32, 64),
    (2, 2, 1, 31, 80, (20, 20), 0, False, True, torch.bfloat16, 64),
    (1, 8, 8, 19, 72, (5, 7, 0), 2, False, False, torch.float16, 500),   # odd sections, an empty one, a tail
    (2, 1, 1, 40, 256, (128,), 2, False, False, torch.float32, 10 ** 6),
    (1, 2, 1, 9, 33, (4, 4, 4, 4), 0, False, True, torch.float32, 77),   # odd head size, four axes
    (2, 40, 8, 3, 96, (16, 16, 16), 2, False, False, torch.bfloat16, 4096),
    (5, 4, 4, 257, 64, (8, 12, 12), 2, False, False, torch.float16, 300),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(str(v).replace("torch.", "") for v in c[:5] + (c[5],)))
def test_rotation_matches_the_formula(case):
    from gguf_train_b200 import _C, rope_axes

    B, H, Hkv, S, D, sections, mode, inter, per, dt, hi = case
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn((B, n, S, D), generator=g).to("cuda", dt) for n in (H, Hkv))
    pos = positions(len(sections), B, S, hi, 2)
    yq, yk = rope_axes(q, pos, sections, k=k, mode=mode, interleaved=inter, per_axis=per, freq_scale=0.75)
    for x, y in ((q, yq), (k, yk)):
        check(y, *reference(x, pos, sections, mode, 10000.0, 0.75, inter, per), dt)
    one = rope_axes(q, pos, sections, mode=mode, interleaved=inter, per_axis=per, freq_scale=0.75)
    assert torch.equal(one, yq)
    assert _C.device_status() == 0


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_views_shared_positions_and_streams(dt):
    """q and k as views of one projection's output, at an offset that is not 16-byte aligned too; positions
    shared by the batch; a call on a side stream."""
    from gguf_train_b200 import rope_axes

    B, S, H, Hkv, D = 2, 29, 6, 2, 64
    sections = (8, 12, 12)
    buf = torch.randn((B, S, (H + 2 * Hkv) * D + 1), device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dt)
    pos = positions(3, 1, S, 4000, 4)
    for off in (0, 1):
        qkv = buf[..., off:off + (H + 2 * Hkv) * D].unflatten(-1, (H + 2 * Hkv, D)).transpose(1, 2)
        q, k = qkv[:, :H], qkv[:, H:H + Hkv]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            yq, yk = rope_axes(q, pos[:, 0], sections, k=k)
            yq3 = rope_axes(q, pos, sections)
        torch.cuda.current_stream().wait_stream(side)
        ref = pos.expand(3, B, S)
        check(yq, *reference(q, ref, sections), dt)
        check(yk, *reference(k, ref, sections), dt)
        assert torch.equal(yq, yq3)


def test_one_axis_agrees_with_rope():
    """With one axis the rotation is rope()'s, up to its f32 accumulation of the angle (i + 1 roundings of an
    angle of at most 50: 50 * 33 * 2^-24 rad)."""
    from gguf_train_b200 import rope, rope_axes

    x = torch.randn((1, 2, 50, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    pos = torch.arange(50, device="cuda", dtype=torch.int32)
    for mode in (0, 2):
        assert (rope_axes(x, pos[None], (32,), mode=mode) - rope(x, pos, mode=mode)).abs().max() < 2 * 50 * 33 * 2.0 ** -24 * 5


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gradient_is_the_rotation_back(dt):
    from gguf_train_b200 import rope_axes

    g = torch.Generator().manual_seed(6)
    q, k = (torch.randn((2, n, 21, 80), generator=g).to("cuda", dt).requires_grad_() for n in (4, 2))
    gq, gk = (torch.randn((2, n, 21, 80), generator=g).to("cuda", dt) for n in (4, 2))
    gq = gq.transpose(1, 2).contiguous().transpose(1, 2)  # a gradient in another layout
    pos = positions(2, 2, 21, 60, 7)
    yq, yk = rope_axes(q, pos, (20, 18), k=k, per_axis=True)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    check(dq, *reference(gq, pos, (20, 18), per_axis=True, sign=-1.0), dt)
    check(dk, *reference(gk, pos, (20, 18), per_axis=True, sign=-1.0), dt)
    # only one of the two is differentiated
    yq, yk = rope_axes(q.detach(), pos, (20, 18), k=k, per_axis=True)
    (dk2,) = torch.autograd.grad(yk, k, gk)
    assert torch.equal(dk2, dk)


def test_gradient_against_differences():
    """The map is linear: L(x + e) - L(x) over a step along a direction equals the gradient's product with it, to f32
    rounding of sums of 2 * 21 * 32 products of order 1 (1e-3)."""
    from gguf_train_b200 import rope_axes

    g = torch.Generator().manual_seed(8)
    x = torch.randn((1, 2, 21, 32), generator=g).cuda().requires_grad_()
    w, e = (torch.randn(x.shape, generator=g).cuda() for _ in range(2))
    pos = positions(3, 1, 21, 50, 9)
    f = lambda z: (rope_axes(z, pos, (4, 6, 6), interleaved=False) * w).double().sum()  # noqa: E731
    (dx,) = torch.autograd.grad(f(x), x)
    num = (f(x.detach() + e) - f(x.detach() - e)) / 2
    assert abs(num.item() - (dx.double() * e.double()).sum().item()) < 1e-3


def test_empty_calls():
    from gguf_train_b200 import rope_axes

    pos = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    assert rope_axes(torch.zeros((2, 3, 0, 16), device="cuda"), pos, (4, 4)).shape == (2, 3, 0, 16)
    pos = torch.zeros((2, 5), dtype=torch.int32, device="cuda")
    assert rope_axes(torch.zeros((0, 3, 5, 16), device="cuda"), pos, (4, 4)).shape == (0, 3, 5, 16)


def test_refusals():
    from gguf_train_b200 import rope_axes

    x = torch.zeros((2, 3, 5, 16), device="cuda")
    pos = torch.zeros((2, 5), dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="sum to between 1 and half"):
        rope_axes(x, pos, (4, 5))
    with pytest.raises(RuntimeError, match="sum to between 1 and half"):
        rope_axes(x, pos, (0, 0))
    with pytest.raises(RuntimeError, match="positions must be"):
        rope_axes(x, pos, (2, 2, 2))
    with pytest.raises(RuntimeError, match="positions must be"):
        rope_axes(x, pos[:, :4], (4, 4))
    with pytest.raises(RuntimeError, match="int32"):
        rope_axes(x, pos.long(), (4, 4))
    with pytest.raises(RuntimeError, match="mode"):
        rope_axes(x, pos, (4, 4), mode=1)
    with pytest.raises(RuntimeError, match="interleaved"):
        rope_axes(x, pos, (1, 5), interleaved=True)
    with pytest.raises(RuntimeError, match="freq_base"):
        rope_axes(x, pos, (4, 4), freq_base=-1.0)
    with pytest.raises(RuntimeError, match="f32, f16 or bf16"):
        rope_axes(x.double(), pos, (4, 4))
    with pytest.raises(RuntimeError, match="do not fit together"):
        rope_axes(x, pos, (4, 4), k=torch.zeros((2, 3, 4, 16), device="cuda"))
    with pytest.raises(RuntimeError, match="1 to 4 sections"):
        rope_axes(x, torch.zeros((5, 5), dtype=torch.int32, device="cuda"), (1, 1, 1, 1, 1))
    with pytest.raises(RuntimeError, match="negative"):
        rope_axes(x, pos, (-1, 4))
