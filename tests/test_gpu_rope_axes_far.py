"""rope_axes at positions near 2^31 against 60-digit arithmetic, and 16-bit heads of 72 (18 + 18 pairs: rows that are not
whole 16-byte pieces).

Tolerance at far positions, for angles whose rest after whole turns is below 2^-6 of a turn (so that neither f32's
rounding of the rest nor of the sine hides the frequency's own error): the frequency's 64-bit fraction is right to 2^-63, 2^-32 of
a turn at 2^31 positions; the product is cut at 2^-32 and rounded to f32 (relative 2^-24); the sine of it, at most
0.1, is right to 4 ulp (2^-25 = 4 ulp of 0.1): (2^-31 + 2^-30) 2 pi + 2^-25 < 4e-8."""

from __future__ import annotations

from decimal import Decimal, getcontext

import pytest
import torch

from test_gpu_rope_axes import check, positions, reference

pytestmark = pytest.mark.gpu

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def _sin(x):
    term = total = x
    for k in range(1, 20):
        term = -term * x * x / ((2 * k) * (2 * k + 1))
        total += term
    return total


@pytest.mark.parametrize("sections,per_axis,scale", [((16, 24, 24), False, 1.0), ((20, 12), True, 0.75), ((32,), False, 0.5)], ids=str)
def test_far_positions_lose_nothing(sections, per_axis, scale):
    from gguf_train_b200 import rope_axes

    getcontext().prec = 60
    P, A, S = sum(sections), len(sections), 4096
    x = torch.zeros((1, 1, S, 2 * P), device="cuda")
    x[..., 0::2] = 1.0  # y = (cos, sin) of every pair
    first = 2 ** 31 - S
    pos = (first + torch.arange(S, dtype=torch.int64)).to("cuda", torch.int32).expand(A, S).contiguous()
    y = rope_axes(x, pos, sections, mode=0, per_axis=per_axis, freq_scale=scale)[0, 0].double().cpu()
    seen, i = 0, 0
    for a, n in enumerate(sections):
        for j in range(n):
            e = Decimal(j) / n if per_axis else Decimal(i) / P
            turns = Decimal(scale) * Decimal(10000) ** -e / (2 * PI)
            for s in range(0, S):
                # (f64 finds the small rests, 60 digits then give their value)
                t = float(turns) * (first + s)
                if abs(t - round(t)) > 2.0 ** -7:
                    continue
                exact = turns * (first + s)
                want = _sin((exact - exact.to_integral_value()) * 2 * PI)
                assert abs(Decimal(y[s, 2 * i + 1].item()) - want) < Decimal("4e-8"), (i, s)
                seen += 1
                if seen % 40 == 0:
                    break
            i += 1
    assert seen > 100


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("mode,per_axis", [(0, True), (2, True), (2, False)])
def test_heads_of_72(dt, mode, per_axis):
    """Forward and gradient, every pair turning, of contiguous tensors and of views of one projection."""
    from gguf_train_b200 import rope_axes

    B, H, S, D, sections = 2, 4, 37, 72, (18, 18)
    g = torch.Generator().manual_seed(11)
    buf = torch.randn((B, S, 3 * H, D), generator=g).to("cuda", dt)
    pos = positions(2, B, S, 60, 12)
    for view in (False, True):
        q, k = (buf[:, :, i * H:(i + 1) * H].transpose(1, 2) for i in (0, 1))
        q, k = (t if view else t.contiguous() for t in (q, k))
        q, k = (t.detach().requires_grad_() for t in (q, k))
        yq, yk = rope_axes(q, pos, sections, k=k, mode=mode, per_axis=per_axis)
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (yq.detach(), yk.detach()))
        for t, y, d in ((q, yq, dq), (k, yk, dk)):
            check(y, *reference(t, pos, sections, mode, per_axis=per_axis), dt)
            check(d, *reference(y, pos, sections, mode, per_axis=per_axis, sign=-1.0), dt)
