"""Derivatives of the rotations beyond the first reverse pass: forward mode is refused (never dropped), and the gradient
is itself differentiable.

Tolerance of the second derivatives (f32): each rotation is right to 6e-7 (|x0| + |x1|) and each product to 2^-24; the
expressions chain three rotations of numbers below 10 with products below 600 (6 y Lw): 600 * 2 * 4e-6 = 5e-3."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def dense(f, shape):
    """The matrix of a linear map on tensors of `shape`, in 64 bits (columns from unit tensors)."""
    n = torch.Size(shape).numel()
    eye = torch.eye(n, device="cuda").reshape(n, *shape)
    return torch.stack([f(e).double().reshape(-1) for e in eye], 1)


def maps():
    from gguf_train_b200 import rope, rope_axes

    pos = torch.tensor([[0, 3, 7], [5, 1, 90]], dtype=torch.int32, device="cuda")
    one = torch.tensor([0, 4, 33], dtype=torch.int32, device="cuda")
    return {
        "rope_axes": lambda x: rope_axes(x, pos, (2, 4)),
        "rope_axes interleaved": lambda x: rope_axes(x, pos, (4, 4), mode=0, interleaved=True),
        "rope": lambda x: rope(x, one, mode=2),
    }


@pytest.mark.parametrize("which", ["rope_axes", "rope_axes interleaved", "rope"])
def test_second_derivative(which):
    """f = sum(y^3) + sum(x^2), y = L x: the gradient is L^T 3 y^2 + 2 x, its derivative along w L^T (6 y (L w)) + 2 w."""
    f = maps()[which]
    shape = (1, 2, 3, 16)
    L = dense(f, shape)
    x, w = (torch.randn(shape, device="cuda", generator=gen(s)) for s in (1, 2))
    x.requires_grad_()
    y = f(x)
    (g,) = torch.autograd.grad((y ** 3).sum() + (x ** 2).sum(), x, create_graph=True)
    (h,) = torch.autograd.grad((g * w).sum(), x)
    xd, wd = x.detach().double().reshape(-1), w.double().reshape(-1)
    want_g = L.T @ (3 * (L @ xd) ** 2) + 2 * xd
    want_h = L.T @ (6 * (L @ xd) * (L @ wd)) + 2 * wd
    assert (g.detach().double().reshape(-1) - want_g).abs().max() < 5e-3
    assert (h.double().reshape(-1) - want_h).abs().max() < 5e-3


def test_second_derivative_of_q_and_k_together():
    from gguf_train_b200 import rope_axes

    pos = torch.tensor([[0, 3, 7], [5, 1, 90]], dtype=torch.int32, device="cuda")
    q, k = (torch.randn((1, n, 3, 16), device="cuda", generator=gen(3 + n)).requires_grad_() for n in (2, 1))
    yq, yk = rope_axes(q, pos, (2, 4), k=k)
    # s = sum of every product of a rotated q value and the rotated k value of its token and dimension, cubed
    gq, gk = torch.autograd.grad(((yq * yk) ** 2).sum(), (q, k), create_graph=True)
    hq, hk = torch.autograd.grad((gq ** 2).sum() + (gk ** 2).sum(), (q, k))
    Lq, Lk = (dense(lambda x: rope_axes(x, pos, (2, 4)), (1, n, 3, 16)) for n in (2, 1))
    qd, kd = (t.detach().double().requires_grad_() for t in (q, k))
    rot = lambda L, t: (L @ t.reshape(-1)).view(t.shape)  # noqa: E731
    wq, wk = torch.autograd.grad(((rot(Lq, qd) * rot(Lk, kd)) ** 2).sum(), (qd, kd), create_graph=True)
    vq, vk = torch.autograd.grad((wq ** 2).sum() + (wk ** 2).sum(), (qd, kd))
    for got, want in ((gq, wq), (gk, wk), (hq, vq), (hk, vk)):
        assert (got.detach().double() - want.detach()).abs().max() <= 2e-5 * want.detach().abs().max()


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    from gguf_train_b200 import rope, rope_axes

    x, t = (torch.randn((1, 2, 3, 16), device="cuda", generator=gen(s)) for s in (7, 8))
    pos = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        d = fwad.make_dual(x, t)
        for call in (lambda: rope_axes(d, pos, (4, 4)), lambda: rope_axes(x, pos, (4, 4), k=d), lambda: rope(d, pos[0])):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        assert rope_axes(x, pos, (4, 4)).shape == x.shape  # nothing dual: as ever
