"""Expanded latent attention and its gradients against the formulas in 64 bits.

Tolerances, with u = eps / 2 of the type: weights w and score gradients ds enter their products rounded once (u of themselves, in f16
at least 2^-25), every result is rounded once, f32 sums of n terms are off by at most n 2^-22 of the sum of magnitudes (two
roundings a term, where the tensor cores cut off a whole step each). An error e of the scores is one of 2 e in the weights.
    out:  u |out| + (u + 2 e) sum w |v|                                              =: t_out
    ds = w (g . v - g . out):  (u + 2 e) |ds| + w (e' + sum |g| t_out),  e' that of the product g . v
    dv:   u |dv| + sum (u + 2 e) w |g|;   dq, dk, dk_rope:  u of themselves + scale sum |error of ds| |other operand|
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _inputs(B, H, Hkv, L, S, Dn, Dr, Dv, dt, seed, lens=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen).to(dt)  # noqa: E731
    q = r(B, L, H, Dn + Dr).transpose(1, 2)
    kv = r(B, S, Hkv, Dn + Dv)
    k, v, kr, g = kv[..., :Dn].transpose(1, 2), kv[..., Dn:].transpose(1, 2), r(B, S, Dr), r(B, H, L, Dv)
    if lens is not None:  # padded tokens hold anything
        pad = torch.arange(S, device="cuda") >= lens[:, None]
        q, k, v, g = (t.masked_fill(pad[:, None, :, None], float("nan")) for t in (q, k, v, g))
        kr = kr.masked_fill(pad[..., None], float("nan"))
    return [t.detach().requires_grad_() for t in (q, k, kr, v)], g


def _exact(q, k, kr, v, g, causal, scale, lens):
    """(value, tolerance) of out, dq, dk, dk_rope, dv."""
    dt, u = q.dtype, torch.finfo(q.dtype).eps / 2
    low = 2.0 ** -25 if dt == torch.float16 else 0.0
    B, H, L, D = q.shape
    Hkv, S, Dn = k.shape[1:]
    G = H // Hkv
    q, k, kr, v, g = (t.detach().double() for t in (q, k, kr, v, g))
    if lens is not None:
        pad = (torch.arange(S, device="cuda") >= lens[:, None])
        q, k, v, g = (t.masked_fill(pad[:, None, :, None], 0.0) for t in (q, k, v, g))
        kr = kr.masked_fill(pad[..., None], 0.0)
    keys = torch.cat((k, kr[:, None].expand(-1, Hkv, -1, -1)), -1).repeat_interleave(G, 1)
    vals = v.repeat_interleave(G, 1)
    x = q @ keys.transpose(2, 3) * scale
    drop = torch.zeros((L, S), dtype=torch.bool, device="cuda")
    if causal:
        drop = torch.arange(S, device="cuda")[None] > torch.arange(L, device="cuda")[:, None]
    drop = drop.expand(B, 1, L, S)
    if lens is not None:
        drop = drop | pad[:, None, None, :] | pad[:, None, :, None]
    x = x.masked_fill(drop, float("-inf"))
    z = torch.logsumexp(x, -1, keepdim=True)
    w = torch.exp(x - z).masked_fill(torch.isinf(z), 0.0)
    out = w @ vals
    n = 2.0 ** -22
    e = D * n * scale * (q.abs() @ keys.abs().transpose(2, 3)).amax()
    wt = (u + 2 * e + S * n) * w + low * w.amax(-1, keepdim=True)
    t_out = u * out.abs() + wt @ vals.abs()
    ds = w * (g @ vals.transpose(2, 3) - (g * out).sum(-1, keepdim=True))
    e2 = v.shape[-1] * n * (g.abs() @ vals.abs().transpose(2, 3))
    t_ds = (u + 2 * e) * ds.abs() + w * (e2 + (g.abs() * (t_out + v.shape[-1] * n * out.abs())).sum(-1, keepdim=True)) + low
    group = lambda t: t.view(B, Hkv, G, *t.shape[2:]).sum(2)  # noqa: E731
    dq, dk, dv = scale * ds @ keys, group(scale * ds.transpose(2, 3) @ q), group(w.transpose(2, 3) @ g)
    t_dq = u * dq.abs() + scale * t_ds @ keys.abs() + S * n * scale * ds.abs() @ keys.abs()
    t_dk = group(scale * t_ds.transpose(2, 3) @ q.abs() + L * n * scale * ds.abs().transpose(2, 3) @ q.abs())
    t_dv = u * dv.abs() + group((wt + L * n * w).transpose(2, 3) @ g.abs())
    dkr, t_dkr = dk[..., Dn:].sum(1), t_dk[..., Dn:].sum(1)
    tiny = torch.finfo(dt).tiny * 2 * u if dt != torch.float32 else 1e-30
    return [(out, t_out + tiny), (dq, t_dq + tiny), (dk[..., :Dn], u * dk[..., :Dn].abs() + t_dk[..., :Dn] + tiny),
            (dkr, u * dkr.abs() + t_dkr + tiny), (dv, t_dv + tiny)]


CASES = [
    # B, H, Hkv, L, S, Dn, Dr, Dv
    (1, 1, 1, 1, 1, 128, 64, 128),
    (2, 3, 3, 70, 70, 128, 64, 128),
    (1, 2, 2, 128, 128, 64, 32, 64),
    (2, 2, 2, 129, 129, 64, 64, 64),
    (1, 4, 2, 65, 65, 128, 32, 128),
    (1, 2, 2, 300, 300, 128, 64, 128),
    (3, 1, 1, 517, 517, 64, 32, 64),
    (1, 3, 3, 1, 200, 128, 64, 128),
    (2, 1, 1, 200, 1, 64, 32, 64),
    (1, 2, 1, 130, 390, 128, 48, 128),
    (1, 2, 2, 390, 130, 128, 16, 128),
    (1, 2, 2, 257, 64, 64, 16, 64),
    # sizes the tensor-core kernels do not take
    (1, 2, 2, 40, 40, 96, 32, 64),
    (1, 2, 2, 33, 50, 48, 16, 80),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_gradients(case, dtype, causal, padded):
    from gguf_train_b200 import _C, latent_sdpa

    B, H, Hkv, L, S, Dn, Dr, Dv = case
    if padded and L != S:
        pytest.skip("lengths go with as many queries as keys")
    lens = None
    if padded:
        lens = torch.tensor([(S * (b + 1) // (B + 1)) if b else S - S // 3 for b in range(B)], dtype=torch.int32, device="cuda")
        lens[-1] = 0 if B > 1 else lens[-1]
    leaves, g = _inputs(B, H, Hkv, L, S, Dn, Dr, Dv, TYPES[dtype], L + S, lens)
    scale = 1.0 / math.sqrt(Dn + Dr)
    out = latent_sdpa(*leaves, is_causal=causal, seq_lens=lens)
    assert out.dtype == leaves[0].dtype and out.shape == (B, H, L, Dv)
    grads = torch.autograd.grad(out, leaves, g)
    assert _C.device_status() == 0
    got = [out.detach(), *grads]
    for name, x, (want, tol) in zip(("out", "dq", "dk", "dk_rope", "dv"), got, _exact(*leaves, g, causal, scale, lens)):
        assert x.dtype == leaves[0].dtype and x.shape == want.shape
        far = float(((x.double() - want).abs() / tol).max())
        assert far <= 1.0, f"{name}: {far:.3g} of the tolerance"
    again = latent_sdpa(*leaves, is_causal=causal, seq_lens=lens)
    assert all(torch.equal(a, b) for a, b in zip(got, [again.detach(), *torch.autograd.grad(again, leaves, g)])) or \
        dtype == "f32" or (Dn, Dv) not in ((128, 128), (64, 64))


def test_gradients_against_differences():
    """Central differences of sum(out * g) in random directions, f32 (whose kernels are those of the general path) and bf16
    against the f32 gradients."""
    from gguf_train_b200 import latent_sdpa

    leaves, g = _inputs(1, 2, 2, 40, 40, 64, 32, 64, torch.float32, 11)
    grads = torch.autograd.grad(latent_sdpa(*leaves, is_causal=True), leaves, g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    f = lambda xs: float((latent_sdpa(*xs, is_causal=True).double() * g.double()).sum())  # noqa: E731
    with torch.no_grad():
        for i, d in enumerate(grads):
            t = torch.randn(d.shape, device="cuda", generator=gen)
            t /= t.norm()
            h = 2.0 ** -5
            xs = [[x + s * h * t if j == i else x for j, x in enumerate(leaves)] for s in (1, -1)]
            num, ana = (f(xs[0]) - f(xs[1])) / (2 * h), float((d.double() * t.double()).sum())
            # the third derivative's part is h^2 / 6 of it (scores move by less than h), f32's rounding 2^-24 |out||g| / h
            assert abs(num - ana) <= h * h * float(d.norm()) + 2.0 ** -24 * 50 / h * math.sqrt(g.numel())
    low = [x.detach().bfloat16().requires_grad_() for x in leaves]
    high = [x.detach().float().requires_grad_() for x in low]
    lg = torch.autograd.grad(latent_sdpa(*low, is_causal=True), low, g.bfloat16())
    hg = torch.autograd.grad(latent_sdpa(*high, is_causal=True), high, g.bfloat16().float())
    for a, b in zip(lg, hg):
        assert float((a.float() - b).norm()) <= 4 * 2.0 ** -8 * float(b.norm())


def test_scale_and_parts():
    """Only some inputs require gradients; a given scale; no gradient asked for."""
    from gguf_train_b200 import latent_sdpa

    leaves, g = _inputs(1, 2, 2, 70, 70, 64, 32, 64, torch.bfloat16, 5)
    full = torch.autograd.grad(latent_sdpa(*leaves, scale=0.3), leaves, g)
    for i in range(4):
        xs = [x.detach().requires_grad_(j == i) for j, x in enumerate(leaves)]
        (one,) = torch.autograd.grad(latent_sdpa(*xs, scale=0.3), xs[i], g)
        assert torch.equal(one, full[i])
    with torch.no_grad():
        assert not latent_sdpa(*leaves, scale=0.3).requires_grad


def test_refusals():
    from gguf_train_b200 import latent_sdpa

    (q, k, kr, v), _ = _inputs(2, 4, 4, 20, 20, 64, 32, 64, torch.bfloat16, 1)
    lens = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    for bad, match in [(lambda: latent_sdpa(q, k, kr[:1], v), "do not"), (lambda: latent_sdpa(q[..., :64], k, kr, v), "do not"),
                       (lambda: latent_sdpa(q, k[:, :3], kr, v[:, :3]), "divisible"),
                       (lambda: latent_sdpa(q, k.half(), kr, v), "one type"),
                       (lambda: latent_sdpa(q.double(), k.double(), kr.double(), v.double()), "one type"),
                       (lambda: latent_sdpa(q, k, kr, v, scale=-1.0), "scale"),
                       (lambda: latent_sdpa(q, k, kr, v, scale=float("nan")), "scale"),
                       (lambda: latent_sdpa(q[:, :, :10], k, kr, v, seq_lens=lens), "as many queries"),
                       (lambda: latent_sdpa(q, k, kr, v, seq_lens=lens.long()), "int32"),
                       (lambda: latent_sdpa(q, k, kr, v, seq_lens=lens[:1]), "int32"),
                       (lambda: latent_sdpa(q, k, kr[:, None], v), "dimensions")]:
        with pytest.raises(RuntimeError, match=match):
            bad()


def test_second_derivatives_are_refused():
    from gguf_train_b200 import latent_sdpa

    leaves, g = _inputs(1, 1, 1, 20, 20, 64, 32, 64, torch.bfloat16, 1)
    (dq,) = torch.autograd.grad(latent_sdpa(*leaves), leaves[0], g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), leaves[1])


def test_gradients_of_other_shapes_and_places():
    """A broadcast output gradient, a rotary key shared by the batch, and saved tensors kept on the host in between."""
    from gguf_train_b200 import latent_sdpa

    leaves, g = _inputs(3, 2, 2, 90, 90, 64, 32, 64, torch.bfloat16, 21)
    one = leaves[2].detach()[:1].clone().requires_grad_()
    out = latent_sdpa(leaves[0], leaves[1], one.expand(3, -1, -1), leaves[3], is_causal=True)
    grads = torch.autograd.grad(out.sum(), (leaves[0], one))
    full = one.detach().expand(3, -1, -1).contiguous().requires_grad_()
    xs = (leaves[0], leaves[1], full, leaves[3])
    want = torch.autograd.grad(latent_sdpa(*xs, is_causal=True), (leaves[0], full), torch.ones_like(g))
    assert torch.equal(grads[0], want[0])
    assert torch.equal(grads[1], want[1].sum(0, keepdim=True))
    want = torch.autograd.grad(latent_sdpa(*leaves, is_causal=True), leaves, g)
    with torch.autograd.graph.save_on_cpu():
        out = latent_sdpa(*leaves, is_causal=True)
    junk = [torch.randn_like(x) for x in leaves for _ in range(4)]  # takes what the saved tensors gave back
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g), want)) and junk
    # inputs that had to be copied to start on 16 bytes
    odd = [torch.randn((*x.shape[:-1], x.shape[-1] + 3), device="cuda").to(torch.bfloat16)[..., 3:].requires_grad_() for x in leaves]
    even = [x.detach().contiguous().requires_grad_() for x in odd]
    with torch.autograd.graph.save_on_cpu():
        a = latent_sdpa(*odd)
    for x, y in zip(torch.autograd.grad(a, odd, g), torch.autograd.grad(latent_sdpa(*even), even, g)):
        assert torch.equal(x, y)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw

    from gguf_train_b200 import latent_sdpa

    leaves, _ = _inputs(1, 1, 1, 20, 20, 64, 32, 64, torch.bfloat16, 1)
    xs = [x.detach() for x in leaves]
    with fw.dual_level(), pytest.raises(Exception):
        latent_sdpa(fw.make_dual(xs[0], torch.ones_like(xs[0])), *xs[1:])


@pytest.mark.parametrize("shape", [(0, 2, 5, 5), (2, 2, 0, 0), (1, 2, 0, 7)])
def test_nothing_to_compute(shape):
    from gguf_train_b200 import latent_sdpa

    B, H, L, S = shape
    r = lambda *s: torch.randn(s, device="cuda").to(torch.bfloat16)  # noqa: E731
    out = latent_sdpa(r(B, H, L, 96), r(B, H, S, 64), r(B, S, 32), r(B, H, S, 64))
    assert out.shape == (B, H, L, 64)
