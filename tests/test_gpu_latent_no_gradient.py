"""The serving calls have no gradient: tensors that require one, or carry a tangent, are refused instead of giving results that silently
have none."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

bf = dict(dtype=torch.bfloat16, device="cuda")


def _cache(batch=2, rows=9):
    from gguf_train_b200 import LatentCache

    return LatentCache(torch.randn((batch, rows, 96), **bf), torch.full((batch,), 5, dtype=torch.int32, device="cuda"), 64)


def _calls():
    """name -> (call of one tensor, that tensor)"""
    from gguf_train_b200 import latent_append, latent_attention

    cache, prefix = _cache(), _cache(1)
    q, c, k = torch.randn((2, 4, 1, 96), **bf), torch.randn((2, 1, 64), **bf), torch.randn((2, 1, 32), **bf)

    def rows(t):
        held = _cache()
        held.rows = t
        return latent_attention(q, held, 0.1)

    def prefix_rows(t):
        prefix.rows = t
        return latent_attention(q, cache, 0.1, prefix=prefix)

    def append_rows(t):
        held = _cache()
        held.rows = t
        return latent_append(held, c, k)

    return {"q": (lambda t: latent_attention(t, cache, 0.1), q), "rows": (rows, cache.rows), "prefix": (prefix_rows, prefix.rows),
            "latent": (lambda t: latent_append(cache, t, k, advance=False), c),
            "k_rope": (lambda t: latent_append(cache, c, t, advance=False, rope=dict(mode=2)), k), "append rows": (append_rows, cache.rows)}


@pytest.mark.parametrize("name", ["q", "rows", "prefix", "latent", "k_rope", "append rows"])
def test_tensors_that_require_a_gradient_are_refused(name):
    call, x = _calls()[name]
    leaf = x.detach().clone().requires_grad_()
    for t in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(t)
        with torch.no_grad():
            call(t)
        with torch.inference_mode():
            call(t)
        call(t.detach())


@pytest.mark.parametrize("name", ["q", "rows", "prefix", "latent", "k_rope", "append rows"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
    import torch.autograd.forward_ad as fw

    call, x = _calls()[name]
    with fw.dual_level(), torch.set_grad_enabled(grad):
        call(x)  # (one without a tangent is taken)
        with pytest.raises(RuntimeError, match="no gradient"):
            call(fw.make_dual(x, torch.ones_like(x)))
