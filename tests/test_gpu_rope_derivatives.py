"""Derivatives of the rotations beyond the first reverse pass: forward mode is refused (never dropped)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


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
