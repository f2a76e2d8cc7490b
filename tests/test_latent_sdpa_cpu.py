"""The C entries of the expanded form without a GPU: sizes and results that are checked before any device work."""

from __future__ import annotations

import ctypes
import re

import pytest


def _t4(*shape):
    from gguf_train_b200 import _C

    stride = [1, 1, 1, 1]
    for i in (2, 1, 0):
        stride[i] = stride[i + 1] * max(shape[i + 1], 1)
    return _C.Tensor4(None, tuple(shape), tuple(stride), _C.GT_BF16)


def _backward(B, H, Hkv, L, S, Dn=64, Dr=32):
    from gguf_train_b200 import _C

    q, k, r, v, o = _t4(B, H, L, Dn + Dr), _t4(B, Hkv, S, Dn), _t4(B, 1, S, Dr), _t4(B, Hkv, S, Dn), _t4(B, H, L, Dn)
    p = ctypes.byref
    return _C.lib.gtb_latent_sdpa_bwd(p(o), p(q), p(k), p(r), p(v), p(o), None, None, 0.1, 0, p(q), p(k), p(r), p(v), None)


def _forward(B, H, Hkv, L, S, Dn=64, Dr=32):
    from gguf_train_b200 import _C

    q, k, r, v, o = _t4(B, H, L, Dn + Dr), _t4(B, Hkv, S, Dn), _t4(B, 1, S, Dr), _t4(B, Hkv, S, Dn), _t4(B, H, L, Dn)
    p = ctypes.byref
    return _C.lib.gtb_latent_sdpa_fwd(p(q), p(k), p(r), p(v), None, 0.1, 0, p(o), None, None)


@pytest.mark.parametrize("B,H,Hkv,L,S", [(2, 0, 3, 5, 5), (2, 0, 0, 5, 5), (2, 0, 3, 0, 5), (1, 2, 2, 0, 7)])
def test_a_backward_that_would_leave_gradients_unwritten_is_refused(B, H, Hkv, L, S):
    """No query anywhere, but keys whose gradients have values."""
    from gguf_train_b200 import _C

    assert _backward(B, H, Hkv, L, S) == -1
    assert re.search("there must be heads, queries and keys|there must be queries and keys", _C.lib.gtb_last_error().decode())


@pytest.mark.parametrize("B,H,Hkv,L,S", [(0, 2, 2, 5, 5), (0, 0, 0, 0, 0), (2, 2, 2, 0, 0), (2, 0, 3, 5, 0), (2, 0, 0, 0, 0)])
def test_nothing_to_write(B, H, Hkv, L, S):
    assert _backward(B, H, Hkv, L, S) == 0
    assert _forward(B, H, Hkv, L, S) == 0


def test_a_forward_without_heads_has_nothing_to_write():
    assert _forward(2, 0, 3, 5, 5) == 0
