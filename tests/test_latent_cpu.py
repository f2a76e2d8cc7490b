"""Latent attention without a GPU: refusals of CPU tensors, and the C entries' checks of sizes and options, which come before
any device work."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch


def _native(**kw):
    from gguf_train_b200 import _C

    f = dict(B=0, Smax=8, R=128, Dr=32, dtype=_C.GT_BF16)
    f.update(kw)
    return _C.Latent(None, None, *(f[n] for n in ("B", "Smax", "R", "Dr", "dtype")))


def _t4(shape, dtype, stride=None):
    from gguf_train_b200 import _C

    if stride is None:
        stride, n = [], 1
        for s in reversed(shape):
            stride.insert(0, n)
            n *= s
    return _C.Tensor4(None, tuple(shape), tuple(stride), dtype)


def _append(c, n=3, dtype=0, mode=2, base=10000.0, **kw):
    from gguf_train_b200 import _C

    x, k = _t4(kw.get("latent", (c.B, 1, n, c.R)), dtype), _t4(kw.get("k_rope", (c.B, 1, n, c.Dr)), kw.get("ktype", dtype))
    return _C.lib.gtb_latent_append(ctypes.byref(c), ctypes.byref(x), ctypes.byref(k), None, None, mode, base, 1.0, 0, None)


def _attend(c, H=4, Lq=2, scale=0.1, prefix=None, **kw):
    from gguf_train_b200 import _C

    q = _t4(kw.get("q", (c.B, H, Lq, c.R + c.Dr)), kw.get("qtype", c.dtype))
    o = _t4(kw.get("out", (c.B, H, Lq, c.R)), kw.get("otype", c.dtype))
    return _C.lib.gtb_latent_attention(ctypes.byref(q), ctypes.byref(c), None if prefix is None else ctypes.byref(prefix), scale,
                                       None, ctypes.byref(o), None, None)


def _refused(rc, match):
    from gguf_train_b200 import _C

    msg = _C.lib.gtb_last_error().decode()
    assert rc == -1 and re.search(match, msg), msg


def test_cpu_tensors_are_refused():
    from gguf_train_b200 import LatentCache, latent_sdpa

    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        LatentCache(torch.zeros((1, 4, 96), dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), 64)
    x = torch.zeros((1, 2, 4, 96))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        latent_sdpa(x, x[..., :64], x[:, 0, :, 64:], x[..., :64])


@pytest.mark.parametrize("change,match", [
    (dict(R=96), "multiple of 64"), (dict(R=576), "multiple of 64"), (dict(R=0), "multiple of 64"),
    (dict(Dr=24), "multiple of 16"), (dict(Dr=80), "multiple of 16"), (dict(Dr=0), "multiple of 16"),
    (dict(Smax=1 << 30), "2\\^30"), (dict(B=-1), "negative"), (dict(Smax=-1), "negative"), (dict(B=1 << 31), "int32"),
    (dict(dtype=0), "f16 or bf16"), (dict(dtype=108), "f16 or bf16"),
])
def test_cache_checks(change, match):
    bad = _native(**change)
    _refused(_append(bad), match)
    _refused(_attend(bad), match)


def test_append_checks():
    from gguf_train_b200 import _C

    c = _native()
    _refused(_append(c, latent=(0, 1, 3, 64)), r"latent must be \(0, 1, n, 128\)")
    _refused(_append(c, k_rope=(0, 1, 2, 32)), "latent must be")
    _refused(_append(c, latent=(0, 2, 3, 128)), "latent must be")
    _refused(_append(c, ktype=_C.GT_F16), "of one type")
    _refused(_append(c, dtype=_C.GT_F64), "of one type")
    _refused(_append(c, mode=1), "rope_mode")
    _refused(_append(c, base=0.0), "freq_base")
    _refused(_append(c, base=float("nan")), "freq_base")
    assert _append(c) == 0 and _append(c, mode=-1, base=0.0) == 0 and _append(c, n=0) == 0


def test_attention_checks():
    from gguf_train_b200 import _C

    c = _native()
    _refused(_attend(c, q=(0, 4, 2, 128)), r"q must be \(0, H, Lq, 160\)")
    _refused(_attend(c, qtype=_C.GT_F16), "of the cache's type")
    _refused(_attend(c, out=(0, 4, 2, 160)), "out must be")
    _refused(_attend(c, otype=_C.GT_F32), "out must be")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _refused(_attend(c, scale=scale), "scale must be positive")
    _refused(_attend(c, H=1 << 16, Lq=1 << 26), "too many query rows")
    # (the prefix's own sizes are checked before its pointers)
    for change in (dict(R=64), dict(Dr=16), dict(dtype=_C.GT_F16), dict(B=0)):
        _refused(_attend(c, prefix=_native(**change)), "prefix must be")
    assert _attend(c) == 0 and _attend(_native(B=0), H=0) == 0
