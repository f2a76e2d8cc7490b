"""The multi-axis rotary embedding and the 8-bit cache without a GPU: refusals of CPU tensors, and the C entries'
checks of sizes and options, which come before any device work."""

from __future__ import annotations

import ctypes

import pytest
import torch


def _native(**kw):
    from gguf_train_b200 import _C

    f = dict(B=0, Hkv=2, Smax=8, D=32, block=16, format=0)
    f.update(kw)
    return _C.KV8(None, None, None, None, None, *(f[n] for n in ("B", "Hkv", "Smax", "D", "block", "format")))


def _err():
    from gguf_train_b200 import _C

    return _C.lib.gtb_last_error().decode()


def test_cpu_tensors_are_refused():
    from gguf_train_b200 import KV8Cache, rope_axes

    x = torch.zeros((1, 1, 4, 16))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rope_axes(x, torch.zeros((2, 4), dtype=torch.int32), (4, 4))
    c = torch.zeros((1, 1, 4, 16), dtype=torch.int8)
    s = torch.zeros((1, 1, 1))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        KV8Cache(c, c.clone(), s, s.clone(), torch.zeros(1, dtype=torch.int32), 16)


@pytest.mark.parametrize("change,match", [
    (dict(block=48), "16, 32, 64 or 128"), (dict(format=2), "int8 or e4m3"), (dict(D=40), "multiple of 16"),
    (dict(D=272), "multiple of 16"), (dict(Smax=1 << 30), "2\\^30"), (dict(B=-1), "negative"),
    (dict(B=1 << 20, Hkv=1 << 20), "int32"),
])
def test_cache_checks(change, match):
    import re

    from gguf_train_b200 import _C

    bad = _native(**change)
    t = _C.Tensor4(None, (0, 2, 1, 32), (0, 0, 32, 1), _C.GT_F32)
    for rc in (_C.lib.gtb_kv8_append(ctypes.byref(bad), ctypes.byref(t), ctypes.byref(t), None, 0, None),
               _C.lib.gtb_kv8_read(ctypes.byref(bad), None, ctypes.byref(t), ctypes.byref(t), None),
               _C.lib.gtb_kv8_attention(ctypes.byref(t), ctypes.byref(bad), 0.0, None, None, None, ctypes.byref(t), None, None),
               _C.lib.gtb_kv8_evict(ctypes.byref(bad), None, 4, 0, ctypes.byref(bad), None, None, None)):
        assert rc == -1 and re.search(match, _err()), _err()


def test_an_empty_batch_needs_no_device():
    from gguf_train_b200 import _C

    c = _native()
    t = _C.Tensor4(None, (0, 2, 1, 32), (0, 0, 32, 1), _C.GT_F32)
    assert _C.lib.gtb_kv8_append(ctypes.byref(c), ctypes.byref(t), ctypes.byref(t), None, 1, None) == 0, _err()
    assert _C.lib.gtb_kv8_read(ctypes.byref(c), None, ctypes.byref(t), ctypes.byref(t), None) == 0, _err()
    assert _C.lib.gtb_kv8_attention(ctypes.byref(t), ctypes.byref(c), 0.0, None, None, None, ctypes.byref(t), None, None) == 0
    assert _C.lib.gtb_kv8_evict(ctypes.byref(c), None, 4, 0, ctypes.byref(c), None, None, None) == 0, _err()


def test_call_checks():
    from gguf_train_b200 import _C

    c = _native()
    t = _C.Tensor4(None, (0, 2, 1, 32), (0, 0, 32, 1), _C.GT_F32)
    wide = _C.Tensor4(None, (0, 2, 1, 64), (0, 0, 64, 1), _C.GT_F32)
    f64 = _C.Tensor4(None, (0, 2, 1, 32), (0, 0, 32, 1), _C.GT_F64)
    ref = ctypes.byref
    assert _C.lib.gtb_kv8_append(ref(c), ref(wide), ref(wide), None, 0, None) == -1 and "n, 32" in _err()
    assert _C.lib.gtb_kv8_append(ref(c), ref(f64), ref(f64), None, 0, None) == -1 and "one type" in _err()
    assert _C.lib.gtb_kv8_append(ref(c), ref(t), None, None, 0, None) == -1
    assert _C.lib.gtb_kv8_append(None, ref(t), ref(t), None, 0, None) == -1
    assert _C.lib.gtb_kv8_read(ref(c), None, ref(wide), ref(wide), None) == -1
    odd = _C.Tensor4(None, (0, 3, 1, 32), (0, 0, 32, 1), _C.GT_F32)
    assert _C.lib.gtb_kv8_attention(ref(odd), ref(c), 0.0, None, None, None, ref(odd), None, None) == -1
    assert "divisible" in _err()
    assert _C.lib.gtb_kv8_attention(ref(t), ref(c), float("inf"), None, None, None, ref(t), None, None) == -1
    assert _C.lib.gtb_kv8_attention(ref(t), ref(c), 0.0, None, None, ctypes.c_void_p(64), ref(t), None, None) == -1
    assert "go together" in _err()
    for budget, recent, match in ((0, 0, "budget must be"), (4, 5, "budget must be"), (9, 0, "fewer than the budget")):
        assert _C.lib.gtb_kv8_evict(ref(c), None, budget, recent, ref(c), None, None, None) == -1 and match in _err()


def test_rope_axes_checks():
    from gguf_train_b200 import _C

    t = _C.Tensor4(None, (0, 2, 5, 32), (0, 0, 32, 1), _C.GT_F32)

    def call(sections, mode=2, flags=0, base=1e4, x=t, y=t, k=None, ko=None):
        arr = (ctypes.c_int32 * len(sections))(*sections)
        p = lambda z: None if z is None else ctypes.byref(z)  # noqa: E731
        return _C.lib.gtb_rope_axes(p(x), p(y), p(k), p(ko), None, 5, 0, arr, len(sections), mode, flags, base, 1.0, 0, None)

    assert call((4, 6, 6)) == 0, _err()
    assert call((4, 6, 7)) == -1 and "half the head dimension" in _err()
    assert call((4, -1)) == -1 and "negative" in _err()
    assert call((4,), mode=3) == -1 and "mode" in _err()
    assert call((4,), flags=4) == -1 and "flags" in _err()
    assert call((2, 14), flags=_C.GTB_ROPE_INTERLEAVED) == -1 and "interleaved" in _err()
    assert call((6, 5, 5), flags=_C.GTB_ROPE_INTERLEAVED) == 0, _err()
    assert call((4,), base=0.0) == -1 and "freq_base" in _err()
    assert call((1, 1, 1, 1, 1)) == -1 and "1 to 4" in _err()
    assert call((4,), k=t) == -1 and "go together" in _err()
    other = _C.Tensor4(None, (0, 2, 6, 32), (0, 0, 32, 1), _C.GT_F32)
    assert call((4,), k=other, ko=other) == -1 and "fit together" in _err()
    assert call((4,), y=other) == -1 and "out must have" in _err()
