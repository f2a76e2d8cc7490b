"""Calls of an empty batch with scores do nothing and need no device."""

from __future__ import annotations

import ctypes


def test_an_empty_batch_with_scores():
    from gguf_train_b200 import _C

    c = _C.KV8(None, None, None, None, None, 0, 2, 8, 32, 16, 0)
    t = _C.Tensor4(None, (0, 2, 1, 32), (0, 0, 32, 1), _C.GT_F32)
    a, b = ctypes.c_void_p(64), ctypes.c_void_p(128)
    for out in (a, b):
        rc = _C.lib.gtb_kv8_attention(ctypes.byref(t), ctypes.byref(c), 0.0, None, a, out, ctypes.byref(t), None, None)
        assert rc == 0, _C.lib.gtb_last_error()
