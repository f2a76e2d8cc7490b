"""The rotation's frequency table is kept from call to call; a call's own arguments are checked all the same."""

from __future__ import annotations

import ctypes


def _call(sections, base, scale, D):
    from gguf_train_b200 import _C

    t = _C.Tensor4(None, (0, 2, 5, D), (0, 0, D, 1), _C.GT_F32)
    arr = (ctypes.c_int32 * max(1, len(sections)))(*sections)
    ref = ctypes.byref(t)
    return _C.lib.gtb_rope_axes(ref, ref, None, None, None, 5, 0, arr, len(sections), 2, 0, base, scale, 0, None)


def test_a_call_without_axes_is_refused_first_and_after_refusals():
    from gguf_train_b200 import _C

    for _ in range(2):
        assert _call((), 0.0, 0.0, 0) == -1
        assert b"1 to 4 sections" in _C.lib.gtb_last_error()
        assert _call((4,), -1.0, 1.0, 16) == -1
        assert b"freq_base" in _C.lib.gtb_last_error()


def test_a_refused_call_is_refused_again():
    from gguf_train_b200 import _C

    assert _call((4, 4), 1e4, 1.0, 16) == 0
    for _ in range(2):
        assert _call((4, 5), 1e4, 1.0, 16) == -1
        assert b"half the head dimension" in _C.lib.gtb_last_error()
    assert _call((4, 4), 1e4, 1.0, 16) == 0
