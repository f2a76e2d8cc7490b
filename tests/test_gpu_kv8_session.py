"""The example session (examples/kv8_session.py) end to end: with nothing evicted the new tokens' outputs are as near to
16-bit attention as 8-bit keys and values allow (relative steps of 4.5 / 127 / sqrt(12) = 1 % of a value for
int8, 2^-4 / sqrt(3) = 3.6 % for e4m3, in keys and in values; scores add about as much again), and evictions in the
middle of decoding leave the outputs finite and close to those of the whole cache."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv8_session.py")


def _session():
    spec = importlib.util.spec_from_file_location("kv8_session", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("e4m3", [False, True])
def test_whole_cache_follows_16_bit_attention(e4m3):
    err = _session().run(batch=2, text=40, rows=6, cols=10, new=20, budget=100, recent=10, capacity=128, e4m3=e4m3, quiet=True)
    assert err < (0.12 if e4m3 else 0.04)


def test_eviction_while_decoding():
    from gguf_train_b200 import _C

    err = _session().run(batch=2, text=60, rows=8, cols=16, new=60, budget=120, recent=30, capacity=144, quiet=True)
    assert math.isfinite(err) and err < 1.0
    assert _C.device_status() == 0
