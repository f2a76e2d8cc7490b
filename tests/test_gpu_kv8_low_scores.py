"""Scores far below zero: what counts is the differences between them, however low all of them lie.

All keys are alike and the values differ, so every weight is 1 / n and the output is the mean of the values; the
log-sum-exp is the score itself, since ln n is below its last bit. Tolerance: weights to 2^-10.5 (f16), the output's
rounding, and 2^-20 of the score for its sums and products."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [1e3, 1e34, 1e37])
@pytest.mark.parametrize("Lq,cap", [(1, 100), (1, 5000), (5, 5000), (40, 300), (80, 300)])
def test_rows_of_low_scores(fmt, dt, size, Lq, cap):
    from gguf_train_b200 import KV8Cache, _C, kv8_attention

    D, n = 64, cap - 1
    g = torch.Generator("cuda").manual_seed(81)
    cache = KV8Cache.empty(1, 1, cap, D, 32, fmt)
    cache.k.copy_(torch.full(cache.k.shape, 64.0, device="cuda").to(fmt))
    cache.k_scale.fill_(2.0 ** -6)  # every key value 1
    v = torch.randint(-8, 9, cache.v.shape, device="cuda", generator=g).float() * 8
    cache.v.copy_(v.to(fmt))
    cache.v_scale.fill_(2.0 ** -6)
    cache.lens.fill_(n)
    q = torch.full((1, 1, Lq, D), -size, device="cuda").to(dt)
    out, lse = kv8_attention(q, cache, scale=2.0 ** -3, need_lse=True)
    s = (q.double().sum(-1) * 2.0 ** -3)
    assert ((lse.double() - s).abs() <= 2.0 ** -20 * s.abs() + 10.0).all()
    vals = v[0, 0].double() * 2.0 ** -6
    for i in range(Lq):
        seen = n - Lq + 1 + i
        want = vals[:seen].mean(0)
        tol = (2.0 ** -10 + 2.0 ** -8) * vals[:seen].abs().mean(0)
        assert ((out[0, 0, i].double() - want).abs() <= tol).all(), i
    assert _C.device_status() == 0
