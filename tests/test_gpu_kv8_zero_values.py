"""Values that are all zero (their blocks' scales are 0) over more cached tokens than 2^20: every score is 0 here, so the
log-sum-exp is ln n and every weight is 1 / n.

Tolerance: a sum of n equal terms in f32, put together from parts of at most 16384 terms a lane and 8192 parts:
relative 24576 * 2^-24 = 1.5e-3 at most, which is also the absolute error of the logarithm."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,H,Lq", [(torch.bfloat16, 1, 1), (torch.float32, 4, 1), (torch.float16, 1, 80)],
                         ids=["bf16 one row", "f32 four rows", "f16 chunk"])
@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
def test_log_sum_exp_and_weights_over_zero_values(fmt, dt, H, Lq):
    from gguf_train_b200 import KV8Cache, _C, kv8_attention

    n = 1_200_000
    cache = KV8Cache.empty(1, 1, n, 16, 64, fmt)
    cache.k.view(torch.uint8).fill_(0x30)
    cache.k_scale.fill_(0.01)
    cache.v.view(torch.uint8).zero_()
    cache.v_scale.zero_()
    cache.lens.fill_(n)
    q = torch.zeros((1, H, Lq, 16), dtype=dt, device="cuda")
    score = torch.zeros((1, 1, n), device="cuda")
    out, lse = kv8_attention(q, cache, score=score, need_lse=True)
    assert (out == 0).all()
    want = torch.log(torch.arange(n - Lq + 1, n + 1, device="cuda", dtype=torch.float64))
    assert ((lse.double() - want).abs() <= 1.5e-3).all()
    # keys before the queries are seen by every row
    weight = H * (1.0 / torch.arange(n - Lq + 1, n + 1, device="cuda", dtype=torch.float64)).sum()
    assert ((score[0, 0, :n - Lq].double() / weight - 1).abs() <= 3e-3).all()
    assert _C.device_status() == 0
