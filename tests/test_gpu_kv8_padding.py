"""Query rows past counts[b] are padding: whatever they hold (NaN, infinities, numbers whose scores overflow), the
outputs, the log-sum-exp and the accumulated weights are those of a call whose padding is zero, to the bit (a padded
row has weight 0 in every sum, and adding 0 changes no sum)."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_kv8 import FMTS, gen, random_cache

pytestmark = pytest.mark.gpu

SHAPES = [
    # B, H, Hkv, Lq, D, cap, block, lens, counts: rows per kv head on both sides of where kept scores end
    (2, 4, 1, 8, 128, 500, 64, [500, 77], [5, 7]),
    (2, 4, 1, 20, 128, 500, 64, [500, 77], [11, 17]),
    (2, 2, 1, 13, 256, 300, 32, [300, 40], [5, 12]),
    (2, 8, 2, 140, 64, 700, 32, [700, 300], [77, 139]),
    (3, 3, 1, 70, 80, 400, 16, [400, 64, 30], [0, 1, 69]),   # the last has fewer rows cached than queries
]


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dt,pad", [(torch.bfloat16, math.nan), (torch.bfloat16, math.inf), (torch.bfloat16, 1e38),
                                    (torch.float16, -math.inf), (torch.float16, 65504.0), (torch.float32, math.nan),
                                    (torch.float32, -3e38)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:7])))
def test_padding_reaches_no_result(fmt, dt, pad, shape):
    from gguf_train_b200 import _C, kv8_attention

    B, H, Hkv, Lq, D, cap, block, lens, counts = shape
    cache = random_cache(B, Hkv, cap, D, block, fmt, lens, 41)
    q = (torch.randn((B, H, Lq, D), device="cuda", generator=gen(42)) * 1.2).to(dt)
    past = torch.arange(Lq, device="cuda")[None] >= torch.tensor(counts, device="cuda")[:, None]
    past = past[:, None, :, None].expand_as(q)
    ct = torch.tensor(counts, dtype=torch.int32, device="cuda")
    base = torch.rand((B, Hkv, cap), device="cuda", generator=gen(43))
    res = []
    for x in (q.masked_fill(past, 0.0), q.masked_fill(past, pad)):
        score = base.clone()
        res.append((*kv8_attention(x, cache, counts=ct, score=score, need_lse=True), score))
    for want, got in zip(*res):
        assert not got.isnan().any() and torch.equal(got, want)
    assert (res[1][0][past] == 0).all() and _C.device_status() == 0
