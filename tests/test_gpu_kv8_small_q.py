"""Query rows whose values are far apart or at the end of their type. The bound is attention_reference's: sums of D exact
products in f32."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv8 import FMTS, check_attention, gen, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D,cap,Lq", [(64, 300, 1), (128, 2600, 1), (128, 700, 3), (128, 400, 70)])
def test_small_values_beside_a_large_one(fmt, dt, D, cap, Lq):
    """The large value meets zeros in every key, so the scores are sums over values 2^-12 as large, and each of those counts
    to its last bit."""
    cache = random_cache(2, 1, cap, D, 64, fmt, [cap, 71], 71)
    cache.k[..., 3] = 0
    q = torch.randn((2, 2, Lq, D), device="cuda", generator=gen(72)) * 2.0 ** -12
    q[..., 3] = 1.9
    check_attention(q.to(dt), cache, scale=2.0 ** 14 / D ** 0.5)


@pytest.mark.parametrize("D,cap", [(64, 300), (128, 2600)])
def test_the_largest_bf16_value_keeps_its_sign(D, cap):
    cache = random_cache(1, 1, cap, D, 64, torch.int8, [cap], 73, dirty=False)
    q = torch.randn((1, 2, 1, D), device="cuda", generator=gen(74)).to(torch.bfloat16)
    q[..., 5] = torch.finfo(torch.bfloat16).max
    cache.k_scale.mul_(2.0 ** -60)
    check_attention(q, cache, scale=2.0 ** -66)
