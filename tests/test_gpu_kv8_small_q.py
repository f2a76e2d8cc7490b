"""Query rows whose values are far apart or at the end of their type. The bound is attention_reference's: sums of D exact
products in f32."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv8 import check_attention, gen, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,cap", [(64, 300), (128, 2600)])
def test_the_largest_bf16_value_keeps_its_sign(D, cap):
    cache = random_cache(1, 1, cap, D, 64, torch.int8, [cap], 73, dirty=False)
    q = torch.randn((1, 2, 1, D), device="cuda", generator=gen(74)).to(torch.bfloat16)
    q[..., 5] = torch.finfo(torch.bfloat16).max
    cache.k_scale.mul_(2.0 ** -60)
    check_attention(q, cache, scale=2.0 ** -66)
