"""A cache's tensors are changed in place or replaced; either way every call works on the ones the cache shows."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_lengths_and_codes_can_be_changed_in_place_or_replaced():
    from gguf_train_b200 import KV8Cache, kv8_append, kv8_attention, kv8_read

    cache = KV8Cache.empty(2, 1, 40, 32, 16)
    x = torch.randn((2, 1, 9, 32), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    q = x[:, :, 5:6]
    kv8_append(cache, x, x)
    want = kv8_attention(q, KV8Cache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.lens - 3, 16))
    cache.lens = cache.lens - 3  # three drafted tokens rejected
    assert cache.lens.tolist() == [6, 6] and torch.equal(kv8_attention(q, cache), want)
    cache.lens += 3
    cache.lens.sub_(3)
    assert cache.lens.tolist() == [6, 6] and torch.equal(kv8_attention(q, cache), want)
    kv8_append(cache, x[:, :, 6:], x[:, :, 6:])
    assert cache.lens.tolist() == [9, 9]
    k, _ = kv8_read(cache, None, 9)
    cache.k, cache.k_scale = -cache.k, cache.k_scale * 2
    assert torch.equal(kv8_read(cache, None, 9)[0], -2 * k)


def test_replacements_that_do_not_fit_are_refused():
    from gguf_train_b200 import KV8Cache

    cache = KV8Cache.empty(2, 1, 40, 32, 16)
    lens = cache.lens
    for name, bad in (("lens", lens.long()), ("lens", lens[:1]), ("lens", lens.cpu()), ("lens", None),
                      ("k", cache.k[:, :, :20]), ("k", cache.k.transpose(2, 3).contiguous().transpose(2, 3)),
                      ("v", cache.v.to(torch.float8_e4m3fn)), ("v_scale", cache.v_scale.double())):
        with pytest.raises(RuntimeError, match=f"KV8Cache: {name}"):
            setattr(cache, name, bad)
    with pytest.raises(AttributeError):
        cache.block = 32
    assert cache.lens is lens and cache.k.shape == (2, 1, 40, 32)
