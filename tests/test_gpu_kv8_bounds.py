"""What the 8-bit cache's calls may touch and take: rows past the capacity reach no memory at all, and the scratch of a
call stays bounded however large the cache's capacity."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from test_gpu_kv8 import FMTS, append_reference, gen, random_cache

pytestmark = pytest.mark.gpu


class _Walled:
    """Tensors inside larger allocations, with a byte pattern on both sides."""

    PAD = 4096

    def __init__(self):
        self.all = []

    def make(self, shape, dtype, fill):
        n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
        buf = torch.full((n + 2 * self.PAD,), 0xA5, dtype=torch.uint8, device="cuda")
        t = buf[self.PAD:self.PAD + n].view(dtype).view(shape)
        t.view(torch.uint8).fill_(fill)
        self.all.append((buf, n))
        return t

    def untouched(self):
        return all((b[:self.PAD] == 0xA5).all() and (b[self.PAD + n:] == 0xA5).all() for b, n in self.all)


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cap,block", [(20, 16), (64, 32), (100, 128)])
def test_rows_past_the_capacity_reach_no_memory(fmt, dt, cap, block):
    """Every (sequence, head, row) holds values of its own; the first sequence overflows, the last fits, the middle one
    is full already."""
    from gguf_train_b200 import KV8Cache, _C, kv8_append

    B, Hkv, D, n = 3, 2, 32, 13
    lens = [cap - 5, cap, cap - n]
    wall = _Walled()
    nb = -(-cap // block)
    k, v = (wall.make((B, Hkv, cap, D), fmt, 0x11) for _ in range(2))
    ks, vs = (wall.make((B, Hkv, nb), torch.float32, 0x3C) for _ in range(2))  # 0x3C3C3C3C: 0.0115
    ln = wall.make((B,), torch.int32, 0)
    ln.copy_(torch.tensor(lens, dtype=torch.int32))
    cache = KV8Cache(k, v, ks, vs, ln, block)
    g = gen(51)
    x = [torch.randn((B, Hkv, n, D), device="cuda", generator=g).to(dt) * (1 + torch.arange(B * Hkv * n, device="cuda").view(B, Hkv, n, 1)).to(dt)
         for _ in range(2)]
    ref = [(c.float().clone(), s.clone()) for c, s in ((k, ks), (v, vs))]
    kv8_append(cache, *x)
    assert _C.device_status() == 61
    for r, xx in zip(ref, x):
        append_reference(r, xx, list(lens), [n] * B, block, fmt)
    for c, s, r in ((k, ks, ref[0]), (v, vs, ref[1])):
        assert torch.equal(c.float(), r[0]) and torch.equal(s, r[1])
    assert ln.tolist() == [cap, cap, cap] and wall.untouched()


def _pool_high(reset=False):
    """The most bytes in use at a time in the device's stream-ordered pool since the last reset (a host-side statistic)."""
    rt = ctypes.CDLL("libcudart.so.12")
    pool, value = ctypes.c_void_p(), ctypes.c_uint64(0)
    assert rt.cudaDeviceGetDefaultMemPool(ctypes.byref(pool), 0) == 0
    torch.cuda.synchronize()
    if reset:
        assert rt.cudaMemPoolSetAttribute(pool, 8, ctypes.byref(value)) == 0  # cudaMemPoolAttrUsedMemHigh
    assert rt.cudaMemPoolGetAttribute(pool, 8, ctypes.byref(value)) == 0
    return value.value


@pytest.mark.parametrize("B,cap", [(40, 1 << 19), (2, 10 << 20)], ids=["many sequences", "long ones"])
def test_scratch_of_weights_is_bounded(B, cap):
    """32 rows a head with weights: kept scores would take 4 * 32 bytes for every row of capacity (2.7 GB here), most of
    it for rows that no sequence holds. A call takes 1 GB of it at most (and a little beside), and the results are those of a
    small cache that holds the same rows."""
    from gguf_train_b200 import KV8Cache, kv8_attention

    H, D, block, small = 32, 16, 128, 1024
    lens = [(97 * b + 300) % small for b in range(B)]
    near = random_cache(B, 1, small, D, block, torch.int8, lens, 52)
    far = KV8Cache.empty(B, 1, cap, D, block)
    for a, b in ((far.k, near.k), (far.v, near.v)):
        a[:, :, :small] = b
    for a, b in ((far.k_scale, near.k_scale), (far.v_scale, near.v_scale)):
        a[:, :, :small // block] = b
    far.lens.copy_(near.lens)
    q = torch.randn((B, H, 1, D), device="cuda", generator=gen(53)).to(torch.bfloat16)
    ss, sf = (torch.zeros((B, 1, c.capacity), device="cuda") for c in (near, far))
    want, wl = kv8_attention(q, near, score=ss, need_lse=True)
    _pool_high(reset=True)
    out, lse = kv8_attention(q, far, score=sf, need_lse=True)
    assert _pool_high() <= 1.2e9
    # the two are cut into parts in other places: f32 sums of the same terms, weights rounded to f16 once
    assert (out.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    assert (lse - wl).abs().nan_to_num(0.0).max() <= 1e-5
    assert ((sf[:, :, :small] - ss).abs() <= 1e-4 * (1e-3 + ss)).all()
    assert (sf[:, :, small:] == 0).all()
