"""The rotation and the 8-bit cache's calls inside one CUDA graph: replayed over changed inputs and a growing cache they
give the bits of the same calls made one by one."""

from __future__ import annotations

import pytest
import torch

from test_gpu_kv8 import FMTS, gen, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("Lq,H,cap", [(1, 4, 300), (1, 8, 9000), (5, 8, 2500), (40, 4, 2500), (40, 32, 900)],
                         ids=lambda v: str(v))
def test_a_step_replayed_from_a_graph(fmt, Lq, H, cap):
    from gguf_train_b200 import KV8Cache, _C, kv8_append, kv8_attention, kv8_evict, rope_axes

    B, Hkv, D, block, steps = 2, 2, 64, 32, 3
    start = random_cache(B, Hkv, cap, D, block, fmt, [cap - steps * Lq - 3, 70], 61)
    g = gen(62)
    xs = [[torch.randn((B, n, Lq, D), device="cuda", generator=g).to(torch.bfloat16) for n in (H, Hkv, Hkv)] for _ in range(steps)]
    pos = [torch.randint(0, 5000, (3, B, Lq), device="cuda", generator=g).to(torch.int32) for _ in range(steps)]

    def fresh():
        cache = KV8Cache(*(t.clone() for t in (start.k, start.v, start.k_scale, start.v_scale, start.lens)), block)
        return cache, torch.zeros((B, Hkv, cap), device="cuda"), KV8Cache.empty(B, Hkv, 50, D, block, fmt)

    def step(q, k, v, p, cache, score, small):
        q, k = rope_axes(q, p, (8, 12, 12), k=k)
        kv8_append(cache, k, v)
        out, lse = kv8_attention(q, cache, score=score, need_lse=True)
        _, s, kept = kv8_evict(cache, score, 50, recent=7, out=small)
        return out, lse, s, kept

    state = fresh()
    want = [[t.clone() for t in (*step(*x, p, *state), state[1], state[2].lens)] for x, p in zip(xs, pos)]
    state = fresh()
    buf, pb = [t.clone() for t in xs[0]], pos[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        res = step(*buf, pb, *state)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for x, p, w in zip(xs, pos, want):
        for a, b in zip(buf, x):
            a.copy_(b)
        pb.copy_(p)
        graph.replay()
        for got, exp in zip((*res, state[1], state[2].lens), w):
            assert torch.equal(got, exp)
    torch.cuda.synchronize()
    del graph
    assert _C.device_status() == 0
