"""A call that is the first work of its thread: autograd's thread starts without a current CUDA context, and the tensor maps of the
tensor-core kernels are made by a driver call, which does not get one by itself."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUN = """
import threading, torch
import gguf_train_b200 as gtb
bf = dict(dtype=torch.bfloat16, device="cuda")
{setup}
g = torch.randn_like(out)
torch.cuda.synchronize()
if {thread}:
    r = []
    t = threading.Thread(target=lambda: r.append({direct}))
    t.start(); t.join()
    assert r, "the thread failed"
else:
    torch.autograd.grad(out, leaves, g)
torch.cuda.synchronize()
assert gtb._C.device_status() == 0
"""

SDPA = ("leaves = [torch.randn((1, 1, 64, 64), **bf).requires_grad_() for _ in range(3)]\n"
        "out = gtb.scaled_dot_product_attention(*leaves, is_causal=True)")
LATENT = ("leaves = [torch.randn(s, **bf).requires_grad_() for s in ((1, 1, 64, 96), (1, 1, 64, 64), (1, 64, 32), (1, 1, 64, 64))]\n"
          "out = gtb.latent_sdpa(*leaves, is_causal=True)")
ABSORBED = ("cache = gtb.LatentCache(torch.randn((1, 64, 96), **bf), torch.tensor([64], dtype=torch.int32, device='cuda'), 64)\n"
            "leaves = []\nq = torch.randn((1, 2, 1, 96), **bf)\nout = q[..., :64].contiguous()")


@pytest.mark.parametrize("setup,thread,direct", [
    (SDPA, False, "None"), (LATENT, False, "None"), (ABSORBED, True, "gtb.latent_attention(q, cache, 0.1)"),
    (LATENT, True, "gtb.latent_sdpa(*[x.detach() for x in leaves])"),
], ids=["sdpa backward", "latent_sdpa backward", "latent_attention", "latent_sdpa"])
def test_first_call_of_a_thread(setup, thread, direct):
    r = subprocess.run([sys.executable, "-c", RUN.format(setup=setup, thread=thread, direct=direct)], cwd=ROOT,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
