"""Work measured for the 8-bit cache operators: multi-axis rotary positions, the block-scaled 8-bit
KV cache (append, attention from one query token to a chunk, eviction by accumulated weight).

`run` computes each in its plain form (32-bit torch operations) or, with `own`, through the package's
entry points. `exact` computes the same outputs in 64 bits.
"""

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FMT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of 64 sequences: the new token's q and k rotated by (time, height, width)
        dict(name="rope_token", op="rope", B=64, H=32, Hkv=8, S=1, D=128, sections="16,24,24", mode=2,
             interleaved=False, per_axis=False, dtype="bf16", grad=False, far=32768),
        # the prompts of a batch, text with an image inside, axes interleaved over the frequencies
        dict(name="rope_prompt", op="rope", B=8, H=32, Hkv=8, S=4096, D=128, sections="24,20,20", mode=2,
             interleaved=True, per_axis=False, dtype="bf16", grad=False, far=1024),
        # training a vision tower: patches of an odd grid, two axes with their own frequencies, f32, with
        # the gradients of q and k
        dict(name="rope_patches_grad", op="rope", B=6, H=16, Hkv=16, S=2047, D=80, sections="20,20", mode=2,
             interleaved=False, per_axis=True, dtype="f32", grad=True, far=1),
        # one decode step of 64 sequences: the new token's k and v into the cache
        dict(name="append_token", op="append", B=64, Hkv=8, n=1, D=128, cap=4096, lo=1, hi=4095, block=64, fmt="int8",
             dtype="bf16", ragged=False),
        # prompts of different lengths appended behind what the cache holds
        dict(name="append_prompt", op="append", B=8, Hkv=8, n=4099, D=128, cap=8192, lo=0, hi=4000, block=32,
             fmt="e4m3", dtype="f16", ragged=True),
        # one short sequence, one token: the latency of a call
        dict(name="attend_short", op="attend", B=1, H=8, Hkv=8, Lq=1, D=64, cap=512, lo=90, hi=512, block=16, fmt="int8",
             dtype="f32", ragged=False, score=False),
        # the decode benchmark's batch: 64 sequences of 1024 to 32768 cached tokens
        dict(name="attend_token", op="attend", B=64, H=32, Hkv=8, Lq=1, D=128, cap=32768, lo=1024, hi=32768, block=64,
             fmt="int8", dtype="bf16", ragged=False, score=False),
        # decode that also accumulates the attention weight of every cached token
        dict(name="attend_token_scored", op="attend", B=16, H=32, Hkv=8, Lq=1, D=128, cap=16384, lo=2000, hi=16384,
             block=32, fmt="e4m3", dtype="f16", ragged=False, score=True),
        # several drafted tokens a sequence, verified in one call
        dict(name="attend_draft", op="attend", B=32, H=32, Hkv=8, Lq=5, D=128, cap=8192, lo=100, hi=8192, block=64,
             fmt="e4m3", dtype="bf16", ragged=True, score=False),
        # a chunk of a long prompt against everything before it
        dict(name="attend_chunk", op="attend", B=4, H=32, Hkv=8, Lq=1021, D=128, cap=8192, lo=4096, hi=8192, block=128,
             fmt="int8", dtype="bf16", ragged=False, score=False),
        # a few short sequences cut to a small budget
        dict(name="evict_short", op="evict", B=2, Hkv=8, D=64, cap=640, lo=200, hi=640, budget=256, recent=32, block=16,
             fmt="int8"),
        # long sequences cut to a quarter of the cache
        dict(name="evict_long", op="evict", B=16, Hkv=8, D=128, cap=16384, lo=3500, hi=16384, budget=4096, recent=128,
             block=64, fmt="int8"),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    n = min(hi, max(lo, n))
    return n if n != 3072 else 3071


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "evict"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 5, 8])
    fmt = rng.choice(["int8", "e4m3"])
    block = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "rope":
        sections = rng.choice(["16,24,24", "32,32", "24,20,20", "8,12,12", "16,16"]) if D == 128 else \
            rng.choice(["8,12,12", "16,16", "10,11,11"])
        # interleaving needs every axis but the first to fit its turns, true of all but a few sections
        interleaved = sections in ("24,20,20", "32,32", "16,16") and rng.random() < 0.5
        S = _log(rng, 1, 8192)
        B = max(1, min(_log(rng, 1, 64), 32768 // S))
        return dict(op=op, B=B, H=Hkv * min(G, 4), Hkv=Hkv, S=S, D=D, sections=sections, mode=rng.choice([0, 2]),
                    interleaved=interleaved, per_axis=rng.random() < 0.4, dtype=dtype, grad=rng.random() < 0.5,
                    far=_log(rng, 1, 100000))
    if op == "append":
        n = rng.choice([1, _log(rng, 1, 4096)])
        B = max(1, min(_log(rng, 1, 64), 32768 // n))
        cap = n + _log(rng, 64, 4000)
        return dict(op=op, B=B, Hkv=Hkv, n=n, D=D, cap=cap, lo=0, hi=cap - n, block=block, fmt=fmt, dtype=dtype,
                    ragged=rng.random() < 0.5)
    if op == "evict":
        cap = _log(rng, 100, 16384)
        budget = _log(rng, 16, max(17, cap // 2))
        return dict(op=op, B=_log(rng, 1, 16), Hkv=Hkv, D=D, cap=cap, lo=max(1, cap // 5), hi=cap, budget=budget,
                    recent=rng.randint(0, budget), block=block, fmt=fmt)
    Lq = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 1000)])
    cap = max(Lq + 1, _log(rng, 32, 32768 if Lq == 1 else 8192))
    B = max(1, min(_log(rng, 1, 64 if Lq < 9 else 4), (1 << 20) // cap))
    return dict(op=op, B=B, H=Hkv * G if Lq < 9 else Hkv * min(G, 32 // Hkv), Hkv=Hkv, Lq=Lq, D=D, cap=cap, lo=max(1, cap // 8),
                hi=cap, block=block, fmt=fmt, dtype=dtype, ragged=rng.random() < 0.5, score=rng.random() < 0.4)


# ------------------------------------------------------------------ inputs

def _codes(shape, fmt, gen):
    """Quantised N(0, 1): what a cache of normal keys and values holds."""
    x = torch.randn(shape, dtype=torch.float16, device="cuda", generator=gen).mul_(TOP[fmt] / 4.3)
    x.clamp_(-TOP[fmt], TOP[fmt])
    return x.round_().to(torch.int8) if fmt == "int8" else x.to(torch.float8_e4m3fn)


def _scales(shape, fmt, gen):
    return (0.7 + 0.6 * torch.rand(shape, device="cuda", generator=gen)) * (4.3 / TOP[fmt])


def _cache(case, gen, lens, dirty):
    """The cache's tensors. Rows at and past the lengths hold zeros, or with `dirty` what earlier
    sequences left: any code (NaN among the e4m3 ones) and any scale."""
    B, Hkv, cap, D, T, fmt = (case[k] for k in ("B", "Hkv", "cap", "D", "block", "fmt"))
    nb = -(-cap // T)
    past = torch.arange(cap, device="cuda")[None, :] >= lens[:, None]
    blocks_past = (torch.arange(nb, device="cuda") * T)[None, :] >= lens[:, None]
    st = {"lens": lens.to(torch.int32)}

    def one():
        c = _codes((B, Hkv, cap, D), fmt, gen)
        c.view(torch.uint8).masked_fill_(past[:, None, :, None], 0x7F if dirty else 0)
        s = _scales((B, Hkv, nb), fmt, gen)
        return c, s.masked_fill(blocks_past[:, None, :], float("nan") if dirty else 0.0)

    st["k"], st["k_scale"] = one()
    st["v"], st["v_scale"] = one()
    return st


def _lens(case, gen):
    B, lo, hi = case["B"], case["lo"], case["hi"]
    n = torch.randint(lo, hi + 1, (B,), device="cuda", generator=gen)
    if hi == case["cap"] and B > 1:
        n[-1] = hi
    return n


def _counts(case, n, gen):
    if not case["ragged"]:
        return None
    c = torch.randint(1, n + 1, (case["B"],), device="cuda", generator=gen)
    c[0] = n
    return c.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    if op == "rope":
        B, S, far = case["B"], case["S"], case["far"]
        sections = [int(x) for x in case["sections"].split(",")]
        A = len(sections)
        at = torch.randint(0, far, (B, 1), device="cuda", generator=gen)
        i = torch.arange(S, device="cuda")[None, :]
        cols = torch.randint(3, 61, (B, 1), device="cuda", generator=gen)
        first = torch.randint(0, S, (B, 1), device="cuda", generator=gen) // (1 if A == 3 else S)
        image = (i >= first) & (i < first + max(1, (S * 3) // 4) + (S if A == 2 else 0))
        j = i - first
        text = at + i
        h = torch.where(image, at + first + j // cols, text)
        w = torch.where(image, at + first + j % cols, text)
        t = torch.where(image, at + first, text)
        pos = torch.stack([t, h, w] if A == 3 else [h, w]).to(torch.int32).contiguous()
        dt = DT[case["dtype"]]
        # q and k as views of a projection's (B, S, heads, D) output
        mk = lambda n: torch.randn((B, S, n, case["D"]), device="cuda", generator=gen).to(dt).transpose(1, 2)  # noqa: E731
        st = {"case": case, "q": mk(case["H"]), "k": mk(case["Hkv"]), "pos": pos, "sections": sections}
        if case["grad"]:
            st["q"].requires_grad_()
            st["k"].requires_grad_()
            st["gq"], st["gk"] = mk(case["H"]).contiguous(), mk(case["Hkv"]).contiguous()
        return st
    lens = _lens(case, gen)
    if op == "append":
        n, T = case["n"], case["block"]
        st = {"case": case, **_cache(case, gen, lens, dirty=False)}
        dt = DT[case["dtype"]]
        # the new rows are views of a (B, n, heads, D) projection
        mk = lambda: (1.2 * torch.randn((case["B"], n, case["Hkv"], case["D"]), device="cuda", generator=gen)).to(dt).transpose(1, 2)  # noqa: E731
        st["xk"], st["xv"] = mk(), mk()
        st["counts"] = _counts(case, n, gen)
        st["start"] = (lens // T * T).to(torch.int32)
        st["rows"] = (n + 2 * T - 2) // T * T
        return st
    if op == "attend":
        st = {"case": case, **_cache(case, gen, lens, dirty=True)}
        B, H, Hkv, Lq, D = (case[k] for k in ("B", "H", "Hkv", "Lq", "D"))
        q = 1.3 * torch.randn((B, Lq, H, D), device="cuda", generator=gen)
        st["q"] = q.to(DT[case["dtype"]]).transpose(1, 2)
        st["counts"] = _counts(case, Lq, gen)
        if case["score"]:
            st["score"] = torch.rand((B, Hkv, case["cap"]), device="cuda", generator=gen) * 3e-4
            st["score_out"] = torch.zeros_like(st["score"])
        return st
    st = {"case": case, **_cache(case, gen, lens, dirty=True)}
    B, Hkv, D, T, budget = (case[k] for k in ("B", "Hkv", "D", "block", "budget"))
    # accumulated weight: most tokens got little, a few much; some exactly nothing
    s = torch.randn((B, Hkv, case["cap"]), device="cuda", generator=gen).mul(1.5).exp()
    s = s.masked_fill(torch.rand(s.shape, device="cuda", generator=gen) < 0.05, 0.0)
    st["score"] = s
    st["out"] = {"k": torch.zeros((B, Hkv, budget, D), dtype=FMT[case["fmt"]], device="cuda"),
                 "v": torch.zeros((B, Hkv, budget, D), dtype=FMT[case["fmt"]], device="cuda"),
                 "k_scale": torch.zeros((B, Hkv, -(-budget // T)), device="cuda"),
                 "v_scale": torch.zeros((B, Hkv, -(-budget // T)), device="cuda"),
                 "lens": torch.zeros(B, dtype=torch.int32, device="cuda")}
    st["score_out"] = torch.zeros((B, Hkv, budget), device="cuda")
    st["zero"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    return st


# ------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    return (_OWN if own else _PLAIN)[op](state)


def _handle(st, name="cache"):
    """The cache handle that a program keeps next to its tensors, made at the first call."""
    if name not in st:
        from gguf_train_b200 import KV8Cache
        t = st if name == "cache" else st["out"]
        st[name] = KV8Cache(t["k"], t["v"], t["k_scale"], t["v_scale"], t["lens"], st["case"]["block"])
    return st[name]


def _own_rope(st):
    from gguf_train_b200 import rope_axes
    c = st["case"]
    yq, yk = rope_axes(st["q"], st["pos"], st["sections"], k=st["k"], mode=c["mode"], interleaved=c["interleaved"],
                       per_axis=c["per_axis"])
    if not c["grad"]:
        return yq, yk
    gq, gk = torch.autograd.grad((yq, yk), (st["q"], st["k"]), (st["gq"], st["gk"]))
    return yq.detach(), yk.detach(), gq, gk


def _own_append(st):
    from gguf_train_b200 import kv8_append, kv8_read
    cache = _handle(st)
    kv8_append(cache, st["xk"], st["xv"], counts=st["counts"], advance=False)
    k, v = kv8_read(cache, st["start"], st["rows"], dtype=st["xk"].dtype)
    return k, v, cache.k_scale, cache.v_scale


def _own_attend(st):
    from gguf_train_b200 import kv8_attention
    if st["case"]["score"]:
        out, lse = kv8_attention(st["q"], _handle(st), counts=st["counts"], score=st["score"],
                                 score_out=st["score_out"], need_lse=True)
        return out, lse, st["score_out"]
    return kv8_attention(st["q"], _handle(st), counts=st["counts"], need_lse=True)


def _own_evict(st):
    from gguf_train_b200 import kv8_evict, kv8_read
    c = st["case"]
    out, score, kept = kv8_evict(_handle(st), st["score"], c["budget"], recent=c["recent"], out=_handle(st, "small"),
                                 score_out=st["score_out"])
    k, v = kv8_read(out, st["zero"], c["budget"], dtype=torch.bfloat16)
    return k, v, out.k_scale, out.v_scale, out.lens, score, kept


_OWN = {"rope": _own_rope, "append": _own_append, "attend": _own_attend, "evict": _own_evict}


# ------------------------------------------------------------------ plain forms, 32 bits

def _pairs(sections, interleaved, per_axis, base=10000.0):
    """(axis, frequency) of every pair of dimensions, as lists."""
    P, A = sum(sections), len(sections)
    if interleaved:
        axis = [i % A if i < A * sections[i % A] else 0 for i in range(P)]
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if per_axis:
        freq = [base ** (-axis[:i].count(a) / sections[a]) for i, a in enumerate(axis)]
    else:
        freq = [base ** (-i / P) for i in range(P)]
    return axis, freq


def _rotate(x, c, s, mode, P):
    x = x.float()
    if mode == 0:
        x0, x1 = x[..., 0:2 * P:2], x[..., 1:2 * P:2]
        y = torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1).flatten(-2)
    else:
        x0, x1 = x[..., :P], x[..., P:2 * P]
        y = torch.cat((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1)
    return torch.cat((y, x[..., 2 * P:]), dim=-1)


def _plain_rope(st):
    c = st["case"]
    axis, freq = _pairs(st["sections"], c["interleaved"], c["per_axis"])
    # the angle as a fraction of a turn in 64-bit fixed point: whole turns fall off in the product, and
    # no 32-bit number has to hold a long position's angle
    turns = [int(round(f / (2 * math.pi) * 2.0 ** 64)) for f in freq]
    turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], device="cuda")
    t = st["pos"].long()[torch.tensor(axis, device="cuda")].permute(1, 2, 0) * turns  # (B, S, P)
    angle = ((t >> 32).float() * (2 * math.pi / 2.0 ** 32))[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    P, mode, dt = len(axis), c["mode"], st["q"].dtype
    ys = tuple(_rotate(st[n].detach(), cos, sin, mode, P).to(dt) for n in ("q", "k"))
    if not c["grad"]:
        return ys
    return ys + tuple(_rotate(st[n], cos, -sin, mode, P).to(dt) for n in ("gq", "gk"))


def _over(x, s):
    return torch.where(s > 0, x / s, torch.zeros_like(x))


def _quantise(x, s, fmt):
    y = _over(x, s).clamp(-TOP[fmt], TOP[fmt])
    return y.round() if fmt == "int8" else y.to(torch.float8_e4m3fn).float()


def _plain_append(st):
    c = st["case"]
    B, Hkv, n, D, T, fmt, cap = (c[k] for k in ("B", "Hkv", "n", "D", "block", "fmt", "cap"))
    rows, nb = st["rows"], st["rows"] // T
    lens, start = st["lens"].long(), st["start"].long()
    counts = torch.full_like(lens, n) if st["counts"] is None else st["counts"].long()
    r = start[:, None] + torch.arange(rows, device="cuda")  # (B, rows): cache rows of the touched blocks
    old = (r < lens[:, None])[:, None, :, None]
    new = ((r >= lens[:, None]) & (r < (lens + counts)[:, None]))[:, None, :, None]
    src = (r - lens[:, None]).clamp(0, n - 1)
    blk = (start // T)[:, None] + torch.arange(nb, device="cuda")
    had = (blk * T < lens[:, None])[:, None]
    touched = (blk * T < (lens + counts)[:, None])[:, None]
    bi = torch.arange(B, device="cuda")[:, None]
    rc, bc = r.clamp(max=cap - 1), blk.clamp(max=st["k_scale"].shape[2] - 1)

    def one(x, codes, scales):
        xr = x.float()[bi, :, src].transpose(1, 2)  # (B, Hkv, rows, D)
        held = codes.view(torch.uint8)[bi, :, rc].transpose(1, 2).contiguous().view(codes.dtype).float()
        kept = scales[bi, :, bc].transpose(1, 2)  # (B, Hkv, nb)
        s_old = torch.where(had, kept, torch.zeros_like(kept))
        amax = torch.where(new, xr.abs(), torch.zeros_like(xr)).reshape(B, Hkv, nb, T * D).amax(-1)
        s = torch.maximum(s_old, amax / TOP[fmt])
        wide = lambda z: z.repeat_interleave(T, dim=2)[..., None]  # noqa: E731
        again = wide(s > s_old)
        q_old = torch.where(again, _quantise(held * wide(s_old), wide(s), fmt), held)
        q_new = _quantise(xr, wide(s), fmt)
        q = torch.where(old, q_old, torch.where(new, q_new, torch.zeros_like(held)))
        # the state's own buffers take the update; rows past the sequence's new end keep what they hold
        live = (old | new).expand(B, Hkv, rows, D).permute(0, 2, 1, 3)[..., 0]
        at = torch.nonzero(live, as_tuple=True)
        codes.view(torch.uint8)[at[0], at[2], r[at[0], at[1]]] = q.to(codes.dtype).view(torch.uint8)[at[0], at[2], at[1]]
        ab = torch.nonzero(touched.expand(B, Hkv, nb), as_tuple=True)
        scales[ab[0], ab[1], blk[ab[0], ab[2]]] = s[ab]
        # values as the cache now stands for them
        s_now = torch.where(touched, s, kept)
        val = torch.where((r < cap)[:, None, :, None], q * wide(s_now), torch.zeros_like(q))
        return val.to(x.dtype)

    k = one(st["xk"], st["k"], st["k_scale"])
    v = one(st["xv"], st["v"], st["v_scale"])
    return k, v, st["k_scale"], st["v_scale"]


def _values(codes, scales, T, valid):
    """Cached values in 32 bits, 0 at and past the lengths."""
    s = scales.repeat_interleave(T, dim=2)[:, :, :codes.shape[2], None]
    return torch.where(valid, codes.float() * s, torch.zeros((), device="cuda"))


def _plain_attend(st):
    c = st["case"]
    B, H, Hkv, Lq, D, T, cap = (c[k] for k in ("B", "H", "Hkv", "Lq", "D", "block", "cap"))
    G = H // Hkv
    lens = st["lens"].long()
    counts = torch.full_like(lens, Lq) if st["counts"] is None else st["counts"].long()
    s_idx, i = torch.arange(cap, device="cuda"), torch.arange(Lq, device="cuda")
    valid = (s_idx < lens[:, None])[:, None, :, None]
    limit = torch.where(i < counts[:, None], lens[:, None] - counts[:, None] + i + 1, torch.zeros_like(i))  # (B, Lq)
    seen = s_idx < limit[:, :, None]  # (B, Lq, cap)
    k = _values(st["k"], st["k_scale"], T, valid)
    q = st["q"].float().reshape(B, Hkv, G * Lq, D)
    x = torch.matmul(q, k.transpose(2, 3)).view(B, Hkv, G, Lq, cap) * (1.0 / math.sqrt(D))
    del k
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del x
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    v = _values(st["v"], st["v_scale"], T, valid)
    out = torch.matmul(p.view(B, Hkv, G * Lq, cap), v).view(B, H, Lq, D).to(st["q"].dtype)
    lse = (torch.log(total) + top)[..., 0].view(B, H, Lq)
    if not c["score"]:
        return out, lse
    w = p.sum((2, 3))
    keep = valid[..., 0].expand(B, Hkv, cap)
    return out, lse, torch.where(keep, st["score"] + w, st["score_out"])


def _plain_evict(st):
    c = st["case"]
    B, Hkv, D, T, fmt, cap, budget, recent = (c[k] for k in ("B", "Hkv", "D", "block", "fmt", "cap", "budget", "recent"))
    lens = st["lens"].long()[:, None, None]
    i = torch.arange(cap, device="cuda")
    cut = lens > budget
    by_score = (i < lens - recent) & cut
    rank_key = torch.where(by_score, torch.nan_to_num(st["score"], nan=float("-inf"), posinf=float("inf")),
                           torch.tensor(float("-inf"), device="cuda"))
    order = torch.sort(rank_key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, i.expand_as(order).contiguous())
    keep = torch.where(cut, ((rank < budget - recent) & by_score) | ((i >= lens - recent) & (i < lens)), i < lens)
    keep = keep.expand(B, Hkv, cap)
    kept = torch.sort((~keep).to(torch.int8), dim=-1, stable=True).indices[..., :budget]
    n_new = lens.clamp(max=budget)  # (B, 1, 1)
    j = torch.arange(budget, device="cuda")[:kept.shape[-1]]
    live = (j < n_new).expand(B, Hkv, -1)
    pad = budget - kept.shape[-1]
    kept = torch.nn.functional.pad(torch.where(live, kept, torch.full_like(kept, -1)), (0, pad), value=-1)
    live = torch.nn.functional.pad(live, (0, pad))
    at = kept.clamp(min=0)
    nb = -(-budget // T)

    def one(codes, scales):
        rows = torch.gather(codes.view(torch.uint8), 2, at[..., None].expand(B, Hkv, budget, D)).view(codes.dtype).float()
        x = torch.where(live[..., None], rows * torch.gather(scales, 2, at // T)[..., None], torch.zeros((), device="cuda"))
        amax = torch.nn.functional.pad(x.abs().amax(-1), (0, nb * T - budget)).view(B, Hkv, nb, T).amax(-1)
        s = amax / TOP[fmt]
        wide = s.repeat_interleave(T, dim=2)[:, :, :budget, None]
        return (_quantise(x, wide, fmt) * wide).to(torch.bfloat16), s

    k, ks = one(st["k"], st["k_scale"])
    v, vs = one(st["v"], st["v_scale"])
    score = torch.where(live, torch.gather(st["score"], 2, at), torch.zeros((), device="cuda"))
    return k, v, ks, vs, n_new.view(B).to(torch.int32), score, kept.to(torch.int32)


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}


# ------------------------------------------------------------------ work of one pass

def work(case):
    c = case
    op = c["op"]
    if op == "rope":
        size = 4 if c["dtype"] == "f32" else 2
        n = c["B"] * (c["H"] + c["Hkv"]) * c["S"] * c["D"]
        A = c["sections"].count(",") + 1
        times = 2 if c["grad"] else 1
        return {"bytes": times * (2 * n * size) + 4 * A * c["B"] * c["S"], "flops": times * 3 * n}
    size = 4 if c.get("dtype") == "f32" else 2
    mean = (c["lo"] + c["hi"]) / 2
    if op == "append":
        share = (c["n"] + 1) / 2 / c["n"] if c["ragged"] else 1.0
        n = 2 * c["B"] * c["Hkv"] * c["n"] * c["D"] * share
        back = 2 * c["B"] * c["Hkv"] * (c["n"] + c["block"]) * c["D"]  # the values read back: codes and output
        return {"bytes": int(n * (size + 1) + back * (1 + size)), "flops": int(4 * n + back)}
    if op == "attend":
        rows = c["H"] * c["Lq"]
        live = (c["Lq"] + 1) / 2 if c["ragged"] else c["Lq"]
        b = c["B"] * mean * c["Hkv"] * (2 * c["D"] + 8 / c["block"]) + 2 * c["B"] * rows * c["D"] * size
        b += c["B"] * c["Hkv"] * mean * 8 if c["score"] else 0
        return {"bytes": int(b), "flops": int(4 * c["D"] * c["B"] * c["H"] * live * max(1.0, mean - live / 2))}
    kept = min(c["budget"], mean)
    rows = c["B"] * c["Hkv"] * kept
    # kept codes read and written, the scores, kept scores and indices, and the values read back in 16 bits
    return {"bytes": int(rows * (4 * c["D"] + 12) + 4 * c["B"] * c["Hkv"] * mean + 2 * rows * c["D"] * 3),
            "flops": int(4 * rows * c["D"])}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """What run returns for these inputs from the operators' definitions in 64 bits. Scales are stored in
    32 bits by definition, so each is rounded to them once."""

    def exact_rope(st, c):
        sections, A = st["sections"], len(st["sections"])
        P = sum(sections)
        pos = st["pos"].double()
        angle = torch.zeros((c["B"], c["S"], P), dtype=torch.float64, device="cuda")
        used = [0] * A
        ends = [sum(sections[:a + 1]) for a in range(A)]
        for i in range(P):
            if c["interleaved"]:
                a = i % A
                a = a if i < A * sections[a] else 0
            else:
                a = next(x for x in range(A) if i < ends[x])
            f = 10000.0 ** (-used[a] / sections[a]) if c["per_axis"] else 10000.0 ** (-i / P)
            used[a] += 1
            angle[..., i] = pos[a] * f

        def turn(x, sign):
            y = x.detach().double().clone()
            for i in range(P):
                u, w = (2 * i, 2 * i + 1) if c["mode"] == 0 else (i, i + P)
                cs, sn = torch.cos(angle[:, None, :, i]), sign * torch.sin(angle[:, None, :, i])
                a, b = x.detach()[..., u].double(), x.detach()[..., w].double()
                y[..., u] = a * cs - b * sn
                y[..., w] = a * sn + b * cs
            return y

        outs = [turn(st["q"], 1.0), turn(st["k"], 1.0)]
        if c["grad"]:
            outs += [turn(st["gq"], -1.0), turn(st["gk"], -1.0)]
        return tuple(outs)

    def exact_codes(y, fmt):
        """The nearest code of each value: whole numbers, or the e4m3 grid (3 bits below the leading one,
        steps of 2^-9 below 2^-6)."""
        y = y.clamp(-TOP[fmt], TOP[fmt])
        if fmt == "int8":
            return torch.round(y)
        e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
        e = torch.where(torch.exp2(e) > y.abs().clamp(min=2.0 ** -6), e - 1, e)
        step = torch.exp2(e - 3)
        return torch.round(y / step) * step

    def exact_append(st, c):
        T, fmt, n, rows, D, cap = c["block"], c["fmt"], c["n"], st["rows"], c["D"], c["cap"]
        outs = []
        for name in ("k", "v"):
            x, codes, scales = st["x" + name], st[name], st[name + "_scale"]
            val = torch.zeros((c["B"], c["Hkv"], rows, D), dtype=torch.float64, device="cuda")
            s_all = scales.double().clone()
            for b in range(c["B"]):
                p = int(st["lens"][b])
                cnt = n if st["counts"] is None else int(st["counts"][b])
                start = p // T * T
                nb = -(-(p + cnt - start) // T)
                page = torch.zeros((c["Hkv"], nb * T, D), dtype=torch.float64, device="cuda")
                s_old = torch.zeros((c["Hkv"], nb), dtype=torch.float64, device="cuda")
                if p > start:
                    s_old[:, 0] = scales[b, :, start // T].double()
                new = page.clone()
                new[:, p - start:p - start + cnt] = x[b, :, :cnt].double()
                amax = new.abs().view(c["Hkv"], nb, T * D).amax(-1)
                s = torch.maximum(s_old, (amax / TOP[fmt]).float().double())  # scales are stored in 32 bits
                sw = s.repeat_interleave(T, dim=1)[..., None]
                page = exact_codes(torch.where(sw > 0, new / sw.clamp(min=1e-300), torch.zeros_like(new)), fmt)
                if p > start:
                    held = codes[b, :, start:p].double()
                    grown = (s[:, 0] > s_old[:, 0])[:, None, None]
                    s0 = s[:, 0].clamp(min=1e-300)[:, None, None]
                    page[:, :p - start] = torch.where(grown, exact_codes(held * s_old[:, 0][:, None, None] / s0, fmt), held)
                m = min(rows, nb * T, cap - start)
                val[b, :, :m] = (page * sw)[:, :m]
                s_all[b, :, start // T:start // T + nb] = s
            outs.append((val, s_all))
        return outs[0][0], outs[1][0], outs[0][1], outs[1][1]

    def exact_attend(st, c):
        B, H, Hkv, Lq, D, T = (c[k] for k in ("B", "H", "Hkv", "Lq", "D", "block"))
        G = H // Hkv
        out = torch.zeros((B, H, Lq, D), dtype=torch.float64, device="cuda")
        lse = torch.full((B, H, Lq), float("-inf"), dtype=torch.float64, device="cuda")
        score = st["score_out"].double().clone() if c["score"] else None
        for b in range(B):
            n = int(st["lens"][b])
            cnt = Lq if st["counts"] is None else int(st["counts"][b])
            row_block = torch.arange(n, device="cuda") // T
            ends = n - cnt + 1 + torch.arange(cnt, device="cuda")
            blocked = torch.arange(n, device="cuda")[None, :] >= ends[:, None]
            for hk in range(Hkv):
                k = st["k"][b, hk, :n].double() * st["k_scale"][b, hk, row_block].double()[:, None]
                v = st["v"][b, hk, :n].double() * st["v_scale"][b, hk, row_block].double()[:, None]
                q = st["q"][b, hk * G:(hk + 1) * G, :cnt].double()
                x = (q @ k.T / math.sqrt(D)).masked_fill(blocked[None], float("-inf"))
                z = torch.logsumexp(x, dim=-1)
                p = torch.where(torch.isinf(z)[..., None], torch.zeros_like(x), torch.exp(x - z[..., None]))
                out[b, hk * G:(hk + 1) * G, :cnt] = p @ v
                lse[b, hk * G:(hk + 1) * G, :cnt] = z
                if score is not None:
                    score[b, hk, :n] = st["score"][b, hk, :n].double() + p.sum((0, 1))
        return (out, lse, score) if c["score"] else (out, lse)

    def exact_evict(st, c):
        B, Hkv, D, T, fmt, budget, recent = (c[k] for k in ("B", "Hkv", "D", "block", "fmt", "budget", "recent"))
        nb = -(-budget // T)
        vals = {n: torch.zeros((B, Hkv, nb * T, D), dtype=torch.float64, device="cuda") for n in ("k", "v")}
        scales = {n: torch.zeros((B, Hkv, nb), dtype=torch.float64, device="cuda") for n in ("k", "v")}
        score = torch.zeros((B, Hkv, budget), dtype=torch.float64, device="cuda")
        kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device="cuda")
        for b in range(B):
            n = int(st["lens"][b])
            for h in range(Hkv):
                if n <= budget:
                    idx = torch.arange(n, device="cuda")
                else:
                    s = st["score"][b, h, :n - recent].double()
                    first = torch.argsort(-s, stable=True)[:budget - recent]
                    idx = torch.cat((torch.sort(first).values, torch.arange(n - recent, n, device="cuda")))
                m = idx.numel()
                kept[b, h, :m] = idx.to(torch.int32)
                score[b, h, :m] = st["score"][b, h, idx].double()
                for name in ("k", "v"):
                    x = torch.zeros((nb * T, D), dtype=torch.float64, device="cuda")
                    x[:m] = st[name][b, h][idx].double() * st[name + "_scale"][b, h, idx // T].double()[:, None]
                    sc = (x.abs().view(nb, T * D).amax(-1) / TOP[fmt]).float().double()
                    sw = sc.repeat_interleave(T)[:, None]
                    vals[name][b, h] = exact_codes(torch.where(sw > 0, x / sw.clamp(min=1e-300), torch.zeros_like(x)), fmt) * sw
                    scales[name][b, h] = sc
        n_new = st["lens"].clamp(max=budget).to(torch.int32)
        return vals["k"][:, :, :budget], vals["v"][:, :, :budget], scales["k"], scales["v"], n_new, score, kept

    st = prepare(case, seed)
    with torch.no_grad():
        return {"rope": exact_rope, "append": exact_append, "attend": exact_attend, "evict": exact_evict}[case["op"]](st, case)
