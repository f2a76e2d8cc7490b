"""Work measured for the latent attention operators: the cache of one latent vector and one rotary key a
token (append), attention over it in the absorbed form from one query token to a chunk, with and without a
prefix that the batch shares, and the expanded form of prompts and training with its gradients.

`run` computes each in its plain form (32-bit torch operations) or, with `own`, through the package's
entry points. `exact` computes the same outputs in 64 bits.
"""

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of 64 sequences: the new token's latent and rotated key into the cache
        dict(name="append_token", op="append", B=64, n=1, R=512, Dr=64, cap=4096, lo=1, hi=4000, mode=2, freq_scale=1.0,
             dtype="bf16", ragged=False),
        # prompts of different lengths written behind what the cache holds, positions scaled for a long context
        dict(name="append_prompt", op="append", B=8, n=4099, R=256, Dr=32, cap=8192, lo=0, hi=4000, mode=0, freq_scale=0.25,
             dtype="f16", ragged=True),
        # one short sequence, one token: the latency of a call
        dict(name="attend_short", op="attend", B=1, H=8, Lq=1, R=128, Dr=32, cap=512, lo=390, hi=511, prefix=0, dtype="f16",
             ragged=False),
        # the decode benchmark's batch: 64 sequences of 1024 to 32768 cached tokens
        dict(name="attend_token", op="attend", B=64, H=16, Lq=1, R=512, Dr=64, cap=32768, lo=1024, hi=32768, prefix=0,
             dtype="bf16", ragged=False),
        # several drafted tokens a sequence, verified in one call
        dict(name="attend_draft", op="attend", B=32, H=20, Lq=5, R=256, Dr=64, cap=8192, lo=100, hi=8192, prefix=0,
             dtype="f16", ragged=True),
        # a chunk of a long prompt against everything before it
        dict(name="attend_chunk", op="attend", B=4, H=32, Lq=509, R=512, Dr=64, cap=8192, lo=4096, hi=8192, prefix=0,
             dtype="bf16", ragged=False),
        # one decode step of a batch whose sequences share a long system prompt
        dict(name="prefix_token", op="attend", B=64, H=16, Lq=1, R=512, Dr=64, cap=2048, lo=1, hi=2048, prefix=16384,
             dtype="bf16", ragged=False),
        # drafts behind a shared document of odd length
        dict(name="prefix_draft", op="attend", B=12, H=12, Lq=3, R=256, Dr=32, cap=640, lo=3, hi=640, prefix=4001,
             dtype="f16", ragged=True),
        # a prompt read with expanded keys and values
        dict(name="prompt", op="sdpa", B=4, H=16, L=4099, S=4099, Dn=128, Dr=64, causal=True, dtype="bf16", ragged=False,
             grad=False),
        # short prompts of different lengths in one padded batch
        dict(name="prompt_ragged", op="sdpa", B=6, H=8, L=517, S=517, Dn=64, Dr=32, causal=True, dtype="f16", ragged=True,
             grad=False),
        # a training step of one layer: output and the gradients of q, k, the shared rotary key and v
        dict(name="train", op="sdpa", B=2, H=16, L=4096, S=4096, Dn=128, Dr=64, causal=True, dtype="bf16", ragged=False,
             grad=True),
        # the same on a padded batch of odd lengths, without a causal mask
        dict(name="train_ragged", op="sdpa", B=3, H=12, L=1023, S=1023, Dn=64, Dr=32, causal=False, dtype="f16",
             ragged=True, grad=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prefix", "sdpa", "sdpa"])
    R, Dr = rng.choice([(128, 32), (192, 32), (256, 32), (256, 64), (320, 48), (512, 64), (512, 64)])
    dtype = rng.choice(["bf16", "f16"])
    ragged = rng.random() < 0.5
    if op == "append":
        n = rng.choice([1, _log(rng, 1, 4096)])
        cap = n + _log(rng, 64, 4000)
        return dict(op=op, B=max(1, min(_log(rng, 1, 64), 32768 // n)), n=n, R=R, Dr=Dr, cap=cap, lo=0, hi=cap - n,
                    mode=rng.choice([0, 2]), freq_scale=rng.choice([1.0, 0.25]), dtype=dtype, ragged=ragged)
    if op == "sdpa":
        Dn, Dr = rng.choice([(128, 64), (128, 64), (128, 32), (64, 32), (64, 64)])
        L = _log(rng, 1, 4096)
        S = L if ragged or rng.random() < 0.6 else _log(rng, 1, 4096)
        H = rng.choice([1, 3, 8, 12, 16])
        B = max(1, min(_log(rng, 1, 16), (4 * 16 * 4096 * 4096) // (L * S * H)))
        return dict(op=op, B=B, H=H, L=L, S=S, Dn=Dn, Dr=Dr, causal=rng.random() < 0.7, dtype=dtype, ragged=ragged,
                    grad=rng.random() < 0.5 and B * H * L * S <= 2 * 16 * 4096 * 4096)
    H = rng.choice([1, 4, 8, 12, 16, 20, 32, 64, 72])
    if op == "prefix":
        Lq = rng.choice([1, 1, rng.randint(2, 6)])
        B = _log(rng, 2, 64)
        cap = _log(rng, max(Lq, 16), 2048)
        P = min(_log(rng, 64, 16384), (1 << 26) // (B * H * Lq))
        return dict(op="attend", B=B, H=H, Lq=Lq, R=R, Dr=Dr, cap=cap, lo=Lq, hi=cap, prefix=P, dtype=dtype, ragged=ragged)
    Lq = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 500)])
    cap = max(Lq + 1, _log(rng, 32, 32768 if Lq == 1 else 8192))
    B = max(1, min(_log(rng, 1, 64 if Lq < 9 else 4), (1 << 20) // cap, (1 << 29) // (cap * H * Lq)))
    return dict(op="attend", B=B, H=H, Lq=Lq, R=R, Dr=Dr, cap=cap, lo=max(Lq, cap // 8), hi=cap, prefix=0, dtype=dtype,
                ragged=ragged)


# ------------------------------------------------------------------ inputs

def _spread(lo, hi, n):
    """n whole numbers from lo to hi at equal distances: a batch's lengths, the same ones for every seed."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _mixed(values, gen):
    order = torch.randperm(len(values), device="cuda", generator=gen)
    return torch.tensor(values, dtype=torch.int32, device="cuda")[order]


def _counts(case, n):
    return _spread(max(1, n // 2), n, case["B"]) if case["ragged"] else None


def _latent_rows(shape, gen, dt):
    """Latents of unit size, as the norm before the cache leaves them, and rotary keys."""
    return torch.randn(shape, dtype=torch.float32 if math.prod(shape) < 1 << 28 else torch.float16, device="cuda",
                       generator=gen).to(dt)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, B, dt = case["op"], case["B"], DT[case["dtype"]]
    st = {"case": case}
    if op == "sdpa":
        H, L, S, Dn, Dr = (case[k] for k in ("H", "L", "S", "Dn", "Dr"))
        # q is a view of a projection's (B, L, heads, size) output, k and v the two parts of another's
        st["q"] = torch.randn((B, L, H, Dn + Dr), device="cuda", generator=gen).to(dt).transpose(1, 2)
        kv = torch.randn((B, S, H, 2 * Dn), device="cuda", generator=gen).to(dt)
        st["k"], st["v"] = kv[..., :Dn].transpose(1, 2), kv[..., Dn:].transpose(1, 2)
        st["k_rope"] = torch.randn((B, S, Dr), device="cuda", generator=gen).to(dt)
        st["seq_lens"] = _mixed(_counts(case, S), gen) if case["ragged"] else None
        if case["grad"]:
            for n in ("q", "k", "k_rope", "v"):
                st[n] = st[n].detach().requires_grad_()
            st["g"] = torch.randn((B, H, L, Dn), device="cuda", generator=gen).to(dt)
        return st
    R, Dr, cap = case["R"], case["Dr"], case["cap"]
    lens = _spread(case["lo"], case["hi"], B)
    st["lens"] = _mixed(lens, gen)
    st["rows"] = _latent_rows((B, cap, R + Dr), gen, dt)
    if op == "append":
        n = case["n"]
        # the latent and the rotary key are the two parts of one projection's output
        x = torch.randn((B, n, R + Dr), device="cuda", generator=gen).to(dt)
        st["latent"], st["k_rope"] = x[..., :R], x[..., R:]
        st["counts"] = _mixed(_counts(case, n), gen) if case["ragged"] else None
        return st
    H, Lq, P = case["H"], case["Lq"], case["prefix"]
    # rows behind the lengths hold what earlier sequences left, NaN among it
    past = torch.arange(cap, device="cuda")[None, :] >= st["lens"][:, None]
    st["rows"].masked_fill_(past[..., None] & (torch.arange(R + Dr, device="cuda") % 3 == 0), float("nan"))
    st["q"] = torch.randn((B, Lq, H, R + Dr), device="cuda", generator=gen).to(dt).transpose(1, 2)
    st["scale"] = 1.0 / math.sqrt(128 + Dr)
    # a sequence has at least as many rows as it has new tokens
    st["counts"] = _mixed(_counts(case, Lq), gen) if case["ragged"] else None
    if P:
        st["prefix_rows"] = _latent_rows((1, P, R + Dr), gen, dt)
        st["prefix_lens"] = torch.full((1,), P, dtype=torch.int32, device="cuda")
    return st


# ------------------------------------------------------------------ one pass

def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _handle(st, name="cache"):
    """The cache handle that a program keeps next to its tensors, made at the first call."""
    if name not in st:
        from gguf_train_b200 import LatentCache
        p = "prefix_" if name == "prefix" else ""
        st[name] = LatentCache(st[p + "rows"], st[p + "lens"], st["case"]["R"])
    return st[name]


def _own_append(st):
    from gguf_train_b200 import latent_append
    c = st["case"]
    latent_append(_handle(st), st["latent"], st["k_rope"], counts=st["counts"], advance=False,
                  rope=dict(mode=c["mode"], freq_scale=c["freq_scale"]))
    return st["rows"]


def _own_attend(st):
    from gguf_train_b200 import latent_attention
    prefix = _handle(st, "prefix") if st["case"]["prefix"] else None
    return latent_attention(st["q"], _handle(st), st["scale"], counts=st["counts"], prefix=prefix, need_lse=True)


def _own_sdpa(st):
    from gguf_train_b200 import latent_sdpa
    c = st["case"]
    out = latent_sdpa(st["q"], st["k"], st["k_rope"], st["v"], is_causal=c["causal"], seq_lens=st["seq_lens"])
    if not c["grad"]:
        return out
    return (out.detach(),) + torch.autograd.grad(out, (st["q"], st["k"], st["k_rope"], st["v"]), st["g"])


_OWN = {"append": _own_append, "attend": _own_attend, "sdpa": _own_sdpa}


# ------------------------------------------------------------------ plain forms, 32 bits

def _plain_append(st):
    c = st["case"]
    B, n, Dr, P = c["B"], c["n"], c["Dr"], c["Dr"] // 2
    i = torch.arange(n, device="cuda")
    at = st["lens"].long()[:, None] + i  # (B, n)
    # a far position's angle does not fit 32 bits
    freq = c["freq_scale"] * 10000.0 ** (-torch.arange(P, dtype=torch.float64, device="cuda") / P)
    angle = at[..., None].double() * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    x = st["k_rope"].float()
    if c["mode"] == 0:
        x0, x1 = x[..., 0::2], x[..., 1::2]
        y = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), dim=-1).flatten(-2)
    else:
        x0, x1 = x[..., :P], x[..., P:]
        y = torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), dim=-1)
    new = torch.cat((st["latent"], y.to(st["latent"].dtype)), dim=-1)
    if st["counts"] is None:
        b = torch.arange(B, device="cuda")[:, None].expand(B, n)
        st["rows"][b, at] = new
    else:
        live = torch.nonzero(i < st["counts"][:, None], as_tuple=True)
        st["rows"][live[0], at[live]] = new[live]
    return st["rows"]


def _plain_attend(st):
    c = st["case"]
    B, H, Lq, R, cap, P = (c[k] for k in ("B", "H", "Lq", "R", "cap", "prefix"))
    lens = st["lens"].long()
    counts = torch.full_like(lens, Lq) if st["counts"] is None else st["counts"].long()
    s, i = torch.arange(cap, device="cuda"), torch.arange(Lq, device="cuda")
    held = (s < lens[:, None])[..., None]
    rows = torch.where(held, st["rows"], torch.zeros((), dtype=st["rows"].dtype, device="cuda")).float()
    q = st["q"].float().reshape(B, H * Lq, -1)
    live = i < counts[:, None]  # (B, Lq)
    limit = torch.where(live, lens[:, None] - counts[:, None] + i + 1, torch.zeros_like(i))
    seen = (s < limit[..., None])[:, None]  # (B, 1, Lq, cap)
    x = torch.matmul(q, rows.transpose(1, 2)).view(B, H, Lq, cap) * st["scale"]
    x = x.masked_fill(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    if P:
        shared = st["prefix_rows"][0].float()
        y = torch.matmul(q.reshape(B * H * Lq, -1), shared.t()).view(B, H, Lq, P) * st["scale"]
        y = y.masked_fill(~live[:, None, :, None], float("-inf"))
        top = torch.maximum(top, y.amax(-1, keepdim=True))
    base = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    x = torch.exp(x - base)
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(B, H * Lq, cap), rows[..., :R]).view(B, H, Lq, R)
    if P:
        y = torch.exp(y - base)
        total = total + y.sum(-1, keepdim=True)
        out = out + torch.matmul(y.view(B * H * Lq, P), shared[:, :R]).view(B, H, Lq, R)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return out.to(st["q"].dtype), (torch.log(total) + top)[..., 0]


def _plain_sdpa(st):
    c = st["case"]
    B, H, L, S, Dn, Dr = (c[k] for k in ("B", "H", "L", "S", "Dn", "Dr"))
    scale = 1.0 / math.sqrt(Dn + Dr)
    t, s = torch.arange(L, device="cuda"), torch.arange(S, device="cuda")
    q, k, v = (st[n].detach().float() for n in ("q", "k", "v"))
    k = torch.cat((k, st["k_rope"].detach().float()[:, None].expand(B, H, S, Dr)), dim=-1)
    drop = s[None, :] > t[:, None] if c["causal"] else torch.zeros((L, S), dtype=torch.bool, device="cuda")
    if st["seq_lens"] is not None:
        pad = s >= st["seq_lens"][:, None]  # (B, S)
        drop = (drop | pad[:, None, :] | pad[:, :, None])[:, None]
        # padded tokens take no part, whatever they hold
        q, k, v = (torch.where(pad[:, None, :, None], torch.zeros_like(z), z) for z in (q, k, v))
    p = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(drop, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(p, v)
    dt = st["q"].dtype
    if not c["grad"]:
        return o.to(dt)
    g = st["g"].float()
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = torch.matmul(g, v.transpose(2, 3)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dk = torch.matmul(ds.transpose(2, 3), q)
    grads = torch.matmul(ds, k), dk[..., :Dn], dk[..., Dn:].sum(1), dv
    return (o.to(dt),) + tuple(z.to(dt) for z in grads)


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "sdpa": _plain_sdpa}


# ------------------------------------------------------------------ exact values, 64 bits

def _exact_append(st):
    c = st["case"]
    rows = st["rows"].double()
    half = c["Dr"] // 2
    pair = torch.arange(half, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        n = c["n"] if st["counts"] is None else int(st["counts"][b])
        first = int(st["lens"][b])
        pos = torch.arange(first, first + n, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((n, half), dtype=torch.float64, device="cuda"),
                           pos[:, None] * c["freq_scale"] * torch.exp(-pair / half * math.log(10000.0)))
        x = st["k_rope"][b, :n].double()
        z = torch.complex(x[:, 0::2], x[:, 1::2]) if c["mode"] == 0 else torch.complex(x[:, :half], x[:, half:])
        z = z * turn
        rows[b, first:first + n, :c["R"]] = st["latent"][b, :n].double()
        if c["mode"] == 0:
            rows[b, first:first + n, c["R"]::2] = z.real
            rows[b, first:first + n, c["R"] + 1::2] = z.imag
        else:
            rows[b, first:first + n, c["R"]:c["R"] + half] = z.real
            rows[b, first:first + n, c["R"] + half:] = z.imag
    return rows


def _exact_attend(st):
    c = st["case"]
    B, H, Lq, R = c["B"], c["H"], c["Lq"], c["R"]
    out = torch.zeros((B, H, Lq, R), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, Lq), float("-inf"), dtype=torch.float64, device="cuda")
    shared = st["prefix_rows"][0].double() if c["prefix"] else None
    for b in range(B):
        n = int(st["lens"][b])
        m = Lq if st["counts"] is None else int(st["counts"][b])
        keys = st["rows"][b, :n].double()
        if shared is not None:
            keys = torch.cat((shared, keys))
        q = st["q"][b, :, :m].double()
        for h0 in range(0, H, 8):
            x = torch.einsum("hid,sd->his", q[h0:h0 + 8], keys) * st["scale"]
            own_end = keys.shape[0] - m + torch.arange(m, device="cuda")
            x.masked_fill_(torch.arange(keys.shape[0], device="cuda") > own_end[:, None], float("-inf"))
            z = torch.logsumexp(x, -1)
            lse[b, h0:h0 + 8, :m] = z
            out[b, h0:h0 + 8, :m] = torch.einsum("his,sd->hid", torch.exp(x - z[..., None]), keys[:, :R])
    return out, lse


def _exact_sdpa(st):
    c = st["case"]
    B, H, L, S, Dn, Dr = (c[k] for k in ("B", "H", "L", "S", "Dn", "Dr"))
    z = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, dq, dk, dkr, dv = z(B, H, L, Dn), z(B, H, L, Dn + Dr), z(B, H, S, Dn), z(B, S, Dr), z(B, H, S, Dn)
    scale = (Dn + Dr) ** -0.5
    for b in range(B):
        n = None if st["seq_lens"] is None else int(st["seq_lens"][b])
        l, m = (L, S) if n is None else (n, n)
        kr = st["k_rope"].detach()[b, :m].double()
        for h in range(H):
            q, k, v = st["q"].detach()[b, h, :l].double(), st["k"].detach()[b, h, :m].double(), st["v"].detach()[b, h, :m].double()
            x = (q[:, :Dn] @ k.t() + q[:, Dn:] @ kr.t()) * scale
            if c["causal"]:
                x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(1), float("-inf"))
            p = torch.softmax(x, -1)
            out[b, h, :l] = p @ v
            if c["grad"]:
                g = st["g"][b, h, :l].double()
                dv[b, h, :m] = p.t() @ g
                dp = g @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[b, h, :l, :Dn], dq[b, h, :l, Dn:] = ds @ k, ds @ kr
                dk[b, h, :m] = ds.t() @ q[:, :Dn]
                dkr[b, :m] += ds.t() @ q[:, Dn:]
    return (out, dq, dk, dkr, dv) if c["grad"] else out


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sdpa": _exact_sdpa}[case["op"]](st)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    """Each input read once and each output written once; products of allowed (query, key) pairs."""
    B = case["B"]
    if case["op"] == "append":
        tokens = sum(_counts(case, case["n"]) or [case["n"]] * B)
        return {"bytes": 2 * 2 * tokens * (case["R"] + case["Dr"]), "flops": 3 * tokens * case["Dr"]}
    if case["op"] == "attend":
        H, Lq, R, Dr, P = (case[k] for k in ("H", "Lq", "R", "Dr", "prefix"))
        lens, counts = _spread(case["lo"], case["hi"], B), _counts(case, Lq) or [Lq] * B
        queries = sum(counts)
        mean = sum(lens) / B
        pairs = sum(P + mean - (m - 1) / 2 for m in counts for _ in range(m))
        return {"bytes": 2 * (R + Dr) * (sum(lens) + P) + H * queries * (2 * (R + Dr) + 2 * R + 4),
                "flops": 2 * H * (2 * R + Dr) * pairs}
    H, L, S, Dn, Dr = (case[k] for k in ("H", "L", "S", "Dn", "Dr"))
    pairs, values = 0, 0
    for n in _counts(case, S) or [None] * B:
        l, m = (L, S) if n is None else (n, n)
        pairs += sum(min(i + 1, m) for i in range(l)) if case["causal"] else l * m
        q, k, r, v, o = H * l * (Dn + Dr), H * m * Dn, m * Dr, H * m * Dn, H * l * Dn
        values += (2 * (q + k + r + v) + 2 * o) if case["grad"] else q + k + r + v + o
    per_pair = 2 * (Dn + Dr + Dn) + (2 * (3 * (Dn + Dr) + 2 * Dn) if case["grad"] else 0)
    return {"bytes": 2 * values, "flops": H * pairs * per_pair}
