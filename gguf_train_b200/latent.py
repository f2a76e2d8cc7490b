"""Latent attention: of each token one latent vector, from which every head's keys and values are made, and one rotary
key that the heads share.

    out = latent_sdpa(q, k, k_rope, v, is_causal=True)                         # prompts and training: keys and values expanded
    cache = LatentCache.empty(batch, capacity, latent_dim=512, rope_dim=64)    # bf16, or dtype=torch.float16
    latent_append(cache, latent, k_rope, rope=dict(mode=2))                    # (B, n, latent_dim), (B, n, rope_dim)
    out = latent_attention(q, cache, scale)                                    # q (B, H, Lq, latent_dim + rope_dim): absorbed

With W_k (heads, Dn, R) and W_v (heads, Dv, R) the up-projections of a latent c, the expanded form attends keys
[W_k c | k_rope] and values W_v c. The absorbed form takes the query through W_k instead, q = [q_nope W_k | q_rope], attends the
cached rows [c | k_rope] themselves, whose latents are the values too, and leaves W_v to the caller's next product: a
decode step reads R + Dr values a cached token for all of its heads. Both give the same attention.

Scores, their maxima and sums, and outputs accumulate in f32. With 16-bit inputs the softmax weights, and in latent_sdpa's backward the
scores' gradients too, are rounded once to the inputs' type before the tensor cores multiply them.

Tensors are torch CUDA tensors; every call runs in the native library on the caller's current stream
(include/gtb_attn.h has the exact definitions). A cache is mutable state: calls that change it, and calls that
read it, are ordered by the streams they are issued on. latent_append and latent_attention serve and have no gradient: they
refuse tensors that require one while gradients are recorded, and those of forward mode; latent_sdpa is differentiable.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.forward_ad import unpack_dual

from . import _C
from .functional import _autocast_lower, _require_cuda, scaled_dot_product_attention
from .kv8 import _CODE, _counts, _stream, _unit_inner

_STORED = (torch.bfloat16, torch.float16)


class LatentCache:
    """The tensors of a latent cache: rows (B, capacity, latent_dim + rope_dim) f16 or bf16, a row a token's latent followed by
    its rotary key, and lens (B) int32, the rows each sequence holds. Contiguous, on one CUDA device; latent_dim a
    multiple of 64 from 64 to 512, rope_dim a multiple of 16 from 16 to 64. Their contents may be changed freely, and a
    tensor may be replaced by one of the same shape and type (cache.lens = cache.lens - rejected)."""

    __slots__ = ("_rows", "_lens", "_latent_dim", "_native")
    latent_dim = property(lambda self: self._latent_dim, doc="size of a latent")
    rope_dim = property(lambda self: self._rows.shape[2] - self._latent_dim, doc="size of a rotary key")
    capacity = property(lambda self: self._rows.shape[1], doc="rows a sequence can hold")

    def __init__(self, rows: torch.Tensor, lens: torch.Tensor, latent_dim: int) -> None:
        _require_cuda("LatentCache", rows, lens)
        latent_dim = int(latent_dim)
        if rows.ndim != 3 or rows.dtype not in _STORED or not rows.is_contiguous():
            raise RuntimeError("LatentCache: rows must be a contiguous f16 or bf16 tensor (B, capacity, latent_dim + rope_dim)")
        rope_dim = rows.shape[2] - latent_dim
        if latent_dim % 64 or not 64 <= latent_dim <= 512:
            raise RuntimeError(f"LatentCache: latent_dim must be a multiple of 64 from 64 to 512, got {latent_dim}")
        if rope_dim % 16 or not 16 <= rope_dim <= 64:
            raise RuntimeError(f"LatentCache: the rotary key must have a multiple of 16 values from 16 to 64, got {rope_dim}")
        if lens.dtype != torch.int32 or tuple(lens.shape) != (rows.shape[0],) or not lens.is_contiguous():
            raise RuntimeError(f"LatentCache: lens must be a contiguous int32 tensor of shape ({rows.shape[0]},)")
        if lens.device != rows.device:
            raise RuntimeError("LatentCache: all tensors must be on one device")
        self._rows, self._lens, self._latent_dim = rows, lens, latent_dim
        self._native = _C.Latent(rows.data_ptr(), lens.data_ptr(), rows.shape[0], rows.shape[1], latent_dim, rope_dim,
                                 _CODE[rows.dtype])

    @classmethod
    def empty(cls, batch: int, capacity: int, latent_dim: int, rope_dim: int, dtype=torch.bfloat16,
              device="cuda") -> "LatentCache":
        """A cache that holds no rows."""
        if dtype not in _STORED:
            raise RuntimeError("LatentCache: dtype must be torch.bfloat16 or torch.float16")
        return cls(torch.empty((batch, capacity, latent_dim + rope_dim), dtype=dtype, device=device),
                   torch.zeros(batch, dtype=torch.int32, device=device), latent_dim)

    def _put(self, slot: str, name: str, t: torch.Tensor) -> None:
        old = getattr(self, slot)
        if not isinstance(t, torch.Tensor) or t.shape != old.shape or t.dtype != old.dtype or t.device != old.device or \
                not t.is_contiguous():
            raise RuntimeError(f"LatentCache: {name} can only be replaced by a contiguous {old.dtype} tensor of shape "
                               f"{list(old.shape)} on {old.device}; make a new LatentCache for others")
        setattr(self._native, name, t.data_ptr())
        setattr(self, slot, t)

    rows = property(lambda self: self._rows, lambda self, t: self._put("_rows", "rows", t))
    lens = property(lambda self: self._lens, lambda self, t: self._put("_lens", "lens", t))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self._rows, self._lens))


def _same_device(name: str, cache: LatentCache, *ts) -> None:
    for t in ts:
        if t is not None and t.device != cache._rows.device:
            raise RuntimeError(f"{name}: a tensor is on {t.device}, the cache on {cache._rows.device}")


def _prefix(name: str, cache: LatentCache, prefix: LatentCache | None) -> None:
    if prefix is None:
        return
    _same_device(name, cache, prefix._rows)
    if prefix._rows.shape[0] != 1 or prefix._rows.shape[2] != cache._rows.shape[2] or \
            prefix._latent_dim != cache._latent_dim or prefix._rows.dtype != cache._rows.dtype:
        raise RuntimeError(f"{name}: the prefix must be a LatentCache of one sequence with the cache's sizes and type")


def _no_gradient(name: str, *ts) -> None:
    """Refuse tensors whose gradients or tangents a serving call would drop."""
    # (a tangent exists only within a level of forward mode: asking the tensors takes 0.9 us each, this 0.1)
    dual = forward_ad._current_level >= 0
    if torch.is_grad_enabled() or dual:
        for t in ts:
            if t.requires_grad and torch.is_grad_enabled() or dual and unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name}: serves and has no gradient; call it under torch.no_grad() or with detached tensors "
                                   f"(latent_sdpa is differentiable)")


def latent_append(cache: LatentCache, latent: torch.Tensor, k_rope: torch.Tensor, counts: torch.Tensor | None = None,
                  advance: bool = True, rope: dict | None = None, prefix: LatentCache | None = None) -> LatentCache:
    """Append latent (B, n, latent_dim) and k_rope (B, n, rope_dim) (f32, f16 or bf16, any layout) behind each sequence's
    cache.lens[b] rows and, with `advance`, increase lens. counts (int32, B) takes only the first counts[b] rows of
    sequence b (prompts padded to one length).

    With `rope` (a dict of mode, 0 or 2, freq_base and freq_scale) k_rope is first rotated for its position, lens[b] + i;
    behind a `prefix` that the batch shares, prefix.lens[0] + lens[b] + i (that length as it is, even where the prefix's tensor
    holds fewer rows). The rotation is rope_axes' over all of rope_dim. Tensors that require a gradient while gradients are
    recorded are refused. Rows past the capacity are dropped and leave status 62 (_C.device_status()). Returns cache."""
    _require_cuda("latent_append", latent, k_rope, counts)
    _same_device("latent_append", cache, latent, k_rope, counts)
    _no_gradient("latent_append", latent, k_rope, cache._rows)
    _prefix("latent_append", cache, prefix)
    B, R, Dr = cache._rows.shape[0], cache._latent_dim, cache.rope_dim
    if latent.ndim != 3 or k_rope.ndim != 3 or (latent.shape[0], latent.shape[2]) != (B, R) or \
            tuple(k_rope.shape) != (B, latent.shape[1], Dr):
        raise RuntimeError(f"latent_append: latent must be ({B}, n, {R}) and k_rope ({B}, n, {Dr}), got "
                           f"{list(latent.shape)} and {list(k_rope.shape)}")
    if latent.dtype not in _CODE or k_rope.dtype != latent.dtype:
        raise RuntimeError("latent_append: latent and k_rope must be f32, f16 or bf16, of one type")
    mode, base, scale = -1, 10000.0, 1.0
    if rope is not None:
        r = {"mode": 0, "freq_base": base, "freq_scale": scale}
        if not set(rope) <= set(r):
            raise RuntimeError(f"latent_append: rope takes {sorted(r)}, got {sorted(rope)}")
        r.update(rope)
        mode, base, scale = int(r["mode"]), float(r["freq_base"]), float(r["freq_scale"])
        if mode not in (0, 2):
            raise RuntimeError(f"latent_append: mode must be 0 (normal) or 2 (NeoX), got {mode}")
    latent, k_rope = _unit_inner(latent), _unit_inner(k_rope)
    code = _CODE[latent.dtype]
    rc = _C.lib.gtb_latent_append(ctypes.byref(cache._native), _C.tensor4(latent[:, None], code),
                                  _C.tensor4(k_rope[:, None], code), _counts("latent_append", counts, B),
                                  None if prefix is None else prefix._lens.data_ptr(), mode, base, scale,
                                  1 if advance else 0, _stream(cache._rows.device))
    _C.check_rc(rc, "latent_append")
    return cache


def _tiled(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its rows do not start on 16 bytes."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and \
            all(n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride())):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(t: torch.Tensor, code: int):
    """_tiled(t), and the tensor4 of it (of k_rope with a dimension for its one head)."""
    s, p = t.stride(), t.data_ptr()
    if s[-1] != 1 or (p | s[0] << 1 | s[1] << 1 | s[-2] << 1) & 15 or min(s) <= 0:
        t = _tiled(t)
        s, p = t.stride(), t.data_ptr()
    n = t.shape
    if len(n) == 4:
        return t, _C._pack4(p, *n, *s, code)
    return t, _C._pack4(p, n[0], 1, n[1], n[2], s[0], s[0], s[1], s[2], code)


def latent_attention(q: torch.Tensor, cache: LatentCache, scale: float, counts: torch.Tensor | None = None,
                     prefix: LatentCache | None = None, need_lse: bool = False):
    """Causal attention of q (B, H, Lq, latent_dim + rope_dim), in the cache's type, over the cache, which already holds the
    queries' own rows: the queries are the last Lq of each sequence's cache.lens[b] tokens (the last counts[b], q's first
    counts[b] rows, where counts is given), and query i attends every row up to its own. scale is that of the expanded
    form, 1 / sqrt(Dn + Dr): the cache does not know it. Lq = 1 is a decode step, a few a draft to verify, many a
    chunk of a prompt. Returns (B, H, Lq, latent_dim), the weights' sums of latents, or (out, lse) with need_lse, lse
    (B, H, Lq) float32; a query with nothing to attend gives 0 and -inf.

    prefix: a LatentCache of one sequence whose rows come before every sequence's own, as those of a system prompt; each
    sequence's cache holds only what follows. Sequences of at most 32 query rows (H * Lq) read the prefix together, as many
    as fill 64 rows; longer ones each for every 64 of their rows.

    No gradient is formed: tensors that require one while gradients are recorded are refused."""
    _require_cuda("latent_attention", q, counts)
    _same_device("latent_attention", cache, q, counts)
    _no_gradient("latent_attention", q, cache._rows, *(() if prefix is None else (prefix._rows,)))
    _prefix("latent_attention", cache, prefix)
    B, _, D = cache._rows.shape
    if q.ndim != 4 or q.shape[0] != B or q.shape[3] != D:
        raise RuntimeError(f"latent_attention: q must be ({B}, H, Lq, {D}), got {list(q.shape)}")
    if q.dtype != cache._rows.dtype:
        raise RuntimeError(f"latent_attention: q must be of the cache's type {cache._rows.dtype}, got {q.dtype}")
    scale = float(scale)
    if not 0.0 < scale < 1e38:
        raise RuntimeError(f"latent_attention: scale must be positive and below 1e38, got {scale}")
    code = _CODE[q.dtype]
    q, qt = _rows(q, code)
    H, Lq = q.shape[1:3]
    out = torch.empty((B, H, Lq, cache._latent_dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Lq), dtype=torch.float32, device=q.device) if need_lse else None
    rc = _C.lib.gtb_latent_attention(qt, ctypes.byref(cache._native),
                                     None if prefix is None else ctypes.byref(prefix._native), scale,
                                     _counts("latent_attention", counts, B), _C.tensor4(out, code),
                                     None if lse is None else lse.data_ptr(), _stream(q.device))
    _C.check_rc(rc, "latent_attention")
    return (out, lse) if need_lse else out


def _sdpa_general(q, k, k_rope, v, is_causal, scale, seq_lens):
    """latent_sdpa by scaled_dot_product_attention, the rotary key repeated for each head."""
    keys = torch.cat((k, k_rope[:, None].expand(-1, k.shape[1], -1, -1)), dim=-1)
    if seq_lens is None:
        return scaled_dot_product_attention(q, keys, v, is_causal=is_causal, scale=scale)
    held = torch.arange(k.shape[2], device=q.device) < seq_lens[:, None]  # (B, S)
    # padded tokens take no part, whatever they hold
    q, keys, v = (torch.where(held[:, None, :, None], t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (q, keys, v))
    out = scaled_dot_product_attention(q, keys, v, held[:, None, None], is_causal=is_causal, scale=scale)
    return torch.where(held[:, None, :, None], out, torch.zeros((), dtype=out.dtype, device=out.device))


def _on_tensor_cores(q, k, k_rope, v) -> bool:
    """The sizes that the native expanded kernels take; others go by scaled_dot_product_attention."""
    Dn, Dr = k.shape[3], k_rope.shape[2]
    return q.dtype in _STORED and Dn in (64, 128) and v.shape[3] == Dn and Dr % 16 == 0 and 16 <= Dr <= 64 and \
        q.shape[0] <= 65535 and q.shape[1] <= 65535 and min(q.shape) > 0 and min(k.shape) > 0


class LatentSDPAFn(torch.autograd.Function):
    """latent_sdpa on the native kernels: apply(q, k, k_rope, v, is_causal, scale, seq_lens). The backward recomputes the weights
    from the saved log-sum-exp."""

    @staticmethod
    def _forward(q, k, k_rope, v, is_causal, scale, seq_lens, need_lse):
        code = _CODE[q.dtype]
        (q, qt), (k, kt), (kr, rt), (v, vt) = _rows(q, code), _rows(k, code), _rows(k_rope, code), _rows(v, code)
        B, H, L, _ = q.shape
        out = torch.empty((B, H, L, v.shape[3]), dtype=q.dtype, device=q.device)
        lse = torch.empty((B, H, L), dtype=torch.float32, device=q.device) if need_lse else None
        rc = _C.lib.gtb_latent_sdpa_fwd(qt, kt, rt, vt, None if seq_lens is None else seq_lens.data_ptr(), scale,
                                        1 if is_causal else 0, _C.tensor4(out, code), None if lse is None else lse.data_ptr(),
                                        _stream(q.device))
        _C.check_rc(rc, "latent_sdpa")
        return q, k, kr, v, out, lse

    @staticmethod
    def forward(ctx, q, k, k_rope, v, is_causal, scale, seq_lens):
        q, k, kr, v, out, lse = LatentSDPAFn._forward(q, k, k_rope, v, is_causal, scale, seq_lens, True)
        ctx.args = is_causal, scale
        ctx.save_for_backward(q, k, kr, v, out, lse, seq_lens)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, kr, v, out, lse, seq_lens = ctx.saved_tensors
        is_causal, scale = ctx.args
        code = _CODE[q.dtype]
        g, gt = _rows(grad_out, code)
        # (hooks on saved tensors may have brought them back in other places)
        (q, qt), (k, kt), (kr, rt), (v, vt), (out, ot) = [_rows(t, code) for t in (q, k, kr, v, out)]
        # (in the inputs' layouts where those are dense, as q's as a view of its projection; all of them start on 16 bytes)
        dq, dk, dkr, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(kr), torch.empty_like(v)
        rc = _C.lib.gtb_latent_sdpa_bwd(gt, qt, kt, rt, vt, ot, lse.data_ptr(),
                                        None if seq_lens is None else seq_lens.data_ptr(), scale, 1 if is_causal else 0,
                                        _C.tensor4(dq, code), _C.tensor4(dk, code), _rows(dkr, code)[1], _C.tensor4(dv, code),
                                        _stream(q.device))
        _C.check_rc(rc, "latent_sdpa_bwd")
        return dq, dk, dkr, dv, None, None, None


def latent_sdpa(q: torch.Tensor, k: torch.Tensor, k_rope: torch.Tensor, v: torch.Tensor, is_causal: bool = False,
                scale: float | None = None, seq_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention whose keys have a part of their own for each head and a rotary part that the heads share: q (B, H, L, Dn + Dr),
    k (B, Hkv, S, Dn), k_rope (B, S, Dr), v (B, Hkv, S, Dv), H a multiple of Hkv; scores scale * (q[..., :Dn] . k +
    q[..., Dn:] . k_rope), scale 1 / sqrt(Dn + Dr) if not given, top-left causal masking as in
    scaled_dot_product_attention. Returns (B, H, L, Dv), differentiable in all four.

    16-bit inputs with Dn = Dv of 64 or 128 and Dr a multiple of 16 up to 64 have kernels of their own, whose gradients have the same
    bits on every run; other sizes, and f32, go by scaled_dot_product_attention with k_rope repeated for each head.

    seq_lens (int32, B; L = S) is for prompts padded to one length: tokens from seq_lens[b] on (which may hold anything) are not
    attended, give 0 and get zero gradients."""
    lowered, cast = _autocast_lower(q, k, k_rope, v)
    if cast:
        with torch.autocast("cuda", enabled=False):
            return latent_sdpa(*lowered, is_causal=is_causal, scale=scale, seq_lens=seq_lens)
    _require_cuda("latent_sdpa", q, k, k_rope, v, seq_lens)
    qs, ks, rs, vs, dt, dev = q.shape, k.shape, k_rope.shape, v.shape, q.dtype, q.device
    if len(qs) != 4 or len(ks) != 4 or len(rs) != 3 or len(vs) != 4:
        raise RuntimeError("latent_sdpa: q, k and v must have four dimensions and k_rope three")
    B, H, L, D = qs
    _, Hkv, S, Dn = ks
    Dr = D - Dn
    if ks[0] != B or vs[:3] != ks[:3] or rs != (B, S, Dr) or Dr < 1 or Dn < 1:
        raise RuntimeError(f"latent_sdpa: q (B, H, L, Dn + Dr), k (B, Hkv, S, Dn), k_rope (B, S, Dr) and v (B, Hkv, S, Dv) do not "
                           f"fit together: {list(qs)}, {list(ks)}, {list(rs)}, {list(vs)}")
    if Hkv == 0 or H % Hkv:
        raise RuntimeError(f"latent_sdpa: num_heads ({H}) must be divisible by num_kv_heads ({Hkv})")
    if k.dtype != dt or k_rope.dtype != dt or v.dtype != dt or dt not in _CODE:
        raise RuntimeError("latent_sdpa: q, k, k_rope and v must be f32, f16 or bf16, of one type")
    if k.device != dev or k_rope.device != dev or v.device != dev or (seq_lens is not None and seq_lens.device != dev):
        raise RuntimeError("latent_sdpa: all tensors must be on one device")
    if seq_lens is not None:
        if L != S:
            raise RuntimeError(f"latent_sdpa: seq_lens needs as many queries as keys, got {L} and {S}")
        if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,) or not seq_lens.is_contiguous():
            raise RuntimeError(f"latent_sdpa: seq_lens must be a contiguous int32 tensor of shape ({B},)")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 1e38:
        raise RuntimeError(f"latent_sdpa: scale must be positive and below 1e38, got {scale}")
    if not _on_tensor_cores(q, k, k_rope, v):
        return _sdpa_general(q, k, k_rope, v, bool(is_causal), scale, seq_lens)
    xs = (q, k, k_rope, v)
    # (tensors of forward mode take the Function too, which refuses them)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or k_rope.requires_grad or v.requires_grad) or \
            any([unpack_dual(t).tangent is not None for t in xs]):
        return LatentSDPAFn.apply(*xs, bool(is_causal), scale, seq_lens)
    return LatentSDPAFn._forward(*xs, bool(is_causal), scale, seq_lens, False)[4]
