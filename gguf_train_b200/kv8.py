"""A KV cache held in 8 bits with one scale for each block of tokens and kv head, and what runs on it.

    cache = KV8Cache.empty(batch, kv_heads, capacity, head_dim, block=64)      # int8, or dtype=torch.float8_e4m3fn
    kv8_append(cache, k, v)                                                    # (B, Hkv, n, D), n from 1 to a prompt
    out = kv8_attention(q, cache, score=score)                                 # q (B, H, Lq, D): the last Lq tokens
    small, score, kept = kv8_evict(cache, score, budget, recent=128)           # by accumulated attention weight

A value is code * scale; the largest code is 127 (int8) or 448 (e4m3). Half the bytes of a 16-bit cache, and
unlike Q8_0 (a scale per 32 values, 34-byte blocks; decode_q8_0) rows stay 16-byte aligned and the scales
cost 4 / (block * D) bytes per value. Tensors are torch CUDA tensors; every call runs in the native library
on the caller's current stream (include/gtb_attn.h has the exact definitions). A cache is mutable state: calls
that change it, and calls that read it, are ordered by the streams they are issued on.
"""

from __future__ import annotations

import ctypes

import torch

from . import _C
from .functional import _require_cuda

_FORMAT = {torch.int8: _C.GTB_KV8_INT8, torch.float8_e4m3fn: _C.GTB_KV8_E4M3}
_CODE = {torch.float32: _C.GT_F32, torch.float16: _C.GT_F16, torch.bfloat16: _C.GT_BF16}
BLOCKS = (16, 32, 64, 128)


def _t4(t: torch.Tensor) -> bytes:
    return _C.tensor4(t, _CODE[t.dtype])


def _stream(dev: torch.device) -> int:
    # the current stream's handle without making a torch.cuda.Stream of it (2 us of a call's 20)
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _unit_inner(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _same_device(name: str, cache: "KV8Cache", *ts) -> None:
    for t in ts:
        if t is not None and t.device != cache._k.device:
            raise RuntimeError(f"{name}: a tensor is on {t.device}, the cache on {cache._k.device}")


def _counts(name: str, counts, batch: int):
    if counts is None:
        return None
    if counts.dtype != torch.int32 or tuple(counts.shape) != (batch,) or not counts.is_contiguous():
        raise RuntimeError(f"{name}: counts must be a contiguous int32 tensor of shape ({batch},)")
    return counts.data_ptr()


def _tensor(name: str):
    """A tensor of a cache. One put in its place has to be like it; the native handle follows."""
    slot = "_" + name

    def get(self) -> torch.Tensor:
        return getattr(self, slot)

    def put(self, t: torch.Tensor) -> None:
        old = getattr(self, slot)
        if not isinstance(t, torch.Tensor) or t.shape != old.shape or t.dtype != old.dtype or t.device != old.device or \
                not t.is_contiguous():
            raise RuntimeError(f"KV8Cache: {name} can only be replaced by a contiguous {old.dtype} tensor of shape "
                               f"{list(old.shape)} on {old.device}; make a new KV8Cache for others")
        setattr(self._native, name, t.data_ptr())
        setattr(self, slot, t)

    return property(get, put)


class KV8Cache:
    """The tensors of an 8-bit cache: k, v (B, Hkv, capacity, D) int8 or float8_e4m3fn codes; k_scale, v_scale
    (B, Hkv, ceil(capacity / block)) float32; lens (B) int32, the rows each sequence holds. All contiguous, on
    one CUDA device; D a multiple of 16 up to 256, block 16, 32, 64 or 128. Their contents may be changed freely, and
    a tensor may be replaced by one of the same shape and type (cache.lens = cache.lens - rejected)."""

    __slots__ = ("_k", "_v", "_k_scale", "_v_scale", "_lens", "_block", "_native")
    k, v, k_scale, v_scale, lens = map(_tensor, ("k", "v", "k_scale", "v_scale", "lens"))
    block = property(lambda self: self._block, doc="tokens that share a scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 lens: torch.Tensor, block: int) -> None:
        _require_cuda("KV8Cache", k, v, k_scale, v_scale, lens)
        if k.ndim != 4 or v.shape != k.shape or k.dtype not in _FORMAT or v.dtype != k.dtype:
            raise RuntimeError("KV8Cache: k and v must be (B, Hkv, capacity, D) tensors of int8 or float8_e4m3fn")
        B, Hkv, cap, D = k.shape
        block = int(block)
        if block not in BLOCKS:
            raise RuntimeError(f"KV8Cache: block must be one of {BLOCKS}, got {block}")
        if D % 16 or not 16 <= D <= 256:
            raise RuntimeError(f"KV8Cache: the head size must be a multiple of 16 up to 256, got {D}")
        want = (B, Hkv, -(-cap // block))
        if tuple(k_scale.shape) != want or tuple(v_scale.shape) != want or k_scale.dtype != torch.float32 or \
                v_scale.dtype != torch.float32:
            raise RuntimeError(f"KV8Cache: k_scale and v_scale must be float32 tensors of shape {want}")
        if lens.dtype != torch.int32 or tuple(lens.shape) != (B,):
            raise RuntimeError(f"KV8Cache: lens must be an int32 tensor of shape ({B},)")
        for t in (k, v, k_scale, v_scale, lens):
            if not t.is_contiguous():
                raise RuntimeError("KV8Cache: all tensors must be contiguous")
            if t.device != k.device:
                raise RuntimeError("KV8Cache: all tensors must be on one device")
        self._k, self._v, self._k_scale, self._v_scale, self._lens, self._block = k, v, k_scale, v_scale, lens, block
        self._native = _C.KV8(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), lens.data_ptr(), B,
                              Hkv, cap, D, block, _FORMAT[k.dtype])

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, block: int = 64, dtype=torch.int8,
              device="cuda") -> "KV8Cache":
        """A cache that holds no rows."""
        if dtype not in _FORMAT:
            raise RuntimeError("KV8Cache: dtype must be torch.int8 or torch.float8_e4m3fn")
        if int(block) not in BLOCKS:
            raise RuntimeError(f"KV8Cache: block must be one of {BLOCKS}, got {block}")
        kv = [torch.empty((batch, kv_heads, capacity, head_dim), dtype=dtype, device=device) for _ in range(2)]
        sc = [torch.zeros((batch, kv_heads, -(-capacity // int(block))), dtype=torch.float32, device=device)
              for _ in range(2)]
        return cls(*kv, *sc, torch.zeros(batch, dtype=torch.int32, device=device), block)

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.lens))


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None,
               advance: bool = True) -> KV8Cache:
    """Append k, v (B, Hkv, n, D; f32, f16 or bf16, any layout) behind each sequence's cache.lens[b] rows and, with
    `advance`, increase lens. counts (int32, B) takes only the first counts[b] rows of sequence b (prompts
    padded to one length). A block's scale grows to hold its largest value, requantising the rows it already
    has where it does. Rows past the capacity are dropped and leave status 61 (_C.device_status()). Returns
    cache."""
    _require_cuda("kv8_append", k, v, counts)
    _same_device("kv8_append", cache, k, v, counts)
    B, Hkv, _, D = cache._k.shape
    if k.ndim != 4 or k.shape != v.shape or (k.shape[0], k.shape[1], k.shape[3]) != (B, Hkv, D):
        raise RuntimeError(f"kv8_append: k and v must be ({B}, {Hkv}, n, {D}), got {list(k.shape)} and {list(v.shape)}")
    if k.dtype not in _CODE or v.dtype != k.dtype:
        raise RuntimeError("kv8_append: k and v must be f32, f16 or bf16, of one type")
    k, v = _unit_inner(k), _unit_inner(v)
    rc = _C.lib.gtb_kv8_append(ctypes.byref(cache._native), _t4(k), _t4(v),
                               _counts("kv8_append", counts, B), 1 if advance else 0, _stream(k.device))
    _C.check_rc(rc, "kv8_append")
    return cache


def kv8_read(cache: KV8Cache, start: torch.Tensor | None, n: int, dtype=torch.float32):
    """Rows start[b] .. start[b] + n - 1 (int32, B; None: 0) of every head as values: (k, v), each (B, Hkv, n, D)
    in `dtype`. Stored rows come back whatever cache.lens says; rows outside the capacity are 0."""
    _require_cuda("kv8_read", start)
    _same_device("kv8_read", cache, start)
    if dtype not in _CODE:
        raise RuntimeError("kv8_read: dtype must be f32, f16 or bf16")
    B, Hkv, _, D = cache._k.shape
    if int(n) < 0:
        raise RuntimeError(f"kv8_read: the number of rows must not be negative, got {n}")
    k = cache._k_scale.new_empty((B, Hkv, int(n), D), dtype=dtype)
    v = torch.empty_like(k)
    rc = _C.lib.gtb_kv8_read(ctypes.byref(cache._native), _counts("kv8_read", start, B), _t4(k), _t4(v),
                             _stream(k.device))
    _C.check_rc(rc, "kv8_read")
    return k, v


def kv8_attention(q: torch.Tensor, cache: KV8Cache, scale: float | None = None, counts: torch.Tensor | None = None,
                  score: torch.Tensor | None = None, score_out: torch.Tensor | None = None, need_lse: bool = False):
    """Causal attention of q (B, H, Lq, D) over the cache, which already holds the queries' own keys: the queries
    are the last Lq of each sequence's cache.lens[b] tokens (the last counts[b], q's first counts[b] rows, where
    counts is given), and query i attends every row up to its own. Lq = 1 is a decode step, a few a draft to
    verify, many a chunk of a prompt. Returns (B, H, Lq, D) in q's dtype, or (out, lse) with need_lse, lse
    (B, H, Lq) float32; a query with nothing to attend gives 0 and -inf.

    score (B, Hkv, capacity) float32 accumulates the attention weight that each cached row got from all
    queries and the kv head's query heads: in place, or into score_out as score + weight for rows below
    cache.lens[b]. It is what kv8_evict goes by."""
    _require_cuda("kv8_attention", q, counts, score, score_out)
    _same_device("kv8_attention", cache, q, counts, score, score_out)
    B, Hkv, cap, D = cache._k.shape
    if q.ndim != 4 or q.shape[0] != B or q.shape[3] != D:
        raise RuntimeError(f"kv8_attention: q must be ({B}, H, Lq, {D}), got {list(q.shape)}")
    if q.dtype not in _CODE:
        raise RuntimeError("kv8_attention: q must be f32, f16 or bf16")
    if score is None and score_out is not None:
        raise RuntimeError("kv8_attention: score_out needs score")
    for t in (score, score_out):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (B, Hkv, cap) or not t.is_contiguous()):
            raise RuntimeError(f"kv8_attention: score must be a contiguous float32 tensor ({B}, {Hkv}, {cap})")
    q = _unit_inner(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty(q.shape[:3], dtype=torch.float32) if need_lse else None
    s_in = None if score is None else score.data_ptr()
    s_out = s_in if score_out is None else score_out.data_ptr()
    rc = _C.lib.gtb_kv8_attention(_t4(q), ctypes.byref(cache._native), 0.0 if scale is None else float(scale),
                                  _counts("kv8_attention", counts, B), s_in, s_out, _t4(out),
                                  None if lse is None else lse.data_ptr(), _stream(q.device))
    _C.check_rc(rc, "kv8_attention")
    return (out, lse) if need_lse else out


def kv8_evict(cache: KV8Cache, score: torch.Tensor, budget: int, recent: int = 0, out: KV8Cache | None = None,
              score_out: torch.Tensor | None = None):
    """Keep at most `budget` rows of every (sequence, kv head): the last `recent`, and of the rows before them those
    of largest accumulated weight (ties to the oldest, NaN last), in their order. They go into `out`, a cache
    of the same batch, heads, head size and format with room for the budget (a new one of capacity `budget` if
    not given), requantised block by block; sequences of at most `budget` rows are kept whole.

    Returns (out, score_out, kept): the kept rows' scores (B, Hkv, out.capacity), 0 past the length, and their
    source rows (B, Hkv, budget) int32, -1 past the length. Keys keep the rotation they were stored with."""
    _require_cuda("kv8_evict", score, score_out)
    _same_device("kv8_evict", cache, score, score_out)
    B, Hkv, cap, D = cache._k.shape
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise RuntimeError(f"kv8_evict: budget must be at least 1 and recent between 0 and budget, got {budget} and {recent}")
    if score.dtype != torch.float32 or tuple(score.shape) != (B, Hkv, cap) or not score.is_contiguous():
        raise RuntimeError(f"kv8_evict: score must be a contiguous float32 tensor ({B}, {Hkv}, {cap})")
    if out is None:
        out = KV8Cache.empty(B, Hkv, budget, D, cache._block, cache._k.dtype, cache._k.device)
    if score_out is None:
        score_out = torch.empty((B, Hkv, out.capacity), dtype=torch.float32, device=score.device)
    elif score_out.dtype != torch.float32 or tuple(score_out.shape) != (B, Hkv, out.capacity) or not score_out.is_contiguous():
        raise RuntimeError(f"kv8_evict: score_out must be a contiguous float32 tensor ({B}, {Hkv}, {out.capacity})")
    kept = torch.empty((B, Hkv, budget), dtype=torch.int32, device=score.device)
    rc = _C.lib.gtb_kv8_evict(ctypes.byref(cache._native), score.data_ptr(), budget, recent, ctypes.byref(out._native),
                              score_out.data_ptr(), kept.data_ptr(), _stream(score.device))
    _C.check_rc(rc, "kv8_evict")
    return out, score_out, kept
