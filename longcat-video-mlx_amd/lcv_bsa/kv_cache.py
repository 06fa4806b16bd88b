"""A KV cache held in 8 bits, and what writes, reads, weighs and shrinks it.

The reference keeps a continuation's cache in 16 bits (longcat_video/models/
attention.py:191-201, 235-275), for every layer through every denoising step.
``KVCache8`` holds e4m3 bytes with one power-of-two scale per block of 64 tokens
and head: half the memory, and half the bytes of every read.

* ``cache_append`` writes new keys and values (at any token, ragged batches);
* ``cached_attention`` attends to it: single tokens, prompts, frames of a video,
  grouped heads, causal or not;
* ``attention_weights`` adds up what attention each cached token got;
* ``cache_evict`` cuts the cache down to its heaviest and its newest tokens.

Lengths and positions are int32 tensors that the kernels read on the device, so
every call can be captured into a graph and replayed as they move on; a plain
int stands for the same number for every item.  There is no gradient through
the cache.
"""

from __future__ import annotations

import functools
import math
from typing import Optional, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from .block_sparse_attention import _dtype_code, _require_device
from .rope_positions import launch, rows_of

__all__ = ["KVCache8", "cache_append", "cached_attention", "attention_weights", "cache_evict"]

BLOCK = 64  # tokens under one scale
_E4M3 = torch.float8_e4m3fn

Ints = Union[int, torch.Tensor]


class KVCache8:
    """Keys ``k8`` ``[B, H, capacity, D]`` and values ``v8`` ``[B, H, capacity / 64,
    D, 64]`` (each block of 64 tokens transposed) in ``float8_e4m3fn``, and the
    blocks' scales ``k_scale``, ``v_scale`` ``[B, H, capacity / 64]``: fp32 powers of
    two in [2^-60, 2^60].  Contiguous, D 64 or 128.  How many tokens of it are in
    use is its user's to say, at every call."""

    __slots__ = ("_tensors", "_shape")

    def __init__(self, k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        _require_device(k8, v8, k_scale, v_scale)
        if k8.dim() != 4:
            raise ValueError(f"k8 must be [B, H, capacity, D], got shape {tuple(k8.shape)}")
        B, H, n, D = k8.shape
        nb = n // BLOCK
        if (D != 64 and D != 128) or n < BLOCK or n % BLOCK or B < 1 or H < 1:
            raise ValueError(f"an 8-bit cache holds head dims 64 and 128 and a multiple of {BLOCK} tokens, "
                             f"got {tuple(k8.shape)}")
        if v8.shape != (B, H, nb, D, BLOCK):
            raise ValueError(f"v8 must be {(B, H, nb, D, BLOCK)}, got {tuple(v8.shape)}")
        if k8.dtype != _E4M3 or v8.dtype != _E4M3:
            raise ValueError(f"k8 and v8 must be {_E4M3}, got {k8.dtype} and {v8.dtype}")
        if (k_scale.shape != (B, H, nb) or v_scale.shape != (B, H, nb)
                or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32):
            raise ValueError(f"k_scale and v_scale must be fp32 {(B, H, nb)}, got {k_scale.dtype} {tuple(k_scale.shape)} "
                             f"and {v_scale.dtype} {tuple(v_scale.shape)}")
        if ((k8.data_ptr() | v8.data_ptr()) % 16 or not k8.is_contiguous() or not v8.is_contiguous()
                or not k_scale.is_contiguous() or not v_scale.is_contiguous()):
            raise ValueError("a cache's tensors must be contiguous, k8 and v8 on 16-byte boundaries")
        self._tensors = k8, v8, k_scale, v_scale
        self._shape = B, H, n, D

    @classmethod
    def _of(cls, k8, v8, k_scale, v_scale) -> "KVCache8":
        """A cache of new tensors, whose shapes need no checks."""
        cache = object.__new__(cls)
        cache._tensors, cache._shape = (k8, v8, k_scale, v_scale), tuple(k8.shape)
        return cache

    @classmethod
    def empty(cls, batch: int, heads: int, capacity: int, head_dim: int, device=None) -> "KVCache8":
        """A cache of zeros with room for ``capacity`` tokens (rounded up to a block)."""
        dev = torch.device("cuda") if device is None else torch.device(device)
        nb = -(-int(capacity) // BLOCK)
        return cls(torch.zeros((batch, heads, nb * BLOCK, head_dim), dtype=torch.uint8, device=dev).view(_E4M3),
                   torch.zeros((batch, heads, nb, head_dim, BLOCK), dtype=torch.uint8, device=dev).view(_E4M3),
                   torch.ones((batch, heads, nb), dtype=torch.float32, device=dev),
                   torch.ones((batch, heads, nb), dtype=torch.float32, device=dev))

    @property
    def k8(self) -> torch.Tensor:
        return self._tensors[0]

    @property
    def v8(self) -> torch.Tensor:
        return self._tensors[1]

    @property
    def k_scale(self) -> torch.Tensor:
        return self._tensors[2]

    @property
    def v_scale(self) -> torch.Tensor:
        return self._tensors[3]

    def _pointers(self) -> _lib.Cache8:
        """The cache as the entry points read it: where its tensors lie now."""
        k8, v8, k_scale, v_scale = self._tensors
        return _lib.Cache8(k8.data_ptr(), v8.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *self._shape)

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """(batch, heads, capacity, head_dim)."""
        return self._shape

    @property
    def capacity(self) -> int:
        return self._shape[2]

    @property
    def device(self) -> torch.device:
        return self.k8.device

    def extended(self, capacity: int, batch: Optional[int] = None) -> "KVCache8":
        """A copy with room for ``capacity`` tokens; a cache of one item may become
        one of ``batch`` equal items.  What lies behind this cache's tokens is not
        initialised."""
        B, H, n, D = self.shape
        batch = B if batch is None else int(batch)
        nb, old = -(-int(capacity) // BLOCK), n // BLOCK
        if batch != B and B != 1:
            raise ValueError(f"a cache of {B} items cannot become one of {batch}")
        if nb < old:
            raise ValueError(f"capacity {capacity} is below this cache's {n}")
        parts = []
        for t, shape in ((self.k8.view(B, H, old, BLOCK, D).view(torch.uint8), (BLOCK, D)),
                         (self.v8.view(torch.uint8), (D, BLOCK)), (self.k_scale, ()), (self.v_scale, ())):
            new = torch.empty((batch, H, nb, *shape), dtype=t.dtype, device=t.device)
            new[:, :, :old] = t
            parts.append(new)
        return self._of(parts[0].view(_E4M3).view(batch, H, nb * BLOCK, D), parts[1].view(_E4M3), *parts[2:])

    def dequantize(self, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[B, H, capacity, D]`` as numbers."""
        B, H, n, D = self.shape
        k = self.k8.float().view(B, H, n // BLOCK, BLOCK, D) * self.k_scale[..., None, None]
        v = self.v8.float().transpose(-1, -2) * self.v_scale[..., None, None]
        return k.reshape(B, H, n, D).to(dtype), v.reshape(B, H, n, D).to(dtype)


def _ints(x: Ints, name: str, B: int, device: torch.device, lo: int, hi: int) -> torch.Tensor:
    """``x`` as the int32 ``[B]`` that the kernels read."""
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.int32 or x.shape != (B,) or x.device != device:
            raise ValueError(f"{name} must be an int or int32 [{B}] on {device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        return x.contiguous()
    x = int(x)
    if not lo <= x <= hi:
        raise ValueError(f"{name}={x} must be in [{lo}, {hi}]")
    return torch.full((B,), x, dtype=torch.int32, device=device)


def no_derivative(what: str, *ts: torch.Tensor) -> None:
    """Raises for tensors that a gradient or a tangent goes through."""
    for t in ts:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError(f"{what} has no forward-mode derivative: call it on detached tensors")


def cache_append(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, start: Ints,
                 counts: Optional[Ints] = None) -> KVCache8:
    """Writes ``k``, ``v`` ``[B, H, S, D]`` (fp16, bf16, fp32; any strides) into the
    cache, in place, from each item's token ``start`` on; of a padded batch the
    first ``counts`` rows of each item (default: all).

    A block's scale becomes the least power of two that brings the largest of its
    new rows within 448, and no less than it was where the block keeps rows before
    ``start`` (those are rounded again if it grows).  To nearest, ties to even;
    infinities, NaN and magnitudes over 448 * 2^60 become NaN.  Rows that would pass
    the capacity and items with a negative start are left out.  Behind the last new
    row the bytes stay, but in its block they stand under the new scale: tokens that
    stood there are lost, so rows are written behind all that is to be kept, or
    instead of it.  Returns the cache."""
    _require_device(cache.k8, k, v)
    no_derivative("cache_append", k, v)
    B, H, n, D = cache.shape
    S = k.shape[2] if k.dim() == 4 else -1
    if k.shape != (B, H, S, D) or v.shape != (B, H, S, D) or k.dtype != v.dtype:
        raise ValueError(f"k, v must be [{B}, {H}, S, {D}] of one dtype, got {tuple(k.shape)} {k.dtype}, "
                         f"{tuple(v.shape)} {v.dtype}")
    code = _dtype_code(k)
    if S > n:
        raise ValueError(f"{S} rows for a cache of {n} tokens")
    rows = S if counts is None else 0 if isinstance(counts, torch.Tensor) else int(counts)  # that a plain start has to fit
    if counts is not None:
        counts = _ints(counts, "counts", B, cache.device, 0, S)
    start = _ints(start, "start", B, cache.device, 0, n - rows)
    if S == 0:
        return cache
    k, ks = rows_of(k, "k")
    v, vs = rows_of(v, "v")
    launch(k, "cache_append", cache._pointers(), k.data_ptr(), v.data_ptr(), code, S, ks, vs, start.data_ptr(),
           None if counts is None else counts.data_ptr())
    return cache


def _queries(what, q, cache, lengths, q_lens, sm_scale, max_len):
    """The arguments that attention and its weights share, checked."""
    _require_device(cache.k8, q)
    no_derivative(what, q)
    B, H, n, D = cache.shape
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D or q.shape[1] < H or q.shape[1] % H:
        raise ValueError(f"q must be [{B}, a multiple of {H}, S, {D}], got {tuple(q.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{what} takes float16 and bfloat16 queries, got {q.dtype}")
    sm_scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0.0 <= sm_scale < math.inf:
        raise ValueError(f"sm_scale={sm_scale} must be finite and not negative")
    max_len = n if max_len is None else min(int(max_len), n)
    if max_len < 0:
        raise ValueError(f"max_len={max_len} is negative")
    lengths = _ints(lengths, "lengths", B, cache.device, 0, n)
    if q_lens is not None:
        q_lens = _ints(q_lens, "q_lens", B, cache.device, 0, q.shape[2])
    return lengths, q_lens, sm_scale, max_len


@functools.lru_cache(maxsize=1024)
def _workspace(entry: str, Hq: int, S: int, B: int, H: int, n: int, D: int, max_len: int) -> int:
    return getattr(_lib.load(), entry)(Hq, S, _lib.Cache8(None, None, None, None, B, H, n, D), max_len)


@functools.lru_cache(maxsize=1024)
def _shared(shape: tuple, strides: tuple, apart: int) -> bool:
    """Whether a tensor of this shape and these strides and one `apart` elements behind it
    have an element in common; apart 0: whether it holds one element twice.  (A layout whose
    dimensions are tangled beyond a few thousand steps of the search counts as one.)"""
    dims = sorted(((st, n) for n, st in zip(shape, strides) if n > 1), reverse=True)
    rest = [sum((n - 1) * st for st, n in dims[i:]) for i in range(len(dims) + 1)]
    steps = 0

    def search(i: int, left: int, moved: bool) -> bool:  # left = sum of d stride, |d| < n, from dims[i] on?
        nonlocal steps
        steps += 1
        if steps > 4096:
            return True
        if abs(left) > rest[i]:
            return False
        if i == len(dims):
            return moved
        st, n = dims[i]
        if st == 0:
            return left == 0
        lo, hi = -((rest[i + 1] - left) // st), (left + rest[i + 1]) // st
        return any(search(i + 1, left - d * st, moved or d != 0) for d in range(max(lo, 1 - n), min(hi, n - 1) + 1))

    return search(0, apart, apart != 0)


def _apart(q: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether rows of ``out`` may be written while others of ``q`` (of its shape and dtype)
    are read: it is q itself, or has no element of another row of it."""
    size = q.element_size()
    first, last = ((t.data_ptr(), t.data_ptr() + size * sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) for t in (q, out))
    if first[1] < last[0] or last[1] < first[0]:
        return True
    strides = tuple(st for n, st in zip(q.shape, q.stride()) if n > 1)
    if strides != tuple(st for n, st in zip(out.shape, out.stride()) if n > 1):
        return False
    apart, odd = divmod(last[0] - first[0], size)
    return not odd and (apart == 0 or not _shared(tuple(n for n in q.shape if n > 1), strides, apart))


def cached_attention(q: torch.Tensor, cache: KVCache8, lengths: Ints, *, q_lens: Optional[Ints] = None,
                     causal: bool = False, sm_scale: Optional[float] = None, max_len: Optional[int] = None,
                     out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """``softmax(sm_scale q k^T) v`` of ``q`` ``[B, Hq, S, D]`` (fp16 / bf16, any
    strides) over the first ``lengths`` tokens of each item's cache; query head h
    reads key head ``h // (Hq / H)``.

    ``q_lens``: how many of the S queries of each item are real (default: all).
    ``causal``: the real queries are the item's last tokens, and query i sees the
    tokens up to ``lengths - q_lens + i``.  Rows that see nothing (padding, empty
    items, queries before the first token) get zeros, as do rows all of whose scores
    are -inf.  ``max_len``: a bound on ``lengths`` known to the caller (longer items
    count as that long); it shapes the launch of many rows, so a close one serves
    short histories in a long cache.

    Sums are fp32.  Before they meet the values, probabilities are rounded to q's type
    once: by half a step of it, in fp16 by up to 2^-22 of the row's largest, however far
    apart the blocks' scales are.  A token whose weight is below 2^-40 of the heaviest's
    may be left out of the row's sum.

    ``out`` may be q, or lie anywhere on its memory; its own elements lie apart.
    Returns it (``[B, Hq, S, D]`` in q's dtype), or ``(out, lse)`` with the fp32
    ``[B, Hq, S]`` log of each row's sum (-inf where nothing is seen)."""
    lengths, q_lens, sm_scale, max_len = _queries("cached_attention", q, cache, lengths, q_lens, sm_scale, max_len)
    B, Hq, S, D = q.shape
    given = out
    if out is None:
        out = q.new_empty((B, Hq, S, D))
    else:
        _require_device(q, out)
        no_derivative("cached_attention", out)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError(f"out must be {tuple(q.shape)} {q.dtype}, got {tuple(out.shape)} {out.dtype}")
        if _shared(tuple(out.shape), out.stride(), 0):
            raise ValueError("out's elements share memory")
    lse = cache.k_scale.new_empty((B, Hq, S)) if return_lse else None
    if q.numel() == 0 or max_len == 0:
        out.zero_()
        if return_lse:
            lse.fill_(-math.inf)
        return (out, lse) if return_lse else out
    # A copy where out's rows cannot be written in place.
    to, os = rows_of(out if given is None or _apart(q, given) else torch.empty_like(out, memory_format=torch.contiguous_format), "out")
    q, qs = rows_of(q, "q")
    size = _workspace("lcv_bsa_cached_attn_workspace_bytes", Hq, S, *cache.shape, max_len)
    ws = torch.empty((size,), dtype=torch.uint8, device=q.device) if size else None
    launch(q, "cached_attn", q.data_ptr(), _dtype_code(q), Hq, S, qs, cache._pointers(), lengths.data_ptr(),
           None if q_lens is None else q_lens.data_ptr(), int(causal), sm_scale, max_len, to.data_ptr(), os,
           None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), size)
    if to is not out:
        out.copy_(to)
    return (out, lse) if return_lse else out


def attention_weights(q: torch.Tensor, cache: KVCache8, lengths: Ints, lse: torch.Tensor, *,
                      q_lens: Optional[Ints] = None, causal: bool = False, sm_scale: Optional[float] = None,
                      max_len: Optional[int] = None, weights: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``weights`` (fp32 ``[B, H, capacity]``; default zeros) plus, for each cached
    token, the attention that these queries gave it: the sum of their softmax over
    the rows of its key head.  ``lse`` and the other arguments are those of
    ``cached_attention``.  ``out`` may be ``weights`` itself, to accumulate in place.
    The same call gives the same bits."""
    lengths, q_lens, sm_scale, max_len = _queries("attention_weights", q, cache, lengths, q_lens, sm_scale, max_len)
    B, Hq, S, D = q.shape
    shape = (B, cache.shape[1], cache.capacity)
    if tuple(lse.shape) != (B, Hq, S) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be fp32 {(B, Hq, S)}, got {lse.dtype} {tuple(lse.shape)}")
    for name, t in (("weights", weights), ("out", out)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32):
            raise ValueError(f"{name} must be fp32 {shape}, got {t.dtype} {tuple(t.shape)}")
    _require_device(q, lse, *(t for t in (weights, out) if t is not None))
    no_derivative("attention_weights", lse, *(t for t in (weights, out) if t is not None))
    if out is None:
        out = lse.new_empty(shape)
    elif not out.is_contiguous():
        raise ValueError("out must be contiguous")
    if q.numel() == 0 or max_len == 0:
        return out.zero_() if weights is None else out.copy_(weights) if out is not weights else out
    if q.stride(2) >= 1 << 25:  # beyond what the kernel's row offsets hold
        q = q.contiguous()
    q, qs = rows_of(q, "q")
    lse = lse.contiguous()
    weights = None if weights is None else weights.contiguous()
    size = _workspace("lcv_bsa_attention_weights_workspace_bytes", Hq, S, *cache.shape, max_len)
    ws = torch.empty((size,), dtype=torch.uint8, device=q.device) if size else None
    launch(q, "attention_weights", q.data_ptr(), _dtype_code(q), Hq, S, qs, cache._pointers(), lengths.data_ptr(),
           None if q_lens is None else q_lens.data_ptr(), int(causal), sm_scale, max_len, lse.data_ptr(),
           None if weights is None else weights.data_ptr(), out.data_ptr(), None if ws is None else ws.data_ptr(), size)
    return out


def cache_evict(cache: KVCache8, lengths: Ints, weights: torch.Tensor, keep: int, *, recent: int = 0):
    """Of each head's ``lengths`` tokens, the newest ``recent`` and the heaviest others
    (by ``weights`` ``[B, H, capacity]`` fp32; equal ones: the lowest token first; NaN
    below everything), ``keep`` in all, in their order, as a new cache.

    Returns ``(cache, weights, kept, lengths)``: the new cache (capacity ``keep``
    rounded up to a block, each block under the least scale for its rows, zeros
    behind the last), the kept tokens' weights (zeros behind), their old indices
    ``[B, H, keep]`` int32 (-1 behind) and the new lengths ``[B]`` int32."""
    _require_device(cache.k8, weights)
    no_derivative("cache_evict", weights)
    B, H, n, D = cache.shape
    if tuple(weights.shape) != (B, H, n) or weights.dtype != torch.float32:
        raise ValueError(f"weights must be fp32 {(B, H, n)}, got {weights.dtype} {tuple(weights.shape)}")
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"keep={keep} must be at least 1 and recent={recent} in [0, keep]")
    lengths = _ints(lengths, "lengths", B, cache.device, 0, n)
    weights = weights.contiguous()
    nb, words, numbers = -(-keep // BLOCK), cache.k8.new_empty, weights.new_empty
    new = KVCache8._of(words((B, H, nb * BLOCK, D)), words((B, H, nb, D, BLOCK)), numbers((B, H, nb)), numbers((B, H, nb)))
    new_weights, kept, left = numbers((B, H, nb * BLOCK)), lengths.new_empty((B, H, keep)), lengths.new_empty((B,))
    launch(weights, "cache_evict", cache._pointers(), lengths.data_ptr(), weights.data_ptr(), keep, recent,
           new._pointers(), new_weights.data_ptr(), kept.data_ptr(), left.data_ptr())
    return new, new_weights, kept, left
