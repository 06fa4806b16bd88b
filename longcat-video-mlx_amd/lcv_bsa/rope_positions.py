"""Rotary positions with several axes at positions given per token, forward and backward.

``rope_3d`` rotates the tokens of one whole latent grid (longcat_video/models/
rope_3d.py:37-128).  ``rope_nd`` takes each token's own position on every axis --
new frames behind a cache, what an eviction left over, rows and columns of an
image, plain text -- and is differentiable.  Same convention: adjacent pairs,
the axes' parts one after another, angle ``position * base^(-2i / dim)``.  The
angles are formed in 64 bits (rope_3d.py:65-93 forms them in fp32), so that far
positions keep theirs.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence

import torch

from . import _lib
from .block_sparse_attention import _dtype_code, _require_device, _stream
from .rope_3d import BASE, rope_dims

__all__ = ["rope_nd", "grid_positions"]

_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


class on_device:
    """Makes ``t``'s device the current one for a launch (nothing where it is)."""

    __slots__ = ("index", "before")

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index

    def __enter__(self):
        now = torch.cuda.current_device()
        self.before = None if now == self.index else now
        if self.before is not None:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before is not None:
            torch.cuda.set_device(self.before)


def rows_of(t: torch.Tensor, name: str) -> tuple[torch.Tensor, _lib.Strides]:
    """``t`` [B, H, S, D] as the kernels read it -- rows dense, on 16-byte
    boundaries, not overlapping -- copied where it is not, and its strides (those
    of dimensions of size one put right)."""
    if t.dim() != 4:
        raise ValueError(f"{name} must be [B, H, S, D], got shape {tuple(t.shape)}")
    B, H, S, D = t.shape
    sb, sh, ss, sd = t.stride()
    sb, sh, ss = sb if B > 1 else D, sh if H > 1 else D, ss if S > 1 else D
    if (sd != 1 and D > 1) or ss < D or (sb | sh | ss) * t.element_size() % 16 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, _lib.Strides(H * S * D, S * D, D)
    return t, _lib.Strides(sb, sh, ss)


def grid_positions(grid: Sequence[int], first: Sequence[int] = (0, 0, 0), device=None) -> torch.Tensor:
    """``[T*H*W, 3]`` int32 positions of a latent grid in t-major token order, the
    first token at ``first``."""
    axes = [torch.arange(a, a + n, dtype=torch.int32, device=device) for a, n in zip(first, grid)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, len(axes))


@functools.lru_cache(maxsize=256)
def _split(D: int, axes: int, dims: Optional[tuple]):
    """The axes' dims (checked; None: the default split) as the entry point reads them."""
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"rope_nd supports head dims that are multiples of 8 up to 256 (got {D})")
    if axes < 1:
        raise ValueError("positions need at least one axis")
    if dims is None:
        dims = rope_dims(D) if axes == 3 else (D // axes,) * axes
    dims = tuple(int(d) for d in dims)
    if len(dims) != axes or min(dims) < 2 or any(d % 2 for d in dims) or sum(dims) != D:
        raise ValueError(f"dims must be {axes} even numbers that sum to {D}, got {dims}")
    return (ctypes.c_int64 * axes)(*dims)


def _rotate(x: torch.Tensor, positions: torch.Tensor, dims, base: float, inverse: bool) -> torch.Tensor:
    B, H, S, D = x.shape
    out = torch.empty_like(x)
    if not x.numel():
        return out
    sb, sh, ss, sd = out.stride()
    if sd != 1 or ss < D:  # x itself is not dense
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        sb, sh, ss, sd = out.stride()
    x, xs = rows_of(x, "x")
    ps = positions.stride()
    with on_device(x):
        st = _lib.load().lcv_bsa_rope_nd(
            x.data_ptr(), _dtype_code(x), B, H, S, D, xs, positions.data_ptr(), _POSITION_TYPES[positions.dtype],
            ps[0] if len(ps) == 3 and positions.shape[0] > 1 else 0, ps[-2], dims, len(dims), base, inverse,
            out.data_ptr(), _lib.Strides(sb if B > 1 else D, sh if H > 1 else D, ss if S > 1 else D), _stream(x))
    _lib.check(st, "rope_nd")
    return out


class _RopeNd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, dims, base, inverse):
        ctx.save_for_backward(positions)
        ctx.how = dims, base, inverse
        return _rotate(x, positions, dims, base, inverse)

    @staticmethod
    def backward(ctx, g):
        dims, base, inverse = ctx.how
        turn = _RopeNd.apply if torch.is_grad_enabled() else _rotate  # a second derivative is wanted, or not
        return turn(g, *ctx.saved_tensors, dims, base, not inverse), None, None, None, None


def rope_nd(x: torch.Tensor, positions: torch.Tensor, dims: Optional[Sequence[int]] = None, *,
            base: float = BASE) -> torch.Tensor:
    """Rotates ``x`` ``[B, H, S, D]`` (fp16, bf16, fp32; D a multiple of 8 up to
    256; any strides) to its tokens' ``positions`` ``[S, axes]`` or ``[B, S, axes]``
    (int32, int64 or fp32; a batch of one is shared).

    ``dims``: the even number of dims that each axis turns, summing to D; by
    default the t / h / w split of ``rope_dims`` for three axes, else equal
    parts.  Differentiable in ``x`` (as often as wanted); positions get no gradient.
    A backward pass that is captured into a graph takes its gradients with
    ``torch.autograd.grad``, while no graph of the same leaves that was made outside
    of the capture is alive: torch would have to order the two streams there."""
    _require_device(x, positions)
    if x.dim() != 4:
        raise ValueError(f"x must be [B, H, S, D], got shape {tuple(x.shape)}")
    _dtype_code(x)
    B, _, S, D = x.shape
    if positions.dim() not in (2, 3) or positions.shape[-2] != S or (positions.dim() == 3 and positions.shape[0] not in (1, B)):
        raise ValueError(f"positions must be [{S}, axes] or [{B} or 1, {S}, axes], got {tuple(positions.shape)}")
    if positions.dtype not in _POSITION_TYPES:
        raise ValueError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    split = _split(D, positions.shape[-1], None if dims is None else tuple(dims))
    if positions.requires_grad:
        positions = positions.detach()
    ps = positions.stride()
    if ps[-1] != 1 or min(ps) < 0:
        positions = positions.contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        return _RopeNd.apply(x, positions, split, float(base), False)
    return _rotate(x, positions, split, float(base), False)
