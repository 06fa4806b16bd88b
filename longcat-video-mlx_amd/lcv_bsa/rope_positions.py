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
from torch.autograd import forward_ad

from . import _lib
from .block_sparse_attention import _dtype_code, _require_device, _stream
from .rope_3d import BASE, rope_dims

__all__ = ["rope_nd", "grid_positions"]

_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


def launch(t: torch.Tensor, name: str, *args) -> None:
    """The entry point ``lcv_bsa_<name>`` with ``t``'s device current, on that device's
    current stream (its last argument)."""
    entry = getattr(_lib.load(), "lcv_bsa_" + name)
    index = t.device.index
    if torch._C._cuda_getDevice() == index:
        status = entry(*args, _stream(t))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _stream(t))
    if status:
        _lib.check(status, name)


@functools.lru_cache(maxsize=4096)
def _row_strides(shape: tuple, strides: tuple, size: int) -> Optional[_lib.Strides]:
    """The strides of [B, H, S, D] as the kernels read it (those of dimensions of size one
    put right); None where its rows are not dense, overlap or leave 16-byte boundaries."""
    (B, H, S, D), (sb, sh, ss, sd) = shape, strides
    sb, sh, ss = sb if B > 1 else D, sh if H > 1 else D, ss if S > 1 else D
    if (sd != 1 and D > 1) or ss < D or (sb | sh | ss) * size % 16:
        return None
    return _lib.Strides(sb, sh, ss)


def rows_of(t: torch.Tensor, name: str) -> tuple[torch.Tensor, _lib.Strides]:
    """``t`` [B, H, S, D] as the kernels read it -- rows dense, on 16-byte
    boundaries, not overlapping -- copied where it is not, and its strides."""
    if t.dim() != 4:
        raise ValueError(f"{name} must be [B, H, S, D], got shape {tuple(t.shape)}")
    strides = _row_strides(t.shape, t.stride(), t.element_size())
    if strides is None or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        _, H, S, D = t.shape
        strides = _lib.Strides(H * S * D, S * D, D)
    return t, strides


def grid_positions(grid: Sequence[int], first: Sequence[int] = (0, 0, 0), device=None) -> torch.Tensor:
    """``[T*H*W, 3]`` int32 positions of a latent grid in t-major token order, the
    first token at ``first``."""
    axes = [torch.arange(a, a + n, dtype=torch.int32, device=device) for a, n in zip(first, grid)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, len(axes))


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


@functools.lru_cache(maxsize=1024)
def _plan(shape: tuple, strides: tuple, dtype: torch.dtype, pshape: tuple, pstrides: tuple, ptype: torch.dtype,
          dims: Optional[tuple]):
    """The checks of a rotation, and what follows from the sizes, strides and types alone:
    (dtype code, position code, positions' strides or None for a copy of them, dims,
    output's strides, whether the output lies in memory like x)."""
    if len(shape) != 4:
        raise ValueError(f"x must be [B, H, S, D], got shape {tuple(shape)}")
    x = torch.empty_strided(shape, strides, dtype=dtype, device="meta")
    code = _dtype_code(x)
    B, H, S, D = shape
    if len(pshape) not in (2, 3) or pshape[-2] != S or (len(pshape) == 3 and pshape[0] not in (1, B)):
        raise ValueError(f"positions must be [{S}, axes] or [{B} or 1, {S}, axes], got {tuple(pshape)}")
    if ptype not in _POSITION_TYPES:
        raise ValueError(f"positions must be int32, int64 or float32, got {ptype}")
    split = _split(D, pshape[-1], dims)
    where = None
    if pshape[-1] == 1 or pstrides[-1] == 1:
        where = (pstrides[0] if len(pshape) == 3 and pshape[0] > 1 else 0, pstrides[-2])
    like = torch.empty_like(x).stride()
    alike = like[3] == 1 and like[2] >= D
    os = _row_strides(shape, like if alike else (H * S * D, S * D, D, 1), x.element_size())
    return code, _POSITION_TYPES[ptype], where, split, os, alike


def _rotate(x: torch.Tensor, positions: torch.Tensor, dims: Optional[tuple], base: float, inverse: bool) -> torch.Tensor:
    shape = x.shape
    code, pcode, where, split, os, alike = _plan(shape, x.stride(), x.dtype, positions.shape, positions.stride(),
                                                 positions.dtype, dims)
    out = torch.empty_like(x) if alike else torch.empty(shape, dtype=x.dtype, device=x.device)
    B, H, S, D = shape
    if not B * H * S:
        return out
    if where is None:
        positions = positions.contiguous()
        where = positions.stride(0) if positions.dim() == 3 and positions.shape[0] > 1 else 0, positions.stride(-2)
    x, xs = rows_of(x, "x")
    launch(x, "rope_nd", x.data_ptr(), code, B, H, S, D, xs, positions.data_ptr(), pcode, *where, split, len(split), base,
           inverse, out.data_ptr(), os)
    return out


def _watched(x: torch.Tensor) -> bool:
    """A derivative of what becomes of ``x`` may be wanted, in reverse or in forward mode."""
    return (x.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0


class _RopeNd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, dims, base, inverse):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.how = dims, base, inverse
        return _rotate(x, positions, dims, base, inverse)

    @staticmethod
    def backward(ctx, g):
        dims, base, inverse = ctx.how
        turn = _RopeNd.apply if torch.is_grad_enabled() or _watched(g) else _rotate  # a further derivative is wanted, or not
        return turn(g, *ctx.saved_tensors, dims, base, not inverse), None, None, None, None

    @staticmethod
    def jvp(ctx, t, *_):
        turn = _RopeNd.apply if t.requires_grad and torch.is_grad_enabled() else _rotate
        return turn(t, *ctx.saved_tensors, *ctx.how)


def rope_nd(x: torch.Tensor, positions: torch.Tensor, dims: Optional[Sequence[int]] = None, *,
            base: float = BASE) -> torch.Tensor:
    """Rotates ``x`` ``[B, H, S, D]`` (fp16, bf16, fp32; D a multiple of 8 up to
    256; any strides) to its tokens' ``positions`` ``[S, axes]`` or ``[B, S, axes]``
    (int32, int64 or fp32; a batch of one is shared).

    ``dims``: the even number of dims that each axis turns, summing to D; by
    default the t / h / w split of ``rope_dims`` for three axes, else equal
    parts.  Differentiable in ``x`` (as often as wanted, and in forward mode);
    positions get no gradient.
    A backward pass that is captured into a graph takes its gradients with
    ``torch.autograd.grad``, while no graph of the same leaves that was made outside
    of the capture is alive: torch would have to order the two streams there."""
    _require_device(x, positions)
    dims = None if dims is None else tuple(dims)
    if positions.requires_grad:
        positions = positions.detach()
    if _watched(x):
        return _RopeNd.apply(x, positions, dims, float(base), False)
    return _rotate(x, positions, dims, float(base), False)
