"""What the attention over an 8-bit cache may lose to rounding, number by number:
value scales far apart, channels that only some blocks fill, queries beside large values
that no key answers."""

from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R
from test_gpu_kv_cache import BF16, F16, _gen, _rows, _within

pytestmark = pytest.mark.gpu


def _head(c, h):
    from lcv_bsa import KVCache8

    return KVCache8(*(t[:, h:h + 1].clone(memory_format=torch.contiguous_format) for t in (c.k8, c.v8, c.k_scale, c.v_scale)))


def _check(q, c, lengths, out, lse, sm_scale=None, least=2.0 ** -25):
    """Each channel by what its own values carry: P is rounded to q's type once (half a step
    u of each; in fp16 no less than `least` of the row's largest, below which it is
    subnormal), the output once, and the scores' fp32 sums as R.attention has them."""
    want, want_lse, _, tol_lse, probs, tol_p = R.attention(q, c, lengths, sm_scale=sm_scale)
    v = R.values(c)[1].abs()
    u = torch.finfo(q.dtype).eps / 2
    size = probs @ v
    tol = u * size + u * want.abs() + tol_p[..., None] * size
    if q.dtype == F16:
        tol += least * probs.amax(-1, keepdim=True) * v[:, :, :lengths[0]].sum(2, keepdim=True)
    _within(out, want, tol + (2.0 ** -25 if q.dtype == F16 else 2.0 ** -134))
    _within(lse, want_lse, tol_lse)


def _values(kind, gen, device, H, n, D):
    """[1, H, n, D] fp32, and the type of the queries."""
    v = torch.randn(1, H, n, D, generator=gen, device=device)
    j = torch.arange(n, device=device) // 64
    if kind in ("outlier, 2e-3", "late outlier, 2e-3", "outlier, 1e-4"):
        v *= float(kind[-4:])
        v[:, :, (10 if kind[0] == "o" else n - 70), 3] = 6e4  # its block's scale is 2^8: the rest there is zero
        return v, F16
    blocks = (n + 63) // 64
    mine = torch.arange(D, device=device) % blocks == j[:, None]  # a channel is filled by one block of `blocks`
    if kind == "steps":
        return v * mine * torch.exp2(14.0 - 32.0 * j[:, None] / (blocks - 1)), F16
    if kind == "rising steps":
        return v * mine * torch.exp2(-18.0 + 32.0 * j[:, None] / (blocks - 1)), F16
    if kind == "near":  # 2^12 apart at the most: one walk, in which the heaviest P may be 2^-3
        return v * mine * torch.exp2(6.0 - 11.0 * j[:, None] / (blocks - 1)), F16
    assert kind in ("far", "far, rising")
    e = 60.0 - 120.0 * j[:, None] / (blocks - 1)
    return v * mine * torch.exp2(e if kind == "far" else -e), BF16


KINDS = ["outlier, 2e-3", "late outlier, 2e-3", "outlier, 1e-4", "steps", "rising steps", "near", "far", "far, rising"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S", [1, 40, 200])
@pytest.mark.parametrize("D", [64, 128])
def test_value_scales_far_apart(device, kind, S, D):
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, S + D)
    n = 576
    v, dtype = _values(kind, gen, device, 1, n, D)
    k = torch.randn(1, 1, n, D, generator=gen, device=device)
    c = cache_append(KVCache8.empty(1, 1, n, D, device), k, v, 0)
    q = _rows(gen, device, 1, 1, S, D, dtype)
    out, lse = cached_attention(q, c, n - 5, return_lse=True)
    _check(q, c, [n - 5], out, lse, least=2.0 ** (-22 if kind == "near" else -25))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
def test_value_scales_far_apart_in_whole_walks(device, kind, D):
    """512 walks of two tiles each, which are not split."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, D)
    H, S, n = 512, 130, 1100
    v, dtype = _values(kind, gen, device, H, n, D)
    k = torch.randn(1, H, n, D, generator=gen, device=device)
    c = cache_append(KVCache8.empty(1, H, n, D, device), k, v, 0)
    q = _rows(gen, device, 1, H, S, D, dtype)
    out, lse = cached_attention(q, c, n - 3, return_lse=True)
    for h in (0, H - 1):
        _check(q[:, h:h + 1], _head(c, h), [n - 3], out[:, h:h + 1], lse[:, h:h + 1],
               least=2.0 ** (-22 if kind == "near" else -25))


@pytest.mark.parametrize("kind", ["far", "far, rising", "near", "outlier, 2e-3"])
@pytest.mark.parametrize("size", [1.0, 12.0])
def test_value_scales_far_apart_in_long_walks(device, kind, size):
    """Walks of 33 blocks of D = 128, for bf16 the form that keeps the keys' bytes; scores
    that pass the room of the first offset in fp16; queries that see the last block in part."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, 8)
    H, S, D, n = 512, 130, 128, 2100
    v, dtype = _values(kind, gen, device, H, n, D)
    k = torch.randn(1, H, n, D, generator=gen, device=device)
    c = cache_append(KVCache8.empty(1, H, n, D, device), k, v, 0)
    q = size * _rows(gen, device, 1, H, S, D, dtype)
    out, lse = cached_attention(q, c, n - 3, return_lse=True)
    for h in (0, H - 1):
        _check(q[:, h:h + 1], _head(c, h), [n - 3], out[:, h:h + 1], lse[:, h:h + 1], least=2.0 ** (-22 if kind == "near" else -25))


@pytest.mark.parametrize("S", [1, 100])
def test_scores_far_below_a_first_block_of_minus_infinity(device, S):
    """The first block's products overflow to -inf; what is left has the whole weight,
    however low its scores are."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    k = torch.zeros(1, 1, 128, 64, device=device)
    k[:, :, :64, 0] = -1.0  # stored as -256
    k[:, :, 64:, 1] = 1.0
    c = cache_append(KVCache8.empty(1, 1, 128, 64, device), k, torch.ones_like(k), 0)
    q = torch.zeros(1, 1, S, 64, dtype=BF16, device=device)
    q[..., 0], q[..., 1] = 2.0 ** 120, -4096.0
    out, lse = cached_attention(q, c, 128, return_lse=True)
    assert bool((out == 1).all())
    assert float((lse - (math.log(64) - 512)).abs().max()) <= 2.0 ** -13  # fp32 near 2^9: 2^-15 a rounding


@pytest.mark.parametrize("S", [1, 100])
@pytest.mark.parametrize("scale", [0.0, 1e-38])
def test_weights_of_minus_infinity_under_a_small_scale(device, S, scale):
    """Products that overflow are scores of -inf whatever the softmax scale, for the weights
    as for the attention."""
    from lcv_bsa import KVCache8, attention_weights, cache_append, cached_attention

    k = torch.zeros(1, 1, 64, 64, device=device)
    k[:, :, :40, 0] = -1.0  # stored as -256
    c = cache_append(KVCache8.empty(1, 1, 64, 64, device), k, torch.ones_like(k), 0)
    q = torch.zeros(1, 1, S, 64, dtype=BF16, device=device)
    q[..., 0] = 2.0 ** 120
    out, lse = cached_attention(q, c, 64, sm_scale=scale, return_lse=True)
    assert bool((out == 1).all())
    w = attention_weights(q, c, 64, lse, sm_scale=scale)[0, 0]
    assert not w[:40].any() and float((w[40:] - S / 24).abs().max()) <= S / 24 * 2.0 ** -18


@pytest.mark.parametrize("scale", [128 ** -0.5, 1.0])
def test_sparse_queries_beside_an_unanswered_value(device, scale):
    """Walks of 32 blocks in bf16, D = 128: rows of one large value in a channel where keys
    are zero and two small ones in each quarter, which are all that the scores hold."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, 9)
    H, S, D, n = 512, 130, 128, 1999
    k, v = (torch.randn(1, H, 2048, D, generator=gen, device=device) for _ in range(2))
    k[..., 5] = 0.0
    at = torch.tensor([3, 20, 35, 60, 70, 90, 100, 127], device=device)
    q = torch.zeros(1, H, S, D, device=device)
    q[..., at] = torch.randn(1, H, S, len(at), generator=gen, device=device) * 2
    sizes = [12, 16, 20, 22, 24, 30, 100]
    for i, e in enumerate(sizes):
        q[:, i::len(sizes), :, 5] = 2.0 ** e
    c = cache_append(KVCache8.empty(1, H, 2048, D, device), k, v, 0)
    q = q.to(BF16)
    out, lse = cached_attention(q, c, n, sm_scale=scale, return_lse=True)
    for h in range(len(sizes)):
        _check(q[:, h:h + 1], _head(c, h), [n], out[:, h:h + 1], lse[:, h:h + 1], scale)


def test_an_infinite_query_over_a_long_walk(device):
    """A row whose only value is infinite and whose scores are all -inf sees nothing."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, 2)
    H, S, D = 512, 130, 128
    k, v = (torch.randn(1, H, 2048, D, generator=gen, device=device) for _ in range(2))
    k[..., 5] = -1.0
    c = cache_append(KVCache8.empty(1, H, 2048, D, device), k, v, 0)
    q = torch.zeros(1, H, S, D, dtype=BF16, device=device)
    q[..., 5] = math.inf
    out, lse = cached_attention(q, c, 2000, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
