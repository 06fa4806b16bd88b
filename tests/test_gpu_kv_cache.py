"""The 8-bit KV cache's operators against their definitions in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rows(gen, device, B, H, S, D, dtype, spread=0.0):
    """[B, H, S, D] views of [B, S, H, D] rows (a projection's layout), whose sizes
    differ by 2^(spread * normal) from block to block."""
    x = torch.randn(B, S, H, D, generator=gen, device=device)
    if spread:
        size = torch.randn(B, (S + 63) // 64, H, 1, generator=gen, device=device).mul_(spread).exp2_()
        x = x * size.repeat_interleave(64, 1)[:, :S]
    return x.to(dtype).transpose(1, 2)


def _cache(gen, device, B, H, capacity, D, spread=1.0, stale=()):
    """A full cache; behind item b's first stale[b] tokens any bytes, NaN among them."""
    from lcv_bsa import KVCache8, cache_append

    c = KVCache8.empty(B, H, capacity, D, device)
    n = c.capacity
    cache_append(c, _rows(gen, device, B, H, n, D, F32), _rows(gen, device, B, H, n, D, F32, spread), 0)
    for b, m in enumerate(stale):
        c.k8.view(torch.uint8)[b, :, m:, ::3] = 127
        c.k8.view(torch.uint8)[b, :, m:, 1::3] = 254
        v = c.v8.view(torch.uint8)
        if m < n:
            v[b, :, m // 64, ::5, m % 64:] = 255
            v[b, :, m // 64, 1::5, m % 64:] = 126
            v[b, :, m // 64 + 1:, ::3] = 127
    return c


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _ints(device, ns):
    return None if ns is None else torch.tensor(ns, dtype=torch.int32, device=device)


def _stored(cache):
    """The stored numbers of k and v [B, H, capacity, D], without scales, and the scales."""
    B, H, n, D = cache.shape
    k = R.TABLE[cache.k8.cpu().view(torch.uint8).long()]
    v = R.TABLE[cache.v8.cpu().view(torch.uint8).long()].transpose(-1, -2).reshape(B, H, n, D)
    return (k, cache.k_scale.cpu().double()), (v, cache.v_scale.cpu().double())


def _same(a, b):
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    assert torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


def _within(got, want, tol):
    got = got.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = torch.isfinite(want)
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0.0, f"over the bound by {float(off.max())}"


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_append_every_value_of_the_type(device, dtype):
    """Rows that run through values of all sizes: the scale, the rounding, ties,
    subnormals, and what cannot be held."""
    from lcv_bsa import KVCache8, cache_append

    if dtype == F32:
        gen = _gen(device, 5)
        bits = torch.randint(0, 1 << 32, (65536,), generator=gen, device=device, dtype=torch.int64).to(torch.int32)
        x = bits.view(torch.float32)
    else:
        x = torch.arange(-32768, 32768, device=device, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x.view(1, 4, 128, 128)
    c = KVCache8.empty(1, 4, 128, 128, device)
    want = R.append(c, x, x, [0])
    cache_append(c, x, x, 0)
    for (a, s), (wa, ws) in zip(_stored(c), want):
        assert torch.equal(s, ws)
        _same(a, wa)
    # One scale throughout: every tie between two stored values, both ways.
    steps = (R.TABLE[:127, None] + torch.tensor([0.0, 0.5])[None] * (R.TABLE[1:128] - R.TABLE[:127]).nan_to_num(0.0)[:, None]).flatten()
    t = torch.zeros(64 * 64, dtype=torch.float64)
    t[:len(steps)], t[len(steps):2 * len(steps)], t[-1] = steps, -steps, 448.0
    t = t.to(dtype).view(1, 1, 64, 64).to(device)
    c = KVCache8.empty(1, 1, 64, 64, device)
    want = R.append(c, t, t, [0])
    cache_append(c, t, t, 0)
    for (a, s), (wa, ws) in zip(_stored(c), want):
        assert torch.equal(s, ws)
        _same(a, wa)


@pytest.mark.parametrize("B,H,D,S,capacity,start,counts", [
    (1, 1, 64, 1, 64, [0], None),
    (1, 2, 128, 1, 128, [63], None),
    (4, 2, 128, 1, 256, [64, 65, 127, 255], None),
    (3, 3, 64, 150, 320, [70, 0, 128], None),
    (4, 2, 128, 130, 256, [126, 1, 64, 60], [130, 0, 5, 3]),
    (2, 1, 64, 64, 128, [64, 32], [64, 64]),
    (5, 1, 64, 100, 128, [100, -1, 128, 27, 500], [100, 100, 100, 200, 1]),  # past the end, before the start
])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_append(device, B, H, D, S, capacity, start, counts, dtype):
    from lcv_bsa import cache_append

    gen = _gen(device, S + capacity)
    c = _cache(gen, device, B, H, capacity, D, spread=4.0)
    k, v = _rows(gen, device, B, H, S, D, dtype, 4.0), 3 * _rows(gen, device, B, H, S, D, dtype, 6.0)
    k[0, 0, 0, 5], v[-1, -1, -1, 7], v[0, 0, 0, 1] = math.inf, math.nan, -math.inf
    before = [t.clone() for t in (c.k8, c.v8)]
    want = R.append(c, k, v, start, counts)
    assert cache_append(c, k, v, _ints(device, start), _ints(device, counts)) is c
    for (a, s), (wa, ws) in zip(_stored(c), want):
        assert torch.equal(s, ws)
        _same(a, wa)
    # bytes behind the last new row, and of items left out, are as they were
    for b in range(B):
        n = min(S, counts[b] if counts else S)
        end = min(start[b] + n, capacity) if start[b] >= 0 and n > 0 else 0
        assert torch.equal(c.k8[b, :, end:].view(torch.uint8), before[0][b, :, end:].view(torch.uint8))


@pytest.mark.parametrize("layout", ["contiguous", "offset", "row stride", "shared heads", "one row", "reversed"])
def test_append_layouts(device, layout):
    from lcv_bsa import KVCache8, cache_append

    gen = _gen(device, 3)
    B, H, S, D = 2, 4, 70, 64
    x = torch.randn(B, H, S, D, generator=gen, device=device).to(BF16)
    if layout == "offset":
        x = torch.randn(B * H * S * D + 3, generator=gen, device=device).to(BF16)[3:].view(B, H, S, D)
    elif layout == "row stride":
        x = torch.randn(B, H, S, D + 4, generator=gen, device=device).to(BF16)[..., :D]
    elif layout == "shared heads":
        x = x[:, :1].expand(B, H, S, D)
    elif layout == "one row":
        x = x[:, :, :1].expand(B, H, S, D)
    elif layout == "reversed":
        x = x.transpose(-1, -2).contiguous().transpose(-1, -2)
    c, d = (KVCache8.empty(B, H, 128, D, device) for _ in range(2))
    cache_append(c, x, x, 3)
    cache_append(d, x.contiguous().clone(), x.contiguous().clone(), torch.tensor([3, 3], dtype=torch.int32, device=device))
    for a, b in ((c.k8, d.k8), (c.v8, d.v8)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(c.k_scale, d.k_scale) and torch.equal(c.v_scale, d.v_scale)


def test_append_token_by_token_is_append_at_once(device):
    """A block filled row by row, largest last, differs from one filled at once only
    below the smallest normal value of its last scale."""
    from lcv_bsa import KVCache8, cache_append

    gen = _gen(device, 8)
    x = torch.randn(1, 2, 70, 64, generator=gen, device=device) * torch.arange(1, 71, device=device).float()[:, None] * 0.01
    a, b = (KVCache8.empty(1, 2, 128, 64, device) for _ in range(2))
    cache_append(a, x, x, 0)
    at = torch.zeros(1, dtype=torch.int32, device=device)
    for i in range(70):
        cache_append(b, x[:, :, i:i + 1], x[:, :, i:i + 1], at)
        at += 1
    assert torch.equal(a.k_scale, b.k_scale)
    for (s, scale), (t, _) in zip(_stored(a), _stored(b)):
        big = s.abs() >= 2.0 ** -6
        assert torch.equal(s[big], t[big])
        assert float((s - t).abs().max()) <= 2.0 ** -9
    ka, va = a.dequantize()
    assert torch.equal(ka.cpu().double(), R.values(a)[0]) and torch.equal(va.cpu().double(), R.values(a)[1])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

CASES = [
    # B, Hq, H, D, S, capacity, lengths, q_lens, causal
    (1, 1, 1, 64, 1, 64, [1], None, False),
    (3, 2, 2, 128, 1, 256, [0, 65, 256], None, False),
    (4, 8, 2, 64, 1, 320, [63, 64, 129, 320], None, True),
    (2, 4, 1, 128, 3, 192, [130, 2], None, True),
    (3, 6, 2, 64, 7, 256, [200, 5, 64], [7, 0, 3], True),
    (2, 5, 5, 128, 33, 128, [128, 100], None, False),
    (2, 4, 2, 64, 70, 320, [300, 40], [70, 65], True),      # item 1: queries before the first token
    (1, 2, 1, 128, 150, 192, [150], None, True),
    (2, 3, 3, 64, 130, 448, [448, 1], [130, 130], False),
    (1, 8, 1, 128, 40, 640, [600], None, False),
    (2, 2, 2, 128, 300, 704, [700, 0], [1, 300], True),
    (70, 1, 1, 64, 1, 1280, [(37 * i * i) % 1281 for i in range(70)], None, False),  # more items than lanes, parts of 8 blocks
    (3, 3, 3, 64, 60, 1344, [1300, 30, 0], [60, 60, 5], True),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(device, case, dtype):
    from lcv_bsa import attention_weights, cached_attention

    B, Hq, H, D, S, capacity, lengths, q_lens, causal = case
    gen = _gen(device, S * 7 + D)
    c = _cache(gen, device, B, H, capacity, D, spread=2.0, stale=lengths)
    q = _rows(gen, device, B, Hq, S, D, dtype)
    out, lse = cached_attention(q, c, _ints(device, lengths), q_lens=_ints(device, q_lens), causal=causal, return_lse=True)
    want, want_lse, tol, tol_lse, probs, tol_p = R.attention(q, c, lengths, q_lens, causal)
    _within(out, want, tol)
    _within(lse, want_lse, tol_lse)
    w = torch.rand(B, H, c.capacity, generator=gen, device=device)
    more = attention_weights(q, c, _ints(device, lengths), lse, q_lens=_ints(device, q_lens), causal=causal, weights=w)
    given, tol_w = R.weights(probs, tol_p, H)
    _within(more, w.cpu().double() + given, tol_w + 2.0 ** -23 * (w.cpu().double() + given))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S", [1, 5, 40, 200])
def test_attention_nan_and_inf(device, S, dtype):
    """A NaN key or value counts for the rows that see it, and for no other; q's own
    NaN and infinities for their rows."""
    from lcv_bsa import cached_attention

    gen = _gen(device, S)
    B, H, D, n = 2, 2, 64, 256
    c = _cache(gen, device, B, H, n, D)
    lengths = [230, 250]
    c.k8.view(torch.uint8)[0, 0, 228, 3] = 127            # seen by the last rows
    v = c.v8.view(torch.uint8)                            # [B, H, nb, D, 64]
    v[1, 1, 248 // 64, 9, 248 % 64] = 255
    v[1, 0, 1, 2, 5] = 127                                # an early token: every row
    v[0, 0, 3, :, 232 - 192] = 127                        # behind the last
    q = _rows(gen, device, B, H, S, D, dtype)
    if S > 2:
        q[0, 1, 1, 4], q[1, 1, 0, 0] = math.nan, math.inf
    for causal in (True, False):
        out = cached_attention(q, c, _ints(device, lengths), causal=causal)
        want, _, tol, *_ = R.attention(q, c, lengths, None, causal)
        _within(out, want, tol)


@pytest.mark.parametrize("S", [1, 90, 130])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_scales(device, S, dtype):
    """Blocks of very different scales, a softmax scale of zero, large scores."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, 2)
    B, H, D, n = 1, 2, 128, 320
    c = KVCache8.empty(B, H, n, D, device)
    size = torch.tensor([1.0, 2.0 ** -30, 2.0 ** 8, 2.0 ** -8, 1.0], device=device).repeat_interleave(64)[:, None]
    k = torch.randn(B, H, n, D, generator=gen, device=device) * size.clamp(max=4)
    v = torch.randn(B, H, n, D, generator=gen, device=device) * size
    cache_append(c, k, v, 0)
    q = _rows(gen, device, B, H, S, D, dtype)
    for sm_scale in (None, 0.0, 3.0):
        out, lse = cached_attention(q, c, 300, sm_scale=sm_scale, return_lse=True)
        want, want_lse, tol, tol_lse, *_ = R.attention(q, c, [300], sm_scale=sm_scale)
        _within(out, want, tol)
        _within(lse, want_lse, tol_lse)


@pytest.mark.parametrize("S", [2, 40, 100])
def test_attention_layouts_and_bounds(device, S):
    """Strides of q and out, max_len, plain ints: the same result."""
    from lcv_bsa import attention_weights, cached_attention

    gen = _gen(device, 4)
    B, Hq, H, D = 2, 4, 2, 64
    c = _cache(gen, device, B, H, 512, D, stale=[190, 190])
    q = _rows(gen, device, B, Hq, S, D, BF16)
    want, lse = cached_attention(q.contiguous(), c, _ints(device, [190, 190]), return_lse=True)
    # Another bound on the lengths may split the walk elsewhere: P is then rounded against
    # another offset, so each result is within u (sum p |v| + |o|) of the exact one, not of
    # the other one.
    exact, _, far, *_ = R.attention(q, c, [190, 190])
    def near(x):
        _within(x, exact, far)
    near(want)
    near(cached_attention(q, c, 190))
    near(cached_attention(q, c, 190, max_len=190))
    near(cached_attention(q, c, 400, max_len=190))
    odd = torch.empty(B * Hq * S * D + 1, dtype=BF16, device=device)[1:].view(B, Hq, S, D).copy_(q)
    near(cached_attention(odd, c, 190))
    to = torch.zeros(B, S, Hq, D, dtype=BF16, device=device)
    assert cached_attention(q, c, 190, out=to.transpose(1, 2)).data_ptr() == to.data_ptr()
    near(to.transpose(1, 2))
    to = torch.zeros(B, Hq, S, D + 3, dtype=BF16, device=device)[..., :D]
    near(cached_attention(q, c, 190, out=to))
    near(to)
    one = q[:, :1].expand(B, Hq, S, D)
    assert torch.equal(cached_attention(one, c, 190), cached_attention(one.contiguous(), c, 190))
    empty, none = cached_attention(q, c, 0, return_lse=True)
    assert not empty.any() and bool((none == -math.inf).all())
    assert cached_attention(q[:, :, :0], c, 190).shape == (B, Hq, 0, D)
    w = attention_weights(q, c, 190, lse)
    assert torch.equal(w, attention_weights(q, c, 190, lse))  # the same bits again
    assert not w[:, :, 190:].any()
    torch.testing.assert_close(w.sum(-1), torch.full((B, H), float(Hq // H * S), device=device), rtol=1e-4, atol=0)
    w2 = w.clone()
    assert attention_weights(q, c, 190, lse, weights=w2, out=w2) is w2
    torch.testing.assert_close(w2, 2 * w, rtol=1e-6, atol=0)


# ---------------------------------------------------------------------------
# evict
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("B,H,D,capacity,lengths,keep,recent,kind", [
    (1, 1, 64, 64, [1], 1, 0, "random"),
    (2, 2, 128, 256, [200, 0], 70, 10, "random"),
    (3, 1, 64, 320, [320, 64, 63], 64, 64, "random"),
    (1, 3, 64, 1600, [1500], 700, 33, "ties"),
    (2, 1, 128, 192, [192, 100], 500, 7, "random"),
    (1, 2, 64, 2560, [2500], 1024, 0, "all equal"),
    (1, 2, 64, 256, [256], 100, 0, "special"),
    (2, 1, 64, 4224, [4200, 1030], 1, 0, "random"),
    (1, 1, 64, 4224, [4220], 4219, 1, "random"),
    (1, 1, 64, 4224, [4200], 2000, 5, "ties"),
    (1, 1, 64, 20544, [20500], 9000, 100, "ties"),
    (1, 1, 64, 20544, [20500], 300, 0, "spread"),
    (1, 1, 64, 66048, [66000], 100, 3, "ties"),
    (1, 1, 64, 66048, [65999], 30000, 0, "spread"),
    (1, 2, 64, 2560, [2500], 1200, 0, "two values"),
    (1, 1, 64, 2560, [2500], 2400, 0, "special"),
])
def test_evict(device, B, H, D, capacity, lengths, keep, recent, kind):
    from lcv_bsa import cache_evict

    gen = _gen(device, keep)
    c = _cache(gen, device, B, H, capacity, D, spread=3.0, stale=lengths)
    w = torch.rand(B, H, capacity, generator=gen, device=device)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "all equal":
        w.fill_(0.25)
    elif kind == "two values":
        w = torch.where(w > 0.5, 1e-38, 3e38)
    elif kind == "spread":  # every exponent, both signs
        w = torch.randint(0, 1 << 32, w.shape, generator=gen, device=device, dtype=torch.int64).to(torch.int32).view(torch.float32)
    elif kind == "special":
        w = w * 2 - 1
        w[..., ::7], w[..., 1::9], w[..., 2::11], w[..., 3::13], w[..., 4::5] = math.nan, math.inf, -math.inf, -0.0, 0.0
    new, new_w, kept, left = cache_evict(c, _ints(device, lengths), w, keep, recent=recent)
    want, stored = R.evict(c, lengths, w.cpu(), keep, recent)
    assert left.tolist() == [min(n, keep) for n in lengths]
    assert new.capacity == -(-keep // 64) * 64 and tuple(kept.shape) == (B, H, keep)
    for b in range(B):
        for h in range(H):
            at = want[b, h]
            assert kept[b, h].tolist() == at + [-1] * (keep - len(at))
            got = new_w[b, h].cpu()
            assert torch.equal(got[:len(at)].nan_to_num(9.0), w[b, h].cpu()[at].nan_to_num(9.0)) and not got[len(at):].any()
    for (a, s), (wa, ws) in zip(_stored(new), stored):
        assert torch.equal(s, ws)
        _same(a, wa)


# ---------------------------------------------------------------------------
# rope
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,H,S,D,dims,kind", [
    (1, 1, 1, 8, (8,), "int32"),
    (2, 3, 17, 128, None, "int32"),
    (1, 5, 65, 96, (32, 64), "int64"),
    (2, 2, 30, 64, (16, 24, 8, 16), "float"),
    (1, 33, 9, 256, (2, 254), "far"),
    (3, 1, 40, 128, (128,), "batch"),
])
def test_rope(device, B, H, S, D, dims, kind, dtype):
    from lcv_bsa import rope_nd

    gen = _gen(device, D)
    axes = 3 if dims is None else len(dims)
    pos = torch.randint(-50, 300, (S, axes), generator=gen, device=device, dtype=torch.int32)
    if kind == "int64":
        pos = pos.long()
    elif kind == "float":
        pos = pos.float() * 0.37
    elif kind == "far":
        pos = pos * 3_000_000
    elif kind == "batch":
        pos = torch.randint(0, 10000, (B, S, axes), generator=gen, device=device, dtype=torch.int32)
    x = torch.randn(B, S, H, D, generator=gen, device=device).to(dtype).transpose(1, 2).requires_grad_(True)
    g = torch.randn(B, H, S, D, generator=gen, device=device).to(dtype)
    y = rope_nd(x, pos, dims)
    d = dims or (D - 4 * (D // 6), 2 * (D // 6), 2 * (D // 6))
    # cos, sin and the angle are off by 2^-22 together (an angle within half a turn
    # in fp32, their own last bits, two products and a sum); the result is rounded once.
    pair = lambda t: t.detach().cpu().double().unflatten(-1, (-1, 2)).abs().sum(-1).repeat_interleave(2, -1)  # noqa: E731
    half = torch.finfo(dtype).eps / 2
    want = R.rope(x, pos, d)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    _within(y, want, half * want.abs() + 2.0 ** -21 * pair(x) + tiny)
    (dx,) = torch.autograd.grad(y, x, g)
    want = R.rope(g, pos, d, sign=-1)
    _within(dx, want, half * want.abs() + 2.0 ** -21 * pair(g) + tiny)


def test_rope_gradients(device):
    """Against differences; twice; of a broadcast input; of an expanded gradient."""
    from lcv_bsa import rope_nd

    gen = _gen(device, 1)
    pos = torch.randint(0, 50, (6, 2), generator=gen, device=device)
    x = torch.randn(1, 2, 6, 16, generator=gen, device=device, requires_grad=True)
    g = torch.randn(1, 2, 6, 16, generator=gen, device=device, requires_grad=True)
    (dx,) = torch.autograd.grad(rope_nd(x, pos), x, g, create_graph=True)
    d = torch.randn(x.shape, generator=gen, device=device)
    slope = ((rope_nd(x + d, pos) - rope_nd(x - d, pos)) * g).sum().double() / 2  # linear: exact up to rounding
    assert abs(float(slope - (dx * d).sum().double())) <= 1e-4
    (dg,) = torch.autograd.grad(dx, g, d)
    torch.testing.assert_close(dg, rope_nd(d, pos), rtol=0, atol=1e-6)
    shared = torch.randn(1, 1, 6, 16, generator=gen, device=device, requires_grad=True)
    rope_nd(shared.expand(1, 4, 6, 16), pos).sum().backward()
    want = 4 * R.rope(torch.ones(1, 1, 6, 16), pos, (8, 8), sign=-1)
    _within(shared.grad, want, torch.full_like(want, 1e-5))
    row = torch.randn(1, 2, 1, 16, generator=gen, device=device, requires_grad=True)
    rope_nd(row.expand(1, 2, 6, 16), pos).sum().backward()
    want = R.rope(torch.ones(1, 1, 6, 16), pos, (8, 8), sign=-1).sum(2, keepdim=True).expand(1, 2, 1, 16)
    _within(row.grad, want, torch.full_like(want, 1e-5))


def test_rope_agrees_with_the_grid(device):
    """On a whole latent grid it is rope_3d (whose angles are fp32)."""
    from lcv_bsa import grid_positions, rope_nd
    from lcv_bsa.rope_3d import rope_3d

    x = torch.randn(1, 4, 3 * 5 * 7, 128, generator=_gen(device, 1), device=device)
    a, _ = rope_3d(x, x, (3, 5, 7))
    torch.testing.assert_close(rope_nd(x, grid_positions((3, 5, 7), device=device)), a, rtol=0, atol=2e-5)
    assert grid_positions((2, 1, 2), (4, 0, 1)).tolist() == [[4, 0, 1], [4, 0, 2], [5, 0, 1], [5, 0, 2]]


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def _decode(c, q, k, v, pos, at, w):
    """One token of every item: turned, appended, attended to, weighed."""
    from lcv_bsa import attention_weights, cache_append, cached_attention, rope_nd

    q, k = rope_nd(q, pos), rope_nd(k, pos)
    cache_append(c, k, v, at)
    n = at + 1
    out, lse = cached_attention(q, c, n, causal=True, return_lse=True)
    attention_weights(q, c, n, lse, weights=w, out=w)
    at.add_(1)
    pos.add_(1)
    return out


def test_a_run_of_them_in_a_graph(device):
    """Decoding captured once and replayed as the lengths move on, against the same
    steps in 64 bits; then an eviction, and on with the shorter cache."""
    from lcv_bsa import KVCache8, cache_append, cache_evict

    gen = _gen(device, 11)
    B, Hq, H, D, steps = 2, 4, 2, 64, 6
    start = [61, 126]

    def state():
        g = _gen(device, 12)
        c = KVCache8.empty(B, H, 256, D, device)
        cache_append(c, _rows(g, device, B, H, 200, D, BF16), _rows(g, device, B, H, 200, D, BF16), 0)
        return c, torch.zeros(B, H, 256, device=device), _ints(device, start), _ints(device, start).view(B, 1, 1).clone()

    tokens = [[_rows(gen, device, B, h, 1, D, BF16) for h in (Hq, H, H)] for _ in range(steps)]
    held = [t.clone() for t in tokens[0]]
    c, w, at, pos = state()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _decode(c, *held, pos, at, w)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    c, w, at, pos = state()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = _decode(c, *held, pos, at, w)
    e, ew, eat, epos = state()
    for i, step in enumerate(tokens):
        for x, y in zip(held, step):
            x.copy_(y)
        graph.replay()
        eager = _decode(e, *step, epos, eat, ew)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(w, ew) and torch.equal(at, eat)
        assert torch.equal(c.k8.view(torch.uint8), e.k8.view(torch.uint8))
        lengths = [n + i + 1 for n in start]
        turned = R.rope(step[0], torch.tensor([[[n + i]] for n in start]), (D,)).to(BF16)
        want, *_ = R.attention(turned, e, lengths, None, True)
        assert float((eager.cpu().double() - want).norm() / want.norm()) < 2.0 ** -6
    lengths = [n + steps for n in start]
    left, lw, kept, n = cache_evict(e, eat, ew, 90, recent=16)
    assert n.tolist() == [min(m, 90) for m in lengths]
    # every query of every step gave one unit to each key head and query head of its group
    torch.testing.assert_close(ew.sum(-1), torch.full((B, H), float(Hq // H * steps), device=device), rtol=1e-4, atol=0)
    n2 = n.clone()
    out = _decode(left, *[t.to(BF16) for t in tokens[0]], pos, n2, lw)
    want, *_ = R.attention(R.rope(tokens[0][0], torch.tensor([[[m]] for m in lengths]), (D,)).to(BF16), left, n2.tolist(), None, True)
    assert float((out.cpu().double() - want).norm() / want.norm()) < 2.0 ** -6


def test_two_streams(device):
    from lcv_bsa import attention_weights, cached_attention

    gen = _gen(device, 6)
    c = _cache(gen, device, 1, 2, 1024, 128)
    qs = [_rows(gen, device, 1, 8, s, 128, F16) for s in (1, 3, 90, 150)]

    def both(q):
        out, lse = cached_attention(q, c, 1000, causal=True, return_lse=True)
        return out, attention_weights(q, c, 1000, lse, causal=True)

    want = [both(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got.append(both(q))
        torch.cuda.synchronize()
        for (a, b), (x, y) in zip(got, want):
            assert torch.equal(a, x) and torch.equal(b, y)


def test_extended(device):
    from lcv_bsa import cached_attention

    gen = _gen(device, 7)
    c = _cache(gen, device, 1, 2, 128, 64)
    d = c.extended(300, batch=3)
    assert d.shape == (3, 2, 320, 64)
    q = _rows(gen, device, 3, 2, 2, 64, BF16)
    out = cached_attention(q, d, 100, max_len=128)
    for b in range(3):
        assert torch.equal(out[b:b + 1], cached_attention(q[b:b + 1], c, 100))
