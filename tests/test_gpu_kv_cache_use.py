"""The 8-bit KV cache's operators as a server or a training loop uses them: in captured
graphs, on several streams, over padded batches, over caches beyond 2^31 bytes."""

from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R
from test_gpu_kv_cache import BF16, F16, F32, _cache, _gen, _ints, _rows, _within

pytestmark = pytest.mark.gpu


def _bits(cache):
    return cache.k8.view(torch.uint8), cache.v8.view(torch.uint8), cache.k_scale, cache.v_scale


def _captured(fn):
    """fn() run once beside the default stream, then captured: (graph, its result)."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


@pytest.mark.parametrize("S", [1, 20, 150])
def test_two_captured_graphs(device, S):
    """Two graphs whose calls split their walks, replayed in turn and beside each other:
    neither works in the other's memory."""
    from lcv_bsa import attention_weights, cached_attention

    gen = _gen(device, S)
    c = _cache(gen, device, 1, 2, 2048, 64)
    qs = [_rows(gen, device, 1, 4, S, 64, F16) for _ in range(2)]
    lengths = _ints(device, [1999])

    def run(q):
        out, lse = cached_attention(q, c, lengths, causal=True, return_lse=True)
        return out, lse, attention_weights(q, c, lengths, lse, causal=True)

    graphs = [_captured(lambda q=q: run(q)) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for step in range(4):
        for q in qs:
            q.normal_(generator=gen)
        lengths.fill_(1990 - 300 * step)
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s if step % 2 else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        for q, (_, got) in zip(qs, graphs):
            for a, b in zip(got, run(q)):
                assert torch.equal(a, b)


def test_captured_append_and_evict(device):
    """The lengths, starts and weights that a replay finds are the ones it uses."""
    from lcv_bsa import cache_append, cache_evict

    gen = _gen(device, 5)
    B, H, D = 2, 2, 128
    start, counts, lengths = (_ints(device, x) for x in ([0, 100], [70, 33], [70, 133]))
    c, e = _cache(gen, device, B, H, 512, D), _cache(_gen(device, 5), device, B, H, 512, D)
    k, v = (_rows(gen, device, B, H, 70, D, BF16) for _ in range(2))
    w = torch.rand(B, H, 512, generator=gen, device=device)

    def run(cache):
        cache_append(cache, k, v, start, counts)
        return cache_evict(cache, lengths, w, 90, recent=20)

    before = [t.clone() for t in _bits(c)]
    graph, (left, lw, kept, n) = _captured(lambda: run(c))
    for t, was in zip(_bits(c), before):
        t.copy_(was)
    for step in range(4):
        k.normal_(generator=gen)
        w.uniform_(generator=gen)
        start.copy_(_ints(device, [50 * step, 400 - 90 * step]))
        counts.copy_(_ints(device, [70 - step, 10 * step]))
        lengths.copy_(_ints(device, [512 - step, 60 + 20 * step]))
        graph.replay()
        want, want_w, want_kept, want_n = run(e)
        torch.cuda.synchronize()
        for a, b in zip((*_bits(c), *_bits(left), lw, kept, n), (*_bits(e), *_bits(want), want_w, want_kept, want_n)):
            assert torch.equal(a, b)


def test_captured_rotary_gradient(device):
    """Forward and backward in one graph, replayed with other values and positions."""
    from lcv_bsa import rope_nd

    gen = _gen(device, 3)
    x = torch.randn(2, 3, 40, 64, generator=gen, device=device, requires_grad=True)
    g = torch.randn(2, 3, 40, 64, generator=gen, device=device)
    pos = torch.randint(0, 999, (2, 40, 2), generator=gen, device=device, dtype=torch.int32)

    def run():
        y = rope_nd(x, pos, (24, 40))
        return y.detach(), torch.autograd.grad(y, x, g)[0]

    graph, (y, dx) = _captured(run)
    for _ in range(4):
        with torch.no_grad():
            x.normal_(generator=gen)
        g.normal_(generator=gen)
        pos.random_(0, 5000, generator=gen)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])


def test_on_another_stream(device):
    """Each step on the stream that is current, its inputs made right before on that stream."""
    from lcv_bsa import KVCache8, attention_weights, cache_append, cache_evict, cached_attention, rope_nd

    def run():
        gen = _gen(device, 9)
        c = KVCache8.empty(1, 2, 4096, 128, device)
        k, q = _rows(gen, device, 1, 2, 4000, 128, BF16), _rows(gen, device, 1, 8, 130, 128, BF16)
        pos = torch.arange(4000, device=device)[:, None]
        cache_append(c, rope_nd(k, pos), k, 0)
        out, lse = cached_attention(rope_nd(q, pos[-130:]), c, 4000, causal=True, return_lse=True)
        w = attention_weights(q, c, 4000, lse, causal=True)
        return (out, lse, w, *_bits(cache_evict(c, 4000, w, 1000, recent=64)[0]))

    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("S", [3, 40, 150])
def test_padded_batch(device, S):
    """Rows behind an item's last hold NaN in q, k, v and lse: nothing of them is seen, and
    nothing behind an item's last token is written."""
    from lcv_bsa import KVCache8, attention_weights, cache_append, cached_attention

    gen = _gen(device, S)
    B, Hq, H, D, n = 3, 4, 2, 64, 512
    counts, start = [S, S // 2, 0], [130, 64, 7]
    c = _cache(gen, device, B, H, n, D)
    before = [t.clone() for t in R.values(c)]
    q, k, v = (_rows(gen, device, B, h, S, D, BF16) for h in (Hq, H, H))
    for t in (q, k, v):
        for b, m in enumerate(counts):
            t[b, :, m:] = math.nan
    cache_append(c, k, v, _ints(device, start), _ints(device, counts))
    lengths = [a + b for a, b in zip(start, counts)]
    held = R.values(c)
    for b, m in enumerate(lengths):
        end = (m + 63) // 64 * 64 if counts[b] else m  # a new scale there
        for x, y in zip(held, before):
            assert not torch.isnan(x[b]).any() and torch.equal(x[b, :, end:], y[b, :, end:])
    out, lse = cached_attention(q, c, _ints(device, lengths), q_lens=_ints(device, counts), causal=True, return_lse=True)
    want, want_lse, tol, tol_lse, probs, tol_p = R.attention(q, c, lengths, counts, True)
    _within(out, want, tol)
    _within(lse, want_lse, tol_lse)
    for b, m in enumerate(counts):
        lse[b, :, m:] = math.nan
    w = attention_weights(q, c, _ints(device, lengths), lse, q_lens=_ints(device, counts), causal=True)
    given, tol_w = R.weights(probs, tol_p, H)
    _within(w, given, tol_w + 2.0 ** -23 * given)


@pytest.mark.parametrize("S", [5, 130])
def test_strides_of_the_queries(device, S):
    """Rows of a projection that holds q, k and v; rows far apart; an lse with other strides."""
    from lcv_bsa import attention_weights, cached_attention

    gen = _gen(device, S)
    c = _cache(gen, device, 1, 2, 256, 64)
    qkv = torch.randn(1, S, 3, 4, 64, generator=gen, device=device).to(F16)
    wide = torch.zeros(1, 4, S, 4096, dtype=F16, device=device)
    plain = qkv[:, :, 1].transpose(1, 2).contiguous()
    wide[..., 64:128] = plain
    out, lse = cached_attention(plain, c, 200, causal=True, return_lse=True)
    w = attention_weights(plain, c, 200, lse, causal=True)
    for q in (qkv[:, :, 1].transpose(1, 2), wide[..., 64:128]):
        a, b = cached_attention(q, c, 200, causal=True, return_lse=True)
        assert torch.equal(a, out) and torch.equal(b, lse)
        assert torch.equal(attention_weights(q, c, 200, lse, causal=True), w)
        strided = lse.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(attention_weights(q, c, 200, strided, causal=True), w)


def test_scores_of_minus_infinity(device):
    """A row all of whose scores are -inf counts as one that sees nothing; a key of score
    -inf among others gets no weight."""
    from lcv_bsa import KVCache8, attention_weights, cache_append, cached_attention

    k = torch.zeros(1, 1, 64, 64, device=device)
    k[..., 0] = -1.0  # stored as -256
    v = torch.ones_like(k)
    none = cache_append(KVCache8.empty(1, 1, 64, 64, device), k, v, 0)
    k[0, 0, 40:, 0] = 0.0
    some = cache_append(KVCache8.empty(1, 1, 64, 64, device), k, v, 0)
    for S in (1, 20, 100):
        q = torch.zeros(1, 1, S, 64, dtype=BF16, device=device)
        q[..., 0] = 2.0 ** 120  # the products are -2^128
        out, lse = cached_attention(q, none, 64, return_lse=True)
        assert not out.any() and bool((lse == -math.inf).all())
        assert not attention_weights(q, none, 64, lse).any()
        out, lse = cached_attention(q, some, 64, return_lse=True)
        assert bool((out == 1).all())
        # exp of log 24, each within 2^-20
        w = attention_weights(q, some, 64, lse)[0, 0]
        assert not w[:40].any() and float((w[40:] - S / 24).abs().max()) <= S / 24 * 2.0 ** -18


@pytest.mark.parametrize("S", [1, 100])
def test_beyond_32_bits(device, S):
    """Two heads of 2^24 tokens: 4 GiB of keys and of values, the second head's all past
    2^31 bytes.  Against the second head's bytes as a cache of its own."""
    from lcv_bsa import KVCache8, attention_weights, cache_append, cache_evict, cached_attention

    gen = _gen(device, 8)
    n, D = 1 << 24, 128
    k8 = torch.randint(0, 256, (1, 2, n, D), generator=gen, device=device, dtype=torch.uint8)
    k8 &= 0xb7  # below 1 in size
    v8 = (k8 & 0x37).view(1, 2, n // 64, D, 64)
    v8[0, 1, :, 1::2] |= 8  # the second head's odd columns are larger
    one = torch.ones(1, 2, n // 64, device=device)
    e4m3 = torch.float8_e4m3fn
    c = KVCache8(k8.view(e4m3), v8.view(e4m3), one * 2.0 ** -4, one.clone())
    tail = [_rows(gen, device, 1, 2, 70, D, BF16) for _ in range(2)]
    cache_append(c, *tail, n - 71)
    half = KVCache8(c.k8[:, 1:], c.v8[:, 1:], c.k_scale[:, 1:], c.v_scale[:, 1:])
    k, v = (x[:, :, -72:] for x in KVCache8(c.k8[:, :, -128:].contiguous(), c.v8[:, :, -2:].contiguous(),
                                           c.k_scale[:, :, -2:].contiguous(), c.v_scale[:, :, -2:].contiguous()).dequantize())
    # half a step of e4m3 at the value, or of its block's smallest
    for x, y, scale in ((k, tail[0], c.k_scale), (v, tail[1], c.v_scale)):
        y = y.float()
        assert bool(((x[:, :, 1:71] - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale[..., -2:].max()).all())
    q = (_rows(gen, device, 1, 2, S, D, BF16) * 0.05).to(BF16)
    out, lse = cached_attention(q, c, n - 1, causal=True, return_lse=True)
    out1, lse1 = cached_attention(q[:, 1:], half, n - 1, causal=True, return_lse=True)
    # The same products, the walk split elsewhere.  A sum goes through at most 2^12 additions
    # in fp32 (a lane's of its part, then the parts'), each result off by 2^-12; P and the
    # output are rounded to bf16, 2^-9 each; the values are positive but for the last 70.
    assert float((lse[:, 1:] - lse1).abs().max()) <= 2 * 2.0 ** -12 + 2.0 ** -18
    off = (out[:, 1:].float() - out1.float()).abs() - (4 * 2.0 ** -9 + 2 * 2.0 ** -12) * out1.float().abs()
    assert float(off.max()) <= 2.0 ** -16
    w = attention_weights(q, c, n - 1, lse, causal=True)
    w1 = attention_weights(q[:, 1:], half, n - 1, lse[:, 1:].contiguous(), causal=True)
    assert torch.equal(w[:, 1:], w1) and not w[:, :, -1].any()
    assert abs(float(w1.double().sum()) - S) <= S * 2.0 ** -8
    few, fw, kept, m = cache_evict(c, n - 1, w, 200, recent=100)
    assert m.tolist() == [200]
    at = kept[0, 1].long()
    assert at[100:].tolist() == list(range(n - 101, n - 1)) and bool((at[1:] > at[:-1]).all())
    old = w[0, 1, :n - 101]
    assert float(old[at[:100]].min()) >= float(old.topk(101).values[-1])
    assert torch.equal(fw[0, 1, :200], w[0, 1][at])
    fk, fv = few.dequantize()
    got_k = c.k8[0, 1][at].float() * c.k_scale[0, 1][at // 64][:, None]
    got_v = c.v8.view(torch.uint8)[0, 1][at // 64, :, at % 64].view(e4m3).float() * c.v_scale[0, 1][at // 64][:, None]
    for x, y, scale in ((fk[0, 1, :200], got_k, few.k_scale), (fv[0, 1, :200], got_v, few.v_scale)):
        assert bool(((x - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale.max()).all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,q_lens", [
    ([500, 0, 3, 129, 512], [300, 7, 0, 129, 1]),
    ([64, 400], [300, 300]),  # item 0: queries before its first token
    ([5, 70, 140, 200, 512, 1, 0, 333, 64], [5, 70, 100, 0, 300, 1, 2, 33, 64]),
])
def test_ragged_batches(device, lengths, q_lens, causal):
    """Every row of every item is answered, whatever the order of the walks."""
    from lcv_bsa import attention_weights, cached_attention

    gen = _gen(device, len(lengths))
    B, S = len(lengths), 300
    c = _cache(gen, device, B, 2, 512, 64, stale=lengths)
    q = _rows(gen, device, B, 4, S, 64, BF16)
    out = torch.full((B, 4, S, 64), math.nan, dtype=BF16, device=device)
    n, m = _ints(device, lengths), _ints(device, q_lens)
    _, lse = cached_attention(q, c, n, q_lens=m, causal=causal, out=out, return_lse=True)
    want, want_lse, tol, tol_lse, probs, tol_p = R.attention(q, c, lengths, q_lens, causal)
    _within(out, want, tol)
    _within(lse, want_lse, tol_lse)
    given, tol_w = R.weights(probs, tol_p, 2)
    _within(attention_weights(q, c, n, lse, q_lens=m, causal=causal), given, tol_w + 2.0 ** -23 * given)


def test_rotary_rows_beyond_32_bits(device):
    """2^31 elements and more: the last heads' rows as on their own."""
    from lcv_bsa import rope_nd

    x = torch.zeros(1, 40, 1 << 20, 64, dtype=F16, device=device)
    x[:, -2:].normal_(generator=_gen(device, 2))
    pos = torch.arange(1 << 20, device=device)[:, None]
    want = rope_nd(x[:, -2:], pos)
    assert torch.equal(rope_nd(x, pos)[:, -2:], want)
    turned = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rope_nd(turned, pos)[:, -2:], want)


@pytest.mark.parametrize("S", [1, 6, 40, 150])
def test_out_may_be_q(device, S):
    """A row is read before it is written, and by its own workgroups alone."""
    from lcv_bsa import cached_attention

    gen = _gen(device, S)
    c = _cache(gen, device, 2, 2, 2048, 64)
    n = _ints(device, [2000, 130])
    q = torch.randn(2, 8, S, 64, generator=gen, device=device).to(BF16)
    want = cached_attention(q, c, n, causal=True)
    assert cached_attention(q, c, n, causal=True, out=q) is q and torch.equal(q, want)


def test_moved_tensors(device):
    """A cache whose tensors were given other memory is read where they are."""
    from lcv_bsa import cached_attention

    gen = _gen(device, 1)
    c = _cache(gen, device, 1, 2, 128, 64)
    q = torch.randn(1, 2, 3, 64, generator=gen, device=device).to(F16)
    want = cached_attention(q, c, 100)
    for t in (c.k8, c.v8, c.k_scale, c.v_scale):
        old = t.detach()  # the memory that it leaves
        t.data = old.view(torch.uint8).clone().view(t.dtype)
        old.view(torch.uint8).zero_()
    assert torch.equal(cached_attention(q, c, 100), want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind", ["plain", "causal", "outlier", "one outlier", "sizes", "tiny", "zeros", "nan"])
def test_long_walks(device, kind, dtype):
    """Walks of 32 blocks of D = 128 that are not split (1024 of them): what the queries hold.

    The reference's bound on a score's error, 136 2^-24 of the largest sum of |k| |q|, has
    room for a q that is held to 2^-22 of its row's largest value where that is a few times
    the others (2^-22 * 4 against 2^-17 of them), not where keys do not answer an outlier."""
    from lcv_bsa import KVCache8, cache_append, cached_attention

    gen = _gen(device, 3)
    H, S, D, n = 512, 130, 128, 1999
    k, v = (torch.randn(1, H, 2048, D, generator=gen, device=device) for _ in range(2))
    q = torch.randn(1, H, S, D, generator=gen, device=device)
    scale, causal = D ** -0.5, kind in ("causal", "nan")
    if kind in ("outlier", "one outlier"):
        k[..., 5] = 0.0
        q[:, :, (slice(None) if kind == "outlier" else 77), 5] = 2.0 ** 15
    elif kind == "sizes":
        q *= torch.randn(1, 1, S, 1, generator=gen, device=device).mul_(3).exp2_()
    elif kind == "tiny":
        small = 2.0 ** (-110 if dtype == BF16 else -12)
        q, scale = q * small, scale / small
    elif kind == "zeros":
        q *= torch.rand(q.shape, generator=gen, device=device) > 0.75
        q[:, :, 100:120] = 0.0
    c = cache_append(KVCache8.empty(1, H, 2048, D, device), k, v, 0)
    if kind == "nan":
        q[:, :, 7, 3], q[:, :, 30, 100] = math.nan, math.inf
        c.k8.view(torch.uint8)[:, :, 1950, 3] = 127
        c.v8.view(torch.uint8)[:, :, 31, 9, 1980 - 31 * 64] = 255
        c.v8.view(torch.uint8)[:, :, 31, 11, 10 + n - 31 * 64] = 127  # behind the last
    q = q.to(dtype)
    out, lse = cached_attention(q, c, n, causal=causal, sm_scale=scale, return_lse=True)
    for h in (0, H - 1):
        part = KVCache8(*(t[:, h:h + 1].clone(memory_format=torch.contiguous_format) for t in (c.k8, c.v8, c.k_scale, c.v_scale)))
        want, want_lse, tol, tol_lse, *_ = R.attention(q[:, h:h + 1], part, [n], None, causal, scale)
        _within(out[:, h:h + 1], want, tol)
        if kind != "nan":
            _within(lse[:, h:h + 1], want_lse, tol_lse)
