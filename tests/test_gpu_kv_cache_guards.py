"""The 8-bit cache beside what watches or changes a layer: norms of other kinds, forward-mode
derivatives, block-sparse continuations; refusals before any work; outputs that share memory
with the queries; appending near the capacity."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from conftest import NORM_CHANGES, changed_norms
from test_gpu_kv_cache import BF16, F32, _cache, _gen, _ints, _stored
from test_gpu_kv_cache_layer import _layer

pytestmark = pytest.mark.gpu

GRID = (2, 8, 8)


def _input(device, C=256, dtype=BF16):
    return torch.randn(1, 128, C, generator=_gen(device, 3), device=device).to(dtype)


def _both(m, x):
    """return_kv with the cache in 16 and in 8 bits: (output, cache) each."""
    with torch.no_grad():
        m.kv_cache_8bit = False
        plain = m(x, GRID, return_kv=True)
        m.kv_cache_8bit = True
        return plain, m(x, GRID, return_kv=True)


def _same_keys(cache, plain):
    """The 8-bit cache holds the 16-bit one's keys after RoPE."""
    from lcv_bsa import KVCache8, cache_append
    from lcv_bsa.rope_3d import rope_3d

    (c, n), (k, v) = cache, plain
    k = rope_3d(k, k, GRID)[1]
    want = cache_append(KVCache8.empty(*k.shape, device=k.device), k, v, 0)
    for (a, s), (b, t) in zip(_stored(c), _stored(want)):
        assert torch.equal(a, b) and torch.equal(s, t)


@pytest.mark.parametrize("what", NORM_CHANGES)
def test_other_norms(device, what):
    m, x = _layer(device, bsa=True), _input(device)
    with changed_norms(what, m):
        (out, plain), (out8, cache) = _both(m, x)
    assert torch.equal(out8, out)
    _same_keys(cache, plain)


def test_norms_of_different_eps(device):
    m, x = _layer(device, bsa=True), _input(device)
    m.k_norm.eps = 0.5
    (out, plain), (out8, cache) = _both(m, x)
    assert torch.equal(out8, out)
    _same_keys(cache, plain)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rope_forward_mode(device, dtype):
    """Linear in x: the tangent is turned as x is, to the bit; through a backward pass too."""
    from lcv_bsa import rope_nd

    gen = _gen(device, 1)
    x, t, g = (torch.randn(1, 3, 20, 64, generator=gen, device=device).to(dtype) for _ in range(3))
    pos = torch.randint(0, 90, (20, 3), generator=gen, device=device)
    want, turned = rope_nd(x, pos), rope_nd(t, pos)
    for leaf in (x, x.clone().requires_grad_(True)):
        with forward_ad.dual_level():
            y, dy = forward_ad.unpack_dual(rope_nd(forward_ad.make_dual(leaf, t), pos))
            assert torch.equal(y, want) and torch.equal(dy, turned)
    with forward_ad.dual_level():  # a tangent that is differentiated in its turn
        r = t.clone().requires_grad_(True)
        dy = forward_ad.unpack_dual(rope_nd(forward_ad.make_dual(x, r), pos)).tangent
        (dr,) = torch.autograd.grad(dy, r, g)
    z = x.clone().requires_grad_(True)
    assert torch.equal(dr, torch.autograd.grad(rope_nd(z, pos), z, g)[0])
    with forward_ad.dual_level():  # no tangent, none made
        assert forward_ad.unpack_dual(rope_nd(x, pos)).tangent is None
        z = x.clone().requires_grad_(True)
        (dx,) = torch.autograd.grad(rope_nd(z, pos), z, forward_ad.make_dual(g, t))
        back, dback = forward_ad.unpack_dual(dx)
    z = x.clone().requires_grad_(True)
    grads = [torch.autograd.grad(rope_nd(z, pos), z, h)[0] for h in (g, t)]
    assert torch.equal(back, grads[0]) and torch.equal(dback, grads[1])


def test_layer_forward_mode(device):
    """A tangent is refused, not lost: where the cache is made and where it is read."""
    m, x = _layer(device), _input(device)
    more = torch.randn(1, 192, 256, generator=_gen(device, 4), device=device).to(BF16)
    with torch.no_grad():
        _, cache = m(x, GRID, return_kv=True)
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="derivative"):
                m(forward_ad.make_dual(x, x), GRID, return_kv=True)
            with pytest.raises(ValueError, match="derivative"):
                m.forward_with_kv_cache(forward_ad.make_dual(more, more), (3, 8, 8), 2, cache)


def test_append_near_the_capacity(device):
    """A plain start stands for the same number in a tensor, also where the rows counted
    alone fit."""
    from lcv_bsa import KVCache8, cache_append

    gen = _gen(device, 2)
    x = torch.randn(2, 2, 10, 64, generator=gen, device=device)
    for counts in (2, _ints(device, [2, 1])):
        a, b = (KVCache8.empty(2, 2, 128, 64, device) for _ in range(2))
        cache_append(a, x, x, 126, counts)
        cache_append(b, x, x, _ints(device, [126, 126]), counts if torch.is_tensor(counts) else _ints(device, [2, 2]))
        for (s, t), (u, w) in zip(_stored(a), _stored(b)):
            assert torch.equal(s, u) and torch.equal(t, w) and bool(s[:, :, 126:127].any())


@pytest.mark.parametrize("bsa", [False, True])
def test_refused_before_any_work(device, bsa, calls):
    """A gradient through the cache, or a head dim that it does not hold."""
    from lcv_bsa import dit_block

    seen = [calls(dit_block, name) for name in ("prepare_qk", "prepare_qkv", "bsa_attention", "dense_attention", "rope_3d")]
    m, x = _layer(device, bsa=bsa), _input(device)
    with pytest.raises(ValueError, match="backward"):
        m(x, GRID, return_kv=True)
    small = _layer(device, heads=8, dim=32, bsa=bsa)
    with torch.no_grad(), pytest.raises(ValueError, match="64 and 128"):
        small(x, GRID, return_kv=True)
    assert not any(seen)
    with torch.no_grad():
        m(x, GRID, return_kv=True)
    assert any(seen)


@pytest.mark.parametrize("S", [1, 4, 40, 130])
def test_out_beside_q(device, S):
    """out over q's memory, some rows on; out between q's rows."""
    from lcv_bsa import cached_attention

    gen = _gen(device, S)
    B, H, D = 2, 4, 64
    c = _cache(gen, device, B, H, 1024, D)
    n = _ints(device, [1000, 70])
    q = torch.randn(B, H, S, D, generator=gen, device=device).to(BF16)
    want = cached_attention(q, c, n)
    size = q.numel()
    for shift in (8, 64, 3 * 64, 64 * S, -64):
        held = torch.zeros(size + 2 * abs(shift), dtype=BF16, device=device)
        a, b = (shift, 2 * shift) if shift > 0 else (-shift, 0)
        src, to = held[a:a + size].view(B, H, S, D), held[b:b + size].view(B, H, S, D)
        src.copy_(q)
        assert cached_attention(src, c, n, out=to) is to and torch.equal(to, want)
    held = torch.zeros(size, dtype=BF16, device=device)
    src, to = held.view(B, H, S, D).copy_(q), held.view(B, S, H, D).transpose(1, 2)
    assert torch.equal(cached_attention(src, c, n, out=to), want)
    packed = torch.zeros(B, S, 3, H, D, dtype=BF16, device=device)
    src, to = packed[:, :, 0].transpose(1, 2), packed[:, :, 1].transpose(1, 2)
    src.copy_(q)
    assert torch.equal(cached_attention(src, c, n, out=to), want)
    assert torch.equal(src, q) and not packed[:, :, 2].any()


@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("dtype", [torch.float16, BF16])
def test_block_sparse_continuation(device, batch, dtype, monkeypatch):
    """BSA between cached and new frames runs from an 8-bit cache as from a 16-bit one: over
    the cached keys as they are stored and the new ones as they are."""
    from lcv_bsa import dit_block

    m = _layer(device, dtype, bsa=True)
    more = torch.randn(batch, 192, 128 * 2, generator=_gen(device, 5), device=device).to(dtype)
    x, shape = _input(device, dtype=dtype), (3,) + GRID[1:]
    with torch.no_grad():
        m.kv_cache_8bit = False
        plain = m(x, GRID, return_kv=True)[1]
        m.kv_cache_8bit = True
        cache = m(x, GRID, return_kv=True)[1]
        dense = m.forward_with_kv_cache(more, shape, 2, cache)
        assert m.last_paths == {"noise": "dense"}
        m.bsa_cond_noise, m.bsa_top_k, m.keep_indices = True, 5, True
        near = lambda a, b: float((a.float() - b.float()).norm() / (b.float() - m.proj.bias.float()).norm()) < 2.0 ** -4  # noqa: E731
        all_blocks = m.forward_with_kv_cache(more, shape, 2, cache)
        assert m.last_paths == {"noise": "bsa"} and near(all_blocks, dense)
        assert near(all_blocks, m.forward_with_kv_cache(more, shape, 2, plain))
        m.bsa_top_k, seen, bsa = 2, [], dit_block.bsa_attention

        def watched(q, k, v, *args, **kw):
            seen.append((q, k, v, kw))
            return bsa(q, k, v, *args, **kw)

        monkeypatch.setattr(dit_block, "bsa_attention", watched)
        out = m.forward_with_kv_cache(more, shape, 2, cache)
    (q, k, v, kw), = seen
    for got, held in zip((k, v), cache[0].dequantize(dtype)):
        assert got.shape == (batch, 2, 320, 128) and torch.equal(got[:, :, :128], held.expand(batch, -1, -1, -1))
    assert kw["kv_shape"] == (5, 8, 8) or kw["kv_shape"] == (1, 1, 320)
    idx = m.last_indices["noise"]
    assert idx.shape[-1] == 2
    # Each block of 64 queries over the keys of its two blocks, in 64 bits on the CPU; P and
    # the output are rounded to 16 bits, and so is the projection's input.
    want = torch.zeros(batch, 192, 2, 128, dtype=torch.float64)
    q, k, v, idx = (t.cpu() for t in (q.double(), k.double(), v.double(), idx.long()))
    for b in range(batch):
        for h in range(2):
            for i in range(3):
                at = (idx[b, h, i][:, None] * 64 + torch.arange(64)).flatten()
                s = q[b, h, 64 * i:64 * i + 64] @ k[b, h, at].T.contiguous() * 128 ** -0.5
                want[b, 64 * i:64 * i + 64, h] = torch.softmax(s, -1) @ v[b, h, at]
    want = want.flatten(2) @ m.proj.weight.detach().cpu().double().T + m.proj.bias.detach().cpu().double()
    assert float((out.cpu().double() - want).norm() / want.norm()) < 2.0 ** -6


def test_block_sparse_continuation_of_the_largest_values(device):
    """fp16's largest numbers round up to 2^16 in e4m3: widened, they are fp16's largest."""
    from lcv_bsa import KVCache8, cache_append

    m = _layer(device, torch.float16, bsa=True)
    gen = _gen(device, 6)
    more = torch.randn(1, 192, 256, generator=gen, device=device).to(torch.float16)
    k, v = (torch.randn(1, 2, 128, 128, generator=gen, device=device) for _ in range(2))
    v[:, :, 10, 3], v[:, 1, 70, 100], k[:, :, 30, 5] = 65504.0, -65000.0, 65504.0
    cache = cache_append(KVCache8.empty(1, 2, 128, 128, device), k, v, 0)
    with torch.no_grad():
        m.proj.weight.mul_(2.0 ** -6)
        m.bsa_cond_noise, m.bsa_top_k = True, 5
        out = m.forward_with_kv_cache(more, (3, 8, 8), 2, (cache, 128))
        assert m.last_paths == {"noise": "bsa"} and bool(torch.isfinite(out).all())
        m.bsa_cond_noise = False
        want = m.forward_with_kv_cache(more, (3, 8, 8), 2, (cache, 128)).float()
    assert float((out.float() - want).norm() / want.norm()) < 2.0 ** -4


def test_captured_block_sparse_continuation(device):
    """Captured once, replayed with other latents and another clip's cache."""
    from test_gpu_kv_cache_layer import _parts

    m, shape = _layer(device, bsa=True), (3, 8, 8)
    m.bsa_cond_noise, m.bsa_top_k = True, 3
    frames = lambda seed, n: torch.randn(1, n, 256, generator=_gen(device, seed), device=device).to(BF16)  # noqa: E731
    with torch.no_grad():
        caches = [m(frames(s, 128), GRID, return_kv=True)[1] for s in (1, 2)]
        held, x = m(frames(1, 128), GRID, return_kv=True)[1], frames(3, 192)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            m.forward_with_kv_cache(x, shape, 2, held)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.forward_with_kv_cache(x, shape, 2, held)
        assert m.last_paths == {"noise": "bsa"}
        for step in range(4):
            x.copy_(frames(20 + step, 192))
            for a, b in zip(_parts(held[0]), _parts(caches[step % 2][0])):
                a.copy_(b)
            graph.replay()
            want = m.forward_with_kv_cache(x, shape, 2, caches[step % 2])
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_continuation_with_gradients_is_refused(device, calls):
    from lcv_bsa import dit_block

    m, x = _layer(device, bsa=True), _input(device)
    more = torch.randn(1, 192, 256, generator=_gen(device, 5), device=device).to(BF16)
    with torch.no_grad():
        cache = m(x, GRID, return_kv=True)[1]
    seen = [calls(dit_block, name) for name in ("bsa_attention", "cached_attention", "rope_nd", "cache_append")]
    for m.bsa_cond_noise in (False, True):
        with pytest.raises(ValueError, match="backward"):
            m.forward_with_kv_cache(more, (3, 8, 8), 2, cache)
    assert not any(seen)
