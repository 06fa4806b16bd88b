"""The DiT layer's KV cache in 8 bits: what return_kv gives, and the continuation from it."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = (2, 6, 7)  # 84 tokens a clip, 42 a frame: the cache ends inside a block


def _layer(device, dtype=torch.bfloat16, heads=2, dim=128, bsa=False):
    from lcv_bsa.dit_block import Attention

    torch.manual_seed(0)
    m = Attention(heads * dim, heads, dtype=dtype, device=device)
    with torch.no_grad():
        for p in (m.q_norm.weight, m.k_norm.weight):
            p.add_(0.1 * torch.randn_like(p))
    m.enable_bsa, m.bsa_shape_policy = bsa, "contiguous"
    m.kv_cache_8bit = True
    return m


def _x(device, B, frames, C, dtype=torch.bfloat16, seed=1):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(B, frames * GRID[1] * GRID[2], C, generator=g, device=device).to(dtype)


def _parts(cache):
    return cache.k8.view(torch.uint8), cache.v8.view(torch.uint8), cache.k_scale, cache.v_scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch", [1, 2])
def test_continuation(device, dtype, dim, batch):
    """Against the 16-bit cache.  Rounded to e4m3, a value is off by 2^-4 / sqrt(12) .. of
    itself in the mean square (under 2^-5), a score by as much of its own spread, so the
    attention's output by less than 2^-4 of its size."""
    m = _layer(device, dtype, 2, dim)
    with torch.no_grad():
        first, more = _x(device, 1, 2, 2 * dim, dtype), _x(device, batch, 3, 2 * dim, dtype, 2)
        out8, cache = m(first, GRID, return_kv=True)
        m.kv_cache_8bit = False
        out, plain = m(first, GRID, return_kv=True)
        assert torch.equal(out8, out)
        assert cache[0].shape == (1, 2, 128, dim) and cache[1] == 84
        want = m.forward_with_kv_cache(more, (3,) + GRID[1:], 2, plain).float()
        before = [t.clone() for t in _parts(cache[0])]
        got = m.forward_with_kv_cache(more, (3,) + GRID[1:], 2, cache)
        off = (got.float() - want).norm() / (want - m.proj.bias.float()).norm()
        assert float(off) < 2.0 ** -4
        # a step of a denoising loop leaves the cache as it was, and the next gives the same
        for a, b in zip(before, _parts(cache[0])):
            assert torch.equal(a, b)
        m.forward_with_kv_cache(100 * more, (3,) + GRID[1:], 2, cache)
        assert torch.equal(got, m.forward_with_kv_cache(more, (3,) + GRID[1:], 2, cache))


def test_keys_are_rotated_once(device):
    """The cache's keys are those of the unquantised path after RoPE."""
    from lcv_bsa.rope_3d import rope_3d

    m = _layer(device)
    with torch.no_grad():
        x = _x(device, 1, 2, 256)
        _, (cache, _) = m(x, GRID, return_kv=True)
        m.kv_cache_8bit = False
        _, (k, v) = m(x, GRID, return_kv=True)
        _, k = rope_3d(k, k, GRID)
        k8, v8 = cache.dequantize()
        for a, b in ((k8[:, :, :84], k), (v8[:, :, :84], v)):
            # half a step of e4m3, or of the block's smallest
            assert bool(((a - b.float()).abs() <= 2.0 ** -4 * b.float().abs() + 2.0 ** -9 * b.float().abs().max() / 448).all())


def test_with_block_sparse_attention(device):
    """64-token blocks: the fused pre-BSA pass fills the same cache."""
    grid = (2, 8, 8)
    m = _layer(device, bsa=True)
    with torch.no_grad():
        x = torch.randn(1, 128, 256, device=device, generator=torch.Generator(device=device).manual_seed(3)).to(torch.bfloat16)
        _, (cache, _) = m(x, grid, return_kv=True)
        assert m.last_path == "bsa"
        m.enable_bsa = False
        _, (plain, _) = m(x, grid, return_kv=True)
        (k, v), (k0, v0) = cache.dequantize(), plain.dequantize()
        assert torch.equal(v, v0)
        # k's norm and rotation round in other places: a step of bf16, then a step of e4m3
        assert float((k - k0).norm() / k0.norm()) < 2.0 ** -6


def test_block(device):
    from lcv_bsa.dit_block import LongCatSingleStreamBlock

    torch.manual_seed(1)
    m = LongCatSingleStreamBlock(256, 2, 4, 64, dtype=torch.bfloat16, device=device)
    g = torch.Generator(device=device).manual_seed(4)
    y = torch.randn(1, 9, 256, generator=g, device=device).to(torch.bfloat16)
    x, more = _x(device, 1, 2, 256), _x(device, 1, 3, 256, seed=5)
    t = torch.randn(1, 3, 64, generator=g, device=device)
    with torch.no_grad():
        _, plain = m(x, y, t[:, :2], [9], GRID, return_kv=True, skip_crs_attn=True)
        want = m(more, y, t, [9], (3,) + GRID[1:], 2, kv_cache=plain).float()
        m.attn.kv_cache_8bit = True
        _, cache = m(x, y, t[:, :2], [9], GRID, return_kv=True, skip_crs_attn=True)
        got = m(more, y, t, [9], (3,) + GRID[1:], 2, kv_cache=cache)
        assert float((got.float() - want).norm() / want.norm()) < 2.0 ** -4


def test_refusals(device):
    m = _layer(device)
    x, more = _x(device, 1, 2, 256), _x(device, 1, 3, 256)
    with pytest.raises(ValueError, match="backward"):
        m(x, GRID, return_kv=True)  # gradients are on
    with torch.no_grad():
        _, cache = m(x, GRID, return_kv=True)
        for shape, ncl in (((3,) + GRID[1:], None), ((3,) + GRID[1:], 3), ((3, 6, 6), 2), ((2,) + GRID[1:], 2)):
            with pytest.raises(ValueError):
                m.forward_with_kv_cache(more, shape, ncl, cache)
        with pytest.raises(ValueError):
            _layer(device, heads=4, dim=64).forward_with_kv_cache(more, (3,) + GRID[1:], 2, cache)


def test_captured_continuation(device):
    """A denoising step captured once, replayed with other latents and another clip's cache."""
    m = _layer(device)
    grid = (3,) + GRID[1:]
    with torch.no_grad():
        x, first = _x(device, 2, 3, 256), [_x(device, 1, 2, 256, seed=s) for s in (1, 7)]
        caches = [m(f, GRID, return_kv=True)[1] for f in first]
        held = m(first[0], GRID, return_kv=True)[1]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            m.forward_with_kv_cache(x, grid, 2, held)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.forward_with_kv_cache(x, grid, 2, held)
        for step in range(4):
            x.copy_(_x(device, 2, 3, 256, seed=20 + step))
            for a, b in zip(_parts(held[0]), _parts(caches[step % 2][0])):
                a.copy_(b)
            graph.replay()
            want = m.forward_with_kv_cache(x, grid, 2, caches[step % 2])
            torch.cuda.synchronize()
            assert torch.equal(out, want)
