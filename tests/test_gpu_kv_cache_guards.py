"""The 8-bit cache beside what watches or changes a layer: norms of other kinds."""

from __future__ import annotations

import pytest
import torch

from conftest import NORM_CHANGES, changed_norms
from test_gpu_kv_cache import BF16, _gen, _stored
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
