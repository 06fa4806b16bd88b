"""A block without its text attention, as when a clip's cache is filled."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_fused_equals_unfused(device):
    """The fused passes against the module's own sequence in fp32, to bf16's rounding: four
    values on the way to the output are rounded, each by at most 2^-8 of itself."""
    from lcv_bsa.dit_block import LongCatSingleStreamBlock

    torch.manual_seed(1)
    m = LongCatSingleStreamBlock(256, 2, 4, 64, dtype=torch.bfloat16, device=device)
    g = torch.Generator(device=device).manual_seed(4)
    x = torch.randn(1, 84, 256, generator=g, device=device).to(torch.bfloat16)
    y = torch.randn(1, 9, 256, generator=g, device=device).to(torch.bfloat16)
    t = torch.randn(1, 2, 64, generator=g, device=device)
    with torch.no_grad():
        got, (k, v) = m(x, y, t, [9], (2, 6, 7), return_kv=True, skip_crs_attn=True)
        m.fused = False
        want, (k0, v0) = m(x, y, t, [9], (2, 6, 7), return_kv=True, skip_crs_attn=True)
    for a, b in ((got, want), (k, k0), (v, v0)):
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 4 * 2.0 ** -8
