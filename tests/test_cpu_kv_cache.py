"""The 8-bit cache's refusals, and its reference's own arithmetic, without a GPU."""

from __future__ import annotations

import math

import pytest
import torch

import cache_reference as R

E4M3 = torch.float8_e4m3fn


@pytest.fixture
def on_cpu(monkeypatch):
    """The operators' checks run on CPU tensors; a launch would raise."""
    from lcv_bsa import _lib, kv_cache, rope_positions

    def no_launch():
        raise AssertionError("reached the library")

    for m in (kv_cache, rope_positions):
        monkeypatch.setattr(m, "_require_device", lambda *ts: None)
    monkeypatch.setattr(_lib, "load", no_launch)


def _parts(B=2, H=2, n=128, D=64):
    return [torch.zeros(B, H, n, D).to(E4M3), torch.zeros(B, H, n // 64, D, 64).to(E4M3), torch.ones(B, H, n // 64), torch.ones(B, H, n // 64)]


def _cache(**kw):
    from lcv_bsa import KVCache8

    return KVCache8(*_parts(**kw))


def test_cpu_tensors_are_refused():
    from lcv_bsa import KVCache8, rope_nd
    from lcv_bsa.block_sparse_attention import BSADeviceError

    with pytest.raises(BSADeviceError):
        KVCache8(*_parts())
    with pytest.raises(BSADeviceError):
        rope_nd(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    lambda p: p.__setitem__(0, p[0][..., :32]),
    lambda p: p.__setitem__(0, p[0][:, :, :100]),
    lambda p: p.__setitem__(0, p[0].float()),
    lambda p: p.__setitem__(0, p[0].view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E4M3)),
    lambda p: p.__setitem__(0, p[0][0]),
    lambda p: p.__setitem__(1, p[1].transpose(-1, -2)[:, :, :1]),
    lambda p: p.__setitem__(1, p[1].view(torch.uint8)),
    lambda p: p.__setitem__(2, p[2].double()),
    lambda p: p.__setitem__(3, p[3][:1]),
    lambda p: p.__setitem__(3, p[3][:1].expand(2, 2, 2)),
])
def test_cache_parts(on_cpu, change):
    from lcv_bsa import KVCache8

    parts = _parts()
    change(parts)
    with pytest.raises(ValueError):
        KVCache8(*parts)


def _i(*ns):
    return torch.tensor(ns, dtype=torch.int32)


def test_append_refusals(on_cpu):
    from lcv_bsa import cache_append

    c, x = _cache(), torch.zeros(2, 2, 10, 64)
    bad = [(x[:1], x[:1], 0, None), (x, x[:, :, :5], 0, None), (x, x.half(), 0, None), (x.double(), x.double(), 0, None),
           (x[..., :32], x[..., :32], 0, None), (x.int(), x.int(), 0, None), (x, x, 119, None), (x, x, -1, None),
           (x, x, _i(0), None), (x, x, torch.tensor([0, 0]), None), (x, x, 0, 11), (x, x, 0, _i(1, 2, 3)), (x, x, 0, -1),
           (torch.zeros(2, 2, 129, 64), torch.zeros(2, 2, 129, 64), 0, None),
           (x.requires_grad_(True) * 1, x.detach(), 0, None)]
    for k, v, start, counts in bad:
        with pytest.raises(ValueError):
            cache_append(c, k, v, start, counts)
    x = x.detach()
    with pytest.raises(AssertionError, match="reached"):
        cache_append(c, x, x, 118)
    assert cache_append(c, x[:, :, :0], x[:, :, :0], 0) is c


def test_attention_refusals(on_cpu):
    from lcv_bsa import attention_weights, cached_attention

    c, q = _cache(), torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16)
    lse, w = torch.zeros(2, 4, 3), torch.zeros(2, 2, 128)
    bad = [dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q[:, :1]), dict(q=q[..., :32]), dict(q=q.float()), dict(q=q[0]), dict(lengths=129),
           dict(lengths=-1), dict(lengths=_i(1)), dict(lengths=torch.tensor([1, 1])), dict(q_lens=4), dict(q_lens=_i(1, 2, 3)),
           dict(sm_scale=-1.0), dict(sm_scale=math.inf), dict(sm_scale=math.nan), dict(max_len=-1),
           dict(q=q.clone().requires_grad_(True))]
    for kw in bad:
        a = dict(dict(q=q, lengths=5), **kw)
        with pytest.raises(ValueError):
            cached_attention(a.pop("q"), c, a.pop("lengths"), **a)
        a = dict(dict(q=q, lengths=5), **kw)
        with pytest.raises(ValueError):
            attention_weights(a.pop("q"), c, a.pop("lengths"), lse, **a)
    for out in (q.float(), q[:, :2], torch.zeros(2, 1, 3, 64, dtype=q.dtype).expand(2, 4, 3, 64)):
        with pytest.raises(ValueError):
            cached_attention(q, c, 5, out=out)
    for kw in (dict(lse=lse[:1]), dict(lse=lse.half()), dict(weights=w[..., :64]), dict(weights=w.double()), dict(out=w[:1]),
               dict(out=torch.zeros(2, 128, 2).transpose(1, 2))):
        a = dict(dict(lse=lse), **kw)
        with pytest.raises(ValueError):
            attention_weights(q, c, 5, a.pop("lse"), **a)
    with pytest.raises(AssertionError, match="reached"):
        cached_attention(q, c, 128)
    out, none = cached_attention(q, c, 0, max_len=0, return_lse=True)
    assert not out.any() and bool((none == -math.inf).all())
    assert cached_attention(q[:, :, :0], c, 3).shape == (2, 4, 0, 64)
    assert torch.equal(attention_weights(q[:, :, :0], c, 3, lse[..., :0], weights=w + 1), w + 1)


def test_evict_refusals(on_cpu):
    from lcv_bsa import cache_evict

    c, w = _cache(), torch.zeros(2, 2, 128)
    for a, kw in (((5, w, 0), {}), ((5, w, 10), dict(recent=11)), ((5, w, 10), dict(recent=-1)), ((5, w[..., :64], 10), {}),
                  ((5, w.double(), 10), {}), ((129, w, 10), {}), ((_i(1), w, 10), {})):
        with pytest.raises(ValueError):
            cache_evict(c, *a, **kw)
    with pytest.raises(AssertionError, match="reached"):
        cache_evict(c, 5, w, 10)


def test_extended_refusals(on_cpu):
    c = _cache()
    for a in ((64,), (128, 3)):
        with pytest.raises(ValueError):
            c.extended(*a)
    assert _cache(B=1).extended(200, 3).shape == (3, 2, 256, 64)


def test_rope_refusals(on_cpu):
    from lcv_bsa import rope_nd

    x, p = torch.zeros(2, 2, 5, 64), torch.zeros(5, 3, dtype=torch.int32)
    bad = [(x[0], p, None), (x, p[:4], None), (x, p[None].expand(3, 5, 3), None), (x, p[0], None), (x, p.double(), None), (x.double(), p, None),
           (x, p[:, :0], None), (x, p, (32, 32)), (x, p, (31, 1, 32)), (x, p, (64, 2, -2)), (x, p, (0, 32, 32)), (x, p, (16, 16, 16)),
           (x[..., :60], p, None), (torch.zeros(2, 2, 5, 264), p, None), (x, torch.zeros(5, 5, dtype=torch.int32), None)]
    for a in bad:
        with pytest.raises(ValueError):
            rope_nd(*a)
    with pytest.raises(AssertionError, match="reached"):
        rope_nd(x, p)
    assert rope_nd(x[:, :, :0], p[:0]).shape == (2, 2, 0, 64)


@pytest.mark.skipif(torch.cuda.is_available(), reason="validation-only calls use fake pointers; CPU container only")
def test_c_entries_refuse_before_a_launch():
    import ctypes

    from lcv_bsa import _lib

    lib, S_, fake = _lib.load(), _lib.Strides, 4096
    C = lambda **kw: _lib.Cache8(**{**dict(k8=fake, v8=fake, k_scale=fake, v_scale=fake, B=1, H=2, capacity=128, D=64), **kw})  # noqa: E731
    st = S_(8192, 4096, 64)
    bad = [(C(k8=None), _lib.ERR_INVALID_ARG), (C(B=0), _lib.ERR_INVALID_ARG), (C(D=96), _lib.ERR_UNSUPPORTED), (C(capacity=100), _lib.ERR_SHAPE),
           (C(capacity=1 << 40), _lib.ERR_UNSUPPORTED), (C(B=1 << 30, H=1 << 30), _lib.ERR_UNSUPPORTED), (C(v8=fake + 8), _lib.ERR_LAYOUT)]
    for c, status in bad:
        assert lib.lcv_bsa_cache_append(c, fake, fake, 1, 4, st, st, fake, None, None) == status
        assert lib.lcv_bsa_cached_attn(fake, 1, 2, 4, st, c, fake, None, 0, 0.1, 64, fake, st, None, None, 0, None) == status
        assert lib.lcv_bsa_attention_weights(fake, 1, 2, 4, st, c, fake, None, 0, 0.1, 64, fake, None, fake, None, 0, None) == status
        assert lib.lcv_bsa_cache_evict(c, fake, fake, 4, 0, C(), fake, fake, fake, None) == status
        assert lib.lcv_bsa_cache_evict(C(), fake, fake, 4, 0, c, fake, fake, fake, None) == status

    def append(k=fake, dtype=1, S=4, ks=st, start=fake):
        return lib.lcv_bsa_cache_append(C(), k, fake, dtype, S, ks, st, start, None, None)

    assert append(k=None) == append(start=None) == append(S=0) == _lib.ERR_INVALID_ARG
    assert append(dtype=5) == _lib.ERR_DTYPE and append(S=129) == _lib.ERR_SHAPE
    assert append(k=fake + 2) == append(ks=S_(8192, 4096, 60)) == append(ks=S_(8192, -1, 64)) == append(ks=S_(8192, 4097, 64)) == _lib.ERR_LAYOUT

    def attn(dtype=1, Hq=2, S=4, scale=0.1, max_len=64, out=fake, lengths=fake, ws=None, size=0, c=C()):
        return lib.lcv_bsa_cached_attn(fake, dtype, Hq, S, st, c, lengths, None, 0, scale, max_len, out, st, None, ws, size, None)

    assert attn(dtype=2) == _lib.ERR_DTYPE and attn(Hq=3) == _lib.ERR_SHAPE
    assert attn(S=0) == attn(max_len=0) == attn(max_len=129) == attn(out=None) == attn(lengths=None) == _lib.ERR_INVALID_ARG
    assert attn(scale=-1.0) == attn(scale=math.inf) == attn(S=1 << 30) == _lib.ERR_UNSUPPORTED
    big = C(capacity=1 << 16)
    assert lib.lcv_bsa_cached_attn_workspace_bytes(2, 1, big, 1 << 16) > 0
    assert attn(S=1, max_len=1 << 16, c=big) == _lib.ERR_INVALID_ARG and b"workspace" in lib.lcv_bsa_last_error()
    assert lib.lcv_bsa_cached_attn_workspace_bytes(0, 1, big, 1 << 16) == 0

    def evict(keep=4, recent=0, dst=None, w=fake, new_w=2 * fake):
        dst = dst or C(k8=2 * fake, v8=2 * fake, k_scale=2 * fake, v_scale=2 * fake)
        return lib.lcv_bsa_cache_evict(C(), fake, w, keep, recent, dst, new_w, fake, fake, None)

    assert evict(keep=0) == evict(keep=129) == evict(recent=5) == evict(recent=-1) == evict(w=None) == evict(new_w=fake) == _lib.ERR_INVALID_ARG
    assert evict(dst=C(H=1)) == _lib.ERR_SHAPE and evict(dst=C(v8=2 * fake)) == _lib.ERR_INVALID_ARG

    def rope(dims, D=64, base=1e4, ptype=0, ps=3, xs=st):
        return lib.lcv_bsa_rope_nd(fake, 1, 1, 2, 4, D, xs, fake, ptype, 0, ps, (ctypes.c_int64 * len(dims))(*dims), len(dims), base, 0, fake, st, None)

    assert rope([32, 16]) == rope([33, 31]) == rope([64, 2]) == rope([-2, 66]) == _lib.ERR_SHAPE
    assert rope([64], base=0.0) == rope([64], base=math.inf) == rope([2] * 33) == _lib.ERR_INVALID_ARG
    assert rope([60], D=60) == _lib.ERR_UNSUPPORTED and rope([64], ptype=3) == _lib.ERR_DTYPE
    assert rope([64], ps=-1) == rope([64], xs=S_(8192, 4096, 63)) == _lib.ERR_LAYOUT


def test_reference_rounds_like_torch():
    """The reference's e4m3 against torch's conversion of every 16-bit value."""
    x = torch.arange(65536).to(torch.int32).to(torch.int16).view(torch.float16).double()
    x = x[x.abs() <= 448]
    got = R.nearest(x, torch.tensor(1.0))
    assert torch.equal(got, x.float().to(E4M3).double())
    assert torch.equal(R.TABLE[torch.arange(256)].nan_to_num(7.0), torch.arange(256).to(torch.uint8).view(E4M3).double().nan_to_num(7.0))
    assert R.least_scale(torch.tensor([448.0])) == 1.0 and R.least_scale(torch.tensor([448.5])) == 2.0
    assert R.least_scale(torch.tensor([0.0])) == 2.0 ** -60 and R.least_scale(torch.tensor([1e30])) == 2.0 ** 60
    assert R.least_scale(torch.tensor([math.inf, 1.0])) == 2.0 ** -8


def test_reference_attention_is_softmax():
    class Cache:
        pass

    c = Cache()
    g = torch.Generator().manual_seed(0)
    c.shape, c.capacity = (1, 1, 64, 64), 64
    c.k8, c.v8 = (torch.randn(1, 1, 64, 64, generator=g).to(E4M3), torch.randn(1, 1, 1, 64, 64, generator=g).to(E4M3))
    c.k_scale = c.v_scale = torch.full((1, 1, 1), 2.0)
    q = torch.randn(1, 2, 3, 64, generator=g).to(torch.bfloat16)
    out, lse, *_ = R.attention(q, c, [50], [2], True)
    k, v = R.values(c)
    t = q.double() @ k.transpose(-1, -2) / 8
    t = t.masked_fill(torch.arange(64) > torch.tensor([48, 49, -1])[:, None], -math.inf)
    want = torch.softmax(t, -1).nan_to_num(0.0) @ v
    torch.testing.assert_close(out, want)
    torch.testing.assert_close(lse, torch.logsumexp(t, -1))


def test_a_cache_keeps_its_tensors(on_cpu):
    """They cannot be exchanged for others, and what is passed on is where they are."""
    c = _cache()
    for name in ("k8", "v8", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
    moved = c.k_scale.clone()
    c.k_scale.data = moved
    p = c._pointers()
    assert (p.k8, p.v8, p.k_scale, p.v_scale) == (c.k8.data_ptr(), c.v8.data_ptr(), moved.data_ptr(), c.v_scale.data_ptr())


@pytest.mark.skipif(torch.cuda.is_available(), reason="validation-only calls use fake pointers; CPU container only")
def test_c_entries_refuse_overlaps():
    import ctypes

    from lcv_bsa import _lib

    lib, fake = _lib.load(), 1 << 20
    st = _lib.Strides(8192, 4096, 64)
    c = _lib.Cache8(k8=fake, v8=fake, k_scale=fake, v_scale=fake, B=1, H=2, capacity=128, D=64)
    for apart in (4, 1020, -4, -1020):  # of 1024 bytes
        assert lib.lcv_bsa_attention_weights(fake, 1, 2, 4, st, c, fake, None, 0, 0.1, 64, fake, fake, fake + apart, None, 0, None) == _lib.ERR_INVALID_ARG
        assert b"overlap" in lib.lcv_bsa_last_error()
    other = _lib.Strides(8192, 64, 128)
    assert lib.lcv_bsa_rope_nd(fake, 1, 1, 2, 4, 64, st, fake, 0, 0, 1, (ctypes.c_int64 * 1)(64), 1, 1e4, 0, fake, other, None) == _lib.ERR_LAYOUT
    assert b"in place" in lib.lcv_bsa_last_error()


def test_tangents_are_refused(on_cpu):
    """Forward-mode derivatives are not dropped; without a tangent the calls go on."""
    from torch.autograd import forward_ad

    from lcv_bsa import attention_weights, cache_append, cache_evict, cached_attention

    c, q, w = _cache(), torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 128)
    x, lse = torch.zeros(2, 2, 3, 64), torch.zeros(2, 4, 3)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda f: cache_append(c, f(x), x, 0), lambda f: cache_append(c, x, f(x), 0),
                     lambda f: cached_attention(f(q), c, 5), lambda f: cached_attention(q, c, 5, out=f(q.clone())),
                     lambda f: attention_weights(f(q), c, 5, lse), lambda f: attention_weights(q, c, 5, f(lse)),
                     lambda f: attention_weights(q, c, 5, lse, weights=f(w)), lambda f: cache_evict(c, 5, f(w), 10)):
            with pytest.raises(ValueError, match="derivative"):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match="derivative"):
                call(dual)
            with pytest.raises(AssertionError, match="reached"):
                call(lambda t: dual(t).detach())


def test_a_plain_start_has_to_fit_the_rows_counted(on_cpu):
    from lcv_bsa import cache_append

    c, x = _cache(), torch.zeros(2, 2, 10, 64)
    for start, counts in ((126, 2), (128, 0), (128, _i(0, 0)), (121, _i(7, 3))):
        with pytest.raises(AssertionError, match="reached"):
            cache_append(c, x, x, start, counts)
    for start, counts in ((127, 2), (129, 0), (129, _i(0, 0)), (-1, 2), (119, None)):
        with pytest.raises(ValueError):
            cache_append(c, x, x, start, counts)


def _addresses(shape, strides, first=0):
    at = torch.tensor([first])
    for n, st in zip(shape, strides):
        at = (at[:, None] + torch.arange(n) * st).flatten()
    return at.tolist()


@pytest.mark.parametrize("shape", [(2, 3, 4, 8), (1, 1, 5, 8), (2, 1, 1, 8), (3, 2, 2, 4)])
def test_shared_elements(shape):
    """Against the lists of addresses, for layouts of every kind."""
    from lcv_bsa.kv_cache import _shared

    layouts = [torch.empty(shape).stride(), torch.empty([shape[i] for i in (0, 2, 1, 3)]).transpose(1, 2).stride(),
               (0, 64, 8, 1), (40, 16, 8, 1), (9, 3, 30, 1), (7, 5, 3, 2), (512, 8, 24, 1), (300, 100, 12, 3), (64, 4, 16, 0)]
    for strides in layouts:
        here = _addresses(shape, strides)
        assert _shared(shape, strides, 0) == (len(set(here)) < len(here))
        for apart in range(-60, 61):
            if apart:
                there = {a + apart for a in here}
                assert _shared(shape, strides, apart) == (not there.isdisjoint(here)), (strides, apart)


def test_overlapping_outputs_are_refused(on_cpu):
    from lcv_bsa import cached_attention

    c, q = _cache(), torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16)
    held = torch.zeros(4096, dtype=torch.bfloat16)
    for strides in ((768, 192, 32, 1), (768, 128, 64, 1), (64, 192, 64, 1), (192, 192, 64, 1), (768, 192, 64, 0)):
        with pytest.raises(ValueError, match="share"):
            cached_attention(q, c, 5, out=held.as_strided(q.shape, strides))
    for strides in ((768, 192, 64, 1), (768, 64, 256, 1), (200, 400, 66, 1), (1, 400, 2, 6)):
        with pytest.raises(AssertionError, match="reached"):
            cached_attention(q, c, 5, out=held.as_strided(q.shape, strides))


@pytest.mark.skipif(torch.cuda.is_available(), reason="validation-only calls use fake pointers; CPU container only")
def test_c_attention_in_place_has_the_same_strides():
    from lcv_bsa import _lib

    lib, fake = _lib.load(), 1 << 20
    c = _lib.Cache8(k8=fake, v8=fake, k_scale=fake, v_scale=fake, B=1, H=2, capacity=128, D=64)
    a, b = _lib.Strides(8192, 4096, 64), _lib.Strides(8192, 64, 128)
    # Strides of a dimension of size one say nothing: such a call goes on to its workspace.
    long = _lib.Cache8(k8=fake, v8=fake, k_scale=fake, v_scale=fake, B=1, H=2, capacity=4096, D=64)
    for S, same in ((4, _lib.Strides(64, 4096, 64)), (1, _lib.Strides(8192, 4096, 128))):
        assert lib.lcv_bsa_cached_attn(fake, 1, 2, S, a, long, fake, None, 0, 0.1, 4096, fake, same, None, None, 0, None) == _lib.ERR_INVALID_ARG
        assert b"workspace" in lib.lcv_bsa_last_error()
    assert lib.lcv_bsa_cached_attn(fake, 1, 2, 4, a, c, fake, None, 0, 0.1, 64, fake, b, None, None, 0, None) == _lib.ERR_LAYOUT
    assert b"in place" in lib.lcv_bsa_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="validation-only calls use fake pointers; CPU container only")
def test_c_weights_refuse_an_out_on_lse():
    from lcv_bsa import _lib

    lib, fake = _lib.load(), 1 << 20
    st = _lib.Strides(8192, 4096, 64)
    c = _lib.Cache8(k8=fake, v8=fake, k_scale=fake, v_scale=fake, B=1, H=2, capacity=128, D=64)
    for apart in (0, 28, -1020):  # lse has 32 bytes, out 1024
        assert lib.lcv_bsa_attention_weights(fake, 1, 2, 4, st, c, fake, None, 0, 0.1, 64, fake, None, fake + apart, None, 0, None) == _lib.ERR_INVALID_ARG
        assert b"lse and out overlap" in lib.lcv_bsa_last_error()
