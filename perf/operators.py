"""The 8-bit KV cache and the rotary positions around it, as timed cases.

A case is one call of an operator:

* ``rope``: ``rope_nd``, several position axes at given positions, forward or (``backward``) a training step's gradient;
* ``append``: ``cache_append``, new keys and values into a cache held in 8 bits;
* ``attend``: ``cached_attention``, queries over such a cache: single tokens, causal prompts, frames of a video;
* ``weights``: ``attention_weights``, how much attention each cached token got from these queries;
* ``evict``: ``cache_evict``, the cache cut down to its heaviest and its newest tokens.

The cache holds keys ``k8`` [B, H, capacity, D] and values ``v8`` [B, H, capacity / 64, D, 64] in e4m3, each block of 64
tokens of a head under one power of two (``k_scale``, ``v_scale`` [B, H, capacity / 64], fp32).

Lists (``lens``, ``q_lens``, ``start``) are texts, one number a batch item.  Sizes are the package's latent grids (45 x 80
tokens a frame at 720p, 30 x 52 at 480p, 32 heads of 128) and generic ones for text.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ESZ = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = 64
BASE = 10000.0


def rope(name, dtype, B, H, D, T, Hl, Wl, axes=3, at=0, backward=False):
    """``at``: the first frame's position; ``axes``: 3 (frame, row, column), 2 (row, column) or 1 (the token's number)."""
    return dict(name=name, kind="rope", dtype=dtype, B=B, H=H, D=D, T=T, Hl=Hl, Wl=Wl, axes=axes, at=at, backward=backward)


def append(name, dtype, H, D, S, start, counts):
    return dict(name=name, kind="append", dtype=dtype, H=H, D=D, S=S, start=start, counts=counts)


def attend(name, dtype, H, Hkv, D, S, lens, q_lens="", causal=False, kind="attend"):
    """S rows of queries an item; ``q_lens``: how many of them are real (all, if empty)."""
    return dict(name=name, kind=kind, dtype=dtype, H=H, Hkv=Hkv, D=D, S=S, lens=lens, q_lens=q_lens, causal=causal)


def evict(name, H, D, lens, keep, recent):
    return dict(name=name, kind="evict", H=H, D=D, lens=lens, keep=keep, recent=recent)


def listed():
    return [
        # Training on a preview-size latent in fp32: the gradient through the rotation, where the launch counts.
        rope("rope_preview_grad_f32", "f32", 1, 2, 128, 8, 16, 16, backward=True),
        # The 720p refinement pass's queries: 16 frames of 45 x 80 tokens, straight from the projection.
        rope("rope_720p_bf16", "bf16", 1, 32, 128, 16, 45, 80),
        # One new token for each of sixteen requests, at different depths (one at a block's start, one at its end).
        append("append_token_f16", "f16", 8, 128, 1, "64,700,1023,5,2048,1999,333,1280,127,850,4000,90,1111,2600,3333,17", ""),
        # Eight 480p frames behind four that are cached: the first of them shares a block with the last cached rows.
        append("append_frames_bf16", "bf16", 32, 128, 12480, "6240", ""),
        # One token over a short history: the smallest call of a decoder.
        attend("token_short_f16", "f16", 8, 8, 64, 1, "501"),
        # One token for each of eight requests over long histories, four query heads to a key head.
        attend("token_long_bf16", "bf16", 32, 8, 128, 1, "32768,17,30011,24576,9000,31999,12345,28000"),
        # A few tokens at once (a draft to be checked), causal among themselves.
        attend("draft_causal_f16", "f16", 32, 8, 128, 6, "8200,4097,1,12000", "6,6,6,3", True),
        # A padded batch of prompts, two of them behind cached text: causal, ragged.
        attend("prompt_causal_bf16", "bf16", 32, 8, 128, 2048, "2048,5000,391,3000", "2048,1999,391,1", True),
        # Video continuation at 480p: eight frames of queries over twelve frames of keys.
        attend("continue_480p_bf16", "bf16", 32, 32, 128, 12480, "18720"),
        # What one token of each request gave to its history.
        attend("weights_token_bf16", "bf16", 32, 8, 128, 1, "16384,9000,15999,4097", kind="weights"),
        # What two 480p frames gave to six.
        attend("weights_frames_f16", "f16", 32, 32, 128, 3120, "9360", kind="weights"),
        # A 480p history of twelve frames cut to half, the newest frame kept whole.
        evict("evict_480p", 32, 128, "18720", 9360, 1560),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(ns):
    return ",".join(str(n) for n in ns)


def _ints(text):
    return [int(t) for t in text.split(",")]


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "token", "token", "weights", "evict"])
    half = rng.choice(["f16", "bf16"])
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    H = Hkv * rng.choice([1, 1, 2, 4, 8])
    if kind == "rope":
        T, Hl, Wl = rng.randint(1, 16), rng.randint(1, 45), rng.randint(1, 80)
        c = rope("", rng.choice(["f16", "bf16", "f32"]), rng.choice([1, 1, 2]) if T * Hl * Wl < 28000 else 1, rng.choice([1, 2, 5, 8, 24]),
                 rng.choice([64, 96, 128, 128]), T, Hl, Wl, rng.choice([1, 2, 3, 3]), rng.choice([0, 7, 100000]), rng.random() < 0.5)
    elif kind == "append":
        B, S = rng.choice([1, 1, 2, 5]), _log(rng, 1, 12000)
        counts = [S] + [rng.randint(0, S) for _ in range(B - 1)]
        c = append("", half, Hkv, D, S, _text(rng.randint(0, 4000) for _ in range(B)), "" if B == 1 else _text(counts))
    elif kind == "token":
        B, S = rng.choice([1, 2, 4, 7]), rng.choice([1, 1, 1, 2, 5])
        c = attend("", half, H, Hkv, D, S, _text(_log(rng, 1, 30000) for _ in range(B)), "", S > 1)
    elif kind == "evict":
        lens = [_log(rng, 70, 18000) for _ in range(rng.choice([1, 1, 3]))]
        keep = rng.randint(1, max(lens))
        c = evict("", Hkv, D, _text(lens), keep, rng.choice([0, keep // 8, keep]))
    else:
        B, S = rng.choice([1, 1, 2, 3]), _log(rng, 17, 3000)
        lens = [_log(rng, 1, 9000) for _ in range(B)]
        q_lens = "" if rng.random() < 0.5 else _text([S] + [rng.randint(0, S) for _ in range(B - 1)])
        c = attend("", half, H, Hkv, D, S, _text(lens), q_lens, rng.random() < 0.5, kind)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# Sizes
# ---------------------------------------------------------------------------

def _blocks(n):
    return -(-n // BLOCK)


def _q_lens(c):
    return _ints(c["q_lens"]) if c["q_lens"] else [c["S"]] * len(_ints(c["lens"]))


def _visible(c):
    """(query, key) pairs of one head over all items."""
    total = 0
    for n, m in zip(_ints(c["lens"]), _q_lens(c)):
        total += sum(range(max(0, n - m + 1), n + 1)) if c["causal"] else m * n
    return total


def work(c):
    if c["kind"] == "rope":
        rows = c["B"] * c["T"] * c["Hl"] * c["Wl"]
        return {"bytes": 2 * rows * c["H"] * c["D"] * ESZ[c["dtype"]] + 4 * c["axes"] * rows // c["B"], "flops": 3 * rows * c["H"] * c["D"]}
    if c["kind"] == "append":
        rows = sum(_ints(c["counts"])) if c["counts"] else c["S"] * len(_ints(c["start"]))
        return {"bytes": 2 * rows * c["H"] * c["D"] * (ESZ[c["dtype"]] + 1), "flops": 6 * rows * c["H"] * c["D"]}
    if c["kind"] == "evict":
        kept = sum(min(n, c["keep"]) for n in _ints(c["lens"])) * c["H"]
        return {"bytes": kept * (4 * c["D"] + 4 + 4) + 4 * sum(_ints(c["lens"])) * c["H"], "flops": 4 * kept * c["D"]}
    keys, rows = sum(n for n, m in zip(_ints(c["lens"]), _q_lens(c)) if m), sum(_q_lens(c))
    if c["kind"] == "weights":
        return {"bytes": keys * c["Hkv"] * (c["D"] + 8) + rows * c["H"] * (2 * c["D"] + 4), "flops": 2 * c["D"] * c["H"] * _visible(c)}
    return {"bytes": 2 * keys * c["Hkv"] * c["D"] + rows * c["H"] * (4 * c["D"] + 4), "flops": 4 * c["D"] * c["H"] * _visible(c)}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _rope_dims(D, axes):
    """Dims of each axis: the package's split for three, halves for two."""
    if axes == 3:
        return (D - 4 * (D // 6), 2 * (D // 6), 2 * (D // 6))
    return (D // 2, D // 2) if axes == 2 else (D,)


def _positions(c, dev):
    """[S, axes] int32."""
    if c["axes"] == 1:
        return (c["at"] + torch.arange(c["T"] * c["Hl"] * c["Wl"], device=dev, dtype=torch.int32))[:, None]
    t, h, w = (torch.arange(n, device=dev, dtype=torch.int32) for n in (c["T"], c["Hl"], c["Wl"]))
    grid = torch.stack(torch.meshgrid(t + c["at"], h, w, indexing="ij"), -1).reshape(-1, 3)
    return (grid if c["axes"] == 3 else grid[:, 1:] + c["at"]).contiguous()


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, within [-60, 60]: 448 = 0.875 * 2^9."""
    m, x = torch.frexp(amax.float())
    return torch.where(amax > 0, x - 9 + (m > 0.875).int(), -60).clamp(-60, 60)


def _to_8(x, e):
    """x * 2^-e in e4m3, to nearest."""
    return torch.ldexp(x.float(), -e).to(torch.float8_e4m3fn)


def _values(gen, dev, B, H, n, D, keys):
    """Keys: normed rows with a few strong channels.  Values: rows whose size drifts from block to block."""
    x = torch.randn(B, H, n, D, generator=gen, device=dev)
    if keys:
        x *= 1 + 3 * (torch.rand(H, 1, D, generator=gen, device=dev) > 0.95)
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True))
    drift = torch.randn(B, H, _blocks(n), 1, generator=gen, device=dev).exp2_()
    return x * drift.repeat_interleave(BLOCK, 2)[:, :, :n]


def _cache(gen, dev, B, H, capacity, D):
    """A cache filled to its capacity."""
    nb = capacity // BLOCK
    k, v = (_values(gen, dev, B, H, capacity, D, keys).view(B, H, nb, BLOCK, D) for keys in (True, False))
    ek, ev = (_exponent(x.abs().amax((-1, -2))) for x in (k, v))
    one = torch.ones((), device=dev)
    return dict(k8=_to_8(k, ek[..., None, None]).view(B, H, capacity, D), v8=_to_8(v.transpose(-1, -2).contiguous(), ev[..., None, None]),
                k_scale=torch.ldexp(one, ek), v_scale=torch.ldexp(one, ev))


def _forget(cache, lens):
    """What stands behind an item's last token is left from earlier requests: any bytes, NaN among them."""
    k, v = cache["k8"].view(torch.uint8), cache["v8"].view(torch.uint8)
    for b, n in enumerate(lens):
        k[b, :, n:, ::7] = 127
        at = n // BLOCK
        if at < v.shape[2]:
            v[b, :, at, ::5, n % BLOCK:] = 255
            v[b, :, at + 1:, ::5] = 127


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if c["kind"] == "rope":
        S = c["T"] * c["Hl"] * c["Wl"]
        x = torch.randn(c["B"], S, c["H"], c["D"], generator=gen, device=dev).to(DTYPES[c["dtype"]]).transpose(1, 2)
        g = torch.randn(c["B"], S, c["H"], c["D"], generator=gen, device=dev).to(DTYPES[c["dtype"]]).transpose(1, 2) if c["backward"] else None
        return dict(kind="rope", x=x, g=g, positions=_positions(c, dev), dims=_rope_dims(c["D"], c["axes"]))

    def ints(ns):
        return torch.tensor(ns, dtype=torch.int32, device=dev)

    if c["kind"] == "append":
        start = _ints(c["start"])
        B, S = len(start), c["S"]
        s = _cache(gen, dev, B, c["H"], BLOCK * _blocks(max(start) + S), c["D"])
        k, v = (_values(gen, dev, B, c["H"], S, c["D"], keys).transpose(1, 2).contiguous().to(DTYPES[c["dtype"]]).transpose(1, 2) for keys in (True, False))
        return dict(kind="append", k=k, v=2 * v, start=ints(start), counts=ints(_ints(c["counts"])) if c["counts"] else None, **s)
    lens = _ints(c["lens"])
    B, longest = len(lens), max(lens)
    if c["kind"] == "evict":
        s = _cache(gen, dev, B, c["H"], BLOCK * _blocks(longest), c["D"])
        weights = torch.rand(B, c["H"], BLOCK * _blocks(longest), generator=gen, device=dev).pow_(4).mul_(8)
        return dict(kind="evict", lengths=ints(lens), weights=weights, keep=c["keep"], recent=c["recent"], **s)
    s = _cache(gen, dev, B, c["Hkv"], BLOCK * (_blocks(longest) + 2), c["D"])
    _forget(s, lens)
    q = (0.7 * torch.randn(B, c["S"], c["H"], c["D"], generator=gen, device=dev)).to(DTYPES[c["dtype"]]).transpose(1, 2)
    s.update(kind=c["kind"], q=q, lengths=ints(lens), q_lens=ints(_q_lens(c)) if c["q_lens"] else None, causal=c["causal"], max_len=longest)
    if c["kind"] == "weights":
        s["weights"] = torch.rand(B, c["Hkv"], s["k8"].shape[2], generator=gen, device=dev)
        s["lse"] = _scores(s)[1]
    return s


# ---------------------------------------------------------------------------
# The plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------

def _rotate(x, positions, dims, sign):
    """Angles in 64 bits (a far position times a frequency), the rest in 32."""
    parts = [positions[:, a, None].double() * BASE ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d) for a, d in enumerate(dims)]
    angle = torch.cat(parts, -1)
    cos, sin = angle.cos().float(), sign * angle.sin().float()
    a, b = x[..., ::2].float(), x[..., 1::2].float()
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).to(x.dtype)


def _append(s):
    """Every block that the new rows touch: read, filled, scaled, rounded and written."""
    k, v, start = s["k"], s["v"], s["start"].long()
    B, H, S, D = k.shape
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(start, S)
    nb, touched = s["k_scale"].shape[2], (S + 2 * BLOCK - 2) // BLOCK
    first = start // BLOCK
    at = (first[:, None] + torch.arange(touched, device=k.device)).clamp(max=nb - 1)  # [B, touched]
    token = (first[:, None] + torch.arange(touched, device=k.device))[..., None] * BLOCK + torch.arange(BLOCK, device=k.device)
    row = (token - start[:, None, None]).flatten(1)  # the new row of each token
    new = ((row >= 0) & (row < counts[:, None])).view(B, 1, touched, BLOCK, 1)
    old = ((row < 0) & (counts > 0)[:, None]).view(B, 1, touched, BLOCK, 1)
    item = torch.arange(B, device=k.device)[:, None]
    live = new.any(-2)[:, 0, :, 0]  # [B, touched]
    for x, name in ((k, "k"), (v, "v")):
        held = s[name + "8"].view(torch.uint8)
        held = held.view(B, H, nb, BLOCK, D) if name == "k" else held
        scale = s[name + "_scale"]
        before = held.transpose(1, 2)[item, at].transpose(1, 2)  # [B, H, touched, ...]
        bytes_ = before if name == "k" else before.transpose(-1, -2)
        was = scale.transpose(1, 2)[item, at].transpose(1, 2)  # [B, H, touched]
        rows = x.float().gather(2, row.clamp(0, S - 1)[:, None, :, None].expand(B, H, -1, D)).view(B, H, touched, BLOCK, D)
        rows = torch.where(new, rows, 0.0)
        e = _exponent(rows.abs().amax((-1, -2)))
        kept = old.any(-2)[..., 0]
        e = torch.where(kept, torch.maximum(e, torch.frexp(was)[1] - 1), e)
        held_rows = bytes_.contiguous().view(torch.float8_e4m3fn).float() * was[..., None, None]
        out = _to_8(torch.where(new, rows, held_rows), e[..., None, None]).view(torch.uint8)
        out = torch.where(new | old, out, bytes_)
        out = out if name == "k" else out.transpose(-1, -2)
        b, j = live.nonzero(as_tuple=True)
        held.transpose(1, 2)[b, at[b, j]] = out.transpose(1, 2)[b, j]
        scale.transpose(1, 2)[b, at[b, j]] = torch.ldexp(torch.ones_like(was), e).transpose(1, 2)[b, j]
    return {n: s[n] for n in ("k8", "v8", "k_scale", "v_scale")}


def _seen(s, S, n):
    """[B, 1, S, n]: whether query i attends to token j."""
    i, j = torch.arange(S, device=s["q"].device)[:, None], torch.arange(n, device=s["q"].device)
    lens = s["lengths"].view(-1, 1, 1, 1)
    q_lens = s["q_lens"].view(-1, 1, 1, 1) if s["q_lens"] is not None else torch.full_like(lens, S)
    seen = (j < lens) & (i < q_lens)
    return seen & (j <= lens - q_lens + i) if s["causal"] else seen


def _held(s, name, groups):
    """[B, H, n, D] fp32: the cached rows of each query head's key head; unused ones are zero."""
    n = s["max_len"]
    B, H, nb = s[name + "_scale"].shape
    x = s["k8"].view(B, H, nb, BLOCK, -1) if name == "k" else s["v8"].transpose(-1, -2)
    x = (x.float() * s[name + "_scale"][..., None, None]).reshape(B, H, nb * BLOCK, -1)[:, :, :n]
    used = torch.arange(n, device=x.device)[:, None] < s["lengths"].view(-1, 1, 1, 1)
    return torch.where(used, x, 0.0).repeat_interleave(groups, 1)


def _scores(s):
    """(scores with -inf where nothing is seen, lse)."""
    q = s["q"]
    k = _held(s, "k", q.shape[1] // s["k_scale"].shape[1])
    t = torch.matmul(q.float(), k.transpose(-1, -2).contiguous()).mul_(q.shape[-1] ** -0.5)
    t = t.masked_fill_(~_seen(s, q.shape[2], k.shape[2]), -math.inf)
    return t, torch.logsumexp(t, -1)


def _probabilities(t, lse):
    return t.sub_(lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp_()


def _attend(s):
    t, lse = _scores(s)
    out = torch.matmul(_probabilities(t, lse), _held(s, "v", t.shape[1] // s["v_scale"].shape[1]))
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _weights(s):
    t = _scores(s)[0]
    B, H, n = s["weights"].shape
    given = _probabilities(t, s["lse"]).sum(-2).view(B, H, -1, t.shape[-1]).sum(2)
    return {"weights": s["weights"] + torch.nn.functional.pad(given, (0, n - given.shape[-1]))}


def _evict(s):
    B, H, n = s["weights"].shape
    D, keep = s["k8"].shape[-1], s["keep"]
    lens = s["lengths"].long()
    j = torch.arange(n, device=lens.device)
    recent = j >= (lens - s["recent"])[:, None]
    rank = torch.where(recent[:, None], math.inf, s["weights"])
    rank = torch.where((j < lens[:, None])[:, None], rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices  # equal weights: the lowest first
    left = lens.clamp(max=keep)
    slot = torch.arange(keep, device=lens.device)
    there = (slot < left[:, None])[:, None]  # [B, 1, keep]
    kept = torch.where(there, order[..., :keep] if keep <= n else torch.nn.functional.pad(order, (0, keep - n)), n).sort(-1).values
    kept = torch.where(there, kept, -1)
    at = kept.clamp(min=0)
    nb = _blocks(keep)
    out = {"kept": kept.int(), "lengths": left.int()}
    more = nb * BLOCK - keep
    out["weights"] = torch.nn.functional.pad(torch.where(there, s["weights"].gather(2, at), 0.0), (0, more))
    for name in ("k", "v"):
        x = s["k8"].view(B, H, n // BLOCK, BLOCK, D) if name == "k" else s["v8"].transpose(-1, -2)
        x = (x.float() * s[name + "_scale"][..., None, None]).reshape(B, H, n, D)
        x = torch.where(there[..., None], x.gather(2, at[..., None].expand(-1, -1, -1, D)), 0.0)
        x = torch.nn.functional.pad(x, (0, 0, 0, more)).view(B, H, nb, BLOCK, D)
        filled = (torch.arange(nb, device=lens.device) * BLOCK < left[:, None])[:, None]
        e = torch.where(filled, _exponent(x.abs().amax((-1, -2))), 0)
        x8 = _to_8(x, e[..., None, None])
        out[name + "8"] = x8.view(B, H, nb * BLOCK, D) if name == "k" else x8.transpose(-1, -2).contiguous()
        out[name + "_scale"] = torch.ldexp(torch.ones((), device=x.device), e)
    return out


def _plain(s):
    if s["kind"] == "rope":
        return {"y": _rotate(s["x"], s["positions"], s["dims"], 1.0)} if s["g"] is None else {"dx": _rotate(s["g"], s["positions"], s["dims"], -1.0)}
    return {"append": _append, "attend": _attend, "weights": _weights, "evict": _evict}[s["kind"]](s)


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------

def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "longcat-video-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import lcv_bsa

    return lcv_bsa


def _call(s):
    P = _package()
    if s["kind"] == "rope":
        if s["g"] is None:
            return {"y": P.rope_nd(s["x"], s["positions"], s["dims"])}
        x = s["x"].detach().requires_grad_(True)
        return {"dx": torch.autograd.grad(P.rope_nd(x, s["positions"], s["dims"]), x, s["g"])[0]}
    cache = P.KVCache8(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
    if s["kind"] == "append":
        P.cache_append(cache, s["k"], s["v"], s["start"], s["counts"])
        return {n: s[n] for n in ("k8", "v8", "k_scale", "v_scale")}
    if s["kind"] == "evict":
        left, weights, kept, lengths = P.cache_evict(cache, s["lengths"], s["weights"], s["keep"], recent=s["recent"])
        return {"kept": kept, "lengths": lengths, "weights": weights, "k8": left.k8, "v8": left.v8, "k_scale": left.k_scale, "v_scale": left.v_scale}
    how = dict(q_lens=s["q_lens"], causal=s["causal"], max_len=s["max_len"])
    if s["kind"] == "attend":
        out, lse = P.cached_attention(s["q"], cache, s["lengths"], return_lse=True, **how)
        return {"out": out, "lse": lse}
    return {"weights": P.attention_weights(s["q"], cache, s["lengths"], s["lse"], weights=s["weights"], **how)}


def run(s):
    return _call(s) if own else _plain(s)


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions: one item and head at a time
# ---------------------------------------------------------------------------

def _exact_rope(s):
    x = (s["x"] if s["g"] is None else s["g"]).double()
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous())
    turn = [s["positions"][:, a].double()[:, None] / BASE ** (torch.arange(d // 2, device=x.device).double() * 2 / d) for a, d in enumerate(s["dims"])]
    turn = torch.cat(turn, 1)
    z = z * torch.polar(torch.ones_like(turn), turn if s["g"] is None else -turn)
    return {"y" if s["g"] is None else "dx": torch.view_as_real(z).flatten(-2)}


def _nearest_8(x, scale):
    """Multiples of x's e4m3 step under ``scale``, to nearest and even, in 64 bits."""
    y = x.double() / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _least_scale(x):
    """The least power of two that brings the rows of x within 448, in [2^-60, 2^60]."""
    e = -60
    top = float(x.abs().max()) if x.numel() else 0.0
    while e < 60 and top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def _exact_append(s):
    B, H = s["k"].shape[:2]
    start = s["start"].tolist()
    counts = s["counts"].tolist() if s["counts"] is not None else [s["k"].shape[2]] * B
    out = {}
    for name in ("k", "v"):
        values = (s["k8"] if name == "k" else s["v8"].transpose(-1, -2).flatten(2, 3)).double()  # [B, H, n, D]
        scales = s[name + "_scale"].double()
        top = s[name].double().abs().amax(-1).cpu()  # [B, H, S]
        held = scales.cpu().clone()
        for b, (p, m) in enumerate(zip(start, counts)):
            for j in range(p // BLOCK, _blocks(p + m) if m else 0):
                lo, hi = max(p, j * BLOCK), min(p + m, (j + 1) * BLOCK)
                for h in range(H):
                    old = held[b, h, j].item()
                    held[b, h, j] = max(_least_scale(top[b, h, lo - p:hi - p]), old if lo > j * BLOCK else 0.0)
            if m:
                each = held[b].to(values.device).repeat_interleave(BLOCK, 1)[..., None]
                was = scales[b].repeat_interleave(BLOCK, 1)[..., None]
                first = p // BLOCK * BLOCK
                values[b, :, first:p] = _nearest_8(values[b, :, first:p] * was[:, first:p], each[:, first:p])
                values[b, :, p:p + m] = _nearest_8(s[name][b, :, :m], each[:, p:p + m])
        out[name + "8"] = values if name == "k" else values.unflatten(2, (-1, BLOCK)).transpose(-1, -2).contiguous()
        out[name + "_scale"] = held.to(values.device)
    return out


def _exact_attend(s, each):
    """Calls each(b, h, rows, probabilities or None, scores' lse) over slices of rows."""
    q = s["q"]
    B, H, S, D = q.shape
    group = H // s["k_scale"].shape[1]
    lens = s["lengths"].tolist()
    q_lens = s["q_lens"].tolist() if s["q_lens"] is not None else [S] * B
    for b in range(B):
        n, m = lens[b], q_lens[b]
        for h in range(H):
            scale = s["k_scale"][b, h // group].double().repeat_interleave(BLOCK)[:n, None]
            keys = (s["k8"][b, h // group, :n].double() * scale).T.contiguous()
            for r in range(0, m, 4096):
                i = torch.arange(r, min(m, r + 4096), device=q.device)
                t = q[b, h, i].double() @ keys / math.sqrt(D)
                if s["causal"]:
                    t = t.masked_fill(torch.arange(n, device=q.device) > (n - m + i)[:, None], -math.inf)
                each(b, h, i, t)


def _exact_out(s):
    q = s["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    group = q.shape[1] // s["v_scale"].shape[1]

    def each(b, h, i, t):
        n = t.shape[1]
        if n:
            v = s["v8"][b, h // group].transpose(-1, -2).double() * s["v_scale"][b, h // group].double()[:, None, None]
            lse[b, h, i] = torch.logsumexp(t, -1)
            out[b, h, i] = torch.softmax(t, -1).nan_to_num(0.0) @ v.flatten(0, 1)[:n]

    _exact_attend(s, each)
    return {"out": out, "lse": lse}


def _exact_weights(s):
    w = s["weights"].double()
    group = s["q"].shape[1] // w.shape[1]

    def each(b, h, i, t):
        given = torch.exp(t - s["lse"][b, h, i].double()[:, None]).nan_to_num(0.0)
        w[b, h // group, :t.shape[1]] += given.sum(0)

    _exact_attend(s, each)
    return {"weights": w}


def _exact_evict(s):
    B, H, n = s["weights"].shape
    keep, nb = s["keep"], _blocks(s["keep"])
    D, dev = s["k8"].shape[-1], s["k8"].device
    out = {"weights": torch.zeros(B, H, nb * BLOCK, dtype=torch.float64, device=dev), "kept": None, "lengths": None}
    chosen = {}
    for b, m in enumerate(s["lengths"].tolist()):
        old = max(0, m - s["recent"])
        for h in range(H):
            newest = torch.arange(old, m, device=dev)[-keep:]
            best = torch.argsort(s["weights"][b, h, :old], descending=True, stable=True)[:max(0, min(m, keep) - len(newest))]
            chosen[b, h] = torch.cat([best, newest]).sort().values
            out["weights"][b, h, :len(chosen[b, h])] = s["weights"][b, h, chosen[b, h]].double()
    for name in ("k", "v"):
        values = torch.zeros(B, H, nb * BLOCK, D, dtype=torch.float64, device=dev)
        scales = torch.ones(B, H, nb, dtype=torch.float64)
        held = (s["k8"] if name == "k" else s["v8"].transpose(-1, -2).flatten(2, 3))
        for (b, h), at in chosen.items():
            rows = held[b, h].double()[at] * s[name + "_scale"][b, h].double()[at // BLOCK][:, None]
            top = rows.abs().amax(-1).cpu()
            for j in range(_blocks(len(at))):
                scales[b, h, j] = _least_scale(top[j * BLOCK:(j + 1) * BLOCK])
            values[b, h, :len(at)] = _nearest_8(rows, scales[b, h].to(dev).repeat_interleave(BLOCK)[:len(at), None])
        out[name + "8"] = values if name == "k" else values.unflatten(2, (-1, BLOCK)).transpose(-1, -2).contiguous()
        out[name + "_scale"] = scales.to(dev)
    return out


def exact(c, seed):
    s = prepare(c, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attend": _exact_out, "weights": _exact_weights, "evict": _exact_evict}[c["kind"]](s)
