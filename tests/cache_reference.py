"""The 8-bit cache's operators in 64 bits on the CPU, element by element from their
definitions, and what rounding allows their results to be off."""

from __future__ import annotations

import math

import torch

BLOCK = 64


def e4m3_table() -> torch.Tensor:
    """The values of the bytes 0 .. 255: sign, 4 exponent bits (bias 7), 3 mantissa
    bits, subnormals at exponent 0, NaN at 0x7f and 0xff."""
    out = []
    for byte in range(256):
        sign, e, m = -1.0 if byte & 128 else 1.0, byte >> 3 & 15, byte & 7
        mag = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out.append(sign * (math.nan if byte & 127 == 127 else mag))
    return torch.tensor(out, dtype=torch.float64)


TABLE = e4m3_table()


def values(cache):
    """k, v [B, H, capacity, D] in 64 bits on the CPU."""
    B, H, n, D = cache.shape
    k = TABLE[cache.k8.cpu().view(torch.uint8).long()].view(B, H, n // BLOCK, BLOCK, D) * cache.k_scale.cpu().double()[..., None, None]
    v = TABLE[cache.v8.cpu().view(torch.uint8).long()].transpose(-1, -2) * cache.v_scale.cpu().double()[..., None, None]
    return k.reshape(B, H, n, D), v.reshape(B, H, n, D)


def nearest(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """x / scale to the nearest e4m3 value (ties to the even mantissa), as numbers;
    NaN where x is not finite or over the largest."""
    y = x.double() / scale
    fine = y.abs() <= 448
    mag = torch.where(fine, y.abs(), 0.0)
    e = torch.floor(torch.log2(mag.clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.where(fine, torch.copysign(torch.round(mag / step) * step, y), math.nan)


def least_scale(x: torch.Tensor) -> float:
    x = x.double().abs()
    x = x[torch.isfinite(x)]
    top, e = (float(x.max()) if x.numel() else 0.0), -60
    while e < 60 and top > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(cache, k, v, start, counts=None):
    """[(stored numbers [B, H, capacity, D], scales [B, H, nb])] of k and of v after the call."""
    B, H, n, D = cache.shape
    out = []
    for x, held, scale in ((k, values(cache)[0], cache.k_scale), (v, values(cache)[1], cache.v_scale)):
        x, scale = x.detach().cpu().double(), scale.cpu().double().clone()
        each = scale.repeat_interleave(BLOCK, 2)[..., None]
        stored = held / each
        for b in range(B):
            p, m = start[b], (counts[b] if counts is not None else x.shape[2])
            m = max(0, min(m, x.shape[2]))
            end = min(p + m, n)
            if p < 0 or m == 0 or p >= n:
                continue
            for h in range(H):
                for j in range(p // BLOCK, -(-end // BLOCK)):
                    lo, hi = max(p, BLOCK * j), min(end, BLOCK * (j + 1))
                    s = least_scale(x[b, h, lo - p:hi - p])
                    old = scale[b, h, j].item()
                    if lo > BLOCK * j:
                        s = max(s, old)
                        stored[b, h, BLOCK * j:lo] = nearest(held[b, h, BLOCK * j:lo], torch.tensor(s))
                    scale[b, h, j] = s
                    stored[b, h, lo:hi] = nearest(x[b, h, lo - p:hi - p], torch.tensor(s))
        out.append((stored, scale))
    return out


def visible(b, i, lengths, q_lens, S, causal):
    m = q_lens[b] if q_lens is not None else S
    if i >= m:
        return 0
    return max(0, min(lengths[b], lengths[b] - m + i + 1)) if causal else lengths[b]


def attention(q, cache, lengths, q_lens=None, causal=False, sm_scale=None):
    """(out, lse, bound on |out|'s error, bound on lse's, probabilities [B, Hq, S, n], bound on their relative error).

    The kernels round, beside fp32 sums: P to q's type (half a step u of each, or
    2^-25 of the row's largest P 2^ev in fp16), and the output (u).  A score of D
    products in fp32 is off by at most (D + 8) 2^-24 of the sum of their sizes; exp2
    and the sums of up to a few thousand values take 2^-18 more."""
    B, H, S, D = q.shape
    Hkv = cache.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    qd = q.detach().cpu().double()
    k, v = values(cache)
    ev = cache.v_scale.cpu().double().repeat_interleave(BLOCK, 2)
    n = cache.capacity
    out = torch.zeros(B, H, S, D, dtype=torch.float64)
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64)
    tol, tol_lse, tol_p = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(lse)
    probs = torch.zeros(B, H, S, n, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            kh, vh, eh = k[b, h * Hkv // H], v[b, h * Hkv // H], ev[b, h * Hkv // H]
            for i in range(S):
                m = visible(b, i, lengths, q_lens, S, causal)
                if m == 0:
                    continue
                t = kh[:m] @ qd[b, h, i] * sm_scale
                e32 = ((D + 8) * 2.0 ** -24 * float((kh[:m].abs() @ qd[b, h, i].abs()).nan_to_num(0.0).max()) * sm_scale
                       + 2.0 ** -18 + 2.0 ** -22 * float(t.abs().nan_to_num(0.0).max()))
                lse[b, h, i] = torch.logsumexp(t, 0)
                p = torch.exp(t - lse[b, h, i])
                probs[b, h, i, :m] = p
                out[b, h, i] = p @ vh[:m]
                size = p @ vh[:m].abs()
                small = 2.0 ** -25 * (p * eh[:m]).max() * (vh[:m].abs() / eh[:m, None]).sum(0) if q.dtype == torch.float16 else 0.0
                tol[b, h, i] = u * size + u * out[b, h, i].abs() + 2 * e32 * size + small + 2.0 ** -25
                tol_lse[b, h, i], tol_p[b, h, i] = 2 * e32 + 2.0 ** -22 * lse[b, h, i].abs(), 2 * e32
    return out, lse, tol, tol_lse, probs, tol_p


def weights(probs, tol_p, Hkv):
    """([B, Hkv, n] sums over each key head's rows, bound on their error)."""
    B, H, S, n = probs.shape
    w = probs.view(B, Hkv, -1, n).sum(2)
    tol = (probs * tol_p[..., None]).view(B, Hkv, -1, n).sum(2) + w * (H * S) * 2.0 ** -24
    return w, tol


def evict(cache, lengths, w, keep, recent):
    """(kept [B, H, keep] lists, stored numbers and scales of k and v)."""
    B, H, n, D = cache.shape
    nb = -(-keep // BLOCK)
    kept, out = {}, []
    for b in range(B):
        for h in range(H):
            m = max(0, min(lengths[b], n))
            tail = min(recent, m)
            old = w[b, h, :m - tail].tolist()
            order = sorted(range(len(old)), key=lambda i: (math.isnan(old[i]), -old[i] if old[i] == old[i] else 0.0, i))
            kept[b, h] = sorted(order[:min(m, keep) - tail]) + list(range(m - tail, m))
    for x in values(cache):
        stored, scale = torch.zeros(B, H, nb * BLOCK, D, dtype=torch.float64), torch.ones(B, H, nb, dtype=torch.float64)
        for (b, h), at in kept.items():
            for j in range(0, len(at), BLOCK):
                rows = x[b, h, at[j:j + BLOCK]]
                s = least_scale(rows)
                scale[b, h, j // BLOCK] = s
                stored[b, h, j:j + len(rows)] = nearest(rows, torch.tensor(s))
        out.append((stored, scale))
    return kept, out


def rope(x, positions, dims, base=10000.0, sign=1):
    """x [B, H, S, D] turned, in 64 bits; positions [B or 1, S, axes]."""
    x, pos = x.detach().cpu().double(), positions.detach().cpu().double()
    pos = pos if pos.dim() == 3 else pos[None]
    angle = torch.cat([pos[..., a, None] * base ** (-2 * torch.arange(d // 2).double() / d) for a, d in enumerate(dims)], -1)
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * torch.polar(torch.ones_like(angle), sign * angle)[:, None]
    return torch.view_as_real(z).flatten(-2)
