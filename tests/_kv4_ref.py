"""Plain forms of the 4-bit paged cache's operators, on the CPU (test helpers).

The packed format is read and written code by code from its definition; attention,
norm and rotation are evaluated in fp64.
"""
from __future__ import annotations

import math

import torch

SHIFT = torch.tensor([4 * (i // 2 + 4 * (i % 2)) for i in range(8)])


def words(D: int, G: int, P: int) -> int:
    return P * (D // 4 + 2 * (D // G))


def key_word(D: int) -> torch.Tensor:
    o = torch.arange(D) // 8
    return (D // 32) * (o % 4) + o // 4


def value_word(D: int) -> torch.Tensor:
    d = torch.arange(D)
    return 64 * (d // 64) + 4 * (d % 16) + d // 16 % 4


def _meta(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    b = w.long()
    half = [torch.where(x > 32767, x - 65536, x).to(torch.int16).view(torch.float16).double()
            for x in (b & 0xFFFF, b >> 16 & 0xFFFF)]
    return half[0], half[1]


def unpack(block: torch.Tensor, D: int, G: int, P: int, parts: bool = False):
    """One block int32 [words] to keys and values fp64 [P, D] (parts: to (codes,
    scales, centres) of both, [P, D] each)."""
    block = block.cpu()
    w = block.long() & 0xFFFFFFFF
    NG, t, d = D // G, torch.arange(P)[:, None], torch.arange(D)
    a, b, c = P * D // 8, P * D // 8 + NG * P, P * D // 4 + NG * P
    kc = (w[t * (D // 8) + key_word(D)] >> SHIFT[d % 8]) & 15
    vc = (w[b + t // 8 * D + value_word(D)] >> SHIFT[t % 8]) & 15
    ks, kz = _meta(block[a + d // G * P + t])
    vs, vz = _meta(block[c + d // G * P + t])
    if parts:
        return (kc, ks, kz), (vc, vs, vz)
    return (kc - 8) * ks + kz, (vc - 8) * vs + vz


def pack(kc, ks, kz, vc, vs, vz, D: int, G: int, P: int) -> torch.Tensor:
    """Codes [P, D] and fp16 groups [P, D / G] to a block int32 [words]."""
    out = torch.zeros(words(D, G, P), dtype=torch.int64)
    NG = D // G
    a, b, c = P * D // 8, P * D // 8 + NG * P, P * D // 4 + NG * P
    for t in range(P):
        for d in range(D):
            out[t * (D // 8) + key_word(D)[d]] |= int(kc[t, d]) << int(SHIFT[d % 8])
            out[b + t // 8 * D + value_word(D)[d]] |= int(vc[t, d]) << int(SHIFT[t % 8])
    for at, s, z in ((a, ks, kz), (c, vs, vz)):
        m = (s.to(torch.float16).view(torch.int16).long() & 0xFFFF) | \
            (z.to(torch.float16).view(torch.int16).long() & 0xFFFF) << 16
        out[at:at + NG * P] = m.t().reshape(-1)
    return torch.where(out > 2**31 - 1, out - 2**32, out).to(torch.int32)


def quantise(x: torch.Tensor, G: int):
    """(codes, scales, centres) of fp32 x [..., D]; fp32 arithmetic as defined."""
    g = x.float().unflatten(-1, (-1, G))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) * (1.0 / 15.0)).half()
    c = (lo + 8.0 * s.float()).half()
    inv = 1.0 / s.float()
    ok = torch.isfinite(inv) & torch.isfinite(c.float()) & torch.isfinite(s.float())
    n = torch.where(ok, ((g - c.float()) * inv).round().clamp(-8, 7), torch.zeros(()))
    return (n + 8).flatten(-2).long(), s.squeeze(-1), c.squeeze(-1)


def norm_rotate32(x, w, cos, sin, positions, eps, interleaved):
    """fp32, every operation rounded by itself, squares summed by halves."""
    y = x.float()
    if w is not None:
        D = y.shape[-1]
        t = (y * y).unflatten(-1, (D // 8, 8))
        for n in (4, 2, 1):
            t = t[..., :n] + t[..., n:]
        t = t.squeeze(-1)
        while t.shape[-1] > 1:
            n = t.shape[-1] // 2
            t = t[..., :n] + t[..., n:]
        # (by way of fp64: torch's fp32 square root is not correctly rounded)
        y = y * (1.0 / (t * (1.0 / D) + eps).double().sqrt().float()) * w.float()
    return _turn(y, cos, sin, positions, interleaved)


def norm_rotate64(x, w, cos, sin, positions, eps, interleaved):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    return _turn(y, cos.double(), sin.double(), positions, interleaved)


def _turn(y, cos, sin, positions, interleaved):
    R = 2 * cos.shape[1]
    c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
    r, rest = y[..., :R], y[..., R:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, rest), -1)


def attention(q, k, v, vres, n, scale, causal, window, sizes):
    """One sequence and kv head, fp64.  q [nq, heads, D]; k, v [n, D]; vres [n, D] =
    |value - centre|; sizes [n, D] bounds of |8 scale| + |centre| of the keys.
    Returns (out, lse, bound of the kernel's error before the last rounding)."""
    nq, heads, D = q.shape
    q = q.double()
    out = torch.zeros(nq, heads, D, dtype=torch.float64)
    lse = torch.full((nq, heads), -math.inf, dtype=torch.float64)
    err = torch.zeros_like(out)
    for i in range(nq):
        pos = n - nq + i
        lo = max(0, pos - window + 1) if window else 0
        hi = min(n, pos + 1) if causal else n
        if hi <= lo:
            continue
        s = q[i] @ k[lo:hi].t() * scale
        m = s.max(-1, keepdim=True)[0]
        p = torch.exp(s - m)
        l = p.sum(-1, keepdim=True)
        p = p / l
        out[i] = p @ v[lo:hi]
        lse[i] = (m + torch.log(l)).squeeze(-1)
        # weights of the values are rounded to 11 bits: 2^-11 of what they multiply;
        # a score is a sum of up to 2 D fp32 terms
        big = (q[i].abs() @ sizes[lo:hi].t()).max(-1, keepdim=True)[0] * scale
        slip = 2.0**-19 * big + 2.0**-19
        err[i] = 2.0**-11 * (p @ vres[lo:hi]) + 2 * slip * (p @ v[lo:hi].abs())
    return out, lse, err
