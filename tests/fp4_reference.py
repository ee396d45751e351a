"""The pool held in 4 bits and attention over it, in 64 bits from the definitions (include/infiniop/ops/paged_caching_fp4.h).
Host tensors in, float64 out; nothing of the package is used."""
from __future__ import annotations

import math

import torch

GROUP = 32
MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantise(x):
    """(codes [.., n / 2], scales [.., n / 32]) uint8 of x [.., n]."""
    g = x.double().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    finite = torch.isfinite(g).all(-1)
    exponent = torch.frexp(torch.where(finite, top, 1.0)).exponent - 1  # floor(log2); 0 has exponent 0 - 1
    exponent = torch.where(top == 0, -1000, exponent)
    s = (exponent - 2).clamp(-23, 13)
    a = (torch.where(finite[..., None], g, 0.0).abs() / torch.pow(2.0, s.double())[..., None]).clamp(max=6.0)
    distance = (a[..., None] - MAGNITUDES).abs()
    nearest = distance.amin(-1, keepdim=True)
    even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    code = even_first[(distance[..., even_first] == nearest).int().argmax(-1)]
    code = code + 8 * torch.signbit(g).long()
    code = torch.where(finite[..., None], code, 0).flatten(-2)
    scales = torch.where(finite, 127 + s, 255)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scales.to(torch.uint8)


def values(codes, scales):
    """What codes [.., n / 2] under scales [.., n / 32] stand for, float64 [.., n]."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).long()
    v = MAGNITUDES[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
    unit = torch.pow(2.0, scales.double() - 127).masked_fill(scales == 255, math.nan)
    return v * unit.repeat_interleave(GROUP, dim=-1)


def sequence(codes, scales, pages, tokens):
    """The first `tokens` rows of the pages, float64 [KV heads, tokens, size]."""
    x = values(codes[pages], scales[pages])  # [pages, heads, rows, size]
    return x.transpose(0, 1).flatten(1, 2)[:, :tokens]


def attention(q, k, v, scale, last, slopes=None):
    """q [n, heads, d] over k, v [KV heads, tokens, d]: row j sees tokens 0 .. last[j] (none where last[j] < 0: the row is
    NaN, to be left out by the caller). A token that a row does not see has no part in it, whatever it holds."""
    n, heads, d = q.shape
    group = heads // k.shape[0]
    out = torch.full((n, heads, v.shape[-1]), math.nan, dtype=torch.float64)
    for j in range(n):
        t = int(last[j]) + 1
        if t <= 0:
            continue
        for h in range(heads):
            s = (k[h // group, :t] @ q[j, h].double()) * scale
            if slopes is not None:
                s = s + slopes[h].double() * (torch.arange(t, dtype=torch.float64) - last[j])
            p = torch.exp(s - s.max())
            out[j, h] = (p / p.sum()) @ v[h // group, :t]
    return out


def make_pool(seed, blocks, heads, page, size, *, spread=1.0):
    """A pool of normal values whose channels differ in size: (k_codes, v_codes, k_scales, v_scales)."""
    gen = torch.Generator().manual_seed(seed)
    made = []
    for _ in range(2):
        channel = torch.exp(spread * torch.randn((heads, 1, size), generator=gen))
        made.append(quantise(torch.randn((blocks, heads, page, size), generator=gen) * channel))
    return made[0][0], made[1][0], made[0][1], made[1][1]
