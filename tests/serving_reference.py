"""Plain 64-bit forms of the serving-step operators, and the error bounds their tests use.

Bounds count every rounding of the kernels: half a step of the 16-bit type
(``finfo.eps / 2``) for each value rounded to it, 2^-24 for an fp32 one.
"""

from __future__ import annotations

import math

import torch

BLOCK = 128


def step_tables(computed, scheduled, offsets, pages, bpp, num_tokens, max_blocks):
    """Lists of the six tables, by the definition, one token at a time."""
    P = BLOCK * bpp
    starts, lens, positions, slots, request, blocks = [0], [], [], [], [], []
    for r, (c, n, o) in enumerate(zip(computed, scheduled, offsets)):
        starts.append(starts[-1] + n)
        lens.append(c + n - o)
        for j in range(n):
            phys = c + j - o
            positions.append(c + j)
            slots.append(pages[r][phys // P] * P + phys % P)
            request.append(r)
        need = -(-(c + n - o) // BLOCK)
        blocks.append([pages[r][i // bpp] * bpp + i % bpp if i < need else -1 for i in range(max_blocks)])
    pad = num_tokens - len(positions)
    return starts, lens, positions + [0] * pad, slots + [-1] * pad, request + [-1] * pad, blocks


def rotate(x, positions, omega, axis):
    """``x`` [N, heads, dim] turned in fp64; positions [axes, N]."""
    f = omega.numel()
    angle = positions[axis.long()].double().t() * omega.double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b, rest = x[..., :f].double(), x[..., f: 2 * f].double(), x[..., 2 * f:].double()
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def rotate_bound(x, omega, dtype):
    """One rounding to 16 bits of a value no larger than |a| + |b|, and fp32 cos, sin and products.

    cos and sin: the reduced half-turn is rounded to fp32 (|u| <= 1: 2^-25 half turns, so pi * 2^-25 in the
    angle), and the function itself is good to 2 ulp (2^-22 of a value of at most 1); each product and the sum
    round once more (2^-24 each).  In all under 2^-20 of |a| + |b|.
    """
    f = omega.numel()
    a, b, rest = x[..., :f].double().abs(), x[..., f: 2 * f].double().abs(), x[..., 2 * f:].double()
    size = torch.cat([a + b, a + b, torch.zeros_like(rest)], -1)
    info = torch.finfo(dtype)
    return size * (info.eps / 2 + 2.0 ** -20) + info.tiny * info.eps


def attention(q, k_cache, v_cache, table, starts, lens, scale, window=0, sinks=0):
    """(out, lse, out bound, lse bound) in fp64, one query row of one head at a time over the keys it sees."""
    N, H, D = q.shape
    kvh = k_cache.shape[2]
    G = H // kvh
    info = torch.finfo(q.dtype)
    u = info.eps / 2
    out = torch.zeros(N, H, D, dtype=torch.float64)
    lse = torch.full((N, H), -math.inf, dtype=torch.float64)
    ob, lb = torch.zeros_like(out), torch.zeros_like(lse)
    for r, length in enumerate(lens):
        n = starts[r + 1] - starts[r]
        if n == 0 or length <= 0:
            continue
        ids = table[r][: -(-length // BLOCK)].long()
        keys = k_cache[ids].flatten(0, 1)[:length].double()
        values = v_cache[ids].flatten(0, 1)[:length].double()
        for j in range(n):
            p = length - n + j
            if p < 0:
                continue
            at = torch.arange(p + 1)
            if window:
                at = at[(at > p - window) | (at < sinks)]
            row = starts[r] + j
            k, v = keys[at], values[at]
            qr = q[row].double().view(kvh, G, D)
            s = torch.einsum("hgd,thd->hgt", qr, k) * scale
            w = torch.softmax(s, -1)
            out[row] = torch.einsum("hgt,thd->hgd", w, v).reshape(H, D)
            lse[row] = torch.logsumexp(s, -1).reshape(H)
            # scores: D products summed in fp32, one more product, and 2^x good to 2^-22 at an argument of at
            # most 2 * peak * log2(e) rounded to fp32: relative error of a weight
            peak = torch.einsum("hgd,thd->hgt", qr.abs(), k.abs()).amax(-1, keepdim=True) * scale
            e = (D + 8) * 2.0 ** -23 * peak + 2.0 ** -20
            spread = torch.einsum("hgt,thd->hgd", w, v.abs())
            # a weight's rounding to 16 bits (half a step; below the normal range half of the smallest
            # subnormal, of weights whose largest is 1), the sums, the normalisation and the output's rounding
            tiny = info.tiny * info.eps / 2 * v.abs().sum(0)[:, None]
            ob[row] = (spread * (u + 2 * e + 2.0 ** -18) + tiny + out[row].view(kvh, G, D).abs() * u).reshape(H, D)
            ob[row] += info.tiny * info.eps
            lb[row] = (e.squeeze(-1) + 2.0 ** -18).reshape(H) + lse[row].abs() * 2.0 ** -22
    return out, lse, ob, lb
