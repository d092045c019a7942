"""Plain 64-bit forms of the KV-pool serving operators, with the error that the
number formats allow beside each value.

Rounding to T is off by at most half a step, ``finfo(T).eps / 2`` of the value
(plus half the smallest subnormal); fp32 sums and products by 2^-24 per step.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of the smallest numbers of the type."""
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).smallest_normal * half_step(dtype)


def plan(lens, new, table, free, cursor, page, tokens, base=0):
    """slots_plan on lists; the table (list of rows) is filled in place."""
    lens_out, cu, slots, positions = [], [0], [], []
    for i, (o, n) in enumerate(zip(lens, new)):
        for p in range(o, o + n):
            if p % page == 0:  # the first token of a page takes it
                table[i][p // page] = free[cursor]
                cursor += 1
            slots.append(table[i][p // page] * page + p % page)
            positions.append(base + p)
        lens_out.append(o + n)
        cu.append(cu[-1] + n)
    pad = tokens - len(slots)
    return slots + [-1] * pad, positions + [0] * pad, cu, lens_out, cursor


def turned(x, w, cos, sin, eps, interleaved):
    """(y, error bound) of [tokens, heads, dim] normed by w and rotated."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    half = cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    y, mag = x.clone(), x.abs()
    a_at = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b_at = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., a_at], x[..., b_at]
    y[..., a_at], y[..., b_at] = a * c - b * s, b * c + a * s
    m = (a * c).abs() + (b * s).abs()
    n = (b * c).abs() + (a * s).abs()
    mag[..., a_at], mag[..., b_at] = m, n
    # sum of squares: dim / 32 lanes' runs and 5 shuffles, then mean, eps, root, quotient, two products,
    # product and sum of the rotation: under 32 roundings of 2^-24
    return y, 32 * F32 * mag


def attention(q, pool, cu, lens, table, page, prefix, prefix_len, scale=None):
    """(o, lse, bound on o, bound on lse) in 64 bits, request by request."""
    T, hq, D = q.shape
    hk = pool.shape[2]
    g = hq // hk
    scale = D ** -0.5 if scale is None else scale
    dt, dev = q.dtype, q.device
    o = torch.zeros(T, hq, D, dtype=torch.float64, device=dev)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=dev)
    tol_o, tol_l = torch.zeros_like(o), torch.zeros_like(lse)
    inner = torch.arange(page, device=dev)

    def flat(pages, n):
        return (pages.long()[:, None] * page + inner).reshape(-1)[:n]

    cu, lens = cu.tolist(), lens.tolist()
    pre = flat(prefix, prefix_len) if prefix_len else torch.zeros(0, dtype=torch.long, device=dev)
    for i, kv in enumerate(lens):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        rec = pool[torch.cat([pre, flat(table[i], kv)])].double()
        keys = torch.arange(prefix_len + kv, device=dev)
        last = prefix_len + kv - (b - a) + torch.arange(b - a, device=dev)
        seen = (keys <= last[:, None]) | (keys < prefix_len)  # the prefix is seen in any case
        for h in range(hk):
            at = slice(h * g, (h + 1) * g)
            x = q[a:b, at].double()
            k, v = rec[:, 0, h], rec[:, 1, h]
            s = (x @ k.T * scale).masked_fill(~seen[:, None], -math.inf)
            big = x.abs() @ k.abs().T * abs(scale)  # what the fp32 dot product's error goes by
            big = torch.where(seen[:, None].expand_as(big), big, 0.0)
            some = seen.any(-1)[:, None]
            if not len(keys):
                continue
            z = torch.logsumexp(s, -1)
            p = torch.where(some[..., None], torch.softmax(s, -1), 0.0)
            lse[a:b, at] = z
            o[a:b, at] = p @ v
            # a score: D products and sums, the scale, the exponent's argument and its power of two
            ds = (D + 16) * F32 * big.amax(-1) + 2.0 ** -20
            n = len(keys)
            weight = p @ v.abs()
            # output rounding + rounding of the probabilities to the type + scores + fp32 sums over the keys;
            # a probability below the type's normal range is off by half a spacing instead, against a sum of
            # at least 2^-9 (probabilities are taken relative to a maximum at most 8 binary places behind)
            tol_o[a:b, at] = half_step(dt) * (1.01 * o[a:b, at].abs() + weight) + tiny(dt) * (
                1 + 512 * v.abs().sum(0)) + (2 * ds + (n / 128 + 256) * F32)[..., None] * weight
            tol_l[a:b, at] = ds + (n / 128 + 256) * F32 + 4 * F32 * torch.where(some, z.abs(), 0.0)
    return o, lse, tol_o, tol_l
