"""A plain 64-bit form, on the CPU, of attention whose scores are capped and biased and whose rows
see a prefix, and the error bound that follows from where the kernels round."""

import math

import torch

from kv_ref import EPS


def attend(q, k, v, first, scale, causal, window, softcap=0.0, slopes=None, prefix=0, coded=False, dtype=None):
    """q [n, heads, dim], k and v [tokens, kv_heads, dim] float64, query i at position first + i
    -> (y, bound).

    With w = p / sum p, an error e_t of every score moves y by at most sum w |v| e + |y| sum w e.
    A score's error: that of a plain one (its f32 sum of dim products, the product with the scale;
    coded keys rounded to f16, 2^-11); a cap does not enlarge it (its slope is at most 1) and adds its
    own: 2^-21 of the cap -- 1 - 2 / (1 + e) with e off by 2^-22 or so of itself, which moves 1 / (1 + e) by
    at most a quarter of that, its sum and reciprocal rounded to 1.5 * 2^-24; above a cap of 256 the series', 2^-22 of
    the score, up to a quarter of the cap; the bias: a slope over a scale, a distance and their product
    rounded (2^-22 of it), and where it is what the f32 sum of the products starts from, as much of it as
    of them is lost there, dim half steps.  The rest is as for plain
    scores: the exponential 2^-21, p rounded to 16 bits, coded values to f16, f32 sums over the tokens,
    the output's half step."""
    n, heads, dim = q.shape
    tokens, group = k.shape[0], heads // k.shape[1]
    y = torch.zeros(n, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(y)
    away = first + torch.arange(n)[:, None] - torch.arange(tokens)[None]
    seen = torch.ones(n, tokens, dtype=torch.bool)
    if causal:
        seen = away >= 0
        seen[:, : max(0, prefix)] = True
    if window > 0:
        seen = seen & (away < window)
    half = EPS[dtype] / 2
    none = torch.zeros((), dtype=torch.float64)
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        z = (q[:, h] @ kh.T) * scale
        e = (q[:, h].abs() @ kh.abs().T) * scale * (dim * 2.0**-24 + 2.0**-22 + (2.0**-11 if coded else 0.0))
        if softcap:
            if softcap <= 256:
                e = e + softcap * 2.0**-21
            else:
                e = e + torch.where(z.abs() < softcap / 4.01, 2.0**-22 * z.abs(), torch.full_like(z, softcap * 2.0**-21))
            z = softcap * torch.tanh(z / softcap)
        if slopes is not None:
            bias = float(slopes[h]) * away.abs().double()
            e = e + 2.0**-22 * z.abs() + bias.abs() * (2.0**-22 + dim * 2.0**-24)
            z = z - bias
        e = torch.where(seen, e + 2.0**-21 + 2.0**-23 * z.abs(), none)
        z = torch.where(seen, z, torch.tensor(-math.inf, dtype=torch.float64))
        some = seen.any(1, keepdim=True)
        m = torch.where(some, z.amax(1, keepdim=True) if tokens else torch.zeros(n, 1, dtype=torch.float64), none)
        p = torch.where(seen, torch.exp(z - m), none)
        total = p.sum(1, keepdim=True)
        w = p / torch.where(total > 0, total, torch.ones_like(total))
        vz = torch.where(seen.any(0)[:, None], vh, none)
        yh = w @ vz
        by = half + (2.0**-11 if coded else 0.0) + 64 * 2.0**-24
        b = (w * e) @ vz.abs() + yh.abs() * (w * e).sum(1, keepdim=True) + by * (w @ vz.abs())
        small = 2.0**-25 * (seen.double() @ vz.abs()) / torch.where(total > 0, total, torch.ones_like(total))
        y[:, h], bound[:, h] = yh, b + (small if dtype == torch.float16 or coded else 0.0)
    return y, bound + half * y.abs() + 2.0**-24 * (2.0**-1 if dtype == torch.float16 else 0.0)
