"""Plain 64-bit forms of rotary positions, the cache's formats and attention over it, on
the CPU, and the error bounds that follow from where the kernels round."""

import math

import numpy as np
import torch

EPS = {torch.float16: 2.0**-10, torch.bfloat16: 2.0**-7, torch.float32: 2.0**-23}
LEVELS = {8: 127, 4: 7}


def rotate(x, positions, freq, interleaved, scale):
    """x [tokens, heads, dim] float64, positions [tokens], freq [pairs] float32."""
    y, r = x.double().clone(), freq.numel()
    t = positions.double()[:, None] * freq.double()
    c, s = (scale * t.cos())[:, None], (scale * t.sin())[:, None]
    i = torch.arange(r)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def rotate_bound(x, freq, interleaved, scale):
    """f32 error of a rotation: cosine and sine each rounded once, two products, a sum --
    three half steps of a sum of magnitudes |a| + |b| (2^-24 each), and one to spare."""
    r = freq.numel()
    i = torch.arange(r)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
    b = torch.zeros_like(x, dtype=torch.float64)
    m = (x.double()[..., ia].abs() + x.double()[..., ib].abs()) * abs(scale) * 4 * 2.0**-24
    b[..., ia], b[..., ib] = m, m
    return b


def quantise(x, bits):
    """(codes int64, scales float16 [..., dim / 32]) of x float32, each step rounded as stated."""
    g = x.float().unflatten(-1, (-1, 32))
    most = g.abs().amax(-1)
    s = (most / LEVELS[bits]).clamp(max=65504.0).half()
    bad = ~torch.isfinite(g).all(-1)
    sf = torch.where((s > 0) & ~bad, s.float(), torch.ones_like(most))
    c = torch.round(g / sf[..., None]).clamp(-LEVELS[bits], LEVELS[bits])
    c = torch.where(((s > 0) & ~bad)[..., None], c, torch.zeros_like(c))
    s = torch.where(bad, torch.tensor(float("nan"), dtype=torch.float16), s)
    return c.flatten(-2).long(), s


def pack(c, bits):
    if bits == 8:
        return (c + 128).to(torch.uint8)
    c = (c + 8).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def unpack(b, bits):
    b = b.long()
    return b - 128 if bits == 8 else torch.stack((b & 15, b >> 4), -1).flatten(-2) - 8


class Pool:
    """A cache on the CPU: tensors in the library's layout, with a place for every sequence."""

    def __init__(self, seed, lens, kv_heads, dim, page, bits, dtype, spare=3, table_pages=None, poison=True, loud=4.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.kv_heads, self.dim, self.page, self.bits, self.dtype = lens, kv_heads, dim, page, bits, dtype
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        width = table_pages or max(1, max(need))
        # entries behind a sequence's pages name no page of the pool
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at : at + n]
            at += n

        def side():
            x = torch.randn(pages, kv_heads, page, dim, generator=g)
            x[..., 5] *= loud
            if bits == 16:
                return x.to(dtype), None
            c, s = quantise(x, bits)
            return pack(c, bits), s.transpose(2, 3).contiguous()

        (self.k, self.ks), (self.v, self.vs) = side(), side()
        if poison:  # slots that no sequence has written hold NaN
            used = torch.zeros(pages, page, dtype=torch.bool)
            for b, n in enumerate(lens):
                for j in range(need[b]):
                    used[self.table[b, j], : min(page, n - j * page)] = True
            dead = ~used[:, None, :].expand(pages, kv_heads, page)
            for x, s in ((self.k, self.ks), (self.v, self.vs)):
                if bits == 16:
                    x[dead] = float("nan")
                else:
                    s.transpose(2, 3)[dead] = float("nan")
                    x[dead] = 255

    def values(self, name, b):
        """Keys or values of sequence b, [tokens, kv_heads, dim] float64."""
        n = self.lens[b]
        rows = self.table[b, : -(-n // self.page)].long()
        x = getattr(self, name)[rows].transpose(1, 2).flatten(0, 1)[:n]
        if self.bits == 16:
            return x.double()
        s = getattr(self, name + "s")[rows].permute(0, 3, 1, 2).flatten(0, 1)[:n].double()
        return unpack(x, self.bits).double() * s.repeat_interleave(32, -1)

    def cuda(self, mlxl3_amd):
        up = lambda t: None if t is None else t.cuda()
        return mlxl3_amd.KvCache(up(self.k), up(self.v), up(self.ks), up(self.vs), bits=self.bits)


def batch(mlxl3_amd, new, lens, table, **kw):
    starts = torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32)
    kw.setdefault("max_q", max(1, max(new)))
    return mlxl3_amd.KvBatch(starts.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                             None if table is None else table.cuda(), **kw)


def attend(q, k, v, first, scale, causal, window, coded=False, dtype=None):
    """q [n, heads, dim], k and v [tokens, kv_heads, dim] float64, query i at position
    first + i -> (y, bound): the result and how far the kernels' roundings may move it.

    With w = p / sum p, a relative error e_t of every p_t moves y by at most
    sum w |v| e + |y| sum w e.  The errors: the score's f32 sum of dim products (dim half
    steps of the sum of magnitudes), its product with the scale and the exponential (2^-22
    of |s| + 1); 8- and 4-bit keys rounded to f16 (2^-11 of the sum of magnitudes); p
    rounded to 16 bits for the product with v, numerator only (half a step of dtype, and
    2^-25 absolute for an f16 p below its normal range, against a largest p of 1 or more);
    8- and 4-bit values rounded to f16 (2^-11); f32 sums over the tokens (2^-24 each, in
    blocks: 64 half steps are ample); the output's own half step."""
    n, heads, dim = q.shape
    tokens, group = k.shape[0], heads // k.shape[1]
    y = torch.zeros(n, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(y)
    t = torch.arange(tokens)[None]
    at = first + torch.arange(n)[:, None]
    seen = torch.ones(n, tokens, dtype=torch.bool)
    if causal:
        seen &= t <= at
    if window > 0:
        seen &= t > at - window
    half = EPS[dtype] / 2
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h] @ kh.T) * scale
        mag = (q[:, h].abs() @ kh.abs().T) * scale
        s = torch.where(seen, s, torch.tensor(-math.inf, dtype=torch.float64))
        mag = torch.where(seen, mag, torch.zeros_like(mag))
        some = seen.any(1, keepdim=True)
        m = torch.where(some, s.amax(1, keepdim=True) if tokens else torch.zeros(n, 1, dtype=torch.float64), torch.zeros(n, 1, dtype=torch.float64))
        p = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
        total = p.sum(1, keepdim=True)
        w = p / torch.where(total > 0, total, torch.ones_like(total))
        e = mag * (dim * 2.0**-24 + 2.0**-22 + (2.0**-11 if coded else 0.0)) + 2.0**-21
        vz = torch.where(seen.any(0)[:, None], vh, torch.zeros_like(vh))
        yh = w @ vz
        by = half + (2.0**-11 if coded else 0.0) + 64 * 2.0**-24
        b = (w * e) @ vz.abs() + yh.abs() * (w * e).sum(1, keepdim=True) + by * (w @ vz.abs())
        small = 2.0**-25 * (seen.double() @ vz.abs()) / torch.where(total > 0, total, torch.ones_like(total))
        y[:, h], bound[:, h] = yh, b + (small if dtype == torch.float16 or coded else 0.0)
    return y, bound + half * y.abs() + 2.0**-24 * (2.0**-1 if dtype == torch.float16 else 0.0)
