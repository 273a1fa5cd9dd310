"""Attention where 16 and 32 bits end: coded values beyond f16's range, values that a row does not
see over coded caches, scores of any size, weights far below the largest, bf16 queries that f16
does not hold.  Against the 64-bit forms of kv_ref.py."""

import math

import pytest
import torch

import kv_ref
from kv_ref import Pool
from test_gpu_attention import BF16, F16, check, run, within

import mlxl3_amd

pytestmark = pytest.mark.gpu

CODED = [(8, F16), (8, BF16), (4, F16), (4, BF16)]


def put_value(pool, seq, t, value):
    """Token t's values in every head: `value` in channel 7 (and its group's scale with it)."""
    row = torch.zeros(pool.kv_heads, pool.dim)
    row[:, 7] = value
    c, s = kv_ref.quantise(row, pool.bits)
    at = int(pool.table[seq, t // pool.page]), slice(None), t % pool.page
    pool.v[at] = kv_ref.pack(c, pool.bits)
    pool.vs.transpose(2, 3)[at] = s
    return s[:, 0].float()


@pytest.mark.parametrize("bits, dtype", CODED)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [math.nan, math.inf, 6.0e4, 6.7e4, -1.0e5, 5.0e5, -8.0e6])
@pytest.mark.parametrize("new", [[1, 3], [40, 33]])
def test_coded_values_that_a_row_does_not_see_do_not_reach_it(bits, dtype, dim, value, new):
    """Groups that are not finite and groups whose largest values f16 does not hold, behind a
    row's position or before its window.  The rows that do not see them are as exact as with
    zeros there."""
    window = 8
    lens = [new[0] + 100, new[1] + 20]
    pool = Pool(44, lens, 2, dim, 16, bits, None)
    for s in range(2):
        for t in (lens[s] - new[s] - window + 1, lens[s] - 1):  # in the first row's window alone; the newest token
            put_value(pool, s, t, value)
    q, _, _, y = run(pool, new, 4, dtype, window=window)
    at = 0
    for s, n in enumerate(new):
        args = q[at : at + n].double(), pool.values("k", s), pool.values("v", s)
        old = lens[s] - n
        for i in range(n):
            sees = [t for t in (old - window + 1, lens[s] - 1) if old + i - window < t <= old + i]
            if not sees:
                lo, hi = old + i - window + 1, old + i + 1
                want, bound = kv_ref.attend(args[0][i : i + 1], args[1][lo:hi], args[2][lo:hi], 0, dim**-0.5, False, 0,
                                            coded=True, dtype=dtype)
                within(y[at + i : at + i + 1], want, bound, f"sequence {s} row {i}")
            elif not math.isfinite(value):
                assert bool(y[at + i, :, :32].isnan().any()), f"sequence {s} row {i} sees it"
        at += n


@pytest.mark.parametrize("bits, dtype", CODED)
@pytest.mark.parametrize("value", [math.nan, 1.0e6])
@pytest.mark.parametrize("new", [[1, 3], [40, 33]])
def test_coded_keys_that_a_row_does_not_see_do_not_reach_it(bits, dtype, value, new):
    """Keys that are not finite, or not as f16, in the newest token: the rows before it are as exact
    as without it."""
    lens = [new[0] + 100, new[1] + 20]
    pool = Pool(53, lens, 2, 128, 16, bits, None)
    clean = Pool(53, lens, 2, 128, 16, bits, None)
    for s in range(2):
        row = torch.zeros(2, 128)
        row[:, 7] = value
        c, scales = kv_ref.quantise(row, bits)
        t = lens[s] - 1
        at = int(pool.table[s, t // 16]), slice(None), t % 16
        pool.k[at] = kv_ref.pack(c, bits)
        pool.ks.transpose(2, 3)[at] = scales
    q, _, _, y = run(pool, new, 4, dtype)
    at = 0
    for s, n in enumerate(new):
        want, bound = kv_ref.attend(q[at : at + n].double(), clean.values("k", s), clean.values("v", s), lens[s] - n, 128**-0.5,
                                    True, 0, coded=True, dtype=dtype)
        within(y[at : at + n - 1], want[:-1], bound[:-1], f"sequence {s}")
        at += n


@pytest.mark.parametrize("bits, dtype", CODED)
@pytest.mark.parametrize("new", [[2], [40]])
def test_the_largest_values_that_f16_holds_are_attended_to(bits, dtype, new):
    """Groups just below the border, seen by some rows: every row within the bound."""
    levels = kv_ref.LEVELS[bits]
    pool = Pool(45, [new[0] + 30], 2, 128, 16, bits, None)
    scales = put_value(pool, 0, pool.lens[0] - 1, 6.4e4)
    assert bool((scales * levels < 65504).all())
    q, _, _, y = run(pool, new, 4, dtype)
    assert bool(y[:-1].isfinite().all())
    check(pool, new, q, y)


def set_side(pool, name, seq, x):
    """A sequence's keys or values: x [tokens, kv_heads, dim]."""
    t = torch.arange(pool.lens[seq])
    at = pool.table[seq, t // pool.page].long(), slice(None), t % pool.page
    if pool.bits == 16:
        getattr(pool, name)[at] = x.to(pool.dtype)
    else:
        c, s = kv_ref.quantise(x, pool.bits)
        getattr(pool, name)[at] = kv_ref.pack(c, pool.bits)
        getattr(pool, name + "s").transpose(2, 3)[at] = s


def set_keys(pool, seq, x):
    """A sequence's keys: x [tokens] times ones, in every head."""
    set_side(pool, "k", seq, x[:, None, None].expand(-1, pool.kv_heads, pool.dim))


ALL = [(16, F16, F16), (16, BF16, BF16)] + [(b, None, t) for b, t in CODED]


@pytest.mark.parametrize("bits, cdtype, dtype", ALL)
@pytest.mark.parametrize("size", [1.0e3, 8.0e3, 3.0e4])
@pytest.mark.parametrize("new, old", [([2], [100]), ([40], [90]), ([3], [2500]), ([70], [2600])])
def test_scores_so_large_that_f32_does_not_resolve_their_neighbours(bits, cdtype, dtype, size, new, old):
    """Scores up to 2^34 (in powers of two), where a rounding is worth 2^10: the tokens of the
    largest score share the whole weight.  Keys of nine levels 9 % apart, so that no
    rounding joins two of them; queries of both signs."""
    lens = [new[0] + old[0]]
    pool = Pool(46, lens, 1, 128, 16, bits, cdtype)
    set_keys(pool, 0, size * (0.2 + 0.09 * (torch.arange(lens[0]) * 7 % 9).float()))
    q = torch.full((new[0], 4, 128), size)
    q[:, 1::2] *= -1
    q = q.to(dtype)
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    y = mlxl3_amd.attention(q.cuda(), pool.cuda(mlxl3_amd), b)
    k, v = pool.values("k", 0), pool.values("v", 0)
    want, _ = kv_ref.attend(q.double(), k, v, old[0], 128**-0.5, True, 0, coded=bits != 16, dtype=dtype)
    mean, _ = kv_ref.attend(q.double(), k, v.abs(), old[0], 128**-0.5, True, 0, coded=bits != 16, dtype=dtype)
    # equal scores are equal bit for bit, so no error of theirs moves the shares: of attend's terms
    # those of the weights (half a step of 16 bits), coded values, sums and the result are left
    half = kv_ref.EPS[dtype] / 2
    rounded = half + (2.0**-11 if bits != 16 else 0.0) + 64 * 2.0**-24
    within(y, want, half * want.abs() + mean * rounded + 2.0**-24, "huge")


@pytest.mark.parametrize("bits, cdtype, dtype", ALL)
@pytest.mark.parametrize("nats", [12.0, 15.0, 16.0, 17.4])
@pytest.mark.parametrize("new, old", [([1], [4000]), ([2], [4000]), ([40], [4000]), ([300], [3700])])
def test_a_long_tail_far_below_one_token(bits, cdtype, dtype, nats, new, old):
    """One key `nats` above thousands of equal ones, with values of zero: the small weights are
    all of the result.  An f16 weight below the normal range is off by up to 2^-25, against a
    largest one of 2^7 or more: 2^-32 of it, not the 2^-25 of weights up to 1."""
    lens = [new[0] + old[0]]
    pool = Pool(47, lens, 1, 128, 64, bits, cdtype)
    x = torch.zeros(lens[0])
    x[0] = nats / 128**0.5
    set_keys(pool, 0, x)
    g = torch.Generator().manual_seed(48)
    v = torch.rand(lens[0], 1, 128, generator=g) + 0.5
    v[0] = 0
    set_side(pool, "v", 0, v)
    q = torch.ones(new[0], 4, 128).to(dtype)
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    y = mlxl3_amd.attention(q.cuda(), pool.cuda(mlxl3_amd), b)
    k, v = pool.values("k", 0), pool.values("v", 0)
    want, bound = kv_ref.attend(q.double(), k, v, old[0], 128**-0.5, True, 0, coded=bits != 16, dtype=dtype)
    if bits != 16 or dtype == F16:
        for i in range(new[0]):
            seen = slice(0, old[0] + i + 1)
            s = (k[seen, 0] @ q[i, 0].double()) * 128**-0.5
            bound[i] -= 2.0**-25 * (1 - 2.0**-7) * v[seen, 0].abs().sum(0) / torch.exp(s - s.max()).sum()
    within(y, want, bound, f"tail {nats} nats below")


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shift", [17, 100, -20, -100])
@pytest.mark.parametrize("new", [[2, 1], [40, 33]])
def test_bf16_queries_beyond_f16_over_codes(bits, dim, shift, new):
    """Queries around 2^shift, which f16 does not hold or only in part, with a scale that gives
    ordinary scores.  One row is zeros."""
    lens = [new[0] + 150, new[1] + 9]
    pool = Pool(49, lens, 2, dim, 16, bits, None)
    scale = 2.0**-shift / dim**0.5
    g = torch.Generator().manual_seed(50)
    q = (torch.randn(sum(new), 6, dim, generator=g) * 2.0**shift).to(BF16)
    q[0, 1] = 0
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    y = mlxl3_amd.attention(q.cuda(), pool.cuda(mlxl3_amd), b, scale=scale)
    check(pool, new, q, y, scale=scale)


def test_a_bf16_query_with_channels_far_apart():
    """One channel of 2^20, whose key's channel is zero: the others count as ever."""
    pool = Pool(51, [300], 1, 128, 16, 8, None)
    codes = pool.k.view(-1, 128)
    codes[:, 64] = 128  # code 0
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(52))
    q[..., 64] = 2.0**20
    q = q.to(BF16)
    y = mlxl3_amd.attention(q.cuda(), pool.cuda(mlxl3_amd), kv_ref.batch(mlxl3_amd, [2], [300], pool.table))
    check(pool, [2], q, y)
