"""Attention with shaped scores where its kernels' ways part: rows that are done again one by one because of
values that others of the workgroup do not see, joined with ranges that were not, over coded caches and
caps beyond 256; and coded keys of f16 queries, which are two f16 and not one rounded one."""

import math

import pytest
import torch

import kv_ref
import scores_ref
from kv_ref import Pool
from test_gpu_attention import F16, FORMATS, within
from test_gpu_scores import geometric, run

import mlxl3_amd

pytestmark = pytest.mark.gpu

KINDS = [dict(softcap=30.0), dict(softcap=1000.0), dict(slopes=geometric(4) / 200), dict(softcap=30.0, slopes=geometric(4) / 200),
         dict(softcap=1000.0, slopes=geometric(4) / 200), dict(prefix=[3, 2])]


def spoil(pool, seq, t, bad):
    """Token t of a sequence: values, or of codes scales, that are not finite or beyond f16."""
    at = int(pool.table[seq, t // pool.page]), slice(None)
    if pool.bits == 16:
        for x in (pool.k, pool.v):
            x[(*at, t % pool.page)] = bad
    else:
        for x in (pool.ks, pool.vs):
            x[(*at, slice(None), t % pool.page)] = bad


def rows_that_do_not_see(pool, new, q, y, spoiled, window=0, **kw):
    """All rows but each sequence's last against the form without the spoiled tokens, which they do not see."""
    at = 0
    for s, n in enumerate(new):
        k, v = pool.values("k", s), pool.values("v", s)
        for t in spoiled[s]:
            k[t] = v[t] = 0
        slopes = kw.get("slopes")
        want, bound = scores_ref.attend(q[at : at + n].double(), k, v, pool.lens[s] - n, pool.dim**-0.5, True, window, kw.get("softcap", 0.0),
                                        None if slopes is None else slopes.float(), kw.get("prefix", [0, 0])[s], coded=pool.bits != 16,
                                        dtype=q.dtype)
        within(y[at : at + n - 1], want[:-1], bound[:-1], f"sequence {s}")
        at += n


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("new", [[2, 3], [40, 33]])
def test_tokens_in_front_of_windows_and_the_newest(bits, cdtype, dtype, kw, new):
    for bad in (math.nan, math.inf) if bits == 16 else (math.nan, math.inf, 65504.0):
        lens = [new[0] + 100, new[1] + 20]
        pool = Pool(43, lens, 2, 128, 16, bits, cdtype)
        spoiled = [(5, n - 1) for n in lens]
        for s in range(2):
            for t in spoiled[s]:
                spoil(pool, s, t, bad)
        q, _, _, y, _ = run(pool, new, 4, dtype, window=8, **kw)
        rows_that_do_not_see(pool, new, q, y, spoiled, window=8, **kw)
        if bad != 65504.0:  # (which counts as infinite or not)
            for s in range(2):
                assert not bool(y[sum(new[: s + 1]) - 1].isfinite().all())


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("new, lens", [([6], [5000]), ([70], [5000]), ([3, 2], [5000, 2900]), ([3, 33], [700, 4000])])
def test_a_range_done_again_and_others_joined(bits, cdtype, dtype, kw, new, lens):
    """Only the newest of a sequence's ranges holds the token: its maxima and sums meet those of ranges that
    were done as usual."""
    if "prefix" in kw:
        kw = dict(prefix=kw["prefix"][: len(new)])
    pool = Pool(44, lens, 2, 128, 16, bits, cdtype)
    spoiled = [(n - 1,) for n in lens]
    for s in range(len(lens)):
        spoil(pool, s, lens[s] - 1, math.nan)
    q, _, _, y, _ = run(pool, new, 4, dtype, **kw)
    rows_that_do_not_see(pool, new, q, y, spoiled, **kw)


def two_keys(bits):
    """Two (code, scale) whose values are 0.4 % apart at most, one of which f16 rounds up and the other one
    down, as much as such a pair can be."""
    codes = torch.arange(64, 128) if bits == 8 else torch.arange(4, 8)
    scales = 1.0 + torch.arange(1024, dtype=torch.float64) / 1024
    x = (codes[:, None] * scales).flatten()
    off = x.half().double() / x - 1
    best = None
    for i in off.argsort(descending=True)[:400].tolist():
        near = (x / x[i] - 1).abs() < 0.004
        j = int(torch.where(near, off, torch.full_like(off, 1.0)).argmin())
        if best is None or off[i] - off[j] > best[0]:
            best = float(off[i] - off[j]), i, j
    assert best[0] > 2.0**-11 * 1.2
    return [(int(codes[i // 1024]), float(scales[i % 1024])) for i in best[1:]]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new, length", [(2, 200), (70, 333), (70, 2500), (3, 4000)])
@pytest.mark.parametrize("size, kw", [
    (200.0, dict(prefix=[3])), (200.0, dict(slopes=geometric(4) / 5000)), (35.0, dict(softcap=50.0)),
    (35.0, dict(softcap=50.0, slopes=geometric(4) / 5000)), (200.0, dict(softcap=1000.0)),
    (200.0, dict(softcap=1000.0, slopes=geometric(4) / 5000)),
])
def test_f16_queries_see_codes_to_15_bits(bits, dim, new, length, size, kw):
    """Keys of two kinds in turn, whose roundings to one f16 would move their scores apart, and values of 1
    and -1: the bound's term for coded keys, 2^-11, shrinks to 2^-15, and one f16 would be beyond it."""
    pool = Pool(72, [length], 2, dim, 16, bits, None)
    kinds = two_keys(bits)
    for t in range(length):
        at = int(pool.table[0, t // 16]), slice(None)
        c, s = kinds[t % 2]
        pool.k[(*at, t % 16)] = c + 128 if bits == 8 else (c + 8) * 17
        pool.ks[(*at, slice(None), t % 16)] = s / 128
        pool.v[(*at, t % 16)] = (64 if t % 2 else -64) + 128 if bits == 8 else (4 if t % 2 else -4) * 17 + 8 * 17
        pool.vs[(*at, slice(None), t % 16)] = 1 / 64 if bits == 8 else 1 / 4
    k, v = pool.values("k", 0), pool.values("v", 0)
    assert bool((v.abs() == 1).all())
    gain = size * math.sqrt(dim) / float(k[0, 0].sum())
    q = torch.full((new, 4, dim), gain).half()
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, [new], [length], pool.table)
    slopes = kw.get("slopes")
    shape = dict(softcap=kw.get("softcap", 0.0), slopes=None if slopes is None else slopes.float().cuda(),
                 prefix=torch.tensor(kw["prefix"], dtype=torch.int32).cuda() if "prefix" in kw else None)
    y = mlxl3_amd.attention(q.cuda(), cache, b, **shape)
    args = (length - new, dim**-0.5, True, 0, kw.get("softcap", 0.0), None if slopes is None else slopes.float(), kw.get("prefix", [0])[0])
    want, exact = scores_ref.attend(q.double(), k, v, *args, dtype=F16)
    rounded = scores_ref.attend(q.double(), k, v, *args, coded=True, dtype=F16)[1]
    bound = exact + (rounded - exact) / 16
    one = scores_ref.attend(q.double(), k.half().double(), v, *args, dtype=F16)[0]
    assert bool(((one - want).abs() > 2 * bound).any(-1).all())  # what the test is for
    within(y, want, bound, "two parts")
