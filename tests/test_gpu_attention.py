"""Rotary positions, the paged cache and attention over it on the GPU, against the 64-bit
forms of kv_ref.py within the bounds derived there from where the kernels round: every
format and head width, page sizes, ragged batches, odd lengths, windows, rows that see
nothing, strides, pages and lengths that the table does not have, slots never written (they
hold NaN throughout), streams and captured graphs."""

import math

import pytest
import torch

import kv_ref
from kv_ref import EPS, Pool

import mlxl3_amd

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def within(y, want, bound, label):
    y = y.detach().cpu().double()
    assert y.shape == want.shape
    off = (y - want).abs()
    ok = off <= bound
    assert bool(ok.all()), f"{label}: off by up to {float((off / bound.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} of the bound"


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens, heads, dim, rot", [
    (1, 1, 64, 64), (1, 32, 128, 128), (7, 5, 128, 64), (33, 3, 256, 64), (130, 2, 128, 32), (5, 3, 80, 20), (6, 2, 96, 96),
    (3, 2, 2, 2), (9, 4, 64, 24),
])
def test_rope(dtype, inter, tokens, heads, dim, rot):
    g = torch.Generator().manual_seed(tokens * 1000 + dim + rot)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype)
    pos = torch.randint(-5000, 200000, (tokens,), generator=g, dtype=torch.int32)
    freq, _ = mlxl3_amd.rope_frequencies(rot, 10000.0)
    scale = 1.0 if dim != 128 else 1.25
    r = mlxl3_amd.Rope(freq.cuda(), interleaved=inter, scale=scale)
    y = r.apply(x.cuda(), pos.cuda())
    want = kv_ref.rotate(x, pos, freq, inter, scale)
    bound = kv_ref.rotate_bound(x, freq, inter, scale) + EPS[dtype] / 2 * want.abs() + 2.0**-25
    assert y.dtype == dtype
    within(y, want, bound, "rope")
    assert torch.equal(y[..., rot:].cpu(), x[..., rot:])
    # in place, and out of / into rows with gaps
    z = x.cuda()
    assert r.apply(z, pos.cuda(), out=z) is z and torch.equal(z, y)
    wide = torch.zeros(tokens, heads + 2, dim, dtype=dtype, device="cuda")
    wide[:, 1:-1] = x.cuda()
    out = torch.full((tokens, heads + 1, dim), 9.0, dtype=dtype, device="cuda")
    r.apply(wide[:, 1:-1], pos.cuda(), out=out[:, :heads])
    assert torch.equal(out[:, :heads], y) and bool((out[:, heads] == 9.0).all())


def test_rope_changes_type_and_far_positions_turn_back():
    x = torch.randn(64, 2, 128, generator=torch.Generator().manual_seed(1))
    pos = torch.arange(64, dtype=torch.int32) * 33000000 + 1
    freq, _ = mlxl3_amd.rope_frequencies(128)
    r = mlxl3_amd.Rope(freq.cuda())
    y = r.apply(x.cuda(), pos.cuda())
    # angles up to 2^31 are rounded to 2^-22 in 64 bits, on both sides alike
    within(y, kv_ref.rotate(x, pos, freq, False, 1.0), kv_ref.rotate_bound(x, freq, False, 1.0) + 2.0**-23 * 5, "far")
    back = r.apply(y, -pos.cuda())
    within(back, x.double(), 3 * kv_ref.rotate_bound(x, freq, False, 1.0) + 8 * 2.0**-24 * 5, "back")
    half = r.apply(x.cuda(), pos.cuda(), dtype=BF16)
    assert half.dtype == BF16 and torch.equal(half, y.to(BF16))


def test_rope_positions_of_a_batch():
    new, lens = [3, 0, 5, 1], [10, 4, 5, 700]
    b = kv_ref.batch(mlxl3_amd, new, lens, None)
    pos = torch.tensor([7, 8, 9, 0, 1, 2, 3, 4, 699], dtype=torch.int32).cuda()
    x = torch.randn(11, 4, 64, device="cuda").half()  # two rows behind the last sequence
    r = mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(64)[0].cuda())
    out = torch.full_like(x, 3.0)
    r.apply(x, batch=b, out=out)
    assert torch.equal(out[:9], r.apply(x[:9], pos)) and bool((out[9:] == 3.0).all())


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
def stored(pool, x, seq_rows, bits, dtype):
    if bits == 16:
        return x.to(dtype).double()
    c, s = kv_ref.quantise(x, bits)
    return c.double() * s.double().repeat_interleave(32, -1)


@pytest.mark.parametrize("bits, cdtype", [(16, F16), (16, BF16), (8, None), (4, None)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim, page, kv_heads, new, old", [
    (128, 16, 2, [1], [0]), (128, 64, 8, [1, 1, 1], [15, 63, 200]), (64, 16, 1, [37, 0, 5], [3, 9, 0]),
    (256, 32, 3, [70, 1], [1, 31]),
])
def test_append_and_read(bits, cdtype, dtype, dim, page, kv_heads, new, old):
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(5, lens, kv_heads, dim, page, bits, cdtype)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    g = torch.Generator().manual_seed(dim + bits)
    n = sum(new)
    k = torch.randn(n, kv_heads, dim, generator=g)
    v = torch.randn(n, kv_heads, dim, generator=g)
    k[..., 3] *= 20
    v[0] = 0  # a token of zeros
    v[-1] *= 2.0**-30  # scales below what f16 holds
    k, v = k.to(dtype), v.to(dtype)
    before = [t.clone() for t in (cache.k, cache.v)]
    cache.append(b, k.cuda(), v.cuda())
    for x, name in ((k, "k"), (v, "v")):
        want = stored(pool, x.float(), None, bits, cdtype)
        for out in (F16, BF16, F32):
            got = dict(zip("kv", cache.read(b, n, out)))[name]
            assert torch.equal(got.cpu(), want.float().to(out)), (name, out)
    # what was there before is as it was
    whole = kv_ref.batch(mlxl3_amd, lens, lens, pool.table)
    got_k, got_v = cache.read(whole, sum(lens), F32)
    at = 0
    for s, (o, t) in enumerate(zip(old, lens)):
        assert torch.equal(got_k[at : at + o].cpu(), pool.values("k", s)[:o].float())
        assert torch.equal(got_v[at : at + o].cpu(), pool.values("v", s)[:o].float())
        at += t
    touched = {(int(pool.table[s, p // page]), p % page) for s, (o, t) in enumerate(zip(old, lens)) for p in range(o, t)}
    keep = torch.ones(cache.pages, page, dtype=torch.bool)
    for pg, sl in touched:
        keep[pg, sl] = False
    keep = keep[:, None].expand(-1, kv_heads, -1).cuda()
    for t, was in zip((cache.k, cache.v), before):
        assert torch.equal(t[keep].view(torch.uint8), was[keep].view(torch.uint8))


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("inter, dim, rot", [(False, 128, 128), (True, 128, 128), (False, 128, 64), (True, 64, 20), (False, 64, 20),
                                             (False, 256, 64)])
def test_append_rotates_keys(bits, inter, dim, rot):
    new, old = [5, 1, 30], [100, 0, 3]
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(6, lens, 2, dim, 16, bits, F16)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    freq, _ = mlxl3_amd.rope_frequencies(rot, 500000.0)
    rope = mlxl3_amd.Rope(freq.cuda(), interleaved=inter, scale=1.1)
    # keys and values as two parts of one projection's rows, with gaps
    both = torch.randn(sum(new), 5, dim, generator=torch.Generator().manual_seed(3)).to(BF16)
    dev = both.cuda()
    k, v = dev[:, :2], dev[:, 3:]
    cache.append(b, k, v, rope=rope)
    got_k, got_v = cache.read(b, sum(new), F32)
    # the rotated keys are exl3_rope's in f32 (bit for bit), then the plain store
    turned = rope.apply(k.float().contiguous(), batch=b).cpu()
    assert torch.equal(got_k.cpu(), stored(pool, turned, None, bits, F16).float())
    assert torch.equal(got_v.cpu(), stored(pool, both[:, 3:].float(), None, bits, F16).float())


def test_groups_that_are_not_finite_and_large_ones():
    pool = Pool(7, [4], 1, 64, 16, 8, None)
    x = torch.zeros(4, 1, 64)
    x[0, 0, 3] = math.nan
    x[1, 0, 40] = math.inf
    x[2, 0, 1], x[2, 0, 2] = 3.0e38, -1.0e6
    x[3] = 1.0e-8
    for bits in (8, 4):
        pool = Pool(7, [4], 1, 64, 16, bits, None)
        cache = pool.cuda(mlxl3_amd)
        b = kv_ref.batch(mlxl3_amd, [4], [4], pool.table)
        cache.append(b, x.cuda(), x.cuda())
        k, _ = cache.read(b, 4, F32)
        k = k.cpu()
        assert k[0, 0, :32].isnan().all() and (k[0, 0, 32:] == 0).all()
        assert (k[1, 0, :32] == 0).all() and k[1, 0, 32:].isnan().all()
        most = kv_ref.LEVELS[bits]
        assert k[2, 0, 1] == 65504.0 * most and k[2, 0, 2] == -65504.0 * min(most, round(1.0e6 / 65504.0))
        assert (k[3] == 0).all()


def test_tokens_without_a_page():
    """Positions behind the table, pages outside the pool, lengths shorter than the new
    tokens, rows behind the last sequence: nothing else is touched, they read as zeros."""
    pool = Pool(8, [40, 20, 9], 2, 64, 16, 16, F16, table_pages=3)
    pool.table[0, 1] = 1 << 30
    pool.table[1, 1] = -1
    cache = pool.cuda(mlxl3_amd)
    new, lens = [40, 20, 9], [40, 20, 4]  # the last says 4 tokens with 9 new ones
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    x = torch.randn(72, 2, 64, device="cuda").half()
    cache.append(b, x, x)
    out = torch.full((72, 2, 64), 5.0, dtype=F16, device="cuda")
    lib = mlxl3_amd.load_library()
    v = torch.full_like(out, 5.0)
    assert lib.exl3_kv_read(cache.handle, b._ref, out.data_ptr(), v.data_ptr(), 9, 72, torch.cuda.current_stream().cuda_stream) == 0
    want = x.clone()
    want[16:32] = 0
    want[40 + 16 : 60] = 0
    want[60:65] = 0
    want[69:] = 5.0
    assert torch.equal(out, want) and torch.equal(v, want)
    past = kv_ref.batch(mlxl3_amd, [2], [49], pool.table[:1])  # 48 positions have a table entry
    k, _ = cache.read(past, 2)
    assert torch.equal(k[0].view(torch.int16), cache.k[int(pool.table[0, 2]), :, 15].view(torch.int16)) and bool((k[1] == 0).all())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def run(pool, new, heads, dtype, seed=11, causal=True, window=0, scale=None, gain=1.0, **kw):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(sum(new), heads, pool.dim, generator=g) * gain).to(dtype)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, new, pool.lens, pool.table, **kw)
    y = mlxl3_amd.attention(q.cuda(), cache, b, scale=scale, causal=causal, window=window)
    return q, cache, b, y


def check(pool, new, q, y, causal=True, window=0, scale=None, label=""):
    scale = 1.0 / math.sqrt(pool.dim) if scale is None else scale
    at = 0
    for s, n in enumerate(new):
        want, bound = kv_ref.attend(q[at : at + n].double(), pool.values("k", s), pool.values("v", s), pool.lens[s] - n, scale,
                                    causal, window, coded=pool.bits != 16, dtype=q.dtype)
        within(y[at : at + n], want, bound, f"{label} sequence {s}")
        at += n


FORMATS = [(16, F16, F16), (16, BF16, BF16), (8, None, F16), (8, None, BF16), (4, None, F16), (4, None, BF16)]


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("dim, kv_heads, group, page, new, old", [
    (128, 1, 1, 16, [1], [0]),                       # a single token that sees itself
    (128, 2, 4, 16, [1], [999]),
    (64, 2, 1, 32, [1, 1, 1], [15, 16, 333]),
    (256, 1, 8, 64, [1, 1], [70, 4]),
    (128, 1, 16, 16, [1], [130]),
    (128, 2, 5, 16, [3, 1, 5], [60, 0, 17]),         # odd groups, short drafts
    (64, 1, 7, 16, [4, 4], [500, 1]),
    (128, 1, 32, 16, [1], [77]),
    (128, 1, 40, 32, [1], [77]),
    (256, 2, 2, 16, [9], [40]),
    (128, 2, 4, 64, [130], [0]),
    (64, 2, 3, 16, [65, 1, 0, 200], [3, 90, 5, 0]),
    (256, 1, 2, 128, [77], [100]),
])
def test_attention(bits, cdtype, dtype, dim, kv_heads, group, page, new, old):
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(dim + sum(lens), lens, kv_heads, dim, page, bits, cdtype)
    q, _, _, y = run(pool, new, kv_heads * group, dtype)
    assert y.dtype == dtype
    check(pool, new, q, y)


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
@pytest.mark.parametrize("causal, window", [(False, 0), (True, 1), (True, 7), (True, 64), (False, 33), (True, 10000)])
@pytest.mark.parametrize("new, old", [([1, 1], [300, 2]), ([6, 3], [200, 0]), ([150, 20], [40, 333])])
def test_windows_and_no_causal_mask(bits, cdtype, dtype, causal, window, new, old):
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(17, lens, 2, 128, 16, bits, cdtype)
    q, _, _, y = run(pool, new, 6, dtype, causal=causal, window=window)
    check(pool, new, q, y, causal, window)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new, old", [([1, 2], [333, 40]), ([150, 60], [0, 500])])
def test_f16_queries_see_codes_to_15_bits(bits, dim, new, old):
    """The bound's terms for coded values (2^-11 each) shrink to 2^-15."""
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(72, lens, 2, dim, 16, bits, None)
    q, _, _, y = run(pool, new, 8, F16, gain=3.0)
    at = 0
    for s, n in enumerate(new):
        args = (q[at : at + n].double(), pool.values("k", s), pool.values("v", s), pool.lens[s] - n, dim**-0.5, True, 0)
        want, exact = kv_ref.attend(*args, dtype=F16)
        rounded = kv_ref.attend(*args, coded=True, dtype=F16)[1]
        within(y[at : at + n], want, exact + (rounded - exact) / 16, f"sequence {s}")
        at += n


@pytest.mark.parametrize("new, old", [([1], [40000]), ([3, 1], [9000, 5]), ([64], [12000])])
@pytest.mark.parametrize("bits, cdtype, dtype", [FORMATS[1], FORMATS[2], FORMATS[4]])
def test_long_contexts(bits, cdtype, dtype, new, old):
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(23, lens, 1, 128, 64, bits, cdtype)
    q, _, _, y = run(pool, new, 4, dtype)
    check(pool, new, q, y)


@pytest.mark.parametrize("gain", [0.0, 12.0])
@pytest.mark.parametrize("new, old", [([1, 2], [200, 77]), ([40, 90], [200, 0])])
def test_flat_and_peaked_scores(gain, new, old):
    lens = [n + o for n, o in zip(new, old)]
    for bits, cdtype, dtype in FORMATS[:3]:
        pool = Pool(29, lens, 2, 128, 16, bits, cdtype, loud=1.0)
        q, _, _, y = run(pool, new, 8, dtype, gain=gain)
        check(pool, new, q, y)


def test_rising_scores():
    """Every block of keys beats those before it: the running maximum moves all the way."""
    for new in ([1], [40]):
        pool = Pool(31, [700], 1, 128, 16, 16, F16, loud=1.0)
        ramp = torch.linspace(0.0, 6.0, 700).half()
        for t in range(700):
            pool.k[int(pool.table[0, t // 16]), 0, t % 16] = ramp[t]
        cache = pool.cuda(mlxl3_amd)
        b = kv_ref.batch(mlxl3_amd, new, [700], pool.table)
        q = torch.full((new[0], 2, 128), 0.5).half()
        y = mlxl3_amd.attention(q.cuda(), cache, b)
        check(pool, new, q, y)


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
def test_rows_that_see_nothing_and_rows_outside(bits, cdtype, dtype):
    """A sequence of length zero and one whose length is below its new tokens: zeros; rows
    in front of the first and behind the last sequence: as they were."""
    for new in ([2, 3, 4], [50, 3, 60]):
        lens = [new[0] + 9, 0, 2]
        pool = Pool(37, [new[0] + 9, 0, 2], 2, 128, 16, bits, cdtype)
        cache = pool.cuda(mlxl3_amd)
        starts = torch.tensor([2, 2 + new[0], 2 + sum(new[:2]), 2 + sum(new)], dtype=torch.int32).cuda()
        b = mlxl3_amd.KvBatch(starts, torch.tensor(lens, dtype=torch.int32).cuda(), pool.table.cuda(), max_q=max(new))
        rows = 2 + sum(new) + 3
        q = torch.randn(rows, 4, 128, generator=torch.Generator().manual_seed(5)).to(dtype)
        out = torch.full((rows, 4, 128), 4.0, dtype=dtype, device="cuda")
        y = mlxl3_amd.attention(q.cuda(), cache, b, out=out)
        assert y is out and bool((y[:2] == 4.0).all()) and bool((y[-3:] == 4.0).all())
        inner = y[2:-3]
        check(pool, [new[0]], q[2 : 2 + new[0]], inner[: new[0]])
        assert bool((inner[new[0] : sum(new) - 2] == 0).all())
        want, bound = kv_ref.attend(q[-5:-3].double(), pool.values("k", 2), pool.values("v", 2), 0, 128**-0.5, True, 0,
                                    coded=bits != 16, dtype=dtype)
        within(inner[-2:], want, bound, "short")


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
@pytest.mark.parametrize("new", [[1, 1], [60, 40]])
def test_pages_outside_the_pool_are_skipped(bits, cdtype, dtype, new):
    lens = [200, 150]
    pool = Pool(41, lens, 2, 128, 16, bits, cdtype, table_pages=13)
    good = pool.table.clone()
    pool.table[0, 2], pool.table[0, 7], pool.table[1, 0] = -1, 1 << 30, pool.k.shape[0]
    q, cache, b, y = run(pool, new, 4, dtype)
    at = 0
    for s, n in enumerate(new):
        keep = torch.ones(lens[s], dtype=torch.bool)
        for j in range(-(-lens[s] // 16)):
            if pool.table[s, j] != good[s, j]:
                keep[16 * j : 16 * j + 16] = False
        pool2 = Pool(41, lens, 2, 128, 16, bits, cdtype, table_pages=13)
        k, v = pool2.values("k", s), pool2.values("v", s)
        for i in range(n):
            see = keep & (torch.arange(lens[s]) <= lens[s] - n + i)
            want, bound = kv_ref.attend(q[at + i : at + i + 1].double(), k[see], v[see], int(see.sum()), 128**-0.5, False, 0,
                                        coded=bits != 16, dtype=dtype)
            within(y[at + i : at + i + 1], want, bound, f"sequence {s} row {i}")
        at += n
    # a length past the table is cut at the table's room
    b2 = kv_ref.batch(mlxl3_amd, [1], [5000], good[1:2, :9])
    y2 = mlxl3_amd.attention(q[:1].cuda(), cache, b2)
    want, bound = kv_ref.attend(q[:1].double(), pool2.values("k", 1)[:144], pool2.values("v", 1)[:144], 4999, 128**-0.5, True, 0,
                                coded=bits != 16, dtype=dtype)
    within(y2, want, bound, "cut")


@pytest.mark.parametrize("new", [[1, 3], [40, 33]])
def test_values_that_a_row_does_not_see_do_not_reach_it(new):
    """NaN and infinities in keys and values behind a row's position or before its window."""
    for bad in (math.nan, math.inf, -math.inf):
        lens = [new[0] + 100, new[1] + 20]
        pool = Pool(43, lens, 2, 128, 16, 16, F16)
        for s, n in enumerate(new):
            for t in (5, lens[s] - 1):  # before every window, and the newest token
                at = int(pool.table[s, t // 16]), slice(None), t % 16
                pool.k[at], pool.v[at] = bad, bad
        q, _, _, y = run(pool, new, 4, F16, window=8)
        at = 0
        for s, n in enumerate(new):
            k, v = pool.values("k", s), pool.values("v", s)
            k[5] = v[5] = 0
            k[-1] = v[-1] = 0
            want, bound = kv_ref.attend(q[at : at + n].double(), k, v, lens[s] - n, 128**-0.5, True, 8, dtype=F16)
            within(y[at : at + n - 1], want[:-1], bound[:-1], f"{bad} sequence {s}")
            assert not bool(y[at + n - 1].isfinite().all())  # the row that does see it
            at += n


def test_strides_and_outputs():
    pool = Pool(47, [90, 33], 2, 128, 16, 16, F16)
    cache = pool.cuda(mlxl3_amd)
    for new in ([1, 2], [33, 30]):
        b = kv_ref.batch(mlxl3_amd, new, pool.lens, pool.table)
        n = sum(new)
        fused = torch.randn(n, 12, 128, generator=torch.Generator().manual_seed(2)).half()
        dev = fused.cuda()
        plain = mlxl3_amd.attention(fused[:, 2:10].contiguous().cuda(), cache, b)
        out = torch.full((n, 10, 128), 7.0, dtype=F16, device="cuda")
        mlxl3_amd.attention(dev[:, 2:10], cache, b, out=out[:, 1:9])
        assert torch.equal(out[:, 1:9], plain) and bool((out[:, 0] == 7.0).all()) and bool((out[:, 9] == 7.0).all())
        # other strides are copied, rows that start at odd addresses read as they are
        turned = fused[:, 2:10].transpose(1, 2).contiguous().transpose(1, 2).cuda()
        assert torch.equal(mlxl3_amd.attention(turned, cache, b), plain)
        odd = torch.zeros(n * 8 * 128 + 3, dtype=F16, device="cuda")
        odd[3:] = fused[:, 2:10].reshape(-1).cuda()
        room = torch.zeros(n * 8 * 128 + 1, dtype=F16, device="cuda")
        got = mlxl3_amd.attention(odd[3:].view(n, 8, 128), cache, b, out=room[1:].view(n, 8, 128))
        assert torch.equal(got, plain)
        with pytest.raises(mlxl3_amd.Exl3Error, match="out must have q's shape"):
            mlxl3_amd.attention(dev[:, 2:10], cache, b, out=out)


def test_max_q_bounds_the_rows_computed():
    """More new tokens than max_q says: rows up to it are right, nothing is read or written
    outside."""
    pool = Pool(53, [60, 50], 1, 128, 16, 16, F16)
    q, cache, _, _ = run(pool, [20, 10], 4, F16)
    b = kv_ref.batch(mlxl3_amd, [20, 10], pool.lens, pool.table, max_q=3)
    y = mlxl3_amd.attention(q.cuda(), cache, b)
    for at, s, n in ((0, 0, 20), (20, 1, 10)):
        want, bound = kv_ref.attend(q[at : at + n].double(), pool.values("k", s), pool.values("v", s), pool.lens[s] - n, 128**-0.5,
                                    True, 0, dtype=F16)
        within(y[at : at + 3], want[:3], bound[:3], f"sequence {s}")


@pytest.mark.parametrize("new", [[2, 4], [20, 40]])
def test_starts_beyond_the_tokens_are_cut(new):
    """The last sequence claims more rows than q has: those there are right, and the memory
    behind them is left as it was."""
    lens = [n + 70 for n in new]
    pool = Pool(56, lens, 1, 64, 16, 16, F16)
    q, cache, b, _ = run(pool, new, 4, F16)
    cut = sum(new) - 3
    out = torch.full((sum(new), 4, 64), 9.0, dtype=F16, device="cuda")
    mlxl3_amd.attention(q[:cut].cuda(), cache, b, out=out[:cut])
    at = 0
    for s, n in enumerate(new):
        want, bound = kv_ref.attend(q[at : at + n].double(), pool.values("k", s), pool.values("v", s), 70, 64**-0.5, True, 0, dtype=F16)
        m = min(n, cut - at)
        within(out[at : at + m], want[:m], bound[:m], f"sequence {s}")
        at += n
    assert bool((out[cut:] == 9.0).all())


@pytest.mark.parametrize("most", [1, 150])
def test_many_sequences(most):
    """More sequences than a wave has lanes, some without new tokens, tiles of many."""
    g = torch.Generator().manual_seed(57)
    new = torch.randint(0, most + 1, (203,), generator=g).tolist()
    lens = [n + int(o) for n, o in zip(new, torch.randint(0, 60, (203,), generator=g))]
    pool = Pool(58, lens, 1, 64, 16, 8, None)
    q, cache, b, y = run(pool, new, 2, BF16)
    check(pool, new, q, y)
    loose = kv_ref.batch(mlxl3_amd, new, lens, pool.table, max_q=2**31 - 1)
    check(pool, new, q, mlxl3_amd.attention(q.cuda(), cache, loose))


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("dim, kv_heads, group, new, old", [
    (128, 8, 4, [1, 1, 1, 0, 1], [5000, 0, 300, 77, 1290]),
    (64, 2, 7, [2, 1, 4, 1], [2, 6000, 40, 700]),
    (256, 4, 2, [1, 3], [200, 3333]),
])
@pytest.mark.parametrize("window", [0, 50000, 700])
def test_ragged_batches_told_long_ones(bits, cdtype, dtype, dim, kv_heads, group, new, old, window):
    """Bounds of 100000 tokens: the ranges go by the tokens that there are."""
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(68, lens, kv_heads, dim, 64, bits, cdtype, table_pages=1600)
    q, _, _, y = run(pool, new, kv_heads * group, dtype, window=window)
    check(pool, new, q, y, window=window)


def test_many_ragged_sequences_told_long_ones():
    g = torch.Generator().manual_seed(69)
    lens = torch.randint(1, 500, (150,), generator=g).tolist()
    lens[77] = 9000
    pool = Pool(70, lens, 1, 64, 64, 16, F16, table_pages=2000)
    new = [min(1 + i % 3, n) for i, n in enumerate(lens)]
    q, _, _, y = run(pool, new, 4, F16)
    check(pool, new, q, y)


@pytest.mark.parametrize("group, new", [(33, [1, 2]), (200, [1, 3]), (129, [2])])
def test_groups_larger_than_a_tile(group, new):
    """The rows of one token fall into several tiles."""
    lens = [n + 90 for n in new]
    pool = Pool(60, lens, 2, 64, 32, 4, None)
    q, _, _, y = run(pool, new, 2 * group, F16)
    check(pool, new, q, y)


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
@pytest.mark.parametrize("new, old, window", [([1], [5000], 1500), ([2, 1], [700, 4000], 900), ([64, 3], [6000, 10], 2500)])
def test_windows_over_several_ranges(bits, cdtype, dtype, new, old, window):
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(62, lens, 1, 128, 64, bits, cdtype)
    q, _, _, y = run(pool, new, 4, dtype, window=window)
    check(pool, new, q, y, window=window)


@pytest.mark.parametrize("bits", [16, 8])
def test_pages_beyond_32_bits(bits):
    """Pages that lie more than 2^32 bytes (and values) into the pool: written, read, attended."""
    dim, heads, page = 128, 8, 64
    pages = 2**32 // (heads * page * dim) + 8
    shape = (pages, heads, page)
    kw = dict(device="cuda")
    if bits == 16:
        cache = mlxl3_amd.KvCache(*(torch.empty(*shape, dim, dtype=F16, **kw) for _ in range(2)))
    else:
        codes = [torch.empty(*shape, dim, dtype=torch.uint8, **kw) for _ in range(2)]
        scales = [torch.empty(pages, heads, dim // 32, page, dtype=F16, **kw) for _ in range(2)]
        cache = mlxl3_amd.KvCache(*codes, *scales, bits=8)
    table = torch.tensor([[pages - 1, 0, pages - 3], [pages - 2, 1, 5]], dtype=torch.int32)
    lens = [150, 131]
    g = torch.Generator().manual_seed(63)
    k, v = (torch.randn(sum(lens), heads, dim, generator=g).to(F16) for _ in range(2))
    cache.append(kv_ref.batch(mlxl3_amd, lens, lens, table), k.cuda(), v.cuda())
    rk, rv = (t.cpu() for t in cache.read(kv_ref.batch(mlxl3_amd, lens, lens, table), sum(lens)))
    for got, x in ((rk, k), (rv, v)):
        if bits == 8:
            c, s = kv_ref.quantise(x, 8)
            x = (c.float() * s.float().repeat_interleave(32, -1)).half()
        assert torch.equal(got, x)
    for new in ([1, 2], [40, 30]):
        q = torch.randn(sum(new), 2 * heads, dim, generator=g).to(F16)
        y = mlxl3_amd.attention(q.cuda(), cache, kv_ref.batch(mlxl3_amd, new, lens, table))
        at = row = 0
        for n, length in zip(new, lens):
            kd, vd = k[row : row + length].double(), v[row : row + length].double()
            if bits == 8:
                kd, vd = (c.double() * s.double().repeat_interleave(32, -1) for c, s in (kv_ref.quantise(kd, 8), kv_ref.quantise(vd, 8)))
            want, bound = kv_ref.attend(q[at : at + n].double(), kd, vd, length - n, dim**-0.5, True, 0, coded=bits == 8, dtype=F16)
            within(y[at : at + n], want, bound, f"{n} new")
            at, row = at + n, row + length


def test_threads_that_share_a_batch():
    """Two threads, each with its stream and cache, and one batch object: a call's workspace
    goes by its own sizes."""
    import threading

    pools = [Pool(65, [3000], 1, dim, 16, 16, F16) for dim in (64, 256)]  # the same pages
    assert torch.equal(pools[0].table, pools[1].table)
    caches = [p.cuda(mlxl3_amd) for p in pools]
    b = kv_ref.batch(mlxl3_amd, [1], [3000], pools[0].table)
    qs = [torch.randn(1, 8, p.dim, generator=torch.Generator().manual_seed(67)).to(F16).cuda() for p in pools]
    want = [mlxl3_amd.attention(q, c, b) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(100):
                    if not torch.equal(mlxl3_amd.attention(qs[i], caches[i], b), want[i]):
                        failed.append(f"thread {i}: another result")
        except Exception as e:  # told to the main thread
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_same_call_same_bits_and_longer_bounds_of_the_launch():
    pool = Pool(59, [3000, 17, 800], 2, 128, 32, 8, None)
    for new in ([1, 1, 1], [40, 17, 2]):
        q, cache, b, y = run(pool, new, 8, BF16)
        assert torch.equal(y, mlxl3_amd.attention(q.cuda(), cache, b))
        for max_kv in (1, 100, 3000, 100000):
            b2 = kv_ref.batch(mlxl3_amd, new, pool.lens, pool.table, max_kv=max_kv)
            check(pool, new, q, mlxl3_amd.attention(q.cuda(), cache, b2))


def test_no_tokens():
    pool = Pool(73, [20], 2, 64, 16, 8, None)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, [0], [20], pool.table)
    rope = mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(64)[0].cuda())
    none = torch.empty(0, 2, 64, dtype=F16, device="cuda")
    before = cache.k.clone()
    cache.append(b, none, none, rope=rope)
    assert torch.equal(cache.k, before)
    assert [t.shape[0] for t in cache.read(b, 0)] == [0, 0]
    assert rope.apply(none, batch=b).shape == none.shape
    assert rope.apply(none, torch.empty(0, dtype=torch.int32, device="cuda")).shape == none.shape
    assert mlxl3_amd.attention(none, cache, b).shape == none.shape
    with pytest.raises(mlxl3_amd.Exl3Error, match="from an array or from a KV batch"):
        rope.apply(none)


@pytest.mark.parametrize("new", [1, 40])
def test_a_graph_told_long_lengths_follows_short_ones(new):
    """Captured once with bounds of 100000 tokens, replayed for lengths that change between
    the replays, eager work beside it; every replay against the eager call."""
    lens = [3000, 90, 700]
    pool = Pool(74, lens, 8, 64, 64, 16, F16, table_pages=1600, poison=False)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, [new] * 3, lens, pool.table)
    q = torch.randn(3 * new, 16, 64, generator=torch.Generator().manual_seed(75)).half().cuda()
    mlxl3_amd.attention(q, cache, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = mlxl3_amd.attention(q, cache, b)
    for now in ([3000, 90, 700], [2999, 40, 641], [1500, 60, 40], [40, 40, 699], [2048, 64, 128]):
        b.kv_lens.copy_(torch.tensor(now, dtype=torch.int32))
        want = mlxl3_amd.attention(q, cache, b)
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), now
        at = 0
        for s, length in enumerate(now):
            w, bound = kv_ref.attend(q[at : at + new].cpu().double(), pool.values("k", s)[:length], pool.values("v", s)[:length],
                                     length - new, 64**-0.5, True, 0, dtype=F16)
            within(y[at : at + new], w, bound, f"{now} sequence {s}")
            at += new


def test_other_streams():
    pool = Pool(61, [2000], 2, 128, 16, 16, BF16)
    q, cache, b, y = run(pool, [1], 8, BF16)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(mlxl3_amd.attention(q.cuda(), cache, b))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)


def test_captured_graphs_follow_the_device_arrays():
    """Append and attention captured once, replayed as the sequences grow, two graphs in
    turn; every replay against the eager calls."""
    lens, steps = [30, 130, 7], 5
    pool = Pool(67, [n + steps for n in lens], 2, 128, 16, 8, None, poison=False)
    table = pool.table.cuda()
    starts = torch.arange(4, dtype=torch.int32).cuda()
    rope = mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(128)[0].cuda())

    class Side:
        def __init__(self):
            self.cache = pool.cuda(mlxl3_amd)
            self.lens = torch.tensor(lens, dtype=torch.int32).cuda()
            self.batch = mlxl3_amd.KvBatch(starts, self.lens, table, max_q=1, max_kv=400)
            self.x = [torch.zeros(3, h, 128, dtype=F16, device="cuda") for h in (8, 2, 2)]

        def step(self):
            q = rope.apply(self.x[0], batch=self.batch)
            self.cache.append(self.batch, self.x[1], self.x[2], rope=rope)
            return mlxl3_amd.attention(q, self.cache, self.batch)

    eager, sides, graphs, outs = Side(), [Side(), Side()], [], []
    eager.step()  # writes what the warm-up steps below write
    for s in sides:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.step())
        graphs.append(g)
    gen = torch.Generator().manual_seed(9)
    for step in range(steps):
        xs = [torch.randn(3, h, 128, generator=gen).half().cuda() for h in (8, 2, 2)]
        for s in [eager] + sides:
            s.lens.copy_(torch.tensor([n + step + 1 for n in lens], dtype=torch.int32))
            for dst, src in zip(s.x, xs):
                dst.copy_(src)
        want = eager.step()
        for g, out, s in zip(graphs, outs, sides):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), step
            assert torch.equal(s.cache.k, eager.cache.k) and torch.equal(s.cache.v_scales, eager.cache.v_scales)


# ---------------------------------------------------------------------------
# the attention block
# ---------------------------------------------------------------------------
def projections(seed, hidden, heads, kv_heads, dim, k, cb, bias):
    from mlxl3_amd import synth

    def one(i, n_in, n_out, with_bias):
        tr, suh, svh, b = synth.linear_layer(seed, i, n_in, n_out, k, bias=with_bias)
        dev = lambda a: None if a is None else torch.from_numpy(a.view("int16") if a.dtype.name == "uint16" else a).cuda()
        return mlxl3_amd.Exl3Linear(dev(tr), dev(suh), dev(svh), dev(b) if with_bias else None, k, cb)

    return [one(0, hidden, heads * dim, bias), one(1, hidden, kv_heads * dim, bias), one(2, hidden, kv_heads * dim, bias),
            one(3, heads * dim, hidden, False)]


@pytest.mark.parametrize("dtype, bits, bias", [(F16, 16, False), (BF16, 16, True), (BF16, 8, True), (F16, 4, True)])
@pytest.mark.parametrize("dim, heads, kv_heads, new, old", [
    (128, 8, 2, [1, 1, 1], [70, 0, 300]), (64, 6, 2, [3, 40], [9, 0]), (256, 2, 1, [2], [33]),
])
def test_attention_block_equals_its_calls(dtype, bits, bias, dim, heads, kv_heads, new, old):
    hidden, rows = 512, sum(new)
    q, k, v, o = projections(3, hidden, heads, kv_heads, dim, 4, 0, bias)
    lens = [n + m for n, m in zip(new, old)]
    pool = Pool(73, lens, kv_heads, dim, 16, bits, dtype, loud=1.0)
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    rope = mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(dim)[0].cuda())
    x = (torch.randn(rows, hidden, generator=torch.Generator().manual_seed(1)) / 8).to(dtype).cuda()
    block = mlxl3_amd.Exl3Attention(q, k, v, o, rope=rope, window=100)
    one, two = pool.cuda(mlxl3_amd), pool.cuda(mlxl3_amd)
    for _ in range(2):
        y = block(x, one, b)
    qs, ks, vs = mlxl3_amd.Exl3Group([q, k, v])(x)
    qr = rope.apply(qs.view(rows, heads, dim), batch=b, dtype=dtype)
    two.append(b, ks.view(rows, kv_heads, dim), vs.view(rows, kv_heads, dim), rope=rope)
    a = mlxl3_amd.attention(qr, two, b, window=100)
    want = o(a.view(rows, heads * dim))
    assert y.dtype == want.dtype and torch.equal(y, want) and bool(y.isfinite().all())
    for name in ("k", "v", "k_scales", "v_scales"):
        if getattr(one, name) is not None:
            assert torch.equal(getattr(one, name).view(torch.uint8), getattr(two, name).view(torch.uint8)), name
    # and the attention inside against 64 bits, from the cache as it now is
    pool.k, pool.v = two.k.cpu(), two.v.cpu()
    pool.ks, pool.vs = (None if t is None else t.cpu() for t in (two.k_scales, two.v_scales))
    check(pool, new, qr.cpu(), a, window=100)


def test_attention_block_in_graphs():
    """Two blocks' steps captured with a workspace each and replayed in turn as the
    sequences grow, against eager calls."""
    hidden, heads, kv_heads, dim = 256, 4, 2, 64
    q, k, v, o = projections(5, hidden, heads, kv_heads, dim, 3, 1, False)
    rope = mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(dim)[0].cuda())
    lens, steps = [40, 3, 260], 4
    pool = Pool(79, [n + steps for n in lens], kv_heads, dim, 16, 4, None, poison=False, loud=1.0)
    table, starts = pool.table.cuda(), torch.arange(4, dtype=torch.int32).cuda()
    block = mlxl3_amd.Exl3Attention(q, k, v, o, rope=rope)

    class Side:
        def __init__(self):
            self.cache = pool.cuda(mlxl3_amd)
            self.lens = torch.tensor(lens, dtype=torch.int32).cuda()
            self.batch = mlxl3_amd.KvBatch(starts, self.lens, table, max_q=1, max_kv=300)
            self.x = torch.zeros(3, hidden, dtype=F16, device="cuda")
            self.ws = torch.zeros(block.workspace_bytes(self.cache, self.batch, 3, F16), dtype=torch.uint8, device="cuda")

        def step(self):
            return block(self.x, self.cache, self.batch, workspace=self.ws)

    eager, sides, graphs, outs = Side(), [Side(), Side()], [], []
    eager.step()
    for s in sides:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.step())
        graphs.append(g)
    gen = torch.Generator().manual_seed(11)
    for step in range(steps):
        x = torch.randn(3, hidden, generator=gen).half().cuda()
        for s in [eager] + sides:
            s.lens.copy_(torch.tensor([n + step + 1 for n in lens], dtype=torch.int32))
            s.x.copy_(x)
        want = eager.step()
        for g, out, s in zip(graphs, outs, sides):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), step
            assert torch.equal(s.cache.v, eager.cache.v)


def test_attention_block_keeps_workspaces_apart():
    """The block's own workspaces: calls on two streams at once, and a captured step whose
    graph is replayed after an eager call that needed a larger one."""
    hidden, heads, kv_heads, dim = 256, 4, 2, 64
    block = mlxl3_amd.Exl3Attention(*projections(7, hidden, heads, kv_heads, dim, 4, 0, False))
    gen = torch.Generator().manual_seed(12)
    pool = Pool(80, [64, 64], kv_heads, dim, 16, 16, F16, poison=False, loud=1.0)

    def side(rows):
        b = kv_ref.batch(mlxl3_amd, [rows], [40 + rows - 1], pool.table[:1], max_kv=64)
        return pool.cuda(mlxl3_amd), b, torch.randn(rows, hidden, generator=gen).half().cuda()

    sides = [side(1), side(20)]
    want = [block(x, c, b) for c, b, x in sides]  # a kept one grows from 1 row's to 20's
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(20):
        for s, (c, b, x), w in zip(streams, sides, want):
            with torch.cuda.stream(s):
                outs.append((block(x, c, b), w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for y, w in outs)

    c, b, x = sides[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = block(x, c, b)
    for rows in (24, 30):
        c2, b2, x2 = side(rows)
        block(x2, c2, b2)
        fill = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")  # takes what a replaced workspace left
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and bool((fill == 255).all())


def test_attention_in_place():
    for new in ([1, 2], [40, 33]):
        pool = Pool(83, [900, 55], 2, 128, 16, 16, F16)
        q, cache, b, y = run(pool, new, 8, F16)
        x = q.cuda()
        assert mlxl3_amd.attention(x, cache, b, out=x) is x and torch.equal(x, y)


def test_python_refusals():
    pool = Pool(71, [20], 2, 128, 16, 16, F16)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, [1], [20], pool.table)
    q = torch.zeros(1, 4, 128, dtype=F16, device="cuda")
    err = mlxl3_amd.Exl3Error
    with pytest.raises(err, match="queries of 64 channels"):
        mlxl3_amd.attention(q[..., :64], cache, b)
    with pytest.raises(err, match="q has dtype"):
        mlxl3_amd.attention(q.float(), cache, b)
    with pytest.raises(err, match="have its type"):
        mlxl3_amd.attention(q.to(BF16), cache, b)
    with pytest.raises(err, match="3 query heads over 2"):
        mlxl3_amd.attention(q[:, :3], cache, b)
    with pytest.raises(err, match="new keys and values have shape"):
        cache.append(b, q, q)
    with pytest.raises(err, match="v has dtype"):
        cache.append(b, q[:, :2], q[:, :2].float())
    with pytest.raises(err, match="positions for 1 tokens"):
        mlxl3_amd.Rope(torch.ones(64, device="cuda")).apply(q, torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(err, match="needs a block table"):
        mlxl3_amd.attention(q, cache, kv_ref.batch(mlxl3_amd, [1], [20], None))
    with pytest.raises(err, match="block_table has one row"):
        mlxl3_amd.KvBatch(b.q_starts, b.kv_lens, pool.table.cuda().repeat(2, 1))
    with pytest.raises(err, match="must be contiguous"):
        mlxl3_amd.KvBatch(b.q_starts, b.kv_lens, pool.table.cuda().repeat(1, 2)[:, ::2])
    with pytest.raises(err, match="k_scales must have shape"):
        codes = torch.zeros(2, 1, 16, 128, dtype=torch.uint8, device="cuda")
        s = torch.zeros(2, 1, 16, 4, dtype=F16, device="cuda")
        mlxl3_amd.KvCache(codes, codes, s, s, bits=8)
    empty = mlxl3_amd.attention(q[:0], cache, b)
    assert empty.shape == (0, 4, 128)
