"""Attention with capped scores, a bias by distance and prefixes on the GPU, against the 64-bit form
of scores_ref.py within the bound derived there: every format and head width, decode, drafts and
prefill, windows, lengths of zero and one, values that a row does not see, graphs and streams."""

import math

import pytest
import torch

import kv_ref
import scores_ref
from kv_ref import Pool
from test_gpu_attention import BF16, F16, F32, FORMATS, projections, within

import mlxl3_amd

pytestmark = pytest.mark.gpu


def geometric(heads):
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float64) / heads)


def run(pool, new, heads, dtype, softcap=0.0, slopes=None, prefix=None, causal=True, window=0, gain=1.0, scale=None, **kw):
    g = torch.Generator().manual_seed(11)
    q = (torch.randn(sum(new), heads, pool.dim, generator=g) * gain).to(dtype)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, new, pool.lens, pool.table, **kw)
    shape = dict(softcap=softcap, slopes=None if slopes is None else slopes.float().cuda(),
                 prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda())
    y = mlxl3_amd.attention(q.cuda(), cache, b, scale=scale, causal=causal, window=window, **shape)
    return q, cache, b, y, shape


def check(pool, new, q, y, softcap=0.0, slopes=None, prefix=None, causal=True, window=0, scale=None, label=""):
    scale = 1.0 / math.sqrt(pool.dim) if scale is None else scale
    at = 0
    for s, n in enumerate(new):
        want, bound = scores_ref.attend(q[at : at + n].double(), pool.values("k", s), pool.values("v", s), pool.lens[s] - n, scale, causal,
                                        window, softcap, None if slopes is None else slopes.float(), 0 if prefix is None else prefix[s],
                                        coded=pool.bits != 16, dtype=q.dtype)
        within(y[at : at + n], want, bound, f"{label} sequence {s}")
        at += n


SHAPES = [
    (128, 1, 1, 16, [1], [0]),
    (128, 2, 4, 16, [1], [999]),
    (64, 2, 1, 32, [1, 1, 1], [15, 16, 333]),
    (256, 1, 8, 64, [1, 1], [70, 4]),
    (128, 2, 5, 16, [3, 1, 5], [60, 0, 17]),
    (64, 1, 7, 16, [4, 4], [500, 1]),
    (128, 1, 32, 16, [1], [77]),
    (256, 2, 2, 16, [9], [40]),
    (128, 2, 4, 64, [130], [0]),
    (64, 2, 3, 16, [65, 1, 0, 200], [3, 90, 5, 0]),
    (256, 1, 2, 128, [77], [100]),
]


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("dim, kv_heads, group, page, new, old", SHAPES)
@pytest.mark.parametrize("kind", ["cap", "bias", "prefix", "all"])
def test_shapes(bits, cdtype, dtype, dim, kv_heads, group, page, new, old, kind):
    lens, heads = [n + o for n, o in zip(new, old)], kv_heads * group
    pool = Pool(dim + sum(lens), lens, kv_heads, dim, page, bits, cdtype)
    kw = {}
    if kind in ("cap", "all"):
        kw["softcap"] = 30.0
    if kind in ("bias", "all"):
        kw["slopes"] = geometric(heads)
    if kind in ("prefix", "all"):
        kw["prefix"] = [(7 * i + 2 * n) // 3 for i, n in enumerate(lens)]
    q, _, _, y, _ = run(pool, new, heads, dtype, gain=4.0 if "softcap" in kw else 1.0, **kw)
    assert y.dtype == dtype
    check(pool, new, q, y, **kw)


@pytest.mark.parametrize("softcap", [2.0**-64, 1e-6, 0.02, 1.0, 15.0, 50.0, 255.0, 257.0, 1000.0, 1e5, 2.0**64])
@pytest.mark.parametrize("gain", [0.05, 1.0, 20.0, 600.0])
@pytest.mark.parametrize("new, old", [([1, 3], [200, 31]), ([40], [100])])
def test_caps_and_scores_of_all_sizes(softcap, gain, new, old):
    """Scores far below, around and far beyond the cap."""
    lens = [n + o for n, o in zip(new, old)]
    pool = Pool(17, lens, 2, 128, 16, 16, F16, loud=1.0)
    q, _, _, y, _ = run(pool, new, 8, F16, softcap=softcap, gain=gain)
    check(pool, new, q, y, softcap=softcap)


def test_a_cap_beyond_the_scores_changes_nothing_much():
    pool = Pool(18, [600], 2, 64, 16, 16, BF16)
    q, cache, b, y, _ = run(pool, [40], 8, BF16, softcap=2.0**60)
    plain = mlxl3_amd.attention(q.cuda(), cache, b)
    assert float((y.float() - plain.float()).abs().max()) <= 2.0**-7 * float(plain.float().abs().max())


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
@pytest.mark.parametrize("slope", [0.0, 1e-4, 0.3, 5.0, 1e4, -0.01])
def test_slopes_of_all_sizes(bits, cdtype, dtype, slope):
    for new, lens in (([1, 2], [700, 33]), ([50], [300])):
        pool = Pool(19, lens, 2, 128, 16, bits, cdtype)
        slopes = slope * torch.linspace(0.5, 1.0, 6, dtype=torch.float64)
        q, _, _, y, _ = run(pool, new, 6, dtype, slopes=slopes)
        check(pool, new, q, y, slopes=slopes)


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("gain", [1e-30, 1e-12, 1e-5, 1e3])
def test_biases_of_queries_of_all_sizes(bits, cdtype, dtype, gain):
    """A bias counts as much whatever the queries' size (f16 ones down to zeros)."""
    for new, lens in (([1, 2], [700, 33]), ([50], [300])):
        pool = Pool(25, lens, 2, 64, 16, bits, cdtype, loud=1.0)
        for kw in (dict(slopes=geometric(6)), dict(slopes=geometric(6), softcap=40.0)):
            q, _, _, y, _ = run(pool, new, 6, dtype, gain=gain, **kw)
            check(pool, new, q, y, **kw)


@pytest.mark.parametrize("scale", [1e-36, 1e-12, 1e-5, 3.0, 1e5, 1e9, 1e30])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_scales_of_all_sizes(bits, scale):
    """Scales that a bias is not divided by, and others; queries of the inverse size."""
    for new, lens in (([1, 2], [300, 33]), ([50], [200])):
        pool = Pool(26, lens, 2, 128, 16, bits, BF16, loud=1.0)
        for kw in (dict(slopes=geometric(4)), dict(softcap=4.0), dict(softcap=4.0, slopes=geometric(4)),
                   dict(softcap=300.0, slopes=geometric(4)), dict(prefix=[20, 5][: len(new)])):
            q, _, _, y, _ = run(pool, new, 4, BF16, gain=0.1 / scale, scale=scale, **kw)
            check(pool, new, q, y, scale=scale, **kw)


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
@pytest.mark.parametrize("causal", [True, False])
def test_distances_count_both_ways(bits, cdtype, dtype, causal):
    """Without a causal mask, and inside a prefix, tokens behind the row are as far as those before it."""
    for new, lens in (([3, 1], [60, 9]), ([90], [200])):
        pool = Pool(20, lens, 2, 64, 16, bits, cdtype)
        slopes, prefix = geometric(4) * 2, [55, 7][: len(new)]
        q, _, _, y, _ = run(pool, new, 4, dtype, slopes=slopes, prefix=prefix, causal=causal)
        check(pool, new, q, y, slopes=slopes, prefix=prefix, causal=causal)


@pytest.mark.parametrize("prefix", [[0, 0], [1, 1], [5, 64], [16, 17], [-4, 3], [10**6, 2**31 - 1], [301, 80]])
@pytest.mark.parametrize("window", [0, 1, 40])
@pytest.mark.parametrize("new", [[1, 1], [4, 2], [301, 80], [60, 30]])
def test_prefixes(prefix, window, new):
    lens = [301, 80]
    for dim, dtype in ((128, F16), (64, BF16)):
        pool = Pool(21, lens, 1, dim, 16, 16, dtype)
        q, _, _, y, _ = run(pool, new, 4, dtype, prefix=prefix, window=window)
        check(pool, new, q, y, prefix=prefix, window=window)


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS)
@pytest.mark.parametrize("new, lens, kw", [
    ([1], [20000], dict(softcap=50.0)), ([1], [9001], dict(slopes=geometric(8))), ([2, 1], [5000, 300], dict(softcap=20.0, slopes=geometric(8))),
    ([1] * 5, [9000, 200, 1, 64, 3000], dict(slopes=geometric(8) / 50)), ([70], [3000], dict(softcap=50.0, prefix=[2990])),
    ([200, 130], [2500, 130], dict(slopes=geometric(8) / 100, prefix=[100, 70], window=900)),
    ([60, 70], [700, 3000], dict(prefix=[650, 2990])), ([1, 2], [9000, 700], dict(prefix=[0, 700])),
    ([90], [2800], dict(softcap=20.0, slopes=geometric(8) / 30)),
])
def test_long_contexts(bits, cdtype, dtype, new, lens, kw):
    """Tokens split over workgroups, evenly and by the batch's sum, and joined."""
    pool = Pool(22, lens, 2, 128, 32, bits, cdtype)
    q, _, _, y, _ = run(pool, new, 8, dtype, gain=4.0 if "softcap" in kw else 1.0, **kw)
    check(pool, new, q, y, **kw)


def test_ragged_batches_by_their_sum():
    """Prefixes count in the batch's sum: prompts whose first rows see far ahead."""
    lens, new = [9000, 40, 3000, 7000], [2, 2, 1, 2]
    pool = Pool(23, lens, 1, 64, 16, 16, F16)
    for window, prefix in ((0, [9000, 40, 0, 6999]), (1500, [9000, 1, 2999, 7000])):
        q, _, _, y, _ = run(pool, new, 4, F16, prefix=prefix, window=window, softcap=30.0, max_kv=100000)
        check(pool, new, q, y, prefix=prefix, window=window, softcap=30.0)


def test_positions_beyond_24_bits():
    """Distances are exact where positions are not f32s: a table whose far pages are missing."""
    first = (1 << 25) + 3
    pool = Pool(24, [64], 1, 64, 1024, 16, F16, spare=0, poison=False)
    pages = first // 1024 + 1
    table = torch.full((1, pages), -1, dtype=torch.int32)
    table[0, -1] = 0
    n = first % 1024 + 1
    cache = pool.cuda(mlxl3_amd)
    slopes = torch.tensor([0.9, 0.25, 0.04, 1.5])
    for new in (1, 40):
        q = torch.randn(new, 4, 64, generator=torch.Generator().manual_seed(1)).half()
        for length in (first + 1, first + 1 + 50):
            used = length - (pages - 1) * 1024
            b = kv_ref.batch(mlxl3_amd, [new], [length], table)
            y = mlxl3_amd.attention(q.cuda(), cache, b, slopes=slopes.cuda())
            k, v = (x[0].transpose(0, 1)[:used].double() for x in (pool.k, pool.v))
            at = length - new - (pages - 1) * 1024  # of the first row in the last page
            want, bound = scores_ref.attend(q.double(), k, v, at, 0.125, True, 0, 0.0, slopes, 0, dtype=F16)
            seen = torch.arange(new) + at >= 0
            within(y[seen], want[seen], bound[seen], f"{new} at {length}")
            assert bool((y[~seen] == 0).all())
    assert n > 0


@pytest.mark.parametrize("kw", [dict(softcap=30.0), dict(slopes=geometric(4)), dict(softcap=10.0, slopes=geometric(4), prefix=[3, 2])])
@pytest.mark.parametrize("new", [[1, 3], [40, 33]])
def test_values_that_a_row_does_not_see_do_not_reach_it(new, kw):
    for bad in (math.nan, math.inf, -math.inf):
        lens = [new[0] + 100, new[1] + 20]
        pool = Pool(43, lens, 2, 128, 16, 16, F16)
        for s, n in enumerate(new):
            for t in (5, lens[s] - 1):  # before every window, and the newest token
                at = int(pool.table[s, t // 16]), slice(None), t % 16
                pool.k[at], pool.v[at] = bad, bad
        q, _, _, y, _ = run(pool, new, 4, F16, window=8, **kw)
        at = 0
        for s, n in enumerate(new):
            k, v = pool.values("k", s), pool.values("v", s)
            k[5] = v[5] = 0
            k[-1] = v[-1] = 0
            want, bound = scores_ref.attend(q[at : at + n].double(), k, v, lens[s] - n, 128**-0.5, True, 8, kw.get("softcap", 0.0),
                                            kw.get("slopes"), kw.get("prefix", [0, 0])[s], dtype=F16)
            within(y[at : at + n - 1], want[:-1], bound[:-1], f"{bad} sequence {s}")
            assert not bool(y[at + n - 1].isfinite().all())  # the row that does see it
            at += n


@pytest.mark.parametrize("bits, cdtype, dtype", FORMATS[:3])
def test_rows_that_see_nothing_and_rows_outside(bits, cdtype, dtype):
    for new in ([2, 3, 4], [50, 3, 60]):
        pool = Pool(37, [new[0] + 9, 0, 2], 2, 128, 16, bits, cdtype)
        cache = pool.cuda(mlxl3_amd)
        starts = torch.tensor([2, 2 + new[0], 2 + sum(new[:2]), 2 + sum(new)], dtype=torch.int32).cuda()
        lens = torch.tensor([new[0] + 9, 0, 2], dtype=torch.int32).cuda()
        b = mlxl3_amd.KvBatch(starts, lens, pool.table.cuda(), max_q=max(new))
        rows = 2 + sum(new) + 3
        q = torch.randn(rows, 4, 128, generator=torch.Generator().manual_seed(5)).to(dtype)
        out = torch.full((rows, 4, 128), 4.0, dtype=dtype, device="cuda")
        slopes = geometric(4)
        prefix = torch.tensor([0, 5, 0], dtype=torch.int32).cuda()
        y = mlxl3_amd.attention(q.cuda(), cache, b, out=out, softcap=20.0, slopes=slopes.float().cuda(), prefix=prefix)
        assert y is out and bool((y[:2] == 4.0).all()) and bool((y[-3:] == 4.0).all())
        inner = y[2:-3]
        check(pool, [new[0]], q[2 : 2 + new[0]], inner[: new[0]], softcap=20.0, slopes=slopes)
        assert bool((inner[new[0] : sum(new) - 2] == 0).all())
        want, bound = scores_ref.attend(q[-5:-3].double(), pool.values("k", 2), pool.values("v", 2), 0, 128**-0.5, True, 0, 20.0,
                                        slopes.float(), 0, coded=bits != 16, dtype=dtype)
        within(inner[-2:], want, bound, "short")


def test_one_call_like_another():
    """Equal bits in repeated calls, in place, into rows with gaps, on other streams, with a workspace."""
    pool = Pool(59, [3000, 17, 800], 2, 128, 32, 8, None)
    kw = dict(softcap=30.0, slopes=geometric(8), prefix=[50, 17, 3])
    for new in ([1, 1, 1], [40, 17, 2]):
        q, cache, b, y, shape = run(pool, new, 8, BF16, **kw)
        check(pool, new, q, y, **kw)
        call = lambda x, **more: mlxl3_amd.attention(x, cache, b, **shape, **more)
        assert torch.equal(call(q.cuda()), y)
        x = q.cuda()
        assert call(x, out=x) is x and torch.equal(x, y)
        wide = torch.full((sum(new), 10, 128), 7.0, dtype=BF16, device="cuda")
        call(q.cuda(), out=wide[:, 1:9])
        assert torch.equal(wide[:, 1:9], y) and bool((wide[:, 0] == 7.0).all()) and bool((wide[:, 9] == 7.0).all())
        need = mlxl3_amd.load_library().exl3_attention_workspace_bytes(cache.handle, b._ref, sum(new), 8)
        assert torch.equal(call(q.cuda(), workspace=torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")), y)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            z = call(q.cuda())
        s.synchronize()
        assert torch.equal(z, y)
        without = kv_ref.batch(mlxl3_amd, new, pool.lens, pool.table)
        told = mlxl3_amd.KvBatch(without.q_starts, without.kv_lens, without.block_table)
        check(pool, new, q, mlxl3_amd.attention(q.cuda(), cache, told, **shape), **kw)


@pytest.mark.parametrize("new", [1, 40])
def test_captured_graphs_follow_the_device_arrays(new):
    """Lengths, prefixes and slopes change between the replays."""
    lens = [3000, 90, 700]
    pool = Pool(74, lens, 8, 64, 64, 16, F16, table_pages=1600, poison=False)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, [new] * 3, lens, pool.table)
    q = torch.randn(3 * new, 16, 64, generator=torch.Generator().manual_seed(75)).half().cuda()
    slopes, prefix = torch.zeros(16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    call = lambda: mlxl3_amd.attention(q, cache, b, softcap=25.0, slopes=slopes, prefix=prefix)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = call()
    for i, now in enumerate(([3000, 90, 700], [2999, 40, 641], [1500, 60, 40], [40, 40, 699])):
        b.kv_lens.copy_(torch.tensor(now, dtype=torch.int32))
        slopes.copy_(geometric(16) * i)
        front = [100 * i, 10 * i, 5]
        prefix.copy_(torch.tensor(front, dtype=torch.int32))
        want = call()
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), now
        at = 0
        for s, length in enumerate(now):
            w, bound = scores_ref.attend(q[at : at + new].cpu().double(), pool.values("k", s)[:length], pool.values("v", s)[:length],
                                         length - new, 64**-0.5, True, 0, 25.0, slopes.cpu(), front[s], dtype=F16)
            within(y[at : at + new], w, bound, f"{now} sequence {s}")
            at += new


@pytest.mark.parametrize("new, lens", [([1, 1], [300, 40]), ([50, 3], [50, 700])])
def test_without_cap_and_bias_scores_are_plain_ones(new, lens):
    """Slopes of zero and a prefix within what rows see anyway: plain attention's result, to a rounding."""
    pool = Pool(81, lens, 2, 128, 16, 16, F16)
    q, cache, b, y, _ = run(pool, new, 8, F16, slopes=torch.zeros(8, dtype=torch.float64), prefix=[1, 0])
    plain = mlxl3_amd.attention(q.cuda(), cache, b)
    assert float((y.float() - plain.float()).abs().max()) <= 2.0**-9 * float(plain.float().abs().max())
    same = mlxl3_amd.attention(q.cuda(), cache, b, softcap=0.0, slopes=None, prefix=None)
    assert torch.equal(same, plain)


@pytest.mark.parametrize("dtype, bits", [(F16, 16), (BF16, 8)])
@pytest.mark.parametrize("new, old", [([1, 1, 1], [70, 0, 300]), ([3, 40], [9, 0])])
def test_attention_block_equals_its_calls(dtype, bits, new, old):
    hidden, rows, heads, kv_heads, dim = 512, sum(new), 8, 2, 64
    q, k, v, o = projections(3, hidden, heads, kv_heads, dim, 4, 0, False)
    lens = [n + m for n, m in zip(new, old)]
    pool = Pool(73, lens, kv_heads, dim, 16, bits, dtype, loud=1.0)
    b = kv_ref.batch(mlxl3_amd, new, lens, pool.table)
    rope = mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(dim)[0].cuda())
    slopes = geometric(heads).float().cuda()
    prefix = torch.tensor([7, 20, 4][: len(new)], dtype=torch.int32).cuda()
    x = (torch.randn(rows, hidden, generator=torch.Generator().manual_seed(1)) / 8).to(dtype).cuda()
    block = mlxl3_amd.Exl3Attention(q, k, v, o, rope=rope, window=100, softcap=5.0, slopes=slopes)
    one, two = pool.cuda(mlxl3_amd), pool.cuda(mlxl3_amd)
    for _ in range(2):
        y = block(x, one, b, prefix=prefix)
    qs, ks, vs = mlxl3_amd.Exl3Group([q, k, v])(x)
    qr = rope.apply(qs.view(rows, heads, dim), batch=b, dtype=dtype)
    two.append(b, ks.view(rows, kv_heads, dim), vs.view(rows, kv_heads, dim), rope=rope)
    a = mlxl3_amd.attention(qr, two, b, window=100, softcap=5.0, slopes=slopes, prefix=prefix)
    assert torch.equal(y, o(a.view(rows, heads * dim))) and bool(y.isfinite().all())
    pool.k, pool.v = two.k.cpu(), two.v.cpu()
    pool.ks, pool.vs = (None if t is None else t.cpu() for t in (two.k_scales, two.v_scales))
    check(pool, new, qr.cpu(), a, window=100, softcap=5.0, slopes=geometric(heads), prefix=prefix.tolist())


def test_python_refusals():
    pool = Pool(71, [20], 2, 128, 16, 16, F16)
    cache = pool.cuda(mlxl3_amd)
    b = kv_ref.batch(mlxl3_amd, [1], [20], pool.table)
    q = torch.zeros(1, 4, 128, dtype=F16, device="cuda")
    err = mlxl3_amd.Exl3Error
    for kw, msg in [
        (dict(softcap=-1.0), "softcap must be 0 or"),
        (dict(softcap=math.nan), "softcap must be 0 or"),
        (dict(softcap=math.inf), "softcap must be 0 or"),
        (dict(softcap=1e-30), "softcap must be 0 or"),
        (dict(softcap="x"), "softcap must be a number"),
        (dict(slopes=torch.zeros(3, device="cuda")), "3 slopes for 4 heads"),
        (dict(slopes=torch.zeros(4)), "slopes must be a device tensor"),
        (dict(slopes=torch.zeros(4, device="cuda", dtype=F16)), "slopes has dtype"),
        (dict(slopes=torch.zeros(8, device="cuda")[::2]), "slopes must be contiguous"),
        (dict(slopes=torch.zeros(2, 2, device="cuda")), "slopes must have 1 dimensions"),
        (dict(prefix=torch.zeros(2, device="cuda", dtype=torch.int32)), "2 prefixes for 1 sequences"),
        (dict(prefix=torch.zeros(1, device="cuda", dtype=torch.int64)), "prefix has dtype"),
        (dict(prefix=[3]), "prefix must be a device tensor"),
    ]:
        with pytest.raises(err, match=msg):
            mlxl3_amd.attention(q, cache, b, **kw)
    none = mlxl3_amd.attention(q[:0], cache, b, softcap=3.0)
    assert none.shape == (0, 4, 128)
