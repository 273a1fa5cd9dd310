"""Root-mean-square norms on the GPU against 64 bits, within what their roundings allow: widths
from one value to the largest, types, residuals, heads among other rows, outputs in place, rows
whose squares f32 does not hold, values that are not finite, streams and captured graphs."""

import math

import pytest
import torch

import mlxl3_amd
from kv_ref import EPS

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def reference(x, weight, eps, residual, dtype):
    """(y, bound) in 64 bits.  s is rounded once (2^-24); the sum of squares takes at most `depth`
    additions one after the other -- 8 in each of a thread's chunks, its chunks in rows that are read
    twice, ten of a tree, 16 of the parts -- with 2^-24 each, half of it in the root; the mean, eps, the
    reciprocal root (2^-23) and two products 2^-24 to 2^-23 each; the output half a step, f16's below the
    normal range 2^-25."""
    s = x.double() if residual is None else x.double() + residual.double()
    width = x.shape[-1]
    y = s / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    depth = 32 + width // 8192 + 26
    rel = EPS[dtype] / 2 + 2.0**-24 * (depth / 2 + 10)
    return y, y.abs() * rel + {F16: 2.0**-25, BF16: 2.0**-133, F32: 2.0**-149}[dtype]


def within(y, want, bound, label=""):
    off = (y.detach().cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"{label}: {float((off / bound).max()):.3g} of the bound"


def rows(seed, *shape, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    x[..., shape[-1] // 3] *= 30
    return x.to(dtype)


WIDTHS = [1, 2, 7, 8, 64, 80, 127, 128, 136, 200, 512, 513, 520, 1000, 2048, 2056, 4096, 4104, 5120, 5121, 8192, 10001, 14336,
          16384, 16392, 32768, 32776, 33001, 131072]


@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width):
    for n, dtype, rtype, wtype in ((1, F16, F16, F16), (5, BF16, F32, BF16), (3, F32, BF16, F32), (17, F16, None, F32),
                                   (2, F32, None, None), (4, F32, F32, F16), (6, BF16, BF16, None)):
        x = rows(width + n, n, width, dtype=dtype)
        r = None if rtype is None else rows(n, n, width, dtype=rtype)
        w = None if wtype is None else rows(99, width, dtype=wtype)
        dev = [None if t is None else t.cuda() for t in (x, r, w)]
        got = mlxl3_amd.rms_norm(dev[0], dev[2], residual=dev[1])
        y, total = got if r is not None else (got, None)
        assert y.dtype == dtype and y.shape == x.shape
        within(y, *reference(x, w, 1e-6, r, dtype), f"{n} x {width} {dtype}")
        if r is not None:
            assert total.dtype == rtype and torch.equal(total.cpu(), (x.float() + r.float()).to(rtype))
            assert torch.equal(dev[0].cpu(), x) and torch.equal(dev[1].cpu(), r)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens, heads, width, gap", [(1, 4, 128, 2), (33, 3, 64, 1), (70, 8, 256, 16), (5, 2, 100, 3), (4, 1, 4096, 1),
                                                       (3, 5, 13, 1), (2, 2, 40000, 1)])
def test_heads_among_others(dtype, tokens, heads, width, gap):
    wide = rows(tokens, tokens, heads + gap, width, dtype=dtype)
    x, w = wide[:, gap:], rows(1, width, dtype=dtype)
    dev = wide.cuda()
    y = mlxl3_amd.rms_norm(dev[:, gap:], w.cuda(), eps=1e-5)
    assert y.is_contiguous()
    within(y, *reference(x, w, 1e-5, None, dtype))
    # into other rows with gaps, and in place
    out = torch.full((tokens, heads + 1, width), 3.0, dtype=dtype, device="cuda")
    assert mlxl3_amd.rms_norm(dev[:, gap:], w.cuda(), eps=1e-5, out=out[:, :heads]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:, :heads], y) and bool((out[:, heads] == 3.0).all())
    assert torch.equal(dev.cpu(), wide)
    view = dev[:, gap:]
    mlxl3_amd.rms_norm(view, w.cuda(), eps=1e-5, out=view)
    assert torch.equal(view, y) and torch.equal(dev[:, :gap].cpu(), wide[:, :gap])


def test_rows_any_distance_apart_and_other_strides():
    for width, pad in ((512, 8), (512, 3), (77, 1), (20000, 24)):
        wide = rows(5, 9, width + pad, dtype=BF16).cuda()
        r = rows(6, 9, width + pad, dtype=F32).cuda()
        x, res = wide[:, pad:], r[:, :width]
        want, total = mlxl3_amd.rms_norm(x.contiguous(), residual=res.contiguous())
        y, t = mlxl3_amd.rms_norm(x, residual=res)
        assert torch.equal(y, want) and torch.equal(t, total)
        turned = x.t().contiguous().t()  # strides that are copied
        assert torch.equal(mlxl3_amd.rms_norm(turned, residual=res)[0], want)
        one = x[:1].expand(9, width)
        assert torch.equal(mlxl3_amd.rms_norm(one), mlxl3_amd.rms_norm(one.contiguous()))
        odd = torch.zeros(9 * width + 1, dtype=BF16, device="cuda")
        odd[1:] = x.reshape(-1)
        within(mlxl3_amd.rms_norm(odd[1:].view(9, width)), *reference(x.cpu(), None, 1e-6, None, BF16))
    deep = rows(7, 2, 3, 5, 64, dtype=F16)
    within(mlxl3_amd.rms_norm(deep.cuda()), *reference(deep, None, 1e-6, None, F16))
    flat = rows(8, 64, dtype=F16)
    within(mlxl3_amd.rms_norm(flat.cuda()), *reference(flat, None, 1e-6, None, F16))


@pytest.mark.parametrize("width", [64, 512, 4096, 5001, 20000, 40000])
def test_in_place(width):
    x, r, w = (rows(i, 6, width, dtype=F16) for i in range(3))
    w = w[0]
    y, total = mlxl3_amd.rms_norm(x.cuda(), w.cuda(), residual=r.cuda())
    for put in ("xr", "rx", "x", "r"):
        a, b = x.cuda(), r.cuda()
        kw = dict(xr=dict(out=a, total=b), rx=dict(out=b, total=a), x=dict(out=a), r=dict(total=b))[put]
        got, sums = mlxl3_amd.rms_norm(a, w.cuda(), residual=b, **kw)
        assert torch.equal(got, y) and torch.equal(sums, total), put
        assert all(t is kw[n] for n, t in (("out", got), ("total", sums)) if n in kw)


def test_output_types():
    x = rows(3, 7, 1024, dtype=F32)
    for dtype in (F16, BF16, F32):
        y = mlxl3_amd.rms_norm(x.cuda(), dtype=dtype)
        assert y.dtype == dtype
        within(y, *reference(x, None, 1e-6, None, dtype))
        out = torch.empty(7, 1024, dtype=dtype, device="cuda")
        assert torch.equal(mlxl3_amd.rms_norm(x.cuda(), out=out), y)


@pytest.mark.parametrize("width", [100, 128, 512, 2048, 8192, 16384, 40000])
def test_large_small_and_zero_rows(width):
    """Rows whose squares f32 does not hold, rows far below eps, rows of zeros."""
    for dtype in (BF16, F32):
        x = rows(11, 6, width, dtype=F32) / 30
        x[1] *= 1e30
        x[2] *= 1e-25
        x[3] = 0
        x[4] *= 3e36
        x = x.to(dtype)
        y = mlxl3_amd.rms_norm(x.cuda())
        within(y, *reference(x, None, 1e-6, None, dtype), f"{dtype}")
        assert bool((y[3] == 0).all()) and bool(y.isfinite().all())
    most = torch.full((2, width), 3.4e38)
    within(mlxl3_amd.rms_norm(most.cuda()), *reference(most, None, 1e-6, None, F32))
    x = torch.full((3, width), 65504.0, dtype=F16)
    r = torch.full((3, width), 65504.0, dtype=F16)
    y, total = mlxl3_amd.rms_norm(x.cuda(), residual=r.cuda())  # the sum is beyond f16, its norm is not
    assert bool(total.isinf().all()) and bool((y == 1.0).all())
    tiny = mlxl3_amd.rms_norm(torch.full((1, width), 1e-18, device="cuda"), eps=2.0**-126)
    within(tiny, *reference(torch.full((1, width), 1e-18), None, 2.0**-126, None, F32))


@pytest.mark.parametrize("width", [64, 300, 4096, 40000])
def test_values_that_are_not_finite_stay_in_their_row(width):
    x = rows(12, 40, width, dtype=F16)
    good = mlxl3_amd.rms_norm(x.cuda())
    x[7, width // 2], x[20, 0], x[33, width - 1] = math.nan, math.inf, -math.inf
    y = mlxl3_amd.rms_norm(x.cuda()).cpu()
    keep = torch.ones(40, dtype=torch.bool)
    keep[[7, 20, 33]] = False
    assert torch.equal(y[keep], good.cpu()[keep])
    assert bool(y[7].isnan().all())
    for row, at in ((20, 0), (33, width - 1)):
        assert bool(y[row, at].isnan()) and int((y[row] != 0).sum()) == 1


def test_many_rows_and_rows_of_no_tokens():
    x = torch.randn(200001, 64, generator=torch.Generator().manual_seed(1)).half()
    within(mlxl3_amd.rms_norm(x.cuda()), *reference(x, None, 1e-6, None, F16))
    for shape in ((0, 64), (3, 0, 8), (0, 2, 128)):
        empty = torch.empty(shape, dtype=F16, device="cuda")
        assert mlxl3_amd.rms_norm(empty).shape == shape
        y, t = mlxl3_amd.rms_norm(empty, residual=empty.float())
        assert y.shape == shape and t.shape == shape and t.dtype == F32


def test_other_streams_and_captured_graphs():
    x, w, r = rows(1, 33, 4096, dtype=F16).cuda(), rows(2, 4096, dtype=F16).cuda(), rows(3, 33, 4096, dtype=F32).cuda()
    y, total = mlxl3_amd.rms_norm(x, w, residual=r)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            outs += [mlxl3_amd.rms_norm(x, w, residual=r) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, y) and torch.equal(b, total) for a, b in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, sums = mlxl3_amd.rms_norm(x, w, residual=r)
    for i in range(4):
        x.copy_(rows(10 + i, 33, 4096, dtype=F16))
        want = mlxl3_amd.rms_norm(x, w, residual=r)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[0]) and torch.equal(sums, want[1])


def test_refusals():
    x = torch.zeros(4, 64, dtype=F16, device="cuda")
    err = mlxl3_amd.Exl3Error
    for kw, msg in [
        (dict(weight=torch.zeros(63, device="cuda")), "weight must have shape"),
        (dict(weight=torch.zeros(64)), "weight must be a device tensor"),
        (dict(weight=torch.zeros(64, device="cuda", dtype=torch.int32)), "weight has dtype"),
        (dict(residual=x[:3]), "residual must have shape"),
        (dict(residual=x.double()), "residual has dtype"),
        (dict(total=x), "a sum needs a residual"),
        (dict(residual=x, total=x.float()), "total must have shape"),
        (dict(residual=x, total=torch.zeros(64, 4, dtype=F16, device="cuda").t()), "total must have contiguous rows"),
        (dict(out=x[:3]), "out must have shape"),
        (dict(out=x.float(), dtype=F16), "out must have shape"),
        (dict(out=torch.zeros(64, 4, dtype=F16, device="cuda").t()), "out must have contiguous rows"),
        (dict(out=torch.zeros(64, dtype=F16, device="cuda").expand(4, 64)), "out must have contiguous rows"),
        (dict(dtype=torch.int8), "unsupported norm output dtype"),
        (dict(eps=0.0), "eps must be"),
        (dict(eps="a"), "eps must be a number"),
    ]:
        with pytest.raises(err, match=msg):
            mlxl3_amd.rms_norm(x, **kw)
    for bad, msg in ((x.long(), "x has dtype"), (x[0, 0], "at least one value"), (x[:, :0], "at least one value")):
        with pytest.raises(err, match=msg):
            mlxl3_amd.rms_norm(bad)
    with pytest.raises(err, match="two outputs"):
        mlxl3_amd.rms_norm(x, residual=x.clone(), out=(o := x.clone()), total=o)


def test_sizes_past_32_bits_are_refused():
    """Not cut to 32 bits: 2^32 + 128 values are no rows of 128, 2^32 + 1 heads not one."""
    for make, msg in (
        (lambda: torch.empty(1, 2**32 + 128, dtype=F16, device="cuda"), "fewer than 2\\^31, got shape"),
        (lambda: torch.empty(2, 2**32 + 2, 1, dtype=F16, device="cuda")[:, 1:], "fewer than 2\\^31 heads"),
    ):
        x = make()
        with pytest.raises(mlxl3_amd.Exl3Error, match=msg):
            mlxl3_amd.rms_norm(x, out=x)  # in place: x stays the only one of its size
        del x
        torch.cuda.empty_cache()
