"""exl3_rms_norm and rms_norm: what is refused before any launch (no GPU needed)."""

import math

import pytest
import torch

import mlxl3_amd

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")
FAKE = 0x1000  # never dereferenced


def norm(**kw):
    a = dict(x=FAKE, xt=9, n=5, heads=1, width=512, xs=512, w=None, wt=0, eps=1e-6, r=None, rt=0, rs=0, total=None, ts=0, y=2 * FAKE,
             yt=9, ys=512)
    a.update(kw)
    lib = mlxl3_amd.load_library()
    rc = lib.exl3_rms_norm(a["x"], a["xt"], a["n"], a["heads"], a["width"], a["xs"], a["w"], a["wt"], a["eps"], a["r"], a["rt"], a["rs"],
                           a["total"], a["ts"], a["y"], a["yt"], a["ys"], None)
    return rc, lib.exl3_last_error().decode()


WITH = dict(r=3 * FAKE, rt=9, rs=512, total=4 * FAKE, ts=512)


@pytest.mark.parametrize("kw, rc, msg", [
    (dict(n=-1), -1, "negative token count"),
    (dict(xt=8), -1, "unsupported norm dtypes 8 and 9"),
    (dict(yt=0), -1, "unsupported norm dtypes 9 and 0"),
    (dict(w=FAKE, wt=7), -1, "unsupported norm weight dtype 7"),
    (dict(r=FAKE, rt=7), -1, "unsupported residual dtype 7"),
    (dict(heads=0), -1, "invalid norm heads: 0"),
    (dict(heads=65537), -1, "invalid norm heads"),
    (dict(width=0), -4, "rows of 1 to 131072 values, got 0"),
    (dict(width=131073, xs=1 << 20, ys=1 << 20), -4, "got 131073"),
    (dict(eps=0.0), -1, "eps must be a positive normal number"),
    (dict(eps=-1e-6), -1, "eps must be a positive normal number"),
    (dict(eps=1e-40), -1, "eps must be a positive normal number"),
    (dict(eps=math.inf), -1, "eps must be a positive normal number"),
    (dict(eps=math.nan), -1, "eps must be a positive normal number"),
    (dict(total=FAKE * 3, ts=512), -1, "a sum needs a residual"),
    (dict(xs=511), -1, "token strides are at least"),
    (dict(ys=0), -1, "token strides are at least"),
    (dict(heads=2), -1, "token strides are at least"),
    (dict(WITH, rs=511), -1, "token strides are at least"),
    (dict(WITH, ts=511), -1, "token strides are at least"),
    (dict(x=None), -1, "null norm input or output"),
    (dict(y=None), -1, "null norm input or output"),
    (dict(WITH, total=2 * FAKE), -1, "two outputs"),
    (dict(y=FAKE, yt=12), -1, "in place keeps the type and the stride"),
    (dict(y=FAKE, ys=1024), -1, "in place keeps the type and the stride"),
    (dict(WITH, y=3 * FAKE, ys=1024), -1, "in place keeps the type and the stride"),
    (dict(WITH, total=3 * FAKE, ts=513), -1, "in place keeps the type and the stride"),
    (dict(WITH, rt=10, total=FAKE), -1, "in place keeps the type and the stride"),
    (dict(n=1 << 40), -4, "too many tokens"),
    (dict(n=1 << 62, xs=1 << 20, ys=1 << 20), -4, "too many tokens"),
])
def test_refusals(kw, rc, msg):
    got, err = norm(**kw)
    assert got == rc and msg in err


def test_no_rows_need_no_memory():
    assert norm(n=0, x=None, y=None)[0] == 0
    assert norm(n=0, x=None, y=None, **dict(WITH, r=None, total=None))[0] == 0


def test_an_armed_launch_fails_before_anything_is_issued():
    lib = mlxl3_amd.load_library()
    lib.exl3_debug_fail_launch(b"RMS norm")
    try:
        assert norm() == (-2, "RMS norm: forced launch failure")
    finally:
        lib.exl3_debug_fail_launch(None)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(mlxl3_amd.Exl3Error, match="x must be a device tensor"):
        mlxl3_amd.rms_norm(x)
    with pytest.raises(mlxl3_amd.Exl3Error, match="x must be a device tensor"):
        mlxl3_amd.rms_norm([1.0, 2.0])
