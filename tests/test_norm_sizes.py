"""Sizes at the end of 64 bits that exl3_rms_norm refuses before any launch (no GPU needed: launches are
armed to fail)."""

import pytest

import mlxl3_amd
from test_norm_api import norm

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")
MOST = 2**63 - 1


@pytest.fixture(autouse=True)
def armed():
    lib = mlxl3_amd.load_library()
    lib.exl3_debug_fail_launch(b"RMS norm")
    yield
    lib.exl3_debug_fail_launch(None)


@pytest.mark.parametrize("heads, width", [(1, 1), (1, 64), (1, 65), (1, 128), (1, 256), (1, 512), (3, 1), (2, 100), (65536, 1), (1, 1 << 17)])
def test_tokens_up_to_64_bits_are_refused(heads, width):
    need = heads * width
    for n in {MOST // need, MOST // need - 1, MOST // need - 14, MOST // need - 30, MOST // need // 2, MOST, MOST - 31}:
        assert norm(n=n, heads=heads, width=width, xs=1 << 40, ys=1 << 40)[0] == -4, n


def test_the_largest_call_is_launched():
    per = {64: 32, 128: 16, 256: 8, 512: 4, 513: 1}
    for width, rows in per.items():
        first = next(e for e in range(1, 64) if norm(n=rows << e, width=width, xs=1 << 20, ys=1 << 20)[0] == -4)
        low, high = rows << (first - 1), rows << first
        while high - low > 1:
            mid = (low + high) // 2
            low, high = (low, mid) if norm(n=mid, width=width, xs=1 << 20, ys=1 << 20)[0] == -4 else (mid, high)
        assert norm(n=low, width=width, xs=1 << 20, ys=1 << 20) == (-2, "RMS norm: forced launch failure")
        assert low % rows == 0 and low // rows < 2**31
