"""exl3_attention_scores and exl3_attn_block_forward_scores: what is refused before any launch (no GPU
needed)."""

import ctypes
import math

import pytest

import mlxl3_amd
from mlxl3_amd import kv
from test_attention_api import FAKE, batch, calls, ref

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")


def attend(h, scores, b=None, n=5, ws=1 << 30, window=0):
    lib = mlxl3_amd.load_library()
    rc = lib.exl3_attention_scores(h, ref(b or batch()), FAKE, 9, n, 4, 512, 0.1, 1, window, ref(scores), FAKE, 512, FAKE, ws, None)
    return rc, lib.exl3_last_error().decode()


@pytest.mark.parametrize("cap", [-1.0, math.nan, math.inf, -math.inf, 2.0**-65, 2.0**65])
def test_caps_out_of_range(cap):
    lib, h = calls()
    try:
        rc, err = attend(h, kv._ScoresC(cap, None, None))
        assert rc == -1 and "softcap must be 0 or 2^-64 to 2^64" in err
        assert attend(h, kv._ScoresC(cap, FAKE, FAKE), n=0)[0] == -1
    finally:
        lib.exl3_kv_cache_destroy(h)


@pytest.mark.parametrize("scores", [None, kv._ScoresC(0.0, None, None), kv._ScoresC(30.0, FAKE, FAKE)])
def test_what_plain_attention_refuses(scores):
    lib, h = calls()
    try:
        assert attend(h, scores, n=-1) == (-1, "negative token count")
        assert attend(h, scores, window=-1)[0] == -1
        assert attend(h, scores, b=batch(max_q=0)) == (-1, "max_q must be positive")
        assert attend(h, scores, n=0)[0] == 0
        assert attend(None, scores) == (-1, "null KV cache")
        long = batch(seqs=1, table_pages=4096, max_q=1)
        need = lib.exl3_attention_workspace_bytes(h, ref(long), 1, 4)
        assert need > 0
        rc, err = attend(h, scores, b=long, n=1, ws=need - 1, window=10)
        assert rc == -1 and "workspace too small" in err
        lib.exl3_debug_fail_launch(b"attention")
        assert attend(h, scores) == (-2, "attention: forced launch failure")
    finally:
        lib.exl3_debug_fail_launch(None)
        lib.exl3_kv_cache_destroy(h)


def test_the_block_refuses_before_its_first_launch():
    lib, h = calls()
    made = []

    def linear(n_in, n_out):
        p = ctypes.c_void_p()
        assert lib.exl3_linear_create(FAKE, n_in, n_out, 4, 0, FAKE, FAKE, None, ctypes.byref(p)) == 0
        made.append(p)
        return p

    parts = [linear(512, 512), linear(512, 256), linear(512, 256), linear(512, 512)]
    try:
        rc = lib.exl3_attn_block_forward_scores(*parts, h, ref(batch()), None, 0.1, 0, ref(kv._ScoresC(-2.0, None, None)), FAKE, 9, 5, FAKE,
                                                FAKE, 1 << 40, None)
        assert rc == -1 and "softcap must be 0 or" in lib.exl3_last_error().decode()
    finally:
        for p in made:
            lib.exl3_linear_destroy(p)
        lib.exl3_kv_cache_destroy(h)


@pytest.mark.parametrize("cap", [1e-60, -1e-60, 5e-324])
def test_a_cap_that_f32_does_not_hold_is_no_call_without_one(cap):
    with pytest.raises(mlxl3_amd.Exl3Error, match="softcap must be 0 or 2\\^-64 to 2\\^64"):
        kv._scores(None, 4, 1, cap, None, None)
