"""What the attention block refuses before its first launch, so that no projection has run and no
page was written: host-only handles, no GPU needed."""

import ctypes

import pytest

import mlxl3_amd
from test_attention_api import FAKE, batch, cache, ref, rope

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")


@pytest.mark.parametrize("what, msg", [
    # attention's grid: 65535 sequences, nearly all without new tokens, of 512 cache heads
    (dict(kv_heads=512, hidden=512, out=512, seqs=65535, rows=5), "too many workgroups"),
    (dict(kv_heads=512, hidden=512, out=512, seqs=65535, rows=20), "too many workgroups"),
    (dict(kv_heads=2, hidden=512, out=512, seqs=65536, rows=5), "up to 65535 sequences"),
    # the o projection's rows x outputs
    (dict(kv_heads=2, hidden=512, out=1 << 21, seqs=2, rows=1024), "input too large: 1024 rows"),
])
def test_sizes_are_refused_before_the_first_launch(what, msg):
    lib = mlxl3_amd.load_library()
    dim, made = 64, []
    rc, h, _ = cache(heads=what["kv_heads"], dim=dim)
    assert rc == 0

    def linear(n_in, n_out):
        p = ctypes.c_void_p()
        assert lib.exl3_linear_create(FAKE, n_in, n_out, 4, 0, FAKE, FAKE, None, ctypes.byref(p)) == 0
        made.append(p)
        return p

    width = what["kv_heads"] * dim
    q, k, v = (linear(what["hidden"], width) for _ in range(3))
    o = linear(width, what["out"])
    launch = b"EXL3 QMV launch" if what["rows"] <= 16 else b"EXL3 QMM launch"
    lib.exl3_debug_fail_launch(launch)  # the first one: nothing is issued either way
    try:
        rc = lib.exl3_attn_block_forward(q, k, v, o, h, ref(batch(seqs=what["seqs"])), ref(rope()), 0.1, 0, FAKE, 9,
                                         what["rows"], FAKE, FAKE, 1 << 40, None)
        err = lib.exl3_last_error().decode()
        assert msg in err and rc in (-1, -4)
    finally:
        lib.exl3_debug_fail_launch(None)
        for p in made:
            lib.exl3_linear_destroy(p)
        lib.exl3_kv_cache_destroy(h)
