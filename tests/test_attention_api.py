"""Rotary positions, the paged cache and attention: what the entry points refuse before
any launch, with host-only handles (no GPU needed), and the rotary frequencies."""

import ctypes
import math

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import kv

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")
FAKE = 0x1000  # never dereferenced


def cache(fmt=9, pages=8, page=16, heads=2, dim=128, k=FAKE, v=FAKE, ks="auto", vs="auto"):
    lib = mlxl3_amd.load_library()
    coded = fmt in (4, 8)
    ks = (FAKE if coded else None) if ks == "auto" else ks
    vs = (FAKE if coded else None) if vs == "auto" else vs
    h = ctypes.c_void_p()
    rc = lib.exl3_kv_cache_create(k, v, ks, vs, fmt, pages, page, heads, dim, ctypes.byref(h))
    return rc, h, lib.exl3_last_error().decode()


@pytest.mark.parametrize("kwargs, rc, msg", [
    (dict(fmt=10), -1, "unknown KV cache format 10"),
    (dict(page=8), -1, "a power of two of 16 to 1024 tokens, got 8"),
    (dict(page=48), -1, "a power of two of 16 to 1024 tokens, got 48"),
    (dict(page=2048), -1, "got 2048"),
    (dict(dim=96), -4, "64, 128 or 256 channels are supported, got 96"),
    (dict(heads=0), -1, "invalid KV head count 0"),
    (dict(pages=0), -1, "invalid KV page count 0"),
    (dict(pages=1 << 31), -1, "invalid KV page count"),
    (dict(k=None), -1, "null KV cache buffer"),
    (dict(fmt=8, vs=None), -1, "null KV cache buffer"),
    (dict(ks=FAKE), -1, "16-bit KV caches have no scales"),
    (dict(v=FAKE + 8), -1, "16-byte aligned"),
])
def test_cache_refusals(kwargs, rc, msg):
    got, h, err = cache(**kwargs)
    assert got == rc and not h.value and msg in err


def batch(**kw):
    a = dict(q_starts=FAKE, kv_lens=FAKE, block_table=FAKE, seqs=2, table_pages=4, max_q=3, max_kv=0)
    a.update(kw)
    return kv._KvBatchC(*(a[n] for n, _ in kv._KvBatchC._fields_))


def rope(**kw):
    a = dict(inv_freq=FAKE, rotary_dim=64, interleaved=0, scale=1.0)
    a.update(kw)
    return kv._RopeC(*(a[n] for n, _ in kv._RopeC._fields_))


def ref(c):
    return None if c is None else ctypes.byref(c)


BAD_BATCHES = [
    (dict(seqs=0), "at least one sequence"),
    (dict(q_starts=None), "null KV batch lengths"),
    (dict(kv_lens=None), "null KV batch lengths"),
    (dict(block_table=None), "needs a block table"),
    (dict(table_pages=0), "needs a block table"),
]


def calls():
    lib = mlxl3_amd.load_library()
    _, h, _ = cache()
    return lib, h


@pytest.mark.parametrize("kw, msg", BAD_BATCHES)
def test_bad_batches_are_refused_everywhere(kw, msg):
    lib, h = calls()
    b = ref(batch(**kw))
    try:
        for rc in (lib.exl3_kv_append(h, b, FAKE, 256, FAKE, 256, 9, 5, None, None),
                   lib.exl3_kv_read(h, b, FAKE, FAKE, 9, 5, None),
                   lib.exl3_attention(h, b, FAKE, 9, 5, 4, 512, 0.1, 1, 0, FAKE, 512, FAKE, 1 << 30, None)):
            assert rc == -1 and msg in lib.exl3_last_error().decode()
    finally:
        lib.exl3_kv_cache_destroy(h)


def append(h, b=None, k=FAKE, ks=256, v=FAKE, vs=256, t=9, n=5, r=None):
    lib = mlxl3_amd.load_library()
    return lib.exl3_kv_append(h, ref(b or batch()), k, ks, v, vs, t, n, ref(r), None), lib.exl3_last_error().decode()


@pytest.mark.parametrize("kw, msg", [
    (dict(k=None), "null KV input"),
    (dict(v=None), "null KV input"),
    (dict(t=7), "unsupported KV input dtype 7"),
    (dict(n=-1), "negative token count"),
    (dict(ks=255), "token strides are at least"),
    (dict(vs=0), "token strides are at least"),
    (dict(r=dict(inv_freq=None)), "null rotary frequencies"),
    (dict(r=dict(rotary_dim=130)), "rotary dimension 130"),
    (dict(r=dict(rotary_dim=7)), "rotary dimension 7"),
    (dict(r=dict(scale=math.inf)), "rotary scale must be finite"),
])
def test_append_refusals(kw, msg):
    lib, h = calls()
    if "r" in kw:
        kw = dict(kw, r=rope(**kw["r"]))
    try:
        rc, err = append(h, **kw)
        assert rc == -1 and msg in err
        assert append(h, n=0)[0] == 0  # nothing to write
        assert lib.exl3_kv_append(None, ref(batch()), FAKE, 256, FAKE, 256, 9, 5, None, None) == -1
        assert lib.exl3_kv_append(h, None, FAKE, 256, FAKE, 256, 9, 5, None, None) == -1
    finally:
        lib.exl3_kv_cache_destroy(h)


def test_read_refusals():
    lib, h = calls()
    b = ref(batch())
    try:
        assert lib.exl3_kv_read(None, b, FAKE, FAKE, 9, 5, None) == -1
        assert lib.exl3_kv_read(h, None, FAKE, FAKE, 9, 5, None) == -1
        assert lib.exl3_kv_read(h, b, FAKE, FAKE, 8, 5, None) == -1
        assert lib.exl3_kv_read(h, b, None, FAKE, 9, 5, None) == -1
        assert lib.exl3_kv_read(h, b, FAKE, FAKE + 2, 9, 5, None) == -1
        assert "16-byte aligned" in lib.exl3_last_error().decode()
        assert lib.exl3_kv_read(h, b, FAKE, FAKE, 9, -1, None) == -1
        assert lib.exl3_kv_read(h, b, None, None, 9, 0, None) == 0
    finally:
        lib.exl3_kv_cache_destroy(h)


@pytest.mark.parametrize("kw, msg", [
    (dict(q=None), "null attention input"),
    (dict(y=None), "null attention input or output"),
    (dict(t=10), "f16 or bf16 queries, got dtype 10"),
    (dict(t=12), "queries of a 16-bit KV cache have its type"),
    (dict(heads=3), "3 query heads over 2 KV heads"),
    (dict(heads=0), "0 query heads"),
    (dict(scale=0.0), "positive and finite"),
    (dict(scale=-0.1), "positive and finite"),
    (dict(scale=math.nan), "positive and finite"),
    (dict(scale=math.inf), "positive and finite"),
    (dict(scale=3e38), "positive and finite"),  # times log2(e) it is infinite
    (dict(window=-1), "negative attention window"),
    (dict(qs=511), "token strides are at least"),
    (dict(ys=1), "token strides are at least"),
    (dict(n=-2), "negative token count"),
    (dict(b=dict(max_q=0)), "max_q must be positive"),
])
def test_attention_refusals(kw, msg):
    lib, h = calls()
    a = dict(b={}, q=FAKE, t=9, n=5, heads=4, qs=512, scale=0.1, window=0, y=FAKE, ys=512)
    a.update(kw)
    run = lambda a: lib.exl3_attention(h, ref(batch(**a["b"])), a["q"], a["t"], a["n"], a["heads"], a["qs"], a["scale"],
                                       1, a["window"], a["y"], a["ys"], FAKE, 1 << 30, None)
    try:
        assert run(a) == -1 and msg in lib.exl3_last_error().decode()
        assert run(dict(a, **dict(b={}, q=None, y=None, t=9, n=0, heads=4, qs=512, ys=512, scale=0.1, window=0))) == 0
        need = lib.exl3_attention_workspace_bytes(h, ref(batch(max_kv=64)), 5, 4)
        if need:
            rc = lib.exl3_attention(h, ref(batch(max_kv=64)), FAKE, 9, 5, 4, 512, 0.1, 1, 0, FAKE, 512, FAKE, need - 1, None)
            assert rc == -1 and "workspace too small" in lib.exl3_last_error().decode()
    finally:
        lib.exl3_kv_cache_destroy(h)


@pytest.mark.parametrize("kw, msg", [
    (dict(x=None), "null rotary input or output"),
    (dict(xt=7), "unsupported rotary dtypes"),
    (dict(yt=0), "unsupported rotary dtypes"),
    (dict(n=-1), "negative token count"),
    (dict(heads=0), "invalid rotary heads"),
    (dict(dim=512), "invalid rotary heads"),
    (dict(xs=511), "token strides are at least"),
    (dict(pos=None), "from an array or from a KV batch"),
    (dict(b=batch()), "from an array or from a KV batch"),
    (dict(r=rope(rotary_dim=0)), "rotary dimension 0"),
    (dict(r=rope(scale=math.nan)), "rotary scale must be finite"),
    (dict(y=FAKE, yt=12), "in place keeps the type"),
    (dict(y=FAKE, ys=1024), "in place keeps the type and the stride"),
])
def test_rope_refusals(kw, msg):
    lib = mlxl3_amd.load_library()
    a = dict(r=rope(), x=FAKE, xt=9, n=5, heads=4, dim=128, xs=512, pos=FAKE, b=None, y=2 * FAKE, yt=9, ys=512)
    a.update(kw)
    rc = lib.exl3_rope(ref(a["r"]), a["x"], a["xt"], a["n"], a["heads"], a["dim"], a["xs"], a["pos"], ref(a["b"]), a["y"],
                       a["yt"], a["ys"], None)
    assert rc == -1 and msg in lib.exl3_last_error().decode()
    assert lib.exl3_rope(None, FAKE, 9, 5, 4, 128, 512, FAKE, None, FAKE, 9, 512, None) == -1


@pytest.mark.parametrize("name, call", [
    ("KV append", lambda lib, h, b: lib.exl3_kv_append(h, b, FAKE, 256, FAKE, 256, 9, 5, None, None)),
    ("KV read", lambda lib, h, b: lib.exl3_kv_read(h, b, FAKE, FAKE, 9, 5, None)),
    ("rotary launch", lambda lib, h, b: lib.exl3_rope(ref(rope()), FAKE, 9, 5, 4, 128, 512, FAKE, None, FAKE, 9, 512, None)),
    ("attention", lambda lib, h, b: lib.exl3_attention(h, b, FAKE, 9, 5, 4, 512, 0.1, 1, 0, FAKE, 512, FAKE, 1 << 30, None)),
])
def test_armed_launches_fail_before_anything_is_issued(name, call):
    lib, h = calls()
    lib.exl3_debug_fail_launch(name.encode())
    try:
        assert call(lib, h, ref(batch())) == -2
        assert f"{name}: forced launch failure" in lib.exl3_last_error().decode()
    finally:
        lib.exl3_debug_fail_launch(None)
        lib.exl3_kv_cache_destroy(h)


def block(**kw):
    """exl3_attn_block_forward with host-only handles; nothing is launched."""
    lib, h = calls()
    made = []

    def linear(n_in, n_out, k=4, bias=None):
        p = ctypes.c_void_p()
        assert lib.exl3_linear_create(FAKE, n_in, n_out, k, 0, FAKE, FAKE, bias, ctypes.byref(p)) == 0
        made.append(p)
        return p

    a = dict(q=(512, 512), k=(512, 256), v=(512, 256), o=(512, 512), kk=4, bias=(None, None, None), r=rope(), scale=0.1,
             window=0, x=FAKE, t=9, rows=5, y=FAKE, ws=FAKE, bytes=1 << 40, b={})
    a.update(kw)
    q, k, v = (linear(*a[n], k=a["kk"] if n == "k" else 4, bias=b) for n, b in zip("qkv", a["bias"]))
    o = linear(*a["o"])
    try:
        b = ref(batch(**a["b"]))
        need = lib.exl3_attn_block_workspace_bytes(q, k, v, o, h, b, a["t"], a["rows"])
        rc = lib.exl3_attn_block_forward(q, k, v, o, h, b, ref(a["r"]), a["scale"], a["window"], a["x"], a["t"], a["rows"],
                                         a["y"], a["ws"], min(a["bytes"], max(need, 1) - 1) if a["bytes"] < 0 else a["bytes"],
                                         None)
        return rc, lib.exl3_last_error().decode(), need
    finally:
        for p in made:
            lib.exl3_linear_destroy(p)
        lib.exl3_kv_cache_destroy(h)


@pytest.mark.parametrize("kw, rc, msg", [
    (dict(k=(512, 384)), -1, "widths differ from the cache's heads"),
    (dict(v=(512, 512)), -1, "widths differ from the cache's heads"),
    (dict(q=(512, 384), o=(384, 512)), -1, "widths differ from the cache's heads"),
    (dict(o=(256, 512)), -1, "widths differ from the cache's heads"),
    (dict(kk=3), -1, "incompatible grouped projections"),
    (dict(t=10), -1, "f16 or bf16 activations, got dtype 10"),
    (dict(t=12), -1, "queries of a 16-bit KV cache have its type"),
    (dict(rows=0), -1, "empty attention block input"),
    (dict(x=None), -1, "null attention block input or output"),
    (dict(y=None), -1, "null attention block input or output"),
    (dict(ws=None), -1, "workspace too small"),
    (dict(bytes=64), -1, "workspace too small"),
    (dict(ws=FAKE + 8), -1, "16-byte aligned"),
    (dict(scale=0.0), -1, "positive and finite"),
    (dict(window=-4), -1, "negative attention window"),
    (dict(r=rope(rotary_dim=256)), -1, "rotary dimension 256"),
    (dict(b=dict(block_table=None)), -1, "needs a block table"),
    (dict(b=dict(max_q=0)), -1, "max_q must be positive"),
    (dict(t=12, bias=(None, FAKE, None)), -4, "both biased or neither"),
    (dict(t=12, bias=(FAKE, FAKE, FAKE), r=None), -4, "need a rotation"),
])
def test_attention_block_refusals(kw, rc, msg):
    got, err, _ = block(**kw)
    assert got == rc and msg in err


def test_attention_block_fails_before_anything_is_issued():
    lib = mlxl3_amd.load_library()
    lib.exl3_debug_fail_launch(b"EXL3 QMV launch")
    try:
        rc, err, need = block()
        assert rc == -2 and "forced launch failure" in err and need > 65536
    finally:
        lib.exl3_debug_fail_launch(None)


def test_python_refuses_host_tensors():
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(mlxl3_amd.Exl3Error, match="q_starts must be a device tensor"):
        mlxl3_amd.KvBatch(i, i[:2], i.view(1, 3))
    with pytest.raises(mlxl3_amd.Exl3Error, match="inv_freq must be a device tensor"):
        mlxl3_amd.Rope(torch.ones(4))
    with pytest.raises(mlxl3_amd.Exl3Error, match="16, 8 or 4 bits"):
        mlxl3_amd.KvCache(torch.zeros(1), torch.zeros(1), bits=5)
    with pytest.raises(mlxl3_amd.Exl3Error, match="k must be a device tensor"):
        mlxl3_amd.KvCache(torch.zeros(1, 1, 16, 64).half(), torch.zeros(1, 1, 16, 64).half())


def test_calls_larger_than_a_launch_are_refused():
    lib, h = calls()
    rc, wide, _ = cache(heads=1024)
    assert rc == 0
    try:
        b = ref(batch())
        assert lib.exl3_kv_append(h, b, FAKE, 256, FAKE, 256, 9, 1 << 29, None, None) == -4
        assert lib.exl3_kv_read(h, b, FAKE, FAKE, 9, 1 << 29, None) == -4
        assert lib.exl3_rope(ref(rope(rotary_dim=256)), FAKE + 2, 9, 1 << 25, 1, 256, 256, FAKE, None, FAKE, 9, 256, None) == -4
        assert lib.exl3_attention(h, b, FAKE, 9, 1 << 31, 4, 512, 0.1, 1, 0, FAKE, 512, FAKE, 1 << 40, None) == -4
        assert "too many tokens" in lib.exl3_last_error().decode()
        b = ref(batch(seqs=65535, max_q=200))
        assert lib.exl3_attention(wide, b, FAKE, 9, 65535 * 200, 1024, 1 << 17, 0.1, 1, 0, FAKE, 1 << 17, FAKE, 1 << 40, None) == -4
        assert "too many workgroups" in lib.exl3_last_error().decode()
        b = ref(batch(seqs=65536))
        assert lib.exl3_attention(h, b, FAKE, 9, 65536, 4, 512, 0.1, 1, 0, FAKE, 512, FAKE, 1 << 40, None) == -4
    finally:
        lib.exl3_kv_cache_destroy(h)
        lib.exl3_kv_cache_destroy(wide)


@pytest.mark.parametrize("window", [-1, 2**31, 2**32])
def test_windows_of_more_than_32_bits_are_refused(window):
    with pytest.raises(mlxl3_amd.Exl3Error, match="attention window"):
        kv._window(window)


# ---------------------------------------------------------------------------
# frequencies
# ---------------------------------------------------------------------------
def test_plain_and_linear_frequencies():
    f, s = mlxl3_amd.rope_frequencies(128, 500000.0)
    assert s == 1.0 and f.dtype == torch.float32 and f.numel() == 64
    want = 500000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    assert torch.equal(f, want.float())
    g, s = mlxl3_amd.rope_frequencies(128, 500000.0, {"rope_type": "linear", "factor": 4.0})
    assert s == 1.0 and torch.equal(g, (want / 4).float())


def test_llama3_frequencies_keep_short_waves_and_stretch_long_ones():
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    f, s = mlxl3_amd.rope_frequencies(128, 500000.0, cfg)
    base = 500000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    wave = 2 * math.pi / base
    assert s == 1.0
    short, long = wave <= 8192 / 4, wave >= 8192
    assert torch.equal(f[short], base[short].float()) and torch.equal(f[long], (base[long] / 8).float())
    for i in (~short & ~long).nonzero().flatten().tolist():
        mix = (8192 / float(wave[i]) - 1.0) / 3.0
        want = mix * float(base[i]) + (1 - mix) * float(base[i]) / 8
        assert abs(float(f[i]) - want) <= 2.0**-23 * want


def test_yarn_frequencies_and_scale():
    cfg = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    f, s = mlxl3_amd.rope_frequencies(128, 1000000.0, cfg)
    assert abs(s - (0.1 * math.log(4.0) + 1.0)) < 1e-12
    base = 1000000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    turns = 32768 * base / (2 * math.pi)
    assert torch.equal(f[turns > 40], base[turns > 40].float())
    assert torch.equal(f[turns < 0.8], (base[turns < 0.8] / 4).float())
    ratio = f.double() / base
    assert bool(((ratio[1:] - ratio[:-1]) <= 1e-7).all()) and float(ratio.min()) >= 0.25 * (1 - 1e-6)
    assert mlxl3_amd.rope_frequencies(128, 1e6, dict(cfg, attention_factor=1.5))[1] == 1.5
    with pytest.raises(mlxl3_amd.Exl3Error, match="unknown rotary scaling"):
        mlxl3_amd.rope_frequencies(128, 1e6, {"rope_type": "other"})
    with pytest.raises(mlxl3_amd.Exl3Error, match="rotary dimension 7"):
        mlxl3_amd.rope_frequencies(7)


@pytest.mark.parametrize("scaling, msg", [
    ({"rope_type": "linear"}, "'linear' rotary scaling takes"),
    ({"type": "llama3", "factor": 8.0}, "'llama3' rotary scaling takes"),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "mscale": 0.7}, "'yarn' rotary scaling takes"),
    ({"rope_type": "linear", "factor": 0.0}, "positive numbers"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
      "original_max_position_embeddings": 8192}, "high_freq_factor must be above"),
])
def test_scalings_that_say_too_little_or_too_much(scaling, msg):
    with pytest.raises(mlxl3_amd.Exl3Error, match=msg):
        mlxl3_amd.rope_frequencies(64, 10000.0, scaling)


def test_absent_and_default_scalings():
    f, s = mlxl3_amd.rope_frequencies(64, 10000.0)
    for scaling in ({}, {"rope_type": "default"}, {"rope_type": None, "factor": None}):
        g, t = mlxl3_amd.rope_frequencies(64, 10000.0, scaling)
        assert torch.equal(f, g) and s == t == 1.0
    with pytest.raises(mlxl3_amd.Exl3Error, match="with base 1.0"):
        mlxl3_amd.rope_frequencies(64, 1.0)
