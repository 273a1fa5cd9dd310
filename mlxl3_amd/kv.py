"""What lies between a layer's q/k/v projections and its output projection: rotary
positions, the paged key/value cache and attention over it (``exl3_rope``,
``exl3_kv_append``, ``exl3_kv_read``, ``exl3_attention``, ``exl3_attention_scores`` of
``include/exl3_hip.h``).

* :class:`KvBatch`   -- the sequences of a call: new tokens, lengths, block table
* :class:`Rope`, :func:`rope_frequencies` -- rotary positions and their frequencies
* :class:`KvCache`   -- pages of f16, bf16, 8- or 4-bit values; append and read
* :func:`attention`  -- new tokens over their sequences' pages
* :class:`Exl3Attention` -- the attention block of a decoder layer
  (``exl3_attn_block_forward``)
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import threading
from typing import Optional

from . import (
    Exl3Error, Exl3Linear, _check, _code_dtype, _dtype_code, _ptr, _stream_ptr, _torch, _vp, _Workspace, load_library,
)

_FORMATS = {8: 8, 4: 4}


class _KvBatchC(ctypes.Structure):
    _fields_ = [
        ("q_starts", _vp),
        ("kv_lens", _vp),
        ("block_table", _vp),
        ("seqs", ctypes.c_int32),
        ("table_pages", ctypes.c_int32),
        ("max_q", ctypes.c_int32),
        ("max_kv", ctypes.c_int32),
    ]


class _RopeC(ctypes.Structure):
    _fields_ = [
        ("inv_freq", _vp),
        ("rotary_dim", ctypes.c_int32),
        ("interleaved", ctypes.c_int32),
        ("scale", ctypes.c_double),
    ]


class _ScoresC(ctypes.Structure):
    _fields_ = [
        ("softcap", ctypes.c_float),
        ("slopes", _vp),
        ("prefix", _vp),
    ]


_FLOATS: dict = {}  # f16, bf16, f32 -> code, and the 16-bit ones: filled on first use
_HALVES: dict = {}


def _floats() -> dict:
    if not _FLOATS:  # the halves first: another thread goes by the floats
        torch = _torch()
        _HALVES.update({t: _dtype_code(t) for t in (torch.float16, torch.bfloat16)})
        _FLOATS.update({t: _dtype_code(t) for t in (torch.float16, torch.bfloat16, torch.float32)})
    return _FLOATS


def _device_tensor(t, name: str, dtypes, dims: int):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise Exl3Error(-1, f"{name} must be a device tensor")
    if t.dtype not in dtypes:
        raise Exl3Error(-1, f"{name} has dtype {t.dtype}, expected one of {tuple(dtypes)}")
    if t.dim() != dims:
        raise Exl3Error(-1, f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    return t


def _plain(t, name: str, dtypes, dims: int):
    """A tensor that the kernels read in place: contiguous."""
    t = _device_tensor(t, name, dtypes, dims)
    if not t.is_contiguous():
        raise Exl3Error(-1, f"{name} must be contiguous")
    return t


def _rows_ok(t) -> bool:
    """Whether the kernels read [tokens, heads, channels] as it is: contiguous heads, tokens
    any distance apart."""
    if t.is_contiguous():
        return True
    n, h, d = t.shape
    return t.stride(2) == 1 and (h == 1 or t.stride(1) == d) and (n == 1 or t.stride(0) >= h * d)


def _heads(t, name: str, dtypes):
    """[tokens, heads, channels] with contiguous heads; copied where its strides are others."""
    t = _device_tensor(t, name, dtypes, 3)
    return t if _rows_ok(t) else t.contiguous()


def _new(t, dtype=None):
    """A contiguous tensor of t's shape."""
    torch = _torch()
    if t.is_contiguous() and (dtype is None or dtype == t.dtype):
        return torch.empty_like(t)  # 0.6 us a call less than from a shape
    return torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device)


def _same(device, t, name: str):
    if t.device != device:
        raise Exl3Error(-1, f"{name} is on {t.device}, expected {device}")


def _launch(device, entry, *args):
    """entry(*args, stream) on the current stream of `device`, which is made the current one
    (launches go to the current device)."""
    torch = _torch()
    if torch._C._cuda_getDevice() == device.index:  # (current_device() looks for the runtime first)
        _check(entry(*args, _stream_ptr(device)))
    else:
        with torch.cuda.device(device):
            _check(entry(*args, _stream_ptr(device)))


class KvBatch:
    """The sequences of a call (``exl3_kv_batch``).

    q_starts int32 [seqs + 1]: rows [q_starts[b], q_starts[b + 1]) of the call's tensors
    are the newest tokens of sequence b; kv_lens int32 [seqs]: its tokens with them;
    block_table int32 [seqs, pages]: the page of every page_tokens positions.  The
    tensors are read on the device at every call (a captured graph can be replayed after
    they were changed in place).  max_q and max_kv bound a sequence's new tokens and its
    length (None: all tokens of a call, and what the table has room for).  Attention is
    launched for max_q tokens of every sequence, and rows past it are not computed: a batch
    of decoded tokens says max_q=1, or pays for rows that it may have.
    """

    def __init__(self, q_starts, kv_lens, block_table=None, max_q: Optional[int] = None,
                 max_kv: Optional[int] = None):
        i32 = (_torch().int32,)
        self.q_starts = _plain(q_starts, "q_starts", i32, 1)
        self.kv_lens = _plain(kv_lens, "kv_lens", i32, 1)
        self.block_table = None if block_table is None else _plain(block_table, "block_table", i32, 2)
        self.seqs = int(self.kv_lens.numel())
        if self.seqs < 1 or self.q_starts.numel() != self.seqs + 1:
            raise Exl3Error(-1, "q_starts has one entry more than kv_lens, which has at least one")
        if block_table is not None and self.block_table.shape[0] != self.seqs:
            raise Exl3Error(-1, "block_table has one row per sequence")
        if not 1 <= int(1 if max_q is None else max_q) < 2**31 or not 0 <= int(max_kv or 0) < 2**31:
            raise Exl3Error(-1, "max_q must be positive, max_kv not negative, both 32 bits")
        self.device = self.kv_lens.device
        _same(self.device, self.q_starts, "q_starts")
        if block_table is not None:
            _same(self.device, self.block_table, "block_table")
        pages = 0 if block_table is None else int(self.block_table.shape[1])
        self._c = _KvBatchC(_ptr(self.q_starts), _ptr(self.kv_lens), _ptr(self.block_table), self.seqs, pages,
                            int(max_q or 1), 0 if max_kv is None else int(max_kv))
        self._ref = ctypes.byref(self._c)
        self._given = max_q is not None
        self._bounded = (None, None, None)  # without max_q: the last attention's tokens, with them as max_q
        self._sized = (None, 0)  # the last attention's sizes and workspace

    def _attended(self, tokens: int):
        """The batch of an attention call of so many tokens."""
        if self._given:
            return self._ref
        bounded = self._bounded  # read once: another thread may replace it
        if bounded[0] != tokens:
            c = _KvBatchC.from_buffer_copy(self._c)
            c.max_q = min(max(1, tokens), 2**31 - 1)
            self._bounded = bounded = (tokens, c, ctypes.byref(c))
        return bounded[2]

    def _workspace_bytes(self, cache: "KvCache", tokens: int, heads: int) -> int:
        key = (cache.kv_heads, cache.head_dim, cache.page_tokens, tokens, heads)
        sized = self._sized  # read once: another thread may replace it
        if sized[0] != key:
            need = load_library().exl3_attention_workspace_bytes(cache.handle, self._attended(tokens), tokens, heads)
            self._sized = sized = (key, int(need))
        return sized[1]


def _ask(batch) -> None:
    """Whether the batch's pages are its sequences' to append to: KvPages knows of those that it made."""
    asked = getattr(batch, "_asked", None)
    if asked is not None:
        asked()


# rope_scaling by type: the keys it needs, and those it may have
_SCALING = {
    "default": (set(), set()),
    "linear": ({"factor"}, set()),
    "llama3": ({"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"}, set()),
    "yarn": ({"factor", "original_max_position_embeddings"}, {"beta_fast", "beta_slow", "attention_factor"}),
}


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None):
    """(inv_freq f32 [rotary_dim / 2], scale) of rotary positions: base^(-2i / rotary_dim),
    changed for a context longer than the trained one as `scaling` says (the keys of a
    checkpoint's rope_scaling):

    * ``{"rope_type": "linear", "factor": s}``: every frequency / s;
    * ``"llama3"`` with factor, low_freq_factor, high_freq_factor and
      original_max_position_embeddings n: wavelengths above n / low are stretched by
      factor, those below n / high kept, in between a linear mix in n / wavelength;
    * ``"yarn"`` with factor, original_max_position_embeddings n and optionally
      beta_fast (32), beta_slow (1), attention_factor: pairs that turn more than
      beta_fast times in n positions are kept, those that turn less than beta_slow times
      stretched, in between a linear mix in the pair's index; scale is attention_factor,
      0.1 ln(factor) + 1 by default.
    """
    torch = _torch()
    if rotary_dim < 2 or rotary_dim % 2 or not base > 1.0:
        raise Exl3Error(-1, f"rotary dimension {rotary_dim} with base {base}")
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    scaling = {key: v for key, v in (scaling or {}).items() if v is not None}
    kind = scaling.pop("rope_type", scaling.pop("type", "default"))
    if kind not in _SCALING:
        raise Exl3Error(-1, f"unknown rotary scaling {kind!r}")
    needed, more = _SCALING[kind]
    if not needed <= set(scaling) or not set(scaling) <= needed | more:
        raise Exl3Error(-1, f"{kind!r} rotary scaling takes {sorted(needed)}, optionally {sorted(more)}")
    scaling = {key: float(v) for key, v in scaling.items()}
    if any(not v > 0.0 for v in scaling.values()):
        raise Exl3Error(-1, "rotary scaling takes positive numbers")
    s, n = scaling.get("factor", 1.0), scaling.get("original_max_position_embeddings", 0.0)
    scale = 1.0
    if kind == "linear":
        freq = [f / s for f in freq]
    elif kind == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        if not high > low:
            raise Exl3Error(-1, "high_freq_factor must be above low_freq_factor")
        mixed = []
        for f in freq:
            turns = n * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            mixed.append(keep * f + (1.0 - keep) * f / s)
        freq = mixed
    elif kind == "yarn":
        def pair(turns):
            return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        first = max(0, math.floor(pair(scaling.get("beta_fast", 32.0))))
        last = min(rotary_dim - 1, math.ceil(pair(scaling.get("beta_slow", 1.0))))
        mixed = []
        for i, f in enumerate(freq):
            stretch = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            mixed.append((1.0 - stretch) * f + stretch * f / s)
        freq = mixed
        scale = scaling.get("attention_factor", 0.1 * math.log(s) + 1.0 if s > 1 else 1.0)
    return torch.tensor(freq, dtype=torch.float64).float(), scale


class Rope:
    """Rotary positions (``exl3_rope``): inv_freq f32 [rotary_dim / 2] on the device,
    pairs (2i, 2i + 1) with interleaved, else (i, i + rotary_dim / 2); cosines and sines
    times `scale`."""

    def __init__(self, inv_freq, interleaved: bool = False, scale: float = 1.0):
        self.inv_freq = _plain(inv_freq, "inv_freq", (_torch().float32,), 1)
        if self.inv_freq.numel() < 1:
            raise Exl3Error(-1, "empty rotary frequencies")
        self.device = self.inv_freq.device
        self.rotary_dim = 2 * int(self.inv_freq.numel())
        self._c = _RopeC(_ptr(self.inv_freq), self.rotary_dim, int(bool(interleaved)), float(scale))
        self._ref = ctypes.byref(self._c)

    def apply(self, x, positions=None, batch: Optional[KvBatch] = None, out=None, dtype=None):
        """x [tokens, heads, channels] (f16, bf16 or f32) rotated by its tokens' positions
        (int32 [tokens], or the batch's) into `out` (x itself: in place; else apart from it) or a
        new tensor of `dtype` (default x's).  Rows outside every sequence of a batch are not
        written."""
        if out is x and not _rows_ok(x):
            raise Exl3Error(-1, "rotation in place needs contiguous heads")
        src = _heads(x, "x", _floats())
        if dtype is not None and dtype not in _FLOATS:
            raise Exl3Error(-1, f"unsupported rotary output dtype {dtype}")
        n, heads, dim = src.shape
        device = src.device
        if out is None:
            out = _new(src, dtype)
        elif out is not x:
            _device_tensor(out, "out", _FLOATS, 3)
            if out.shape != src.shape or not _rows_ok(out):
                raise Exl3Error(-1, "out must have x's shape and contiguous heads")
            _same(device, out, "out")
        where = None
        if positions is not None:
            _plain(positions, "positions", (_torch().int32,), 1)
            if positions.numel() != n:
                raise Exl3Error(-1, f"{positions.numel()} positions for {n} tokens")
            _same(device, positions, "positions")
            where = positions.data_ptr()
        if batch is not None:
            _same(device, batch.kv_lens, "batch")
        _same(device, self.inv_freq, "inv_freq")
        if n == 0 and (where is not None) != (batch is not None):
            return out  # no tokens: an empty tensor's address is null
        _launch(device, load_library().exl3_rope, self._ref, src.data_ptr(), _FLOATS[src.dtype], n, heads, dim,
                src.stride(0), where, None if batch is None else batch._ref, out.data_ptr(), _FLOATS[out.dtype],
                out.stride(0))
        return out


class KvCache:
    """A pool of pages of keys and values (``exl3_kv_cache``).

    k, v: [pages, kv_heads, page_tokens, head_dim] f16 or bf16 (bits=16), or uint8 codes
    of head_dim bytes (bits=8) or head_dim / 2 bytes (bits=4) with k_scales, v_scales f16
    [pages, kv_heads, head_dim / 32, page_tokens].  The tensors are used in place.
    """

    def __init__(self, k, v, k_scales=None, v_scales=None, bits: int = 16):
        torch = _torch()
        if bits not in (16, 8, 4):
            raise Exl3Error(-1, f"KV caches hold 16, 8 or 4 bits a value, got {bits}")
        kinds = (torch.float16, torch.bfloat16) if bits == 16 else (torch.uint8,)
        self.k, self.v = _plain(k, "k", kinds, 4), _plain(v, "v", kinds, 4)
        if self.k.shape != self.v.shape or self.k.dtype != self.v.dtype:
            raise Exl3Error(-1, "keys and values of a cache have one shape and type")
        self.pages, self.kv_heads, self.page_tokens, width = (int(d) for d in self.k.shape)
        self.head_dim = 2 * width if bits == 4 else width
        self.bits, self.device = bits, self.k.device
        self.k_scales, self.v_scales = k_scales, v_scales
        if bits == 16:
            if k_scales is not None or v_scales is not None:
                raise Exl3Error(-1, "16-bit KV caches have no scales")
        else:
            want = (self.pages, self.kv_heads, self.head_dim // 32, self.page_tokens)
            for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
                if tuple(_plain(s, name, (torch.float16,), 4).shape) != want:
                    raise Exl3Error(-1, f"{name} must have shape {want}")
        for name, t in (("v", v), ("k_scales", k_scales), ("v_scales", v_scales)):
            if t is not None:
                _same(self.device, t, name)
        fmt = _FORMATS.get(bits) or _dtype_code(self.k.dtype)
        h = _vp()
        lib = load_library()
        self._destroy = lib.exl3_kv_cache_destroy
        _check(lib.exl3_kv_cache_create(
            _ptr(self.k), _ptr(self.v), _ptr(k_scales), _ptr(v_scales), fmt, self.pages, self.page_tokens,
            self.kv_heads, self.head_dim, ctypes.byref(h)))
        self._handle = h

    @classmethod
    def zeros(cls, pages: int, page_tokens: int, kv_heads: int, head_dim: int, dtype=None, bits: int = 16,
              device="cuda") -> "KvCache":
        """A new pool of zeros: `dtype` (default float16) with bits=16, else codes and scales."""
        torch = _torch()
        shape = (pages, kv_heads, page_tokens)
        if bits == 16:
            dtype = dtype or torch.float16
            return cls(*(torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(2)))
        codes = [torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(pages, kv_heads, head_dim // 32, page_tokens, dtype=torch.float16, device=device)
                  for _ in range(2)]
        return cls(*codes, *scales, bits=bits)

    @property
    def handle(self):
        return self._handle

    def __del__(self):
        h = getattr(self, "_handle", None)
        if h is not None and h.value:
            self._destroy(h)
            self._handle = None

    def append(self, batch: KvBatch, k, v, rope: Optional[Rope] = None) -> None:
        """Writes the batch's new tokens, k and v [tokens, kv_heads, head_dim] (f16, bf16
        or f32), to their pages, keys rotated by `rope` first."""
        k, v = _heads(k, "k", _floats()), _heads(v, "v", (k.dtype,))
        if k.shape != v.shape or k.shape[1] != self.kv_heads or k.shape[2] != self.head_dim:
            raise Exl3Error(-1, f"new keys and values have shape [tokens, {self.kv_heads}, {self.head_dim}]")
        device = self.device
        _same(device, k, "k")
        _same(device, v, "v")
        _same(device, batch.kv_lens, "batch")
        if rope is not None:
            _same(device, rope.inv_freq, "rope")
        _ask(batch)
        _launch(device, load_library().exl3_kv_append, self._handle, batch._ref, k.data_ptr(), k.stride(0),
                v.data_ptr(), v.stride(0), _FLOATS[k.dtype], k.shape[0], None if rope is None else rope._ref)

    def read(self, batch: KvBatch, tokens: int, dtype=None):
        """(k, v) [tokens, kv_heads, head_dim] of the batch's newest tokens in `dtype`
        (default: the cache's, float16 for codes).  Rows behind the last sequence are not
        written."""
        torch = _torch()
        dtype = dtype or (self.k.dtype if self.bits == 16 else torch.float16)
        if dtype not in _floats():
            raise Exl3Error(-1, f"unsupported KV output dtype {dtype}")
        device, tokens = self.device, int(tokens)
        if tokens < 0:
            raise Exl3Error(-1, "negative token count")
        _same(device, batch.kv_lens, "batch")
        shape = (tokens, self.kv_heads, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
        _launch(device, load_library().exl3_kv_read, self._handle, batch._ref, k.data_ptr(), v.data_ptr(),
                _FLOATS[dtype], tokens)
        return k, v


def _window(window) -> int:
    if not 0 <= int(window) < 2**31:
        raise Exl3Error(-1, f"attention window {window}")
    return int(window)


def _scores(device, heads: int, seqs: int, softcap, slopes, prefix):
    """The C form of shaped scores, or None without any."""
    try:
        softcap = float(softcap)
    except (TypeError, ValueError):
        raise Exl3Error(-1, f"attention softcap must be a number, got {softcap!r}") from None
    if slopes is not None:
        _plain(slopes, "slopes", (_torch().float32,), 1)
        if slopes.numel() != heads:
            raise Exl3Error(-1, f"{slopes.numel()} slopes for {heads} heads")
        _same(device, slopes, "slopes")
    if prefix is not None:
        _plain(prefix, "prefix", (_torch().int32,), 1)
        if prefix.numel() != seqs:
            raise Exl3Error(-1, f"{prefix.numel()} prefixes for {seqs} sequences")
        _same(device, prefix, "prefix")
    if softcap == 0.0 and slopes is None and prefix is None:
        return None
    scores = _ScoresC(softcap, _ptr(slopes), _ptr(prefix))
    if softcap != 0.0 and scores.softcap == 0.0:  # (what else is out of range the call refuses)
        raise Exl3Error(-1, f"attention softcap must be 0 or 2^-64 to 2^64, got {softcap:g}")
    return scores


def attention(q, cache: KvCache, batch: KvBatch, scale: Optional[float] = None, causal: bool = True,
              window: int = 0, out=None, workspace=None, softcap: float = 0.0, slopes=None, prefix=None):
    """Attention of the batch's new tokens over the cache (``exl3_attention``): q
    [tokens, heads, head_dim] (f16 or bf16, the cache's type where it is 16-bit) -> the
    same shape and type.  scale defaults to 1 / sqrt(head_dim); causal: a token sees the
    positions up to its own; window > 0: only the last `window` of them.  `out` may be q and is
    apart from it else.  Rows outside every sequence and past the batch's max_q are not
    written (in a new tensor they hold anything).

    Shaped scores (``exl3_attention_scores``): softcap > 0: a score z = scale q.k becomes
    softcap * tanh(z / softcap); slopes (f32 [heads], finite, counted up to 2^32): then slope
    times the distance of the token's position and the row's is taken off it; prefix (int32
    [seqs], with causal): every row sees the first prefix[b] tokens of its sequence too, as far
    as the window lets it."""
    torch = _torch()
    _floats()
    q = _heads(q, "q", _HALVES)
    n, heads, dim = q.shape
    device = cache.device
    if dim != cache.head_dim:
        raise Exl3Error(-1, f"queries of {dim} channels over a cache of {cache.head_dim}")
    _same(device, q, "q")
    _same(device, batch.kv_lens, "batch")
    window = _window(window)
    if out is None:
        out = _new(q)
    elif (not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or not out.is_cuda
          or not _rows_ok(out)):
        raise Exl3Error(-1, "out must have q's shape and type and contiguous heads")
    else:
        _same(device, out, "out")
    space, room = None, 0
    if workspace is None:
        room = batch._workspace_bytes(cache, n, heads)
        if room:
            workspace = torch.empty(room, dtype=torch.uint8, device=device)
    else:
        _plain(workspace, "workspace", (torch.uint8,), 1)
        _same(device, workspace, "workspace")
        room = workspace.numel()
    if workspace is not None:
        space = workspace.data_ptr()
    shape = None
    if slopes is not None or prefix is not None or softcap != 0.0:
        shape = _scores(device, heads, batch.seqs, softcap, slopes, prefix)
    if shape is None:
        _launch(device, load_library().exl3_attention, cache._handle, batch._attended(n), q.data_ptr(), _HALVES[q.dtype],
                n, heads, q.stride(0), dim**-0.5 if scale is None else float(scale), 1 if causal else 0, window,
                out.data_ptr(), out.stride(0), space, room)
    else:
        _launch(device, load_library().exl3_attention_scores, cache._handle, batch._attended(n), q.data_ptr(),
                _HALVES[q.dtype], n, heads, q.stride(0), dim**-0.5 if scale is None else float(scale), 1 if causal else 0,
                window, ctypes.byref(shape), out.data_ptr(), out.stride(0), space, room)
    return out


_MOST_STREAMS = 40  # that a block keeps a workspace for; PyTorch's own pool has 32 of a device


class Exl3Attention:
    """The attention block of a decoder layer (``exl3_attn_block_forward``): the q/k/v
    projections of x as a group, keys rotated and appended with the values, queries rotated,
    causal attention over the cache (softcap and slopes as :func:`attention` takes them), the o
    projection."""

    def __init__(self, q: Exl3Linear, k: Exl3Linear, v: Exl3Linear, o: Exl3Linear, rope: Optional[Rope] = None,
                 scale: Optional[float] = None, window: int = 0, softcap: float = 0.0, slopes=None):
        if len({(m.in_features, m.k, m.cb) for m in (q, k, v)}) != 1:
            raise Exl3Error(-1, "incompatible grouped projections")
        if o.in_features != q.out_features or k.out_features != v.out_features:
            raise Exl3Error(-1, "attention block widths differ")
        self.q, self.k, self.v, self.o = q, k, v, o
        self.device = None  # of the projections; not known of those loaded to "cuda"
        for name, m in zip("qkvo", (q, k, v, o)):
            at = m.device if m.trellis is None else m.trellis.device
            if at.index is not None:
                if self.device not in (None, at):
                    raise Exl3Error(-1, f"projection {name} is on {at}, others on {self.device}")
                self.device = at
        self.rope, self.scale, self.window = rope, scale, _window(window)
        self.softcap, self.slopes = softcap, slopes
        self._ws: dict = {}  # (lock, workspace) by stream, the last used one last
        self._ws_lock = threading.Lock()

    def workspace_bytes(self, cache: KvCache, batch: KvBatch, rows: int, dtype) -> int:
        _floats()
        if dtype not in _HALVES:
            raise Exl3Error(-1, f"attention blocks take f16 or bf16 activations, got {dtype}")
        return int(load_library().exl3_attn_block_workspace_bytes(
            self.q.handle, self.k.handle, self.v.handle, self.o.handle, cache.handle, batch._attended(int(rows)),
            _HALVES[dtype], int(rows)))

    def _kept(self, device):
        """The lock and the workspace of the current stream.  A call is several launches, which
        leave their results to each other in the workspace: the lock keeps those of one call
        together in the stream.  Those of the streams used longest ago are dropped (their memory
        goes back to the allocator, which reuses it in the same stream's order)."""
        key = device, _stream_ptr(device)
        with self._ws_lock:
            kept = self._ws.pop(key, None) or (threading.Lock(), _Workspace())
            self._ws[key] = kept
            while len(self._ws) > _MOST_STREAMS:
                del self._ws[next(iter(self._ws))]
        return kept

    def forward(self, x, cache: KvCache, batch: KvBatch, workspace=None, prefix=None):
        """x [rows, in] (f16 or bf16) -> [rows, out] in the o projection's result dtype;
        the cache's pages get the rows' keys and values.  `workspace`: a zero-filled uint8
        tensor of :meth:`workspace_bytes`, of which two calls that run at once need one each;
        by default one that the block keeps for the stream (threads on one stream take turns), and
        in a captured graph one of the graph's, all of which every replay clears first (a given
        one saves that).  `prefix`: as :func:`attention` takes it."""
        torch = _torch()
        _floats()
        x = _device_tensor(x, "x", _HALVES, 2).contiguous()
        rows, device = x.shape[0], cache.device
        if x.shape[1] != self.q.in_features or rows < 1:
            raise Exl3Error(-1, f"invalid attention block input for {self.q.in_features} inputs")
        _same(device, x, "x")
        _same(device, batch.kv_lens, "batch")
        if self.device is not None:
            _same(device, self, "projections")
        if self.rope is not None:
            _same(device, self.rope.inv_freq, "rope")
        _ask(batch)
        shape = None
        if self.slopes is not None or prefix is not None or self.softcap != 0.0:
            shape = _scores(device, self.q.out_features // cache.head_dim, batch.seqs, self.softcap, self.slopes, prefix)
        lib, code = load_library(), _HALVES[x.dtype]
        y = torch.empty(rows, self.o.out_features, device=device,
                        dtype=_code_dtype(lib.exl3_linear_output_dtype(self.o.handle, code)))
        turn = contextlib.nullcontext()
        if workspace is None:
            need = self.workspace_bytes(cache, batch, rows, x.dtype)
            if torch.cuda.is_current_stream_capturing():  # a kept one could be replaced before a replay
                workspace = torch.zeros(max(need, 256), dtype=torch.uint8, device=device)
            else:
                turn, kept = self._kept(device)
        else:
            _plain(workspace, "workspace", (torch.uint8,), 1)
            _same(device, workspace, "workspace")
        scale = cache.head_dim**-0.5 if self.scale is None else float(self.scale)
        with turn:
            if workspace is None:
                workspace = kept.get(need, device)
            args = (self.q.handle, self.k.handle, self.v.handle, self.o.handle, cache.handle, batch._attended(rows),
                    None if self.rope is None else self.rope._ref, scale, self.window)
            more = (x.data_ptr(), code, rows, y.data_ptr(), workspace.data_ptr(), workspace.numel())
            if shape is None:
                _launch(device, lib.exl3_attn_block_forward, *args, *more)
            else:
                _launch(device, lib.exl3_attn_block_forward_scores, *args, ctypes.byref(shape), *more)
        return y

    __call__ = forward
