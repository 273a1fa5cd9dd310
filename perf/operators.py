"""The operators between a layer's q/k/v projections and its output projection, as cases that can be timed.

Kinds:
  rope    Rope.apply                       rotary positions of queries or keys
  store   KvCache.append, KvCache.read     new keys (rotated where `rope`) and values into a paged cache of
                                           16-, 8- or 4-bit values, and the same tokens read back
  read    KvCache.read                     whole sequences read back from the cache
  attend  attention                        new tokens of each sequence over its pages

Sequence b of a batch has n_b new tokens, the last n_b of the L_b tokens that the cache holds of it with them;
its pages are scattered over the pool.  Keys and values are N(0, 1) with one channel in fifty 8 times larger
(keys of real models have such channels), queries N(0, 1).  The plain forms compute in 32 bits (angles in 64) and
round once; cached 8- and 4-bit values are code * scale with one f16 scale per 32 values of a head,
scale = f16(max|x| / most), code = rint(x / scale), most = 127 or 7.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_MOST = {8: 127, 4: 7}


def listed():
    return [
        # the queries of one decoded token: the smallest rotation there is
        dict(name="rope_m1", kind="rope", tokens=1, heads=32, dim=128, rot=128, inter=False, scale=1.0, far=4000, dtype="f16"),
        # the queries of a long prefill chunk far into a scaled context, half of each head rotated, neighbours paired
        dict(name="rope_m4096", kind="rope", tokens=4096, heads=40, dim=128, rot=64, inter=True, scale=1.2, far=131072, dtype="bf16"),
        # one decoded token into an 8-bit cache
        dict(name="store_m1", kind="store", seqs=1, new=1, ctx=700, kv_heads=8, dim=128, page=16, bits=8, rope=True, dtype="f16"),
        # a batch of decoded tokens into a 4-bit cache
        dict(name="store_b64", kind="store", seqs=64, new=1, ctx=3000, kv_heads=8, dim=128, page=32, bits=4, rope=True, dtype="bf16"),
        # a prefill chunk into an 8-bit cache, from an odd place on
        dict(name="store_m4096", kind="store", seqs=1, new=4096, ctx=9001, kv_heads=8, dim=128, page=64, bits=8, rope=True, dtype="f16"),
        # a long 4-bit context read back whole (to move it, or for a kernel that wants plain values)
        dict(name="read_32k", kind="read", seqs=2, ctx=32771, kv_heads=8, dim=128, page=32, bits=4, dtype="f16"),
        # one decoded token after a short prompt: the smallest attention there is
        dict(name="attend_m1", kind="attend", seqs=1, new=1, ctx=1000, heads=32, kv_heads=8, dim=128, page=16, bits=16, window=0, dtype="f16"),
        # a batch of decodes of all lengths over an 8-bit cache, five query heads to a key head
        dict(name="attend_b32", kind="attend", seqs=32, new=1, ctx=8192, heads=40, kv_heads=8, dim=128, page=32, bits=8, window=0, dtype="f16"),
        # one decoded token at the end of a long context
        dict(name="attend_long", kind="attend", seqs=1, new=1, ctx=131071, heads=32, kv_heads=8, dim=128, page=64, bits=16, window=0, dtype="bf16"),
        # short drafts of several sequences verified over a 4-bit cache
        dict(name="attend_draft", kind="attend", seqs=4, new=5, ctx=6001, heads=32, kv_heads=8, dim=128, page=16, bits=4, window=0, dtype="bf16"),
        # a prefill chunk late in a long prompt
        dict(name="attend_m2048", kind="attend", seqs=1, new=2048, ctx=16384, heads=32, kv_heads=8, dim=128, page=64, bits=16, window=0, dtype="bf16"),
        # prompts of unequal lengths from their first token, small heads and a sliding window
        dict(name="attend_prompts", kind="attend", seqs=6, new=1500, ctx=1500, heads=32, kv_heads=8, dim=64, page=16, bits=16, window=512, dtype="f16"),
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------
_MAX_FLOPS = 2.5e11  # attention, below the largest listed case
_MAX_CACHE = 2.0e8   # cached values a case may read
_MAX_ROWS = 2.0e7    # values a rotation or an append may touch


def _log_int(rng, lo, hi):
    hi = max(lo, int(hi))
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "store", "store", "read", "attend", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
    if kind == "rope":
        heads = rng.choice([4, 8, 16, 32, 40])
        return dict(kind=kind, tokens=_log_int(rng, 1, _MAX_ROWS / (heads * dim)), heads=heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, dim // 4]), inter=rng.random() < 0.4, scale=rng.choice([1.0, 1.0, 1.2]),
                    far=_log_int(rng, 100, 1000000), dtype=rng.choice(["f16", "bf16", "f32"]))
    seqs, bits = _log_int(rng, 1, 64), rng.choice([16, 8, 4])
    if kind == "store":
        new = _log_int(rng, 1, _MAX_ROWS / (seqs * kv_heads * dim)) if rng.random() < 0.6 else 1
        return dict(kind=kind, seqs=seqs, new=new, ctx=new + _log_int(rng, 1, 4000), kv_heads=kv_heads, dim=dim, page=page,
                    bits=bits, rope=rng.random() < 0.6, dtype=dtype)
    ctx = _log_int(rng, 30, min(131072, _MAX_CACHE / (2 * seqs * kv_heads * dim)))
    if kind == "read":
        return dict(kind=kind, seqs=seqs, ctx=ctx, kv_heads=kv_heads, dim=dim, page=page, bits=bits, dtype=dtype)
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8])
    most = _MAX_FLOPS / (4.0 * dim * heads * seqs * ctx)
    new = rng.choice([1, _log_int(rng, 2, 16), _log_int(rng, 16, 4096)])
    new = max(1, min(new, ctx, int(most), int(4.0e9 / (4.0 * heads * seqs * ctx))))
    return dict(kind=kind, seqs=seqs, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, bits=bits,
                window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]), dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, tokens with them) of each sequence: the first has all, the others between 30 and 100 %."""
    part = [1.0 if b == 0 else 0.3 + 0.7 * ((b * 2654435761) % 1000) / 1000 for b in range(case["seqs"])]
    new = [max(1, int(case.get("new", case["ctx"]) * p)) for p in part]
    old = [int((case["ctx"] - case.get("new", case["ctx"])) * p) for p in part]
    return new, [n + o for n, o in zip(new, old)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _values(g, n, heads, dim, dtype):
    x = torch.randn(n, heads, dim, device="cuda", generator=g)
    loud = torch.rand(heads, dim, device="cuda", generator=g) < 0.02
    return torch.where(loud, 8.0 * x, x).to(dtype)


def _quantised(x, bits):
    """Scales [..., dim / 32] and whole numbers [..., dim] of x [..., dim] in 32 bits."""
    g = x.float().unflatten(-1, (-1, 32))
    s = (g.abs().amax(-1) / _MOST[bits]).clamp(max=65504.0).half()
    c = torch.round(g / torch.where(s > 0, s.float(), 1.0).unsqueeze(-1)).clamp(-_MOST[bits], _MOST[bits])
    c = torch.where((s > 0).unsqueeze(-1), c, 0.0)
    return s, c.flatten(-2)


def _codes(c, bits):
    """Whole numbers as they are stored: offset by 128 in a byte, or by 8 in half a byte, the low half first."""
    if bits == 8:
        return (c + 128).to(torch.uint8)
    c = (c + 8).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _pool(g, pages, case, dtype):
    """Keys or values of a pool of pages that earlier sequences have filled, and their scales."""
    x = _values(g, pages * case["page"], case["kv_heads"], case["dim"], dtype)
    x = x.unflatten(0, (pages, case["page"])).transpose(1, 2).contiguous()
    if case["bits"] == 16:
        return x, None
    s, c = _quantised(x, case["bits"])
    return _codes(c, case["bits"]), s.transpose(2, 3).contiguous()


def _frequencies(rot):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def prepare(case, seed):
    g, dtype = _generator(seed), _DTYPES[case["dtype"]]
    if case["kind"] == "rope":
        return dict(case=case, x=_values(g, case["tokens"], case["heads"], case["dim"], dtype), freq=_frequencies(case["rot"]),
                    positions=torch.randint(0, case["far"], (case["tokens"],), dtype=torch.int32, device="cuda", generator=g))
    new, lens = _lengths(case)
    need = [-(-n // case["page"]) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    state = dict(case=case, dtype=dtype, table=table, starts=starts, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 tokens=sum(new), max_q=max(new), max_kv=max(lens))
    state["k"], state["ks"] = _pool(g, pages, case, dtype)
    state["v"], state["vs"] = _pool(g, pages, case, dtype)
    if case["kind"] == "store":
        state["k_new"] = _values(g, sum(new), case["kv_heads"], case["dim"], dtype)
        state["v_new"] = _values(g, sum(new), case["kv_heads"], case["dim"], dtype)
        state["freq"] = _frequencies(case["dim"])
    if case["kind"] == "attend":
        state["q"] = torch.randn(sum(new), case["heads"], case["dim"], device="cuda", generator=g).to(dtype)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _rotated(x, positions, freq, inter, scale):
    """x [tokens, heads, dim] in 32 bits with its first 2 * len(freq) channels rotated."""
    r = freq.numel()
    angle = positions.double().unsqueeze(1) * freq.double()
    cos, sin = ((f * scale).float().unsqueeze(1) for f in (angle.cos(), angle.sin()))
    x = x.float()
    a, b = (x[..., 0 : 2 * r : 2], x[..., 1 : 2 * r : 2]) if inter else (x[..., :r], x[..., r : 2 * r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * r :]), -1)


def _places(state):
    """Sequence, index among its new tokens and position of every new token."""
    starts, lens = state["starts"].long(), state["lens"].long()
    n = torch.arange(state["tokens"], device="cuda")
    seq = torch.searchsorted(starts, n, right=True) - 1
    j = n - starts[seq]
    return seq, j, lens[seq] - (starts[seq + 1] - starts[seq]) + j


def _gathered(pool, scales, page, slot, bits):
    """Cached heads [..., kv_heads, dim] in 32 bits of the tokens at (page, slot)."""
    x = pool[page, :, slot]
    if bits == 16:
        return x.float()
    if bits == 4:
        x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
    s = scales[page, :, :, slot].float()
    return ((x.float() - (128 if bits == 8 else 8)).unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _read(state):
    case = state["case"]
    seq, _, pos = _places(state)
    page, slot = state["table"].long()[seq, pos // case["page"]], pos % case["page"]
    return [_gathered(state[n], state[n + "s"], page, slot, case["bits"]).to(state["dtype"]) for n in ("k", "v")]


def _store(state):
    case = state["case"]
    seq, _, pos = _places(state)
    page, slot = state["table"].long()[seq, pos // case["page"]], pos % case["page"]
    k, v = state["k_new"].float(), state["v_new"].float()
    if case["rope"]:
        k = _rotated(k, pos, state["freq"], False, 1.0)

    def put(name, x):
        if case["bits"] == 16:
            state[name][page, :, slot] = x.to(state["dtype"])
            return
        s, c = _quantised(x, case["bits"])
        state[name][page, :, slot] = _codes(c, case["bits"])
        state[name + "s"][page, :, :, slot] = s

    put("k", k)
    put("v", v)
    return _read(state)


def _attend(state):
    case = state["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seqs, most_q, most_kv = case["seqs"], state["max_q"], state["max_kv"]
    seq, j, _ = _places(state)
    lens, starts = state["lens"].long(), state["starts"].long()
    t = torch.arange(most_kv, device="cuda")
    pages = state["table"].long()[:, t // page]
    slots = (t % page).expand(seqs, -1)
    k, v = (_gathered(state[n], state[n + "s"], pages, slots, case["bits"]).permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    q = torch.zeros(seqs, most_q, heads, dim, device="cuda")
    q[seq, j] = state["q"].float()
    q = q.unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).reshape(seqs * kv_heads, -1, dim)
    k, v = k.flatten(0, 1), v.flatten(0, 1)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(dim))
    at = (lens - (starts[1:] - starts[:-1])).unsqueeze(1) + torch.arange(most_q, device="cuda")
    seen = (t <= at.unsqueeze(-1)) & (t < lens.view(-1, 1, 1))
    if case["window"]:
        seen &= t > at.unsqueeze(-1) - case["window"]
    s = s.view(seqs, kv_heads, -1, most_q, most_kv).masked_fill_(~seen.view(seqs, 1, 1, most_q, most_kv), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3.0e38))
    total = p.sum(-1, keepdim=True)
    y = torch.bmm(p.view(seqs * kv_heads, -1, most_kv), v).view(seqs, kv_heads, -1, most_q, dim)
    y = (y / torch.where(total > 0, total, 1.0)).permute(0, 3, 1, 2, 4).reshape(seqs, most_q, heads, dim)
    return y[seq, j].to(state["dtype"])


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _handles(state):
    """The cache and the batch that a serving program makes once and keeps for all layers' calls."""
    if "cache" not in state:
        import mlxl3_amd

        case = state["case"]
        state["cache"] = mlxl3_amd.KvCache(state["k"], state["v"], state["ks"], state["vs"], bits=case["bits"])
        state["batch"] = mlxl3_amd.KvBatch(state["starts"], state["lens"], state["table"], max_q=state["max_q"], max_kv=state["max_kv"])
        if case.get("rope"):
            state["rope"] = mlxl3_amd.Rope(state["freq"])
    return state["cache"], state["batch"]


def _own(state):
    import mlxl3_amd

    case = state["case"]
    if case["kind"] == "rope":
        if "rope" not in state:
            state["rope"] = mlxl3_amd.Rope(state["freq"], interleaved=case["inter"], scale=case["scale"])
        return state["rope"].apply(state["x"], state["positions"])
    cache, batch = _handles(state)
    if case["kind"] == "attend":
        return mlxl3_amd.attention(state["q"], cache, batch, window=case["window"])
    if case["kind"] == "store":
        cache.append(batch, state["k_new"], state["v_new"], rope=state.get("rope"))
    return list(cache.read(batch, state["tokens"], state["dtype"]))


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["kind"] == "rope":
        return _rotated(state["x"], state["positions"], state["freq"], case["inter"], case["scale"]).to(state["x"].dtype)
    return {"store": _store, "read": _read, "attend": _attend}[case["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * size * n + 4 * case["tokens"], "flops": 3 * n * case["rot"] // case["dim"]}
    new, lens = _lengths(case)
    width = case["kv_heads"] * case["dim"]
    cached = 2 * width * (2.0 if case["bits"] == 16 else case["bits"] / 8 + 2 / 32)  # bytes of a token's keys and values
    if case["kind"] != "attend":
        plain = 2 * size * width * sum(new)
        ways = 2 if case["kind"] == "store" else 1
        return {"bytes": ways * (plain + cached * sum(new)), "flops": 4 * width * sum(new)}
    pairs = seen = 0
    for n, total in zip(new, lens):
        first = total - n
        w = case["window"] or total
        seen += total - max(0, first - w + 1)
        full = max(0, min(n, w - first))  # rows whose window still reaches the first token
        pairs += full * first + full * (full + 1) // 2 + (n - full) * w
    return {"bytes": 2 * size * sum(new) * case["heads"] * case["dim"] + cached * seen, "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _turn64(x, positions, freq, inter, scale):
    y, r = x.double().clone(), freq.numel()
    angle = positions.double()[:, None, None] * freq.double()
    z = torch.polar(torch.full_like(angle, scale), angle)
    first, second = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if inter else (slice(0, r), slice(r, 2 * r))
    w = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _stored64(x, bits):
    """What the cache holds of x [tokens, kv_heads, dim] (64 bits)."""
    if bits == 16:
        return x
    groups = x.reshape(x.shape[0], x.shape[1], -1, 32)
    scale = (groups.abs().max(-1, keepdim=True).values / _MOST[bits]).clamp(max=65504).half().double()
    whole = torch.where(scale > 0, (groups / scale).round().clamp(-_MOST[bits], _MOST[bits]), torch.zeros_like(groups))
    return (whole * scale).reshape(x.shape)


def _sequence64(state, name, b):
    """Keys or values of sequence b in the cache, [tokens, kv_heads, dim] in 64 bits."""
    case, total = state["case"], int(state["lens"][b])
    rows = state["table"][b, : -(-total // case["page"])].long()
    x = state[name][rows].transpose(1, 2).flatten(0, 1)[:total]
    if case["bits"] == 16:
        return x.double()
    if case["bits"] == 4:
        low = x.to(torch.int64) % 16
        x = torch.stack((low, (x.to(torch.int64) - low) // 16), -1).flatten(-2) - 8
    else:
        x = x.to(torch.int64) - 128
    s = state[name + "s"][rows].permute(0, 3, 1, 2).flatten(0, 1)[:total].double()
    return x.double() * s.repeat_interleave(32, -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return _turn64(state["x"], state["positions"], state["freq"], case["inter"], case["scale"])
    new, lens = _lengths(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if case["kind"] == "store":
        k, v = state["k_new"].double(), state["v_new"].double()
        if case["rope"]:
            pos = torch.cat([torch.arange(total - n, total) for n, total in zip(new, lens)]).cuda()
            k = _turn64(k, pos, state["freq"], False, 1.0)
        return [_stored64(k, case["bits"]), _stored64(v, case["bits"])]
    if case["kind"] == "read":
        return [torch.cat([_sequence64(state, name, b) for b in range(len(lens))]) for name in ("k", "v")]
    group = case["heads"] // case["kv_heads"]
    y = torch.zeros(starts[-1], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    for b, (n, total) in enumerate(zip(new, lens)):
        k, v = _sequence64(state, "k", b), _sequence64(state, "v", b)
        at = torch.arange(total - n, total, device="cuda")[:, None]
        t = torch.arange(total, device="cuda")[None]
        hidden = t > at
        if case["window"]:
            hidden = hidden | (t <= at - case["window"])
        for h in range(case["heads"]):
            q = state["q"][starts[b] : starts[b + 1], h].double()
            s = (q @ k[:, h // group].T) / math.sqrt(case["dim"])
            w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            y[starts[b] : starts[b + 1], h] = w @ v[:, h // group]
    return y
