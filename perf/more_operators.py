"""More operators of a decoder layer around its projections, as cases that can be timed.

Kinds:
  attend  attention        new tokens of each sequence over its pages, scores capped, with a bias by distance,
                           with a prefix that all rows see
  copy    KvPages.copy     pages of the caches of all layers copied: filled slots when sequences are forked,
                           whole pages when a pool is compacted
  norm    rms_norm         root-mean-square norm of rows or heads, with the residual's addition

A score is z = q.k / sqrt(dim), capped it is cap * tanh(z / cap), the bias takes slope_h * |i - t| off it (row at
position i, token t).  A row sees the tokens up to its own position and those of its sequence's prefix, and with a
window only the last `window` positions up to its own and whatever the prefix has behind it.  Sequence b of a batch
has n_b new tokens, the last n_b of the L_b tokens that the cache holds of it with them; its pages are scattered over
the pool.  Keys and values are N(0, 1) with one channel in fifty 8 times larger (keys of real models have such
channels), queries N(0, gain^2).  8- and 4-bit values are code * scale with one f16 scale per 32 values of a head.
A norm is x / sqrt(mean(x^2) + eps) * weight of a row x, or of x + residual, which is given out too.

The plain forms compute in 32 bits and round once.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_MOST = {8: 127, 4: 7}
_EPS = 1.0e-6


def listed():
    return [
        # one decoded token after a short prompt, capped scores: the smallest attention there is
        dict(name="capped_m1", kind="attend", seqs=1, new=1, ctx=1000, heads=32, kv_heads=8, dim=128, page=16, bits=16, window=0,
             cap=50.0, bias=False, prefix=0.0, gain=4.0, dtype="f16"),
        # a batch of decodes of all lengths over an 8-bit cache, biased by distance
        dict(name="biased_b32", kind="attend", seqs=32, new=1, ctx=8192, heads=40, kv_heads=8, dim=128, page=32, bits=8, window=0,
             cap=0.0, bias=True, prefix=0.0, gain=1.0, dtype="f16"),
        # one decoded token at the end of a long context, capped scores
        dict(name="capped_long", kind="attend", seqs=1, new=1, ctx=131071, heads=32, kv_heads=8, dim=128, page=64, bits=16, window=0,
             cap=50.0, bias=False, prefix=0.0, gain=4.0, dtype="bf16"),
        # short drafts of several sequences verified over a 4-bit cache, biased by distance
        dict(name="biased_draft", kind="attend", seqs=4, new=5, ctx=6001, heads=32, kv_heads=8, dim=128, page=16, bits=4, window=0,
             cap=0.0, bias=True, prefix=0.0, gain=1.0, dtype="bf16"),
        # a prefill chunk late in a long prompt, capped scores
        dict(name="capped_m2048", kind="attend", seqs=1, new=2048, ctx=16384, heads=32, kv_heads=8, dim=128, page=64, bits=16, window=0,
             cap=50.0, bias=False, prefix=0.0, gain=4.0, dtype="bf16"),
        # prompts of unequal lengths from their first token: a prefix (an image, a task) seen by all rows, bias by distance
        dict(name="prefix_prompts", kind="attend", seqs=6, new=1500, ctx=1500, heads=32, kv_heads=8, dim=64, page=16, bits=16, window=0,
             cap=0.0, bias=True, prefix=0.5, gain=1.0, dtype="f16"),
        # one sequence forked: the filled part of its last page, in every layer's cache
        dict(name="fork_1", kind="copy", layers=32, pairs=1, used=0, kv_heads=8, dim=128, page=16, bits=16, part=True, dtype="f16"),
        # a batch of sequences forked for sampling over 8-bit caches
        dict(name="fork_b48", kind="copy", layers=16, pairs=48, used=0, kv_heads=8, dim=128, page=32, bits=8, part=True, dtype="f16"),
        # a pool compacted: whole pages moved into the holes in front of them
        dict(name="compact", kind="copy", layers=4, pairs=230, used=40, kv_heads=8, dim=128, page=32, bits=16, part=False, dtype="bf16"),
        # the hidden state of one decoded token, with the residual
        dict(name="norm_m1", kind="norm", tokens=1, heads=1, width=4096, residual="f16", gap=0, weight="f16", dtype="f16"),
        # a prefill chunk's hidden states, the residual kept in 32 bits
        dict(name="norm_m4096", kind="norm", tokens=4096, heads=1, width=4096, residual="f32", gap=0, weight="bf16", dtype="bf16"),
        # the query heads among a projection's q, k and v rows
        dict(name="norm_heads", kind="norm", tokens=2001, heads=32, width=128, residual="", gap=16, weight="f32", dtype="f16"),
    ]


# ---------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------
_MAX_FLOPS = 4.0e11  # attention, below the largest listed case
_MAX_CACHE = 2.0e8   # cached values an attention may read
_MAX_POOL = 2.5e8    # bytes of all layers' pools
_MAX_ROWS = 1.6e7    # values a norm may touch


def _log_int(rng, lo, hi):
    hi = max(lo, int(hi))
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "copy", "copy", "norm", "norm"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "norm":
        if rng.random() < 0.3:
            heads, width, gap, residual = rng.choice([1, 4, 8, 32, 40]), rng.choice([64, 128, 256]), rng.choice([0, 2, 16]), ""
        else:
            heads, gap, residual = 1, 0, rng.choice(["", dtype, "f32"])
            width = _log_int(rng, 8, 20000) if rng.random() < 0.3 else rng.choice([1024, 2048, 4096, 5120, 7168, 8192, 14336])
        return dict(kind=kind, tokens=_log_int(rng, 1, _MAX_ROWS / (heads * width)), heads=heads, width=width, residual=residual, gap=gap,
                    weight=rng.choice(["", "f16", "bf16", "f32"]), dtype=rng.choice([dtype, dtype, dtype, "f32"]))
    dim, kv_heads = rng.choice([64, 128, 128, 128, 256]), rng.choice([1, 2, 4, 8, 8])
    page, bits = rng.choice([16, 32, 64, 128]), rng.choice([16, 8, 4])
    if kind == "copy":
        layers = _log_int(rng, 1, 64)
        size = layers * 2 * kv_heads * page * dim * (2.0 if bits == 16 else bits / 8 + 2 / 32)
        pages = int(max(3, min(600, _MAX_POOL / size)))  # in three parts: left alone, copied, copied to
        return dict(kind=kind, layers=layers, pairs=_log_int(rng, 1, pages / 3), used=_log_int(rng, 1, pages / 3), kv_heads=kv_heads,
                    dim=dim, page=page, bits=bits, part=rng.random() < 0.6, dtype=dtype)
    seqs = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 30, min(131072, _MAX_CACHE / (2 * seqs * kv_heads * dim)))
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8])
    most = _MAX_FLOPS / (4.0 * dim * heads * seqs * ctx)
    new = rng.choice([1, _log_int(rng, 2, 16), _log_int(rng, 16, 4096)])
    new = max(1, min(new, ctx, int(most), int(4.0e9 / (4.0 * heads * seqs * ctx))))
    cap, bias = rng.choice([(20.0, False), (50.0, False), (50.0, False), (0.0, True), (0.0, True), (30.0, True), (0.0, False)])
    prefix = round(rng.uniform(0.05, 0.95), 2) if rng.random() < 0.3 or not (cap or bias) else 0.0
    return dict(kind=kind, seqs=seqs, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, bits=bits,
                window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]), cap=cap, bias=bias, prefix=prefix,
                gain=round(rng.uniform(1.0, 5.0), 1) if cap else 1.0, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, tokens with them) of each sequence: the first has all, the others between 30 and 100 %."""
    part = [1.0 if b == 0 else 0.3 + 0.7 * ((b * 2654435761) % 1000) / 1000 for b in range(case["seqs"])]
    new = [max(1, int(case["new"] * p)) for p in part]
    old = [int((case["ctx"] - case["new"]) * p) for p in part]
    return new, [n + o for n, o in zip(new, old)]


def _prefixes(case):
    """Tokens of each sequence that all its rows see: none, or a part of it that differs by sequence."""
    return [int(case["prefix"] * (0.5 + 0.5 * ((b * 40503) % 64) / 64) * n) for b, n in enumerate(_lengths(case)[1])]


def _slots(case):
    """Slots of each copied page that are copied."""
    return [1 + (i * 40503 + 8) % case["page"] if case["part"] else case["page"] for i in range(case["pairs"])]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _values(g, n, heads, dim, dtype):
    x = torch.randn(n, heads, dim, device="cuda", generator=g)
    loud = torch.rand(heads, dim, device="cuda", generator=g) < 0.02
    return torch.where(loud, 8.0 * x, x).to(dtype)


def _pool(g, pages, case, dtype):
    """Keys or values of a pool of pages that earlier sequences have filled, and their scales."""
    x = _values(g, pages * case["page"], case["kv_heads"], case["dim"], dtype)
    x = x.unflatten(0, (pages, case["page"])).transpose(1, 2).contiguous()
    bits = case["bits"]
    if bits == 16:
        return x, None
    groups = x.float().unflatten(-1, (-1, 32))
    s = (groups.abs().amax(-1) / _MOST[bits]).clamp(max=65504.0).half()
    c = torch.round(groups / torch.where(s > 0, s.float(), 1.0).unsqueeze(-1)).clamp(-_MOST[bits], _MOST[bits]).flatten(-2)
    c = (c + (128 if bits == 8 else 8)).to(torch.uint8)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c, s.transpose(2, 3).contiguous()


def _prepare_attend(case, g):
    dtype = _DTYPES[case["dtype"]]
    new, lens = _lengths(case)
    need = [-(-n // case["page"]) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    i32 = dict(dtype=torch.int32, device="cuda")
    state = dict(case=case, dtype=dtype, table=table, lens=torch.tensor(lens, **i32), tokens=sum(new), max_q=max(new), max_kv=max(lens),
                 starts=torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).cuda())
    state["k"], state["ks"] = _pool(g, pages, case, dtype)
    state["v"], state["vs"] = _pool(g, pages, case, dtype)
    state["q"] = (case["gain"] * torch.randn(sum(new), case["heads"], case["dim"], device="cuda", generator=g)).to(dtype)
    h = torch.arange(1, case["heads"] + 1, dtype=torch.float64)
    state["slopes"] = (2.0 ** (-8.0 * h / case["heads"])).float().cuda() if case["bias"] else None
    state["prefix"] = torch.tensor(_prefixes(case), **i32) if case["prefix"] else None
    return state


def _prepare_copy(case, g):
    pages = case["used"] + 2 * case["pairs"] + 1
    state = dict(case=case, layers=[])
    for _ in range(case["layers"]):
        state["layers"].append([*_pool(g, pages, case, _DTYPES[case["dtype"]]), *_pool(g, pages, case, _DTYPES[case["dtype"]])])
    # which pages is known on the host: a program keeps its free pages and its sequences' pages there
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(case["pairs"])).tolist()
    state["src"], state["dst"] = order[: case["pairs"]], order[case["pairs"] : 2 * case["pairs"]]
    state["slots"] = _slots(case) if case["part"] else None
    return state


def _prepare_norm(case, g):
    dtype, heads, width = _DTYPES[case["dtype"]], case["heads"], case["width"]
    x = _values(g, case["tokens"], heads + case["gap"], width, dtype)[:, :heads]
    x = x if heads > 1 or case["gap"] else x.squeeze(1)
    state = dict(case=case, x=x, residual=None, weight=None)
    if case["residual"]:
        state["residual"] = (5.0 * torch.randn(case["tokens"], width, device="cuda", generator=g)).to(_DTYPES[case["residual"]])
    if case["weight"]:
        state["weight"] = (1.0 + 0.3 * torch.randn(width, device="cuda", generator=g)).to(_DTYPES[case["weight"]])
    return state


def prepare(case, seed):
    return {"attend": _prepare_attend, "copy": _prepare_copy, "norm": _prepare_norm}[case["kind"]](case, _generator(seed))


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _gathered(pool, scales, page, slot, bits):
    """Cached heads [..., kv_heads, dim] in 32 bits of the tokens at (page, slot)."""
    x = pool[page, :, slot]
    if bits == 16:
        return x.float()
    if bits == 4:
        x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
    s = scales[page, :, :, slot].float()
    return ((x.float() - (128 if bits == 8 else 8)).unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _attend(state):
    case = state["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seqs, most_q, most_kv = case["seqs"], state["max_q"], state["max_kv"]
    lens, starts = state["lens"].long(), state["starts"].long()
    n = torch.arange(state["tokens"], device="cuda")
    seq = torch.searchsorted(starts, n, right=True) - 1
    j = n - starts[seq]
    t = torch.arange(most_kv, device="cuda")
    pages = state["table"].long()[:, t // page]
    slots = (t % page).expand(seqs, -1)
    k, v = (_gathered(state[n], state[n + "s"], pages, slots, case["bits"]).permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    q = torch.zeros(seqs, most_q, heads, dim, device="cuda")
    q[seq, j] = state["q"].float()
    q = q.unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).reshape(seqs * kv_heads, -1, dim)
    k, v = k.flatten(0, 1), v.flatten(0, 1)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(dim))
    if case["cap"]:
        s.div_(case["cap"]).tanh_().mul_(case["cap"])
    s = s.view(seqs, kv_heads, -1, most_q, most_kv)
    at = (lens - (starts[1:] - starts[:-1])).unsqueeze(1) + torch.arange(most_q, device="cuda")
    if case["bias"]:
        s -= state["slopes"].view(1, kv_heads, -1, 1, 1) * (at.unsqueeze(-1) - t).abs().float().view(seqs, 1, 1, most_q, most_kv)
    seen = t <= at.unsqueeze(-1)
    if case["prefix"]:
        seen |= t < state["prefix"].view(-1, 1, 1)
    seen &= t < lens.view(-1, 1, 1)
    if case["window"]:
        seen &= t > at.unsqueeze(-1) - case["window"]
    s.masked_fill_(~seen.view(seqs, 1, 1, most_q, most_kv), -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True).clamp(min=-3.0e38)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.bmm(p.view(seqs * kv_heads, -1, most_kv), v).view(seqs, kv_heads, -1, most_q, dim)
    y = (y / torch.where(total > 0, total, 1.0)).permute(0, 3, 1, 2, 4).reshape(seqs, most_q, heads, dim)
    return y[seq, j].to(state["dtype"])


def _copy(state):
    case = state["case"]
    src, dst = (torch.tensor(state[n], device="cuda") for n in ("src", "dst"))
    if not case["part"]:
        for layer in state["layers"]:
            for x in layer:
                if x is not None:
                    x[dst] = x[src]
        return _copied(state)
    slots = torch.tensor(state["slots"], device="cuda")
    pair = torch.repeat_interleave(torch.arange(case["pairs"], device="cuda"), slots)
    slot = torch.arange(pair.numel(), device="cuda") - (slots.cumsum(0) - slots)[pair]
    a, b = src[pair], dst[pair]
    for k, ks, v, vs in state["layers"]:
        for x in (k, v):
            x[b, :, slot] = x[a, :, slot]
        for s in (ks, vs):
            if s is not None:
                s[b, :, :, slot] = s[a, :, :, slot]
    return _copied(state)


def _copied(state):
    return [x for layer in state["layers"] for x in layer if x is not None]


def _norm(state):
    x = state["x"].float()
    if state["residual"] is not None:
        x = x + state["residual"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    if state["weight"] is not None:
        y = y * state["weight"].float()
    y = y.to(state["x"].dtype)
    return y if state["residual"] is None else (y, x.to(state["residual"].dtype))


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(state):
    import mlxl3_amd

    case = state["case"]
    if case["kind"] == "norm":
        return mlxl3_amd.rms_norm(state["x"], state["weight"], eps=_EPS, residual=state["residual"])
    if "kept" not in state:  # the handles that a serving program makes once
        if case["kind"] == "copy":
            state["kept"] = mlxl3_amd.KvPages([mlxl3_amd.KvCache(k, v, ks, vs, bits=case["bits"]) for k, ks, v, vs in state["layers"]])
        else:
            state["kept"] = (
                mlxl3_amd.KvCache(state["k"], state["v"], state["ks"], state["vs"], bits=case["bits"]),
                mlxl3_amd.KvBatch(state["starts"], state["lens"], state["table"], max_q=state["max_q"], max_kv=state["max_kv"]),
            )
    if case["kind"] == "copy":
        state["kept"].copy(state["src"], state["dst"], state["slots"])
        return _copied(state)
    cache, batch = state["kept"]
    return mlxl3_amd.attention(state["q"], cache, batch, window=case["window"], softcap=case["cap"], slopes=state["slopes"],
                               prefix=state["prefix"])


def run(state):
    if own:
        return _own(state)
    return {"attend": _attend, "copy": _copy, "norm": _norm}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
_SIZE = {"f16": 2, "bf16": 2, "f32": 4, "": 0}


def _token_bytes(case):
    """Of a token's keys and values in one cache."""
    return 2 * case["kv_heads"] * case["dim"] * (2.0 if case["bits"] == 16 else case["bits"] / 8 + 2 / 32)


def work(case):
    if case["kind"] == "norm":
        n = case["tokens"] * case["heads"] * case["width"]
        return {"bytes": n * 2 * (_SIZE[case["dtype"]] + _SIZE[case["residual"]]) + case["width"] * _SIZE[case["weight"]],
                "flops": n * (4 + bool(case["residual"]))}
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * _token_bytes(case) * sum(_slots(case)), "flops": 0}
    new, lens = _lengths(case)
    prefix = _prefixes(case)
    pairs = seen = 0
    for n, total, pre in zip(new, lens, prefix):
        first, pre = total - n, min(pre, total)
        w = case["window"] or total
        seen += total - max(0, first - w + 1)
        for i in range(first, total):
            pairs += max(i + 1, pre) - max(0, i - w + 1)
    return {"bytes": 2 * _SIZE[case["dtype"]] * sum(new) * case["heads"] * case["dim"] + _token_bytes(case) * seen,
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
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


def _attend64(case, state):
    new, lens = _lengths(case)
    prefix = _prefixes(case)
    group = case["heads"] // case["kv_heads"]
    y = torch.zeros(sum(new), case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        k, v = _sequence64(state, "k", b), _sequence64(state, "v", b)
        away = torch.arange(total - n, total, device="cuda")[:, None] - torch.arange(total, device="cuda")
        hidden = away < 0
        hidden[:, : prefix[b]] = False
        if case["window"]:
            hidden |= away >= case["window"]
        for h in range(case["heads"]):
            z = (state["q"][start : start + n, h].double() @ k[:, h // group].T) / math.sqrt(case["dim"])
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if case["bias"]:
                z = z - float(state["slopes"][h]) * away.abs().double()
            y[start : start + n, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
        start += n
    return y


def _copy64(case, state):
    slots = _slots(case)
    for layer in state["layers"]:
        for i, x in enumerate(layer):
            if x is None:
                continue
            for a, b, n in zip(state["src"], state["dst"], slots):
                if i % 2:
                    x[b, :, :, :n] = x[a, :, :, :n]
                else:
                    x[b, :, :n] = x[a, :, :n]
    return _copied(state)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attend":
        return _attend64(case, state)
    if case["kind"] == "copy":
        return _copy64(case, state)
    rows = state["x"].double()
    if state["residual"] is not None:
        rows = rows + state["residual"].double()
    size = torch.linalg.vector_norm(rows, dim=-1, keepdim=True) ** 2 / case["width"]
    y = rows / (size + _EPS).sqrt()
    if state["weight"] is not None:
        y = y * state["weight"].double()
    return y if state["residual"] is None else (y, rows)
