"""Decoder layers as a serving program puts them together -- norm, attention block with capped and biased
scores, norm with the residual, feed-forward -- over sequences that KvPages keeps: prompts with a prefix,
forks, drafts that are cut, a compaction, captured steps."""

import pytest
import torch

import mlxl3_amd
import scores_ref
from mlxl3_amd import KvCache, KvPages, synth
from test_gpu_attention import F16, projections
from test_gpu_norm import reference
from test_gpu_norm import within as near

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, DIM = 512, 8, 2, 64


def mlp(seed):
    def one(i, n_in, n_out):
        tr, suh, svh, _ = synth.linear_layer(seed, i, n_in, n_out, 4)
        dev = lambda a: torch.from_numpy(a.view("int16") if a.dtype.name == "uint16" else a).cuda()
        return mlxl3_amd.Exl3Linear(dev(tr), dev(suh), dev(svh), None, 4, 0)

    return mlxl3_amd.Exl3Mlp(one(10, HIDDEN, 1024), one(11, HIDDEN, 1024), one(12, 1024, HIDDEN))


class Layer:
    def __init__(self, seed, softcap, biased):
        g = torch.Generator().manual_seed(seed)
        self.softcap = softcap
        self.slopes = (2.0 ** -torch.arange(1, HEADS + 1).float()).cuda() if biased else None
        rope = None if biased else mlxl3_amd.Rope(mlxl3_amd.rope_frequencies(DIM)[0].cuda())
        # the synthetic projections multiply by 30 to 40; f16 holds 65504
        self.norms = [((1 + 0.2 * torch.randn(HIDDEN, generator=g)) / 32).half().cuda() for _ in range(2)]
        self.parts = projections(seed, HIDDEN, HEADS, KV_HEADS, DIM, 4, 0, False)
        self.rope = rope
        self.block = mlxl3_amd.Exl3Attention(*self.parts, rope=rope, softcap=softcap, slopes=self.slopes)
        self.mlp = mlp(seed)

    def __call__(self, part, h, cache, batch, prefix=None):
        """What is still to be added to the stream h, which is updated in place."""
        if part is None:
            x = mlxl3_amd.rms_norm(h, self.norms[0], dtype=F16)
        else:
            x, _ = mlxl3_amd.rms_norm(part, self.norms[0], residual=h, total=h)
        a = self.block(x, cache, batch, prefix=prefix)
        x, _ = mlxl3_amd.rms_norm(a, self.norms[1], residual=h, total=h)
        return self.mlp(x)


class Model:
    def __init__(self):
        self.layers = [Layer(1, 5.0, False), Layer(2, 0.0, True), Layer(3, 20.0, True)]
        self.norm = torch.full((HIDDEN,), 0.5, device="cuda")

    def __call__(self, x, caches, batch, prefix=None):
        h, part = x.float(), None  # the stream is kept in 32 bits
        for layer, cache in zip(self.layers, caches):
            part = layer(part, h, cache, batch, prefix)
        return mlxl3_amd.rms_norm(part, self.norm, residual=h)[0]


@pytest.fixture(scope="module")
def model():
    return Model()


def tokens(seed, n):
    return torch.randn(n, HIDDEN, generator=torch.Generator().manual_seed(seed)).half().cuda()


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bits", [16, 8])
def test_sequences_that_share_pages_answer_as_those_that_do_not(model, bits):
    """Prompts with prefixes, forks that go on differently, a draft of which two tokens are kept, an end, a
    compaction: bit for bit what sequences with pages of their own give."""
    shared = [KvCache.zeros(30, 16, KV_HEADS, DIM, bits=bits) for _ in model.layers]
    apart = [KvCache.zeros(90, 16, KV_HEADS, DIM, bits=bits) for _ in model.layers]
    pages, single, to = KvPages(shared), KvPages(apart), {}

    def new():
        s = pages.new()
        to[s] = single.new()
        return s

    def fork(s):
        t = pages.fork(s)
        n = single.tokens(to[s])
        to[t] = single.new(n)
        single.copy(single.pages_of(to[s]), single.pages_of(to[t]))
        return t

    def step(seed, seqs, new_tokens, prefix=None):
        pages.grow(seqs, new_tokens)
        single.grow([to[s] for s in seqs], new_tokens)
        x = tokens(seed, sum(new_tokens))
        y = model(x, shared, pages.batch(seqs, new_tokens), prefix)
        z = model(x, apart, single.batch([to[s] for s in seqs], new_tokens), prefix)
        assert torch.equal(y, z) and bool(y.isfinite().all()), seed
        return y

    a, b = new(), new()
    step(1, [a, b], [70, 21], i32(30, 21))
    free = pages.free_pages
    forks = [fork(a) for _ in range(3)]
    assert pages.free_pages == free
    step(2, [a] + forks, [1] * 4)
    assert pages.free_pages == free - 3  # of four that shared the last page, three copied it
    step(3, [b, forks[0], forks[1]], [1, 5, 1])
    pages.cut(forks[0], 73)
    single.cut(to[forks[0]], 73)
    for s in (a, forks[2]):
        pages.free(s)
        single.free(to.pop(s))
    step(4, [forks[0], b, forks[1]], [1, 1, 1])
    pages.compact()
    c = fork(forks[0])
    for seed in range(5, 9):
        step(seed, [c, forks[0], b, forks[1]], [1] * 4)
    step(9, [b, c], [40, 1], i32(60, 0))


@pytest.mark.parametrize("layer", [0, 1, 2])
def test_a_layer_against_64_bits(model, layer):
    """Norm, block and norm of one layer for a prompt with a prefix and a decoded token, each from its own
    inputs."""
    it = model.layers[layer]
    cache = KvCache.zeros(20, 16, KV_HEADS, DIM)
    pages = KvPages(cache)
    a, b = pages.new(90), pages.new(33)
    prefix = i32(40, 0)
    for new in ([90, 33], [1, 1]):
        if new == [1, 1]:
            pages.grow([a, b])
        n = sum(new)
        part, h = tokens(20 + n, n), tokens(30 + n, n).float() * 3
        batch = pages.batch([a, b], new)
        x, total = mlxl3_amd.rms_norm(part, it.norms[0], residual=h)
        near(x, *reference(part.cpu(), it.norms[0].cpu(), 1e-6, h.cpu(), F16), "norm")
        assert torch.equal(total, part.float() + h)
        y = it.block(x, cache, batch, prefix=prefix)
        q = mlxl3_amd.Exl3Group(it.parts[:3])(x)[0].view(n, HEADS, DIM)
        q = q if it.rope is None else it.rope.apply(q, batch=batch)
        att = mlxl3_amd.attention(q, cache, batch, softcap=it.softcap, slopes=it.slopes, prefix=prefix)
        assert torch.equal(y, it.parts[3](att.view(n, HEADS * DIM)))
        at = 0
        for s, m, pre in ((a, new[0], 40), (b, new[1], 0)):
            length = pages.tokens(s)
            k, v = (t.cpu().double() for t in cache.read(pages.batch(s, length), length))
            want, bound = scores_ref.attend(q[at : at + m].cpu().double(), k, v, length - m, DIM**-0.5, True, 0, it.softcap,
                                            None if it.slopes is None else it.slopes.cpu(), pre, dtype=F16)
            near(att[at : at + m], want, bound, "attention")
            at += m


def test_captured_steps(model):
    """One decode step of all layers captured, replayed as the sequences grow, other work between the
    replays, against eager steps over caches of their own."""
    steps, lens = 5, [37, 90, 12]

    class Side:
        def __init__(self):
            self.caches = [KvCache.zeros(40, 16, KV_HEADS, DIM, bits=8) for _ in model.layers]
            self.pages = KvPages(self.caches)
            self.seqs = [self.pages.new(n) for n in lens]
            model(tokens(1, sum(lens)), self.caches, self.pages.batch(self.seqs, lens))
            self.pages.grow(self.seqs, [steps] * 3)
            self.batch = self.pages.batch(self.seqs, 1, max_kv=200)
            self.x = torch.zeros(3, HIDDEN, dtype=F16, device="cuda")

        def step(self):
            return model(self.x, self.caches, self.batch)

    eager, graphed = Side(), Side()
    for s in (eager, graphed):
        s.batch.kv_lens.copy_(i32(*(n + 1 for n in lens)))
        s.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = graphed.step()
    for i in range(steps):
        for s in (eager, graphed):
            s.batch.kv_lens.copy_(i32(*(n + 1 + i for n in lens)))
            s.x.copy_(tokens(50 + i, 3))
        want = eager.step()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
        for one, two in zip(eager.caches, graphed.caches):
            assert torch.equal(one.k, two.k) and torch.equal(one.v_scales, two.v_scales)
