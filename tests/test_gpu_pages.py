"""Copies of cache pages on the GPU: every format, filled slots and whole pages, many layers and many
pages, layers of differing shapes, everything else as it was; sequences that are forked, grown, cut and
compacted read what was appended to them."""

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import KvCache, KvPages

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def cache(seed, pages, page, heads, dim, bits, dtype=F16):
    """A cache of random bytes (any code, any scale, NaNs among 16-bit values)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    some = lambda *shape: torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
    if bits == 16:
        k, v = (some(pages, heads, page, 2 * dim).view(dtype) for _ in range(2))
        return KvCache(k, v)
    k, v = (some(pages, heads, page, dim * bits // 8) for _ in range(2))
    return KvCache(k, v, *(some(pages, heads, dim // 32, 2 * page).view(F16) for _ in range(2)), bits=bits)


def tensors(c):
    return [t.view(torch.uint8) if t.dtype == torch.uint8 else t.view(torch.int16) for t in (c.k, c.v, c.k_scales, c.v_scales) if t is not None]


def check(caches, src, dst, slots=None):
    before = [[t.clone() for t in tensors(c)] for c in caches]
    KvPages(caches).copy(src, dst, slots)
    for c, old in zip(caches, before):
        for i, (t, w) in enumerate(zip(tensors(c), old)):
            for a, b, n in zip(src, dst, slots or [c.page_tokens] * len(src)):
                if i < 2:
                    w[b, :, :n] = w[a, :, :n]
                else:
                    w[b, :, :, :n] = w[a, :, :, :n]
            assert torch.equal(t, w), i


@pytest.mark.parametrize("bits, dtype", [(16, F16), (16, BF16), (8, F16), (4, F16)])
@pytest.mark.parametrize("page, heads, dim", [(16, 1, 64), (16, 8, 128), (32, 3, 256), (128, 2, 128), (1024, 1, 64), (64, 5, 64)])
def test_formats_and_slots(bits, dtype, page, heads, dim):
    caches = [cache(page + i, 12, page, heads, dim, bits, dtype) for i in range(3)]
    check(caches, [3], [7])
    check(caches, [0, 11, 5, 0], [1, 2, 8, 9])
    for n in {1, 2, 7, 8, 9, 15, 16, page // 2 + 1, page - 1, page}:
        check(caches, [4], [6], [n])
    check(caches, [0, 11, 5, 0, 3], [1, 2, 8, 9, 10], [page, 1, page - 1, 0, 9])
    check(caches, [0], [1], [0])
    check(caches, [], [])


def test_more_pages_and_caches_than_a_launch_names():
    caches = [cache(i, 700, 16, 1, 64, 4) for i in range(70)]
    order = torch.randperm(700, generator=torch.Generator().manual_seed(1)).tolist()
    check(caches, order[:340], order[340:680])
    check(caches, order[:340], order[340:680], [i % 17 for i in range(340)])
    check(caches[:1], [5] * 600, [p for p in range(601) if p != 5])


def test_layers_of_differing_shapes():
    caches = [cache(1, 9, 32, 8, 128, 16), cache(2, 9, 32, 2, 256, 8), cache(3, 9, 32, 8, 128, 16, BF16), cache(4, 9, 32, 8, 128, 16),
              cache(5, 9, 32, 2, 256, 4), cache(6, 9, 32, 2, 64, 8), cache(7, 9, 32, 2, 256, 8)]
    check(caches, [0, 8], [4, 5], [32, 11])


def test_a_cache_listed_twice_and_lists_of_other_kinds():
    c = cache(1, 9, 16, 2, 64, 8)
    check([c, c], [1], [2])
    was = [t.clone() for t in tensors(c)]
    KvPages([c]).copy(torch.tensor([3], dtype=torch.int64), (4,), torch.tensor([5]).numpy())
    assert torch.equal(c.k[4, :, :5], was[0][3, :, :5]) and torch.equal(c.k[4, :, 5:], was[0][4, :, 5:])
    with pytest.raises(mlxl3_amd.Exl3Error, match="on the host"):
        KvPages([c]).copy(torch.tensor([3], device="cuda"), [4])


def test_pages_beyond_32_bits():
    """A pool of more than 4 GiB a side."""
    n = (1 << 32) // (16 * 8 * 256) + 40
    c = KvCache.zeros(n, 16, 8, 128, dtype=BF16)
    c.k[n - 1] = 1.5
    c.v[3] = 2.5
    KvPages([c]).copy([n - 1, 3], [0, n - 2], [16, 9])
    assert bool((c.k[0] == 1.5).all()) and bool((c.v[n - 2, :, :9] == 2.5).all()) and bool((c.v[n - 2, :, 9:] == 0).all())
    assert bool((c.k[1] == 0).all()) and bool((c.k[n - 2, :, :9] == 0).all()) and bool((c.v[0] == 0).all())


def test_other_streams_and_captured_graphs():
    c = cache(1, 40, 32, 4, 128, 8)
    pages = KvPages([c])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pages.copy([1], [2])
        pages.copy([2], [3], [9])
    s.synchronize()
    assert torch.equal(c.k[2], c.k[1]) and torch.equal(c.k[3, :, :9], c.k[1, :, :9])
    lists = [5, 6], [7, 8], [32, 5]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pages.copy(*lists)
    lists[0][:] = [0, 0]  # the graph keeps its own
    for i in range(3):
        c.k[5], c.v[6] = i + 1, i + 2
        was = c.v[8, :, 5:].clone()
        g.replay()
        torch.cuda.synchronize()
        assert bool((c.k[7] == i + 1).all()) and bool((c.v[8, :, :5] == i + 2).all()) and torch.equal(c.v[8, :, 5:], was)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_forked_sequences_read_what_was_appended_to_them(bits):
    """Two layers, one pool: prompts, forks, tokens appended to some, drafts cut, ends, a compaction; every
    sequence reads what a cache of its own holds."""
    layers = [KvCache.zeros(40, 16, 2, 64, bits=bits) for _ in range(2)]
    alone = [KvCache.zeros(200, 16, 2, 64, bits=bits) for _ in range(2)]
    pages, single = KvPages(layers), KvPages(alone)
    gen, want = torch.Generator().manual_seed(bits), {}

    def append(seqs, new):
        new = [new] * len(seqs)
        pages.grow(seqs, new)
        single.grow([want[s] for s in seqs], new)
        a, b = pages.batch(seqs, new), single.batch([want[s] for s in seqs], new)
        for one, two in zip(layers, alone):
            k, v = (torch.randn(sum(new), 2, 64, generator=gen).half().cuda() for _ in range(2))
            one.append(a, k, v)
            two.append(b, k, v)

    def copied(seq):
        """The sequence `single` keeps for it, page by page its own."""
        n = single.tokens(seq)
        other = single.new(n)
        if n:
            single.copy(single.pages_of(seq), single.pages_of(other))
        return other

    def same():
        for s, w in want.items():
            n = pages.tokens(s)
            assert n == single.tokens(w)
            if n == 0:
                continue
            for one, two in zip(layers, alone):
                for x, y in zip(one.read(pages.batch(s, n), n), two.read(single.batch(w, n), n)):
                    assert torch.equal(x, y), s

    def new():
        s = pages.new()
        want[s] = single.new()
        return s

    def fork(s):
        t = pages.fork(s)
        want[t] = copied(want[s])
        return t

    a, b = new(), new()
    append([a], 37)
    append([b], 16)
    same()
    forks = [fork(a) for _ in range(3)] + [fork(b)]
    append(forks[:2] + [a], 1)      # three of four that share a page write to it
    same()
    append(forks, 5)
    same()
    for s, n in ((a, 33), (forks[0], 20), (forks[3], 16)):
        pages.cut(s, n)
        single.cut(want[s], n)
    c = fork(forks[0])
    append([a, forks[0], c, forks[3]], 3)
    same()
    for s in (forks[1], b):
        pages.free(s)
        del want[s]
    same()
    used = 40 - pages.free_pages
    pages.compact()
    assert 40 - pages.free_pages == used and all(p < used for s in want for p in pages.pages_of(s))
    same()
    append(list(want), 20)
    same()
