"""Appends to pages that sequences share, on the GPU: what is refused writes nothing, what the oldest
sequence fills all that share it read."""

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import KvCache, KvPages

pytestmark = pytest.mark.gpu


def some(seed, n):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, 2, 64, generator=g).half().cuda() for _ in range(2)]


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_room_made_before_a_fork(bits):
    cache = KvCache.zeros(12, 16, 2, 64, bits=bits)
    alone = KvCache.zeros(12, 16, 2, 64, bits=bits)
    pages, single = KvPages(cache), KvPages(alone)
    held = lambda: [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]
    read = lambda s: cache.read(pages.batch(s, pages.tokens(s)), pages.tokens(s))
    a, w = pages.new(20), single.new(20)
    b = pages.fork(a)
    was = held()
    for seqs, n in (([a, b], 40), ([b], 20), ([a, a], 40)):
        with pytest.raises(mlxl3_amd.Exl3Error, match="shared|twice"):
            cache.append(pages.batch(seqs, 20), *some(1, n))
    assert all(torch.equal(x, y) for x, y in zip(held(), was))
    k, v = some(2, 20)
    cache.append(pages.batch(a, 20), k, v)
    alone.append(single.batch(w, 20), k, v)
    want = alone.read(single.batch(w, 20), 20)
    for s in (a, b):
        assert all(torch.equal(x, y) for x, y in zip(read(s), want))
    pages.grow([a, b], 3)  # their own from here on
    cache.append(pages.batch([a, b], 3), *some(3, 6))
    more = [[x[:3] for x in some(3, 6)], [x[3:] for x in some(3, 6)]]
    for s, (k, v) in zip((a, b), more):
        single.grow(w, 3)
        alone.append(single.batch(w, 3), k.contiguous(), v.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(read(s), alone.read(single.batch(w, 23), 23)))
        single.cut(w, 20)
