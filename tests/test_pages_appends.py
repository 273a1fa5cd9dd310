"""Which sequence appends to a page that several share, without a GPU: room made before a fork is the
oldest one's to fill, nothing is appended through a batch whose pages are others' by now."""

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import Exl3Attention, KvBatch, KvPages, kv
from test_pages import HostCache

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")
PAGE = 16


class Cache(HostCache):
    """A cache that notes what is appended to it."""

    kv_heads, head_dim = 2, 64


@pytest.fixture
def launched(monkeypatch):
    """The entries that calls would launch: tensors stay on the host."""
    names = []
    monkeypatch.setattr(kv, "_device_tensor", lambda t, *a: t)
    monkeypatch.setattr(kv, "_launch", lambda device, entry, *args: names.append(entry.__name__))
    return names


def made():
    caches = [Cache(12, PAGE) for _ in range(2)]
    return caches, KvPages(caches)


def append(caches, batch):
    n = int(batch.q_starts[-1])
    k = torch.zeros(n, 2, 64, dtype=torch.float16)
    for c in caches:
        c.append(batch, k, k)


def refused(caches, batch, names, match):
    names.clear()
    with pytest.raises(mlxl3_amd.Exl3Error, match=match):
        append(caches, batch)
    assert not names


def test_room_made_before_a_fork_is_filled_once(launched):
    caches, pages = made()
    a = pages.new(20)
    b = pages.fork(a)
    c = pages.fork(b)
    refused(caches, pages.batch([a, b], 20), launched, "shared")  # every slot from two rows at once
    refused(caches, pages.batch([b], 20), launched, "shared")
    append(caches, pages.batch([a], 20))
    assert launched == ["exl3_kv_append"] * 2
    refused(caches, pages.batch([b, c], [3, 0]), launched, "shared")
    append(caches, pages.batch([b, c], 0))  # reads, and what appends nothing, of pages that are shared
    pages.grow([a, b, c], [1, 2, 3])  # their own from here on
    append(caches, pages.batch([a, b, c], [1, 2, 3]))


def test_a_draft_s_room(launched):
    """A fork between a growth and its append: the draft is the older one's, the younger one's after a cut."""
    caches, pages = made()
    a = pages.new(20)
    append(caches, pages.batch(a, 20))
    pages.grow(a, 5)
    b = pages.fork(a)
    refused(caches, pages.batch([a, b], 5), launched, "shared")
    pages.cut(b, 20)
    pages.grow(b, 5)
    append(caches, pages.batch([a, b], 5))


def test_pages_are_the_oldest_holder_s(launched):
    caches, pages = made()
    a = pages.new(20)
    b, c = pages.fork(a), pages.fork(a)
    pages.free(a)
    refused(caches, pages.batch([c], 20), launched, "shared")
    append(caches, pages.batch([b], 20))
    pages.free(b)
    append(caches, pages.batch([c], 20))  # nobody else's now


def test_a_sequence_that_is_listed_twice(launched):
    caches, pages = made()
    a = pages.new(20)
    refused(caches, pages.batch([a, a], 1), launched, "twice")
    append(caches, pages.batch([a, a], [1, 0]))


def test_batches_made_before_the_pages_changed(launched):
    caches, pages = made()
    a = pages.new(40)
    b = pages.new(20)
    old = pages.batch([a, b], [40, 20])
    append(caches, old)
    pages.new(3)
    pages.grow(a, 30)
    append(caches, old)  # what others do to their pages does not matter
    cut = pages.batch([a], 30)
    pages.cut(a, 10)
    refused(caches, cut, launched, "before")
    last = pages.batch([b], 1)
    pages.compact()
    refused(caches, last, launched, "before")
    last = pages.batch([b], 1)
    pages.free(b)
    refused(caches, last, launched, "before")


def test_the_block_asks_too(launched, monkeypatch):
    """Before anything is launched."""
    caches, pages = made()

    class Part:
        k = cb = 0
        in_features = out_features = 128
        trellis, device, handle = None, torch.device("cpu"), None

    block = Exl3Attention(*[Part()] * 4)
    b = pages.fork(pages.new(20))
    x = torch.zeros(20, 128, dtype=torch.float16)
    with pytest.raises(mlxl3_amd.Exl3Error, match="shared"):
        block(x, caches[0], pages.batch([b], 20))
    assert not launched


def test_batches_of_others_are_not_asked(launched):
    caches, _ = made()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    append(caches, KvBatch(i32(0, 2, 4), i32(2, 2), i32(0, 0).view(2, 1), max_q=2))
    assert launched == ["exl3_kv_append"] * 2
