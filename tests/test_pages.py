"""KvPages and exl3_kv_copy_pages without a GPU: what is refused before any launch, and the
bookkeeping against sequences that are kept as plain lists (copies are done on the host)."""

import ctypes
import random

import pytest
import torch

import mlxl3_amd
from mlxl3_amd import KvCache, KvPages, kv

pytestmark = pytest.mark.skipif(not mlxl3_amd.LIB_PATH.exists(), reason="libexl3_hip.so not built")
FAKE = 0x1000  # never dereferenced


def handle(pages=8, page=16, heads=2, dim=128, fmt=9):
    h = ctypes.c_void_p()
    coded = FAKE if fmt in (4, 8) else None
    assert mlxl3_amd.load_library().exl3_kv_cache_create(FAKE, FAKE, coded, coded, fmt, pages, page, heads, dim, ctypes.byref(h)) == 0
    return h


def copy(handles, src, dst, slots=None, pairs=None, count=None):
    lib = mlxl3_amd.load_library()
    c = None if handles is None else (ctypes.c_void_p * len(handles))(*[None if h is None else h.value for h in handles])
    ints = lambda a: None if a is None else (ctypes.c_int32 * len(a))(*a)
    rc = lib.exl3_kv_copy_pages(c, len(handles or ()) if count is None else count, ints(src), ints(dst), ints(slots),
                                len(src or ()) if pairs is None else pairs, None)
    return rc, lib.exl3_last_error().decode()


@pytest.mark.parametrize("src, dst, slots, kw, msg", [
    ([0], [8], None, {}, "page 8 of a pool of 8"),
    ([-1], [1], None, {}, "page -1 of a pool of 8"),
    ([8], [1], None, {}, "page 8 of a pool of 8"),
    ([0], [0], None, {}, "page 0 is copied and copied to"),
    ([0, 1], [2, 2], None, {}, "page 2 is copied to twice"),
    ([0, 1], [1, 2], None, {}, "page 1 is copied and copied to"),
    ([3, 2, 7], [6, 5, 3], None, {}, "page 3 is copied and copied to"),
    ([0], [1], [17], {}, "17 slots of a page of 16"),
    ([0], [1], [-1], {}, "-1 slots of a page of 16"),
    ([0], [1], None, dict(pairs=-1), "negative page count"),
    ([0] * 9, list(range(9)), None, {}, "9 copies among 8 pages"),
    (None, [1], None, dict(pairs=1), "null page list"),
    ([1], None, None, dict(pairs=1), "null page list"),
])
def test_refused_lists(src, dst, slots, kw, msg):
    h = handle()
    try:
        rc, err = copy([h], src, dst, slots, **kw)
        assert rc == -1 and msg in err
    finally:
        mlxl3_amd.load_library().exl3_kv_cache_destroy(h)


def test_long_lists_are_refused_alike():
    h = handle(pages=1000)
    try:
        src, dst = list(range(400)), list(range(400, 800))
        dst[399] = dst[3]
        assert "page 403 is copied to twice" in copy([h], src, dst)[1]
        dst[399] = 17
        assert "page 17 is copied and copied to" in copy([h], src, dst)[1]
    finally:
        mlxl3_amd.load_library().exl3_kv_cache_destroy(h)


def test_refused_caches():
    lib = mlxl3_amd.load_library()
    made = [handle(), handle(pages=9), handle(page=32), handle(heads=4, fmt=8)]
    try:
        assert copy([made[0], made[1]], [0], [1]) == (-1, "KV caches whose pages are copied together have as many pages of as many tokens")
        assert copy([made[0], made[2]], [0], [1])[0] == -1
        assert copy([made[0], None], [0], [1]) == (-1, "null KV cache")
        assert copy(None, [0], [1], count=1)[0] == -1
        assert "at least one KV cache" in copy([], [0], [1])[1]
        assert copy([made[0], made[3]], [], [])[0] == 0  # nothing to copy
        lib.exl3_debug_fail_launch(b"KV page copy")
        assert copy([made[0], made[3]], [0], [1]) == (-2, "KV page copy: forced launch failure")
    finally:
        lib.exl3_debug_fail_launch(None)
        for h in made:
            lib.exl3_kv_cache_destroy(h)


class HostCache(KvCache):
    """What KvPages asks of a cache, on the host."""

    def __init__(self, pages, page, device="cpu"):
        self.pages, self.page_tokens, self.device = pages, page, torch.device(device)
        self._handle = handle(pages, page)
        self._destroy = mlxl3_amd.load_library().exl3_kv_cache_destroy


class HostPages(KvPages):
    """Copies what the caches would hold, one number a slot, and checks the lists as the library does."""

    def __init__(self, pages=12, page=16):
        super().__init__([HostCache(pages, page) for _ in range(2)])
        self.slots = [[None] * page for _ in range(pages)]
        self.copied = 0
        self.fail = False

    def copy(self, src, dst, tokens=None):
        if self.fail:
            raise mlxl3_amd.Exl3Error(-2, "forced")
        tokens = [self.page_tokens] * len(src) if tokens is None else tokens
        assert len(set(dst)) == len(dst) and not set(src) & set(dst) and len(src) == len(dst) == len(tokens)
        for a, b, n in zip(src, dst, tokens):
            assert 0 <= n <= self.page_tokens
            self.slots[b][:n] = self.slots[a][:n]
        self.copied += len(src)


def read(pages, seq):
    p = pages.page_tokens
    return [pages.slots[pages.pages_of(seq)[t // p]][t % p] for t in range(pages.tokens(seq))]


def write(pages, seq, n, value):
    """What an append of the newest n tokens writes."""
    p, total = pages.page_tokens, pages.tokens(seq)
    for t in range(total - n, total):
        pages.slots[pages.pages_of(seq)[t // p]][t % p] = (value, t)


def consistent(pages):
    uses = [0] * pages.pages
    for s in pages.sequences:
        held = pages.pages_of(s)
        assert len(held) == -(-pages.tokens(s) // pages.page_tokens)
        for p in held:
            uses[p] += 1
    assert uses == pages._uses
    assert sorted(pages._free) == [p for p in range(pages.pages) if uses[p] == 0] and pages.free_pages == len(pages._free)


@pytest.mark.parametrize("seed", range(6))
def test_sequences_keep_their_tokens(seed):
    """Random forks, growth, cuts, ends and compactions: every sequence holds what was written to it."""
    rng = random.Random(seed)
    pages = HostPages(rng.choice([6, 20, 60]), rng.choice([16, 32]))
    want: dict = {}
    for step in range(400):
        act = rng.choice(["new", "grow", "grow", "grow", "fork", "fork", "cut", "free", "compact"])
        alive = list(want)
        if act == "new":
            n = rng.choice([0, 1, 15, 16, 17, 70])
            if -(-n // pages.page_tokens) <= pages.free_pages:
                s = pages.new(n)
                write(pages, s, n, step)
                want[s] = [(step, t) for t in range(n)]
            else:
                with pytest.raises(mlxl3_amd.Exl3Error, match="pages needed"):
                    pages.new(n)
        elif act == "compact":
            before = pages.free_pages
            pages.compact()
            assert pages.free_pages == before
            assert all(p < pages.pages - before for s in want for p in pages.pages_of(s))
        elif not alive:
            continue
        elif act == "grow":
            some = rng.sample(alive, rng.randint(1, len(alive)))
            more = [rng.choice([0, 1, 1, 5, 16, 40]) for _ in some]
            try:
                pages.grow(some, more)
            except mlxl3_amd.Exl3Error as e:
                assert "pages needed" in str(e)
            else:
                for i, (s, n) in enumerate(zip(some, more)):
                    write(pages, s, n, (step, i))
                    want[s] += [((step, i), len(want[s]) + t) for t in range(n)]
        elif act == "fork":
            s = rng.choice(alive)
            copied = pages.copied
            want[pages.fork(s)] = list(want[s])
            assert pages.copied == copied
        elif act == "cut":
            s = rng.choice(alive)
            n = rng.randint(0, len(want[s]))
            pages.cut(s, n)
            del want[s][n:]
        else:
            s = rng.choice(alive)
            pages.free(s)
            del want[s]
        assert pages.sequences == list(want)
        consistent(pages)
        for s, w in want.items():
            assert read(pages, s) == w, (step, act)


def test_a_failed_copy_changes_nothing():
    pages = HostPages()
    a = pages.new(20)
    b = pages.fork(a)
    c = pages.new(40)
    pages.free(a)
    pages.grow(b, 0)
    a = pages.fork(b)
    pages.fail = True
    state = lambda: ([pages.pages_of(s) for s in pages.sequences], [pages.tokens(s) for s in pages.sequences], list(pages._uses),
                     sorted(pages._free))
    before = state()
    with pytest.raises(mlxl3_amd.Exl3Error, match="forced"):
        pages.grow([a, c], [3, 30])
    assert state() == before
    pages.free(a)
    pages.free(b)
    before = state()
    with pytest.raises(mlxl3_amd.Exl3Error, match="forced"):
        pages.compact()
    assert state() == before
    with pytest.raises(mlxl3_amd.Exl3Error, match="pages needed"):
        pages.new(1000)
    assert state() == before and pages.sequences == [c]


def test_batches():
    pages = HostPages()
    a, b = pages.new(40), pages.new(3)
    c = pages.fork(a)
    batch = pages.batch([b, c, a], new=[3, 2, 0])
    assert batch.q_starts.tolist() == [0, 3, 5, 5] and batch.kv_lens.tolist() == [3, 40, 40]
    assert batch.block_table.tolist()[1] == pages.pages_of(a) and batch.block_table.tolist()[0][:1] == pages.pages_of(b)
    assert (batch._c.max_q, batch._c.max_kv, batch._c.table_pages) == (3, 40, 3)
    one = pages.batch(a)
    assert one.q_starts.tolist() == [0, 1] and one._c.max_q == 1
    empty = pages.new()
    assert pages.batch([empty], 0).kv_lens.tolist() == [0]
    assert pages.batch([a], max_kv=1000)._c.max_kv == 1000


@pytest.fixture
def host_batches(monkeypatch):
    monkeypatch.setattr(kv, "_device_tensor", lambda t, *a: t)


test_batches = pytest.mark.usefixtures("host_batches")(test_batches)


def test_refusals(host_batches):
    err = mlxl3_amd.Exl3Error
    pages = HostPages()
    a = pages.new(20)
    for call, msg in [
        (lambda: pages.grow(a + 5), "unknown sequence"),
        (lambda: pages.grow([a, a]), "a sequence is listed once"),
        (lambda: pages.grow([a], [1, 2]), "for each sequence"),
        (lambda: pages.grow(a, -1), "not negative"),
        (lambda: pages.grow(a, 1.5), "whole numbers"),
        (lambda: pages.grow("a"), "whole numbers"),
        (lambda: pages.grow(a, 2**31 - 1), "fewer than 2"),
        (lambda: pages.grow(a, 2**40), "32 bits"),
        (lambda: pages.new(-3), "not negative"),
        (lambda: pages.cut(a, 21), "21 of 20 tokens"),
        (lambda: pages.cut(a, -1), "-1 of 20 tokens"),
        (lambda: pages.cut(a, None), "whole numbers"),
        (lambda: pages.fork([a]), "unknown sequence"),
        (lambda: pages.free(None), "unknown sequence"),
        (lambda: pages.tokens(7), "unknown sequence"),
        (lambda: pages.batch([]), "at least one sequence"),
        (lambda: pages.batch([a], 21), "among its tokens"),
        (lambda: pages.batch([a], [1, 2]), "at least one sequence"),
        (lambda: KvPages([]), "at least one KvCache"),
        (lambda: KvPages([1]), "at least one KvCache"),
        (lambda: KvPages([HostCache(8, 16), HostCache(9, 16)]), "as many pages"),
        (lambda: KvPages([HostCache(8, 16), HostCache(8, 32)]), "as many pages"),
        (lambda: KvPages([HostCache(8, 16), HostCache(8, 16, "meta")]), "a cache is on meta"),
    ]:
        with pytest.raises(err, match=msg):
            call()
    assert pages.sequences == [a] and pages.tokens(a) == 20
    consistent(pages)


def test_lists_that_copy_refuses(monkeypatch):
    from mlxl3_amd import pages as module

    monkeypatch.setattr(module._kv, "_launch", lambda device, entry, *args: kv._check(entry(*args, None)))
    pages = KvPages(HostCache(8, 16))
    err = mlxl3_amd.Exl3Error
    for args, msg in [
        (([0], [1, 2]), "as many sources"),
        (([0], [1], [1, 2]), "as many sources"),
        (([0.5], [1]), "whole numbers"),
        (([2**32], [1]), "32 bits"),
        ((torch.tensor([0.0]), [1]), "on the host"),
        ((torch.tensor([[0]]), [1]), "on the host"),
        ((3, [1]), "whole numbers"),
        (([0], [8]), "page 8 of a pool of 8"),
        (([0, 0], [1, 1]), "copied to twice"),
        (([0, 1], [1, 2]), "copied and copied to"),
        (([0], [1], [17]), "17 slots"),
    ]:
        with pytest.raises(err, match=msg):
            pages.copy(*args)
    pages.copy([], [])
    pages.copy(torch.tensor([], dtype=torch.int32), [], [])
