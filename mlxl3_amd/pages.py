"""Which pages of a model's caches belong to which sequence: sequences share pages, are forked, cut
and freed, pools are compacted.  The bookkeeping is on the host; what has to move is copied in
all layers' caches at once (``exl3_kv_copy_pages`` of ``include/exl3_hip.h``)."""

from __future__ import annotations

import array
import ctypes
import heapq
import operator
import threading
from typing import Optional, Sequence

from . import Exl3Error, _torch, _vp, load_library
from . import kv as _kv
from .kv import KvBatch, KvCache


def _ints(values, name: str):
    """A list, an array or a host tensor of whole numbers of 32 bits."""
    torch = _torch()
    if isinstance(values, torch.Tensor):
        if values.is_cuda or values.is_floating_point() or values.dim() != 1:
            raise Exl3Error(-1, f"{name} must be a list of whole numbers on the host")
        values = values.tolist()
    try:
        return array.array("i", values)
    except (TypeError, ValueError, OverflowError):
        raise Exl3Error(-1, f"{name} must be a list of whole numbers of 32 bits") from None


def _several(values, name: str, each: int = 1) -> list:
    """A list of numbers, or a number `each` times."""
    try:
        value = operator.index(values)
    except TypeError:
        return list(_ints(values, name))
    return list(_ints([value] * each, name))


def _pointer(a):
    return a.buffer_info()[0] if len(a) else None


class _Held:
    """A sequence: its pages in order and its tokens."""

    __slots__ = ("pages", "tokens")

    def __init__(self, pages, tokens):
        self.pages, self.tokens = pages, tokens


class _Appended:
    """What an append of a batch is asked: the pages that it writes, (sequence, number of the first
    page, pages), and the state of the bookkeeping in which they were found to be right."""

    __slots__ = ("owner", "parts", "right")

    def __init__(self, owner, parts):
        self.owner, self.parts, self.right = owner, parts, None

    def __call__(self) -> None:
        if self.right != self.owner._changes:  # asked once, not by every layer
            self.right = self.owner._check_appended(self.parts)


class KvPages:
    """The pages of `caches`, one :class:`KvCache` per layer (as many pages of as many tokens each,
    on one device), handed out to sequences, which are named by numbers.

    A sequence's pages are the same in every cache.  Its tokens are those that it has room for:
    :meth:`new` and :meth:`grow` count them before they are appended, and nothing here knows whether
    they were.  :meth:`fork` shares the pages; a shared page that is only partly filled is copied before
    :meth:`grow` makes room in it, so that room belongs to one sequence.  Room that was made before a
    fork is in shared pages: the oldest of the sequences that share a page fills it, once, for all of
    them and before one of them grows (a copy takes what is there), and an append through another one's
    :meth:`batch` is refused.  Copies go to the current stream, like the calls that write and read the
    caches.  Methods may be called from any thread."""

    def __init__(self, caches: Sequence[KvCache]):
        caches = [caches] if isinstance(caches, KvCache) else list(caches)
        if not caches or not all(isinstance(c, KvCache) for c in caches):
            raise Exl3Error(-1, "pages are those of at least one KvCache")
        first = caches[0]
        for c in caches:
            if (c.pages, c.page_tokens) != (first.pages, first.page_tokens):
                raise Exl3Error(-1, "KV caches whose pages are copied together have as many pages of as many tokens")
            if c.device != first.device:
                raise Exl3Error(-1, f"a cache is on {c.device}, expected {first.device}")
        self.caches, self.device = caches, first.device
        self.pages, self.page_tokens = first.pages, first.page_tokens
        self._handles = (_vp * len(caches))(*[c.handle.value for c in caches])
        self._uses = [0] * self.pages
        self._free = list(range(self.pages))  # a heap: the first free page is taken first
        self._held: dict = {}
        self._next = 0
        self._changes = 0  # of which pages belong to whom
        self._lock = threading.RLock()

    # -- copies ---------------------------------------------------------------
    def copy(self, src, dst, tokens=None) -> None:
        """Copies page src[i] to page dst[i] in every cache, or its first tokens[i] slots.  The
        lists are whole numbers on the host and may be changed after the call.  A page may be copied
        to several, none is copied to twice or copied and copied to.  In a captured graph the lists
        are those of the capture."""
        src, dst = _ints(src, "src"), _ints(dst, "dst")
        slots = None if tokens is None else _ints(tokens, "tokens")
        if len(src) != len(dst) or (slots is not None and len(slots) != len(src)):
            raise Exl3Error(-1, "a copy of pages takes as many sources as destinations, and as many token counts")
        _kv._launch(self.device, load_library().exl3_kv_copy_pages, self._handles, len(self._handles), _pointer(src),
                    _pointer(dst), None if slots is None else _pointer(slots), len(src))

    # -- sequences ------------------------------------------------------------
    def _sequence(self, seq) -> _Held:
        try:
            return self._held[seq]
        except (KeyError, TypeError):
            raise Exl3Error(-1, f"unknown sequence {seq!r}") from None

    @property
    def free_pages(self) -> int:
        """Pages that no sequence has."""
        return len(self._free)

    @property
    def sequences(self) -> list:
        """The sequences' numbers, oldest first."""
        with self._lock:
            return list(self._held)

    def tokens(self, seq) -> int:
        """The tokens of a sequence."""
        with self._lock:
            return self._sequence(seq).tokens

    def pages_of(self, seq) -> list:
        """The pages of a sequence, in order."""
        with self._lock:
            return list(self._sequence(seq).pages)

    def new(self, tokens: int = 0) -> int:
        """A new sequence with room for `tokens` tokens; returns its number."""
        with self._lock:
            seq = self._next
            self._held[seq] = _Held([], 0)
            try:
                self.grow([seq], tokens)
            except BaseException:
                del self._held[seq]
                raise
            self._next += 1
            return seq

    def grow(self, seqs, tokens=1) -> None:
        """Room for `tokens` more tokens (a number, or one per sequence) of each of the sequences
        `seqs` (a number, or a list), which are to be appended next: new pages, and a copy of a last
        page that is shared.  Without enough free pages nothing changes."""
        with self._lock:
            seqs = _several(seqs, "sequences")
            more = _several(tokens, "tokens", len(seqs))
            if len(more) != len(seqs) or any(n < 0 for n in more):
                raise Exl3Error(-1, "growth is a number of tokens that is not negative for each sequence")
            if len(set(seqs)) != len(seqs):
                raise Exl3Error(-1, "a sequence is listed once")
            page = self.page_tokens
            uses: dict = {}  # of shared last pages, as they get fewer
            plan = []  # (sequence, tokens it will have, whether its last page is copied, pages it takes)
            for seq, n in zip(seqs, more):
                held = self._sequence(seq)
                total = held.tokens + n
                if total >= 2**31:
                    raise Exl3Error(-1, f"a sequence has fewer than 2^31 tokens, got {total}")
                last = held.pages[-1] if n and held.tokens % page else None
                shared = last is not None and uses.setdefault(last, self._uses[last]) > 1
                if shared:
                    uses[last] -= 1
                plan.append((held, total, shared, -(-total // page) - len(held.pages) + shared))
            need = sum(p[3] for p in plan)
            if need > len(self._free):
                raise Exl3Error(-1, f"{need} pages needed, {len(self._free)} of {self.pages} free")
            taken = heapq.nsmallest(need, self._free)
            at, src, dst, slots = 0, [], [], []
            for held, _, shared, n in plan:
                if shared:
                    src.append(held.pages[-1])
                    dst.append(taken[at])
                    slots.append(held.tokens % page)
                at += n
            if src:
                self.copy(src, dst, slots)
            self._changes += 1
            for _ in taken:
                heapq.heappop(self._free)
            at = 0
            for held, total, shared, n in plan:
                if shared:
                    self._uses[held.pages.pop()] -= 1
                for p in taken[at : at + n]:
                    self._uses[p] = 1
                held.pages += taken[at : at + n]
                held.tokens, at = total, at + n

    def fork(self, seq) -> int:
        """A new sequence with the tokens of `seq`, whose pages it shares: append those that there is
        room for first."""
        with self._lock:
            held = self._sequence(seq)
            self._changes += 1
            for p in held.pages:
                self._uses[p] += 1
            self._held[self._next] = _Held(list(held.pages), held.tokens)
            self._next += 1
            return self._next - 1

    def cut(self, seq, tokens: int) -> None:
        """Keeps the first `tokens` tokens of a sequence (of a draft, say, the accepted ones)."""
        with self._lock:
            held = self._sequence(seq)
            tokens = _ints([tokens], "tokens")[0]
            if not 0 <= tokens <= held.tokens:
                raise Exl3Error(-1, f"{tokens} of {held.tokens} tokens kept")
            keep = -(-tokens // self.page_tokens)
            self._changes += 1
            self._drop(held.pages[keep:])
            del held.pages[keep:]
            held.tokens = tokens

    def free(self, seq) -> None:
        """Ends a sequence; its pages that no other one shares are free."""
        with self._lock:
            self._drop(self._sequence(seq).pages)
            self._changes += 1
            del self._held[seq]

    def _drop(self, pages) -> None:
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                heapq.heappush(self._free, p)

    def compact(self) -> int:
        """Moves pages to the front of the pool, so that the pages in use are its first ones;
        returns how many moved.  Batches made before name the old ones; nothing is appended through
        them."""
        with self._lock:
            used = self.pages - len(self._free)
            src = [p for p in range(used, self.pages) if self._uses[p]]
            if not src:
                return 0
            dst = sorted(p for p in self._free if p < used)
            page, filled = self.page_tokens, dict.fromkeys(src, 0)
            for held in self._held.values():
                for i, p in enumerate(held.pages):
                    if p in filled:
                        filled[p] = max(filled[p], min(page, held.tokens - i * page))
            self.copy(src, dst, [filled[p] for p in src])
            self._changes += 1
            to = dict(zip(src, dst))
            for held in self._held.values():
                held.pages = [to.get(p, p) for p in held.pages]
            for a, b in to.items():
                self._uses[b], self._uses[a] = self._uses[a], 0
            self._free = list(range(used, self.pages))  # sorted: a heap
            return len(src)

    def batch(self, seqs, new=1, max_kv: Optional[int] = None) -> KvBatch:
        """The :class:`KvBatch` of a call with the `new` newest tokens (a number, or one per
        sequence) of each of the sequences `seqs`, to read or to append them: made and uploaded anew by
        every call, so one of a step is for all its layers.  An append through it asks whether their
        pages are the sequences' to write, as they are then.  A captured graph asks at its capture, and
        nobody looks at what the program writes to the batch's tensors: one that makes room ahead and
        captures a step sets kv_lens to the tokens of each replay."""
        torch = _torch()
        with self._lock:
            seqs = _several(seqs, "sequences")
            new = _several(new, "new", len(seqs))
            held = [self._sequence(s) for s in seqs]
            if not seqs or len(new) != len(seqs):
                raise Exl3Error(-1, "a batch has at least one sequence, and new tokens for each")
            if any(not 0 <= n <= h.tokens for n, h in zip(new, held)):
                raise Exl3Error(-1, "a sequence's new tokens are among its tokens")
            starts = [0]
            for n in new:
                starts.append(starts[-1] + n)
            wide = max(1, max(len(h.pages) for h in held))
            rows = [p for h in held for p in h.pages + [0] * (wide - len(h.pages))]
            lens = [h.tokens for h in held]
            page = self.page_tokens
            parts = [(s, (h.tokens - n) // page, h.pages[(h.tokens - n) // page :]) for s, n, h in zip(seqs, new, held) if n]
        # one transfer: starts, lengths, table
        both = torch.frombuffer(_ints(starts + lens + rows, "tokens"), dtype=torch.int32).to(self.device)
        n = len(seqs)
        batch = KvBatch(both[: n + 1], both[n + 1 : 2 * n + 1], both[2 * n + 1 :].view(n, wide), max_q=max(1, max(new)),
                        max_kv=max(lens) if max_kv is None else max_kv)
        batch._asked = _Appended(self, parts)
        return batch

    def _check_appended(self, parts) -> int:
        """Refuses an append to `parts` (:class:`_Appended`) that would write what another sequence
        has, or a slot twice; returns the state that it was asked in."""
        with self._lock:
            if len({seq for seq, _, _ in parts}) != len(parts):
                raise Exl3Error(-1, "a sequence whose tokens are appended is listed twice")
            for seq, first, pages in parts:
                held = self._held.get(seq)
                if held is None or held.pages[first : first + len(pages)] != pages:
                    raise Exl3Error(-1, f"a batch that was made before the pages of sequence {seq} changed")
                for i, p in enumerate(pages, first):
                    # (a shared page has one place in all that share it; the oldest come first)
                    if self._uses[p] > 1 and seq != next(
                            s for s, h in self._held.items() if i < len(h.pages) and h.pages[i] == p):
                        raise Exl3Error(-1, f"page {p} is shared: an older sequence than {seq} appends to it")
            return self._changes
