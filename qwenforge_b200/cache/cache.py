"""The sequence cache: what a model keeps between steps, per sequence.

A *slot* stands for one live sequence. It is taken when the sequence starts, holds the
sequence's own length, and is given back when the sequence ends; the next sequence that
starts takes it again.

What is kept per slot is declared by the model's mixers, one *need* per schedule entry:

  KvNeed     keys and values of every position (window 0), of the last `window` positions, or of the positions of
             the current block of `chunk` (a mask that cuts a sequence into blocks counted from its position 0); or
             one row per position that serves as both, `planes=1`.
             Storage is handed out in pages of PAGE_TOKENS positions, so a sequence holds
             ceil(length / PAGE_TOKENS) pages and nothing more: the cache is sized by the
             number of live tokens, not by slots x longest sequence.
             `every` > 1: one row per `every` positions instead of one per position (the means of whole blocks of
             positions: a sequence of n positions holds n // every rows, and pages by rows). `pool` > 0 on a windowed
             need: positions also stay until their block of `pool` positions is complete, so that whoever forms that
             block's row can still read them.
  StateNeed  a tensor of fixed shape per sequence (a recurrent state, a running statistic),
             zeroed when the slot is taken.
  BundleNeed several of these under names, for a schedule entry that keeps more than one thing (keys and values, the
             rows of whole blocks beside them, and the last inputs of a short convolution).

Entries with the same need share a *group*; each group has storage of its own (its own
pages, page table and page allocator). A group with a window gives pages back as soon as
every position on them has left the window, so in steady state a sequence holds about
window / PAGE_TOKENS + 1 pages there.

A sequence may be forked (`fork`): the new ones hold its whole pages with it (a page counts its holders) and get copies of the page
that is still being filled and of the fixed-size state. So a page at or behind a sequence's length is always its own, and no write
reaches a page that two sequences hold. `rewind` drops a sequence's last positions, `compact` moves the held pages to the front.

Keys and values may be kept in 8 bits (`kv_dtype`): a page then holds e4m3 codes, and the group a power of two for each page, plane and
head beside them. They travel together: a copied page takes its scales with it. A group has one more storage there, of the model's own
dtype and one entry's size: the values that a prompt's attention reads back, under the same page numbers, one schedule entry after
another.

The state that decoding itself keeps per sequence (latest token, position, step count, budget)
lives in the decode graph's own device buffers (`engine/graphs.py`); this cache holds only what
the model's mixers declare.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from .. import ops
from .allocators import CacheFull, CacheMisuse, PageAllocator, SlotAllocator

PAGE_TOKENS = 64

def round_up(n: int, multiple: int) -> int:
    return (n + multiple - 1) // multiple * multiple


@dataclass(frozen=True)
class KvNeed:
    kv_heads: int
    head_dim: int
    window: int = 0  # 0: every earlier position
    planes: int = 2  # rows kept per position and head: keys and values, or 1 for a mixer whose keys are its values
                     # (the shared latent of a latent attention)
    chunk: int = 0   # > 0: a query sees only the positions of its own block of `chunk` positions
    every: int = 1   # > 1: one row per `every` positions (row b stands for positions b * every .. b * every + every - 1)
    pool: int = 0    # > 0: a position also stays until its block of `pool` positions is complete

    def first_visible(self, position: int) -> int:
        """Lowest position that a query at `position` sees."""
        first = max(0, position - self.window + 1) if self.window > 0 else 0
        return max(first, position // self.chunk * self.chunk) if self.chunk > 0 else first

    def first_kept(self, length: int) -> int:
        """Lowest position that is still needed when the sequence holds `length` positions: by the next query's mask, or
        by the block of `pool` positions that is not complete yet."""
        first = self.first_visible(length)
        return min(first, length // self.pool * self.pool) if self.pool > 0 else first

    def rows(self, length: int) -> int:
        """Rows that a sequence of `length` positions holds."""
        return length // self.every

    def fits(self, dtype: torch.dtype) -> bool:
        """Whether a cache of this dtype (8 bits) has a form for these rows: keys and values, one row of each per position."""
        return (dtype == torch.float8_e4m3fn and self.planes == 2 and self.chunk == 0 and self.every == 1 and self.pool == 0
                and self.head_dim in ops.E4M3_HEAD_DIMS)

    def merged(self, other: "KvNeed") -> "KvNeed":
        """What serves this need and a reader with a mask of its own over the same rows: where the masks differ, every
        position is kept."""
        if (other.kv_heads, other.head_dim, other.planes) != (self.kv_heads, self.head_dim, self.planes):
            raise ValueError(f"a layer that reads another layer's cache needs rows of the same shape: {other} against {self}")
        if (other.window, other.chunk, other.every, other.pool) == (self.window, self.chunk, self.every, self.pool):
            return self
        if other.every != self.every:
            raise ValueError(f"a layer that reads another layer's cache needs rows for the same positions: {other} against {self}")
        return KvNeed(self.kv_heads, self.head_dim, 0, self.planes, 0, self.every)


@dataclass(frozen=True)
class StateNeed:
    shape: tuple
    dtype: torch.dtype = torch.float32


@dataclass(frozen=True)
class BundleNeed:
    """Several needs of one schedule entry: ((name, need), ...); a need may itself be a bundle. The entry's site is then a
    `BundleSite` with one site per name."""
    items: tuple

    def flat(self, prefix: tuple = ()):
        """(path of names, need) for every KvNeed and StateNeed in the bundle."""
        for name, need in self.items:
            if isinstance(need, BundleNeed):
                yield from need.flat(prefix + (name,))
            elif need is not None:
                yield prefix + (name,), need


def tokens_for_continuations(needs: Sequence[Optional[object]], sequences: Sequence[tuple[int, int]], continuations: int, max_seqs: int) -> int:
    """Cache tokens that the groups of one row per several positions ask for where every sequence, (prompt length, longest length), is continued
    `continuations` times: such a group has its share of the cache's pages and one more per sequence, while each continuation holds a copy of the page
    that its prompt has begun and those behind it."""
    flat = [inner for need in needs for inner in ([n for _, n in need.flat()] if isinstance(need, BundleNeed) else [need])]
    tokens = 0
    for every in {need.every for need in flat if isinstance(need, KvNeed) and need.every > 1}:
        pages = 0
        for prompt, total in sequences:
            rows, begun = total // every, prompt // every // PAGE_TOKENS * PAGE_TOKENS
            pages += round_up(rows, PAGE_TOKENS) // PAGE_TOKENS + (continuations - 1) * (round_up(rows - begun, PAGE_TOKENS) // PAGE_TOKENS)
        tokens = max(tokens, PAGE_TOKENS * max(pages, every * (pages - max_seqs)))
    return tokens


class BundleSite:
    """The sites of a schedule entry that keeps several things, by the names its `BundleNeed` gave them."""

    def __init__(self):
        self._sites: dict = {}

    def __getitem__(self, name: str):
        try:
            return self._sites[name]
        except KeyError:
            raise KeyError(f"this schedule entry keeps nothing called {name!r}; it keeps {', '.join(sorted(self._sites)) or 'nothing'}") from None

    def get(self, name: str, default=None):
        return self._sites.get(name, default)

    def put(self, path: tuple, site) -> None:
        if len(path) == 1:
            self._sites[path[0]] = site
        else:
            self._sites.setdefault(path[0], BundleSite()).put(path[1:], site)


class KvSite:
    """One schedule entry's view of its group: its own storage, the group's shared page table."""

    def __init__(self, group: "KvGroup", index: int):
        self.group = group
        self.storage = group.storage[index]  # [pages, planes, kv_heads, PAGE_TOKENS, head_dim]
        self.scales = None if group.scales is None else group.scales[index]  # [pages, planes, kv_heads], of a cache in 8 bits
        self.table = group.table
        self.kv_heads = group.need.kv_heads
        self.head_dim = group.need.head_dim
        self.window = group.need.window
        self._codes = None

    def codes(self):
        """What the kernels of a cache in 8 bits address it by (checked once)."""
        if self._codes is None:
            self._codes = ops.E4m3SiteArgs(self.storage, self.scales, self.table, self.kv_heads, self.head_dim)
        return self._codes


class KvGroup:
    def __init__(self, need: KvNeed, entries: Sequence[int], n_pages: int, n_slots: int, pages_per_seq: int,
                 dtype: torch.dtype, device, kv_dtype: Optional[torch.dtype] = None):
        self.need = need
        self.entries = list(entries)
        self.pages = PageAllocator(n_pages)
        self.pages_per_seq = pages_per_seq
        # zeroed once: no kernel reads beyond a sequence's length, stale data is finite anyway
        shape = (len(self.entries), n_pages, need.planes, need.kv_heads, PAGE_TOKENS, need.head_dim)
        self.storage = torch.zeros(shape, dtype=dtype if kv_dtype is None else kv_dtype, device=device)
        self.scales = self.values = None
        if kv_dtype is not None:
            self.scales = torch.zeros(shape[:4], dtype=torch.float32, device=device)
            self.values = torch.zeros(shape[1:], dtype=dtype, device=device)
        self.table = torch.full((n_slots, pages_per_seq), -1, dtype=torch.int32, device=device)
        self._host_table = torch.full((n_slots, pages_per_seq), -1, dtype=torch.int32)
        self._held: list[dict[int, int]] = [dict() for _ in range(n_slots)]  # slot -> {logical page: page id}
        self._dirty: set[int] = set()

    def pages_missing(self, slot: int, first_pos: int, end_pos: int) -> list[int]:
        """Logical pages covering positions [first_pos, end_pos) that the slot does not hold."""
        if end_pos <= first_pos:
            return []
        held = self._held[slot]
        return [lp for lp in range(first_pos // PAGE_TOKENS, (end_pos - 1) // PAGE_TOKENS + 1) if lp not in held]

    def first_needed(self, length: int) -> int:
        """Lowest ROW that is still needed when the sequence holds `length` positions."""
        return self.need.first_kept(length) // self.need.every

    def grant(self, slot: int, logical_pages: Sequence[int]) -> None:
        ids = self.pages.take(len(logical_pages))
        for lp, page in zip(logical_pages, ids):
            if lp >= self.pages_per_seq:
                self.pages.give_back(ids)
                raise CacheFull(f"position {lp * PAGE_TOKENS} is beyond the cache's longest sequence "
                                f"({self.pages_per_seq * PAGE_TOKENS} positions)")
            self._held[slot][lp] = page
            self._host_table[slot, lp] = page
        if logical_pages:
            self._dirty.add(slot)

    def trim(self, slot: int, length: int) -> None:
        """Give back pages all of whose positions have left the window of every later query."""
        if (self.need.window <= 0 and self.need.chunk <= 0) or self.need.every > 1:
            return
        keep_from = self.first_needed(length) // PAGE_TOKENS
        gone = [lp for lp in self._held[slot] if lp < keep_from]
        if gone:
            self.pages.give_back([self._held[slot].pop(lp) for lp in gone])
            for lp in gone:
                self._host_table[slot, lp] = -1
            self._dirty.add(slot)

    def release(self, slot: int) -> None:
        held = self._held[slot]
        if held:
            self.pages.give_back(list(held.values()))
            held.clear()
            self._host_table[slot].fill_(-1)
            self._dirty.add(slot)

    def pages_held(self, slot: int) -> int:
        return len(self._held[slot])

    def _put(self, slot: int, logical: int, page: int) -> None:
        self._held[slot][logical] = page
        self._host_table[slot, logical] = page
        self._dirty.add(slot)

    def filling(self, slot: int, length: int) -> Optional[int]:
        """The logical page that a sequence of `length` positions has begun and not filled (None: there is none, or it is not held)."""
        rows = self.need.rows(length)
        return rows // PAGE_TOKENS if rows % PAGE_TOKENS and rows // PAGE_TOKENS in self._held[slot] else None

    def fork(self, slot: int, length: int, forks: Sequence[int]) -> None:
        """The slots of `forks` (which hold nothing) get the pages that `slot` has filled, and a copy each of the one it is filling."""
        held, whole = self._held[slot], self.need.rows(length) // PAGE_TOKENS
        kept = {lp: page for lp, page in held.items() if lp < whole}
        self.pages.share(kept.values(), len(forks))
        partial = self.filling(slot, length)
        copies = self.pages.take(len(forks)) if partial is not None else []
        for i, fork in enumerate(forks):
            for lp, page in kept.items():
                self._put(fork, lp, page)
            if partial is not None:
                self._put(fork, partial, copies[i])
        if copies:
            self._copy([(held[partial], page, self.need.rows(length) % PAGE_TOKENS) for page in copies])

    def _copy(self, moves: list) -> None:
        """Rows of pages to other pages, with their pages' scales: (from, to, rows) or (from, to)."""
        ops.copy_pages(self.storage, moves)
        if self.scales is not None:
            ops.copy_pages(self.scales, [move[:2] for move in moves])

    def rewind_missing(self, slot: int, length: int) -> bool:
        """Whether a page that a sequence of `length` positions still needs has been given back."""
        first = self.first_needed(length)
        rows = self.need.rows(length)
        return rows > first and bool(self.pages_missing(slot, first, rows))

    def shares_filling(self, slot: int, length: int) -> bool:
        """Whether the page in which `length` ends is one that other sequences hold too."""
        partial = self.filling(slot, length)
        return partial is not None and self.pages.holders(self._held[slot][partial]) > 1

    def rewind(self, slot: int, length: int) -> None:
        """Back to `length` positions: pages behind it are given back, and the one it ends in becomes the slot's own."""
        held, rows = self._held[slot], self.need.rows(length)
        if self.shares_filling(slot, length):
            partial = rows // PAGE_TOKENS
            old, (new,) = held[partial], self.pages.take(1)
            self._copy([(old, new, rows % PAGE_TOKENS)])
            self.pages.give_back([old])
            self._put(slot, partial, new)
        gone = [lp for lp in held if lp * PAGE_TOKENS >= rows]
        if gone:
            self.pages.give_back([held.pop(lp) for lp in gone])
            for lp in gone:
                self._host_table[slot, lp] = -1
            self._dirty.add(slot)

    def compact(self) -> int:
        """Held pages to the front of the storage; returns how many moved."""
        moves = self.pages.compact()
        if moves:
            self._copy(moves)
            to = dict(moves)
            for slot, held in enumerate(self._held):
                for lp, page in held.items():
                    if page in to:
                        self._put(slot, lp, to[page])
        return len(moves)

    def flush(self) -> None:
        """Bring the device page table up to date with the host's (rows that changed since the last call)."""
        if not self._dirty:
            return
        rows = sorted(self._dirty)
        self._dirty.clear()
        if len(rows) == 1 or rows[-1] - rows[0] + 1 == len(rows):
            lo, hi = rows[0], rows[-1] + 1
            # through a copy of the rows: `trim` and `release` may rewrite the host table as soon as this returns,
            # and a copy from that pageable snapshot has left the host when the call returns
            self.table[lo:hi].copy_(self._host_table[lo:hi].clone())
        else:
            index = torch.tensor(rows, dtype=torch.long)
            self.table.index_copy_(0, index.to(self.table.device), self._host_table[index].to(self.table.device))


class StateGroup:
    def __init__(self, need: StateNeed, entries: Sequence[int], n_slots: int, device):
        self.need = need
        self.entries = list(entries)
        self.storage = torch.zeros((len(self.entries), n_slots, *need.shape), dtype=need.dtype, device=device)

    def reset(self, slot: int) -> None:
        self.storage[:, slot].zero_()

    def fork(self, slot: int, forks: Sequence[int]) -> None:
        ops.copy_pages(self.storage, [(slot, fork) for fork in forks])


class StateSite:
    """One schedule entry's fixed-size state: `storage[slot]` belongs to the sequence in `slot`."""

    def __init__(self, group: StateGroup, index: int):
        self.group = group
        self.storage = group.storage[index]  # [slots, *shape]


class SequenceCache:
    """Slots and groups of one model on one device.

    needs        one entry per schedule entry: KvNeed, StateNeed or None (that entry keeps nothing,
                 or reads another entry's cache)
    max_tokens   the most tokens that live sequences hold at any time, each sequence's count
                 rounded up to PAGE_TOKENS; sizes every KV group
    max_seqs     number of slots
    max_len      the longest sequence a slot can hold (sizes the page tables)
    kv_dtype     None: keys and values in `dtype`; torch.float8_e4m3fn: in 8 bits (every position's own keys and values, of head
                 sizes that the kernels have)
    """

    _serials = 0

    def __init__(self, needs: Sequence[Optional[object]], max_tokens: int, max_seqs: int, max_len: int,
                 dtype: torch.dtype, device, kv_dtype: Optional[torch.dtype] = None):
        self.device = torch.device(device)
        self.dtype = dtype
        self.kv_dtype = kv_dtype
        SequenceCache._serials += 1
        self.serial = SequenceCache._serials  # tells caches apart for whoever keeps things per cache (captured graphs)
        n_pages = max(1, round_up(max_tokens, PAGE_TOKENS) // PAGE_TOKENS)
        self.n_pages = n_pages
        self.max_seqs = max(1, min(max_seqs, n_pages))
        self.max_len = min(round_up(max_len, PAGE_TOKENS), n_pages * PAGE_TOKENS)
        pages_per_seq = self.max_len // PAGE_TOKENS
        self.slots = SlotAllocator(self.max_seqs)
        self.lengths = [0] * self.max_seqs
        self._shared: dict = {}   # batch (slots) -> what its sequences share

        # who keeps what: (schedule entry, path of names inside its bundle; () for an entry with one need) per need
        by_need: dict[object, list[tuple]] = {}
        for entry, need in enumerate(needs):
            if isinstance(need, BundleNeed):
                for path, inner in need.flat():
                    by_need.setdefault(inner, []).append((entry, path))
            elif need is not None:
                by_need.setdefault(need, []).append((entry, ()))
        self.kv_groups: list[KvGroup] = []
        self.state_groups: list[StateGroup] = []
        self._sites: dict[int, object] = {}

        def place(entry: int, path: tuple, site) -> None:
            if path:
                self._sites.setdefault(entry, BundleSite()).put(path, site)
            else:
                self._sites[entry] = site

        for need, keepers in by_need.items():
            if isinstance(need, KvNeed):
                if kv_dtype is not None and not need.fits(kv_dtype):
                    raise ValueError(f"a cache in {kv_dtype} does not hold {need}")
                # a group of one row per `every` positions is sized by rows: fewer pages, each sequence's last one partly empty
                pages = n_pages if need.every <= 1 else min(n_pages, n_pages // need.every + self.max_seqs)
                group = KvGroup(need, keepers, pages, self.max_seqs, pages_per_seq, dtype, self.device, kv_dtype)
                self.kv_groups.append(group)
                for i, (entry, path) in enumerate(keepers):
                    place(entry, path, KvSite(group, i))
            elif isinstance(need, StateNeed):
                group = StateGroup(need, keepers, self.max_seqs, self.device)
                self.state_groups.append(group)
                for i, (entry, path) in enumerate(keepers):
                    place(entry, path, StateSite(group, i))
            else:
                raise TypeError(f"unknown cache need {need!r}")

    # ------------------------------------------------------------------ sites
    def site(self, entry: int):
        """The storage view of schedule entry `entry` (None if it keeps nothing)."""
        return self._sites.get(entry)

    # ------------------------------------------------------------------ sequences
    def open(self) -> int:
        """Start a sequence: take a slot with length 0 and zeroed fixed-size state."""
        slot = self.slots.take()
        self.lengths[slot] = 0
        for group in self.state_groups:
            group.reset(slot)
        return slot

    def _check_held(self, slot: int) -> None:
        if not self.slots.is_held(slot):
            raise CacheMisuse(f"slot {slot} is not held by a live sequence")

    def reserve(self, requests: Sequence[tuple[int, int]]) -> None:
        """Make sure that each (slot, total_length) has pages for positions up to total_length.

        All or nothing: if the pages for all requests together are not free, CacheFull is
        raised and nothing has changed.
        """
        plans = []
        for group in self.kv_groups:
            wanted = 0
            plan = []
            for slot, total in requests:
                self._check_held(slot)
                if total > self.max_len:
                    raise CacheFull(f"a sequence of {total} tokens exceeds the cache's longest sequence ({self.max_len})")
                held = group.need.rows(self.lengths[slot])
                first = min(group.first_needed(self.lengths[slot]), held)
                missing = group.pages_missing(slot, first, group.need.rows(total))
                wanted += len(missing)
                plan.append((slot, missing))
            if wanted > group.pages.n_free:
                raise CacheFull(f"{wanted} cache pages wanted ({wanted * PAGE_TOKENS} tokens), "
                                f"{group.pages.n_free} of {group.pages.n_pages} free")
            plans.append((group, plan))
        for group, plan in plans:
            for slot, missing in plan:
                group.grant(slot, missing)

    def advance(self, slot: int, n_tokens: int) -> None:
        """The sequence grew by n_tokens (a step wrote them); windowed groups drop what no later query sees."""
        self._check_held(slot)
        self.lengths[slot] += n_tokens
        for group in self.kv_groups:
            group.trim(slot, self.lengths[slot])

    def close(self, slot: int) -> None:
        """End a sequence: its pages and its slot become free."""
        self._check_held(slot)
        for group in self.kv_groups:
            group.release(slot)
        self.lengths[slot] = 0
        self.slots.give_back(slot)
        self._shared.clear()

    # ------------------------------------------------------------------ branches
    def fork(self, slot: int, count: int = 1) -> list[int]:
        """Start `count` sequences that continue where `slot` stands: its positions (whole pages shared, the begun one copied) and its
        fixed-size state. Pages that `slot` has reserved ahead stay its own. All or nothing: CacheFull leaves everything as it was."""
        self._check_held(slot)
        if count < 0:
            raise ValueError("fork: count must be >= 0")
        if count > self.slots.n_free:
            raise CacheFull(f"{count} sequence slots wanted, {self.slots.n_free} of {self.max_seqs} free")
        length = self.lengths[slot]
        for group in self.kv_groups:
            if group.filling(slot, length) is not None and count > group.pages.n_free:
                raise CacheFull(f"{count} cache pages wanted, {group.pages.n_free} of {group.pages.n_pages} free")
        if count == 0:
            return []
        forks = [self.slots.take() for _ in range(count)]
        for group in self.kv_groups:
            group.fork(slot, length, forks)
        for group in self.state_groups:
            group.fork(slot, forks)
        for fork in forks:
            self.lengths[fork] = length
        self._shared.clear()
        return forks

    def rewind(self, slot: int, length: int) -> None:
        """Drop the positions of `slot` from `length` on (drafted tokens that were refused); pages behind it become free, those that were
        reserved ahead among them. Not possible where something cannot go back: a fixed-size state, or positions that a window has
        given up since. All or nothing."""
        self._check_held(slot)
        if not 0 <= length <= self.lengths[slot]:
            raise ValueError(f"rewind: length {length} outside 0 .. {self.lengths[slot]}")
        if length < self.lengths[slot]:
            if self.state_groups:
                raise CacheMisuse("rewind: a state of fixed size cannot go back")
            if any(group.rewind_missing(slot, length) for group in self.kv_groups):
                raise CacheMisuse(f"rewind: positions that a query at {length} sees have left their window and were given up")
        for group in self.kv_groups:
            if group.shares_filling(slot, length) and not group.pages.n_free:
                raise CacheFull(f"1 cache page wanted, 0 of {group.pages.n_pages} free")
        for group in self.kv_groups:
            group.rewind(slot, length)
        self.lengths[slot] = length
        self._shared.clear()

    def compact(self) -> int:
        """Move the held pages of every group to the front of its storage, so that all behind them is free; the page tables on the
        device follow at once. Returns how many pages moved."""
        moved = sum(group.compact() for group in self.kv_groups)
        self.flush()
        return moved

    def pages_used(self) -> list[int]:
        """Per group of keys and values, the held pages (a shared one counts once)."""
        return [group.pages.n_pages - group.pages.n_free for group in self.kv_groups]

    def shared_groups(self, slots: Sequence[int]) -> list[tuple]:
        """Which sequences of a batch begin with the same pages: (batch entries, pages) for every two or more that do, as
        `ops.SharedPrefix` takes them. Only positions that every later query sees count (keys and values without a window)."""
        group = next((g for g in self.kv_groups if g.need.window <= 0 and g.need.chunk <= 0 and g.need.every == 1), None)
        if group is None or not group.pages.n_shared:
            return []
        families: dict = {}
        for entry, slot in enumerate(slots):
            if slot >= 0 and 0 in group._held[slot]:
                families.setdefault(group._held[slot][0], []).append(entry)
        found = []
        for entries in families.values():
            if len(entries) < 2:
                continue
            whole = min(self.lengths[slots[e]] for e in entries) // PAGE_TOKENS
            rows = group._host_table[[slots[e] for e in entries], :whole]
            same = (rows == rows[0]).all(0)
            pages = whole if bool(same.all()) else int(same.to(torch.int8).argmin())
            if pages > 0:
                found.append((entries, pages))
        return found

    def shared_prefix(self, slots: Sequence[int]):
        """`ops.SharedPrefix` of a batch whose sequences begin with the same pages, or None. Kept for a batch that comes back, until a
        sequence is forked, rewound or closed."""
        key = tuple(slots)
        if key not in self._shared:
            if len(self._shared) >= 256:
                self._shared.clear()
            groups = self.shared_groups(key)
            self._shared[key] = ops.SharedPrefix(groups, len(key), self.device) if groups else None
        return self._shared[key]

    def shared_worth_reading(self, slots: Sequence[int]):
        """`shared_prefix`, where an attention layer is faster for reading it once (`ops.attention_shared_pays`); else None. (A cache in
        8 bits is read by every sequence for itself.)"""
        if self.kv_dtype is not None:
            return None
        share = self.shared_prefix(slots)
        if share is None or any(ops.attention_shared_pays(share, g.storage.dtype, g.need.kv_heads, g.need.head_dim) for g in self.kv_groups):
            return share
        return None

    def flush(self) -> None:
        for group in self.kv_groups:
            group.flush()

    # ------------------------------------------------------------------ accounting
    def tokens_free(self) -> int:
        if not self.kv_groups:
            return self.n_pages * PAGE_TOKENS
        return min(g.pages.n_free * g.need.every for g in self.kv_groups) * PAGE_TOKENS

    def live_slots(self) -> list[int]:
        return [s for s in range(self.max_seqs) if self.slots.is_held(s)]

    def read_bytes(self, lengths: Sequence[int]) -> int:
        """Bytes of keys and values that one single-token step reads for sequences of these lengths."""
        total = 0
        for g in self.kv_groups:
            per_token = len(g.entries) * g.need.planes * g.need.kv_heads * g.need.head_dim * g.storage.element_size()
            if g.need.every > 1:
                total += per_token * sum(g.need.rows(n) for n in lengths)
            else:
                total += per_token * sum(n - g.need.first_visible(n - 1) for n in lengths if n > 0)
        return total

    def storage_bytes(self) -> int:
        total = sum(t.numel() * t.element_size() for g in self.kv_groups for t in (g.storage, g.scales, g.values) if t is not None)
        total += sum(g.storage.numel() * g.storage.element_size() for g in self.state_groups)
        return total
