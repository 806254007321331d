"""Forks of sequences, rewound and compacted ones: the bookkeeping, on the CPU, with a plain copy in the kernel's place; and what the
entries of the kernels refuse before any of them runs."""
import random

import numpy as np
import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.cache import PAGE_TOKENS, BundleNeed, CacheFull, CacheMisuse, KvNeed, PageAllocator, SequenceCache, StateNeed


def plain_copy(storage, moves):
    n_rows = storage.shape[-2] if storage.dim() >= 4 else 1
    checked = ops.page_moves(moves, storage.shape[1], n_rows)
    for source, target, rows in checked.tolist():
        if storage.dim() >= 4:
            storage[:, target, ..., :rows, :] = storage[:, source, ..., :rows, :]
        else:
            storage[:, target] = storage[:, source]


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(ops, "copy_pages", plain_copy)


NEEDS = {
    "full": [KvNeed(2, 4), KvNeed(2, 4)],
    "window": [KvNeed(2, 4), KvNeed(1, 4, window=70)],
    "pooled": [BundleNeed((("kv", KvNeed(1, 4, window=20, pool=16)), ("blocks", KvNeed(1, 4, every=16))))],
    "state": [KvNeed(1, 4), StateNeed((3, 2))],
}


def grow(cache, slot, values, base):
    """Append positions whose rows hold `value` in every group; pooled rows hold their block's last value."""
    start = cache.lengths[slot]
    cache.reserve([(slot, start + len(values))])
    for g in cache.kv_groups:
        for i, v in enumerate(values):
            p = start + i
            if g.need.every > 1:
                if (p + 1) % g.need.every:
                    continue
                p = p // g.need.every
            page = int(g._host_table[slot, p // PAGE_TOKENS])
            assert page >= 0 and g.pages.holders(page) == 1   # what is written is the sequence's own
            g.storage[:, page, :, :, p % PAGE_TOKENS] = float(v)
    for g in cache.state_groups:
        g.storage[:, slot] = float(values[-1])
    cache.advance(slot, len(values))
    base.setdefault(slot, []).extend(values)


def check(cache, base):
    for g in cache.kv_groups:
        held = [p for slot in base for p in g._held[slot].values()]
        counts = {p: held.count(p) for p in set(held)}
        assert all(g.pages.holders(p) == counts.get(p, 0) for p in range(g.pages.n_pages))
        assert g.pages.n_free == g.pages.n_pages - len(counts) and sorted(set(g.pages._free)) == sorted(g.pages._free)
        assert g.pages.n_shared == sum(c > 1 for c in counts.values())
        for slot, values in base.items():
            assert cache.lengths[slot] == len(values)
            for row in range(min(g.first_needed(len(values)), g.need.rows(len(values))), g.need.rows(len(values))):
                page = int(g._host_table[slot, row // PAGE_TOKENS])
                want = values[row] if g.need.every == 1 else values[row * g.need.every + g.need.every - 1]
                assert (g.storage[:, page, :, :, row % PAGE_TOKENS] == float(want)).all()
    for g in cache.state_groups:
        for slot, values in base.items():
            assert (g.storage[:, slot] == float(values[-1] if values else 0)).all()


@pytest.mark.parametrize("kind", list(NEEDS))
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_sequences_keep_their_rows_through_forks_rewinds_and_compactions(kind, seed):
    rng = random.Random(seed)
    cache = SequenceCache(NEEDS[kind], 40 * PAGE_TOKENS, 6, 12 * PAGE_TOKENS, torch.float32, "cpu")
    base, count = {}, 0
    for _ in range(80):
        live = list(base)
        what = rng.random()
        try:
            if not live or what < 0.15:
                slot = cache.open()
                base[slot] = []
                grow(cache, slot, [count + i for i in range(rng.choice([1, 63, 64, 65, 200]))], base)
                count += 200
            elif what < 0.5:
                slot = rng.choice(live)
                n = rng.choice([1, 2, 17, 64, 100])
                if len(base[slot]) + n <= cache.max_len:
                    grow(cache, slot, [count + i for i in range(n)], base)
                    count += n
            elif what < 0.7:
                slot = rng.choice(live)
                for fork in cache.fork(slot, rng.choice([0, 1, 2])):
                    base[fork] = list(base[slot])
            elif what < 0.8:
                slot = rng.choice(live)
                length = max(0, len(base[slot]) - rng.choice([0, 1, 5, 64, 130]))
                cache.rewind(slot, length)
                base[slot] = base[slot][:length]
            elif what < 0.9:
                cache.compact()
                for g in cache.kv_groups:
                    assert all(p < g.pages.n_pages - g.pages.n_free for slot in base for p in g._held[slot].values())
            else:
                slot = rng.choice(live)
                cache.close(slot)
                del base[slot]
        except (CacheFull, CacheMisuse) as e:
            assert "wanted" in str(e) or "in use" in str(e) or "cannot go back" in str(e) or "left their window" in str(e)
            base = {slot: values for slot, values in base.items() if len(values) == cache.lengths[slot]} if not live else base
            for slot in list(base):
                if not base[slot] and cache.lengths[slot] == 0 and slot not in live:
                    cache.close(slot)
                    del base[slot]
        check(cache, base)
    cache.flush()
    for g in cache.kv_groups:
        assert torch.equal(g.table, g._host_table)


def test_fork_is_all_or_nothing():
    cache = SequenceCache(NEEDS["full"], 4 * PAGE_TOKENS, 4, 4 * PAGE_TOKENS, torch.float32, "cpu")
    slot, base = cache.open(), {}
    grow(cache, slot, list(range(100)), base)
    with pytest.raises(CacheFull, match="pages"):
        cache.fork(slot, 3)   # two pages are free, three forks need one each
    with pytest.raises(CacheFull, match="slots"):
        cache.fork(slot, 4)
    check(cache, base)
    forks = cache.fork(slot, 2)
    base.update({f: list(base[slot]) for f in forks})
    check(cache, base)
    with pytest.raises(CacheFull):
        cache.rewind(slot, 30)   # into the page that all three hold, with none free
    check(cache, base)
    cache.close(forks[0])
    del base[forks[0]]
    cache.rewind(slot, 30)
    base[slot] = base[slot][:30]
    check(cache, base)
    with pytest.raises(CacheMisuse):
        cache.fork(forks[0], 1)
    with pytest.raises(ValueError):
        cache.rewind(slot, 31)


def test_what_cannot_go_back_is_refused():
    cache = SequenceCache(NEEDS["state"], 4 * PAGE_TOKENS, 2, 4 * PAGE_TOKENS, torch.float32, "cpu")
    base = {}
    slot = cache.open()
    grow(cache, slot, [1, 2, 3], base)
    with pytest.raises(CacheMisuse, match="fixed size"):
        cache.rewind(slot, 2)
    cache = SequenceCache(NEEDS["window"], 16 * PAGE_TOKENS, 2, 8 * PAGE_TOKENS, torch.float32, "cpu")
    base = {}
    slot = cache.open()
    for i in range(5):
        grow(cache, slot, list(range(60)), base)
    with pytest.raises(CacheMisuse, match="window"):
        cache.rewind(slot, 150)
    check(cache, base)
    cache.rewind(slot, 298)
    base[slot] = base[slot][:298]
    check(cache, base)


def test_shared_groups():
    cache = SequenceCache(NEEDS["full"], 64 * PAGE_TOKENS, 8, 8 * PAGE_TOKENS, torch.float32, "cpu")
    base, slot, other = {}, cache.open(), cache.open()
    grow(cache, slot, list(range(130)), base)
    grow(cache, other, list(range(70)), base)
    assert cache.shared_groups([slot, other]) == [] and cache.shared_prefix([slot, other]) is None
    a, b = cache.fork(slot, 2)
    base.update({f: list(base[slot]) for f in (a, b)})
    assert cache.shared_groups([other, a, -1, b, slot]) == [([1, 3, 4], 2)]
    grow(cache, b, list(range(100)), base)
    c = cache.fork(b)[0]
    base[c] = list(base[b])
    assert cache.shared_groups([b, c]) == [([0, 1], 3)]
    assert cache.shared_groups([a, b, c]) == [([0, 1, 2], 2)]
    share = cache.shared_prefix([a, other, b, c])
    assert share.groups == [([0, 2, 3], 2)] and share.entry_pages.tolist() == [2, 0, 2, 2] and share.least_pages == 0
    assert cache.shared_prefix([a, other, b, c]) is share
    cache.rewind(c, 70)
    base[c] = base[c][:70]
    assert cache.shared_prefix([a, other, b, c]).groups == [([0, 2, 3], 1)]
    check(cache, base)


def test_page_allocator_counts_holders():
    pages = PageAllocator(6)
    a = pages.take(3)
    pages.share(a[:2], 2)
    assert [pages.holders(p) for p in a] == [3, 3, 1] and pages.n_shared == 2
    pages.give_back(a)
    assert pages.n_free == 4 and pages.n_shared == 2
    pages.give_back([a[0], a[0], a[1]])
    assert pages.n_free == 5 and pages.n_shared == 0
    with pytest.raises(CacheMisuse):
        pages.give_back([a[0]])
    with pytest.raises(CacheMisuse):
        pages.share([a[0]])
    b = pages.take(5)
    pages.give_back([p for p in b if p < 4])
    keep = [p for p in range(6) if pages.holders(p)]
    moves = pages.compact()
    assert [m[0] for m in moves] == [p for p in keep if p >= len(keep)] and all(pages.holders(p) == (p < len(keep)) for p in range(6))
    assert pages.take(1) == [len(keep)]


@pytest.mark.parametrize("moves, what", [
    ([(0, 4)], "outside 0 .. 3"), ([(-1, 2)], "outside"), ([(0, 1, 9)], "rows"), ([(0, 1, -1)], "rows"), ([(0, 1), (2, 1)], "target of two"),
    ([(0, 1), (1, 2)], "source of one"), ([(0, 0)], "source of one"), ([(0,)], "moves are"), ([(0, 1, 2, 3)], "moves are"), ([0, 1], "moves are")])
def test_moves_that_are_refused(moves, what):
    with pytest.raises(ops.KernelError, match=what):
        ops.page_moves(moves, 4, 8)


def test_moves_that_are_taken():
    assert ops.page_moves([], 4, 8).shape == (0, 3)
    assert ops.page_moves([(0, 1), (0, 2)], 4, 8).tolist() == [[0, 1, 8], [0, 2, 8]]
    assert ops.page_moves(np.array([[3, 0, 0]]), 4, 8).tolist() == [[3, 0, 0]]


def test_groups_that_are_refused():
    for groups, n in (([([0, 0], 1)], 2), ([([0], 1), ([0, 1], 2)], 2), ([([2], 1)], 2), ([([-1], 1)], 2), ([([], 1)], 2), ([([0], -1)], 2), ([], 0)):
        with pytest.raises(ops.KernelError):
            ops.SharedPrefix(groups, n, "cpu")
    assert len(ops.SharedPrefix([([0, 1], 0)], 2, "cpu")) == 0


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(ops.KernelError, match="CUDA"):
        from qwenforge_b200.ops import branches
        branches.copy_pages(torch.zeros(1, 4, 1, 1, 8, 4), [(0, 1)])
    share, i32 = ops.SharedPrefix([([0, 1], 1)], 2, "cpu"), torch.zeros(3, dtype=torch.int32)
    site = ops.KvSiteArgs(torch.zeros(2, 2, 1, 64, 32), torch.zeros(2, 2, dtype=torch.int32), 1, 32)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.attention_shared(torch.zeros(2, 32), torch.zeros(2, 32), i32, i32[:2], i32[:2], site, 1, 2, 1.0, share, ops.SharedScratch("cpu"), i32[:1])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.verify_drafts(torch.zeros(2, 8), None, i32[:1], i32[:2], torch.zeros(1), 1.0, 0, torch.zeros(1, dtype=torch.int64), i32[:1], i32[:1], i32[:2].view(1, 2))


def test_when_shared_reading_pays():
    many = ops.SharedPrefix([(range(64), 64)], 64, "cpu")
    assert many.saved_pages == 63 * 64
    assert ops.attention_shared_pays(many, torch.bfloat16, 2, 64) and not ops.attention_shared_pays(many, torch.bfloat16, 2, 300)
    few = ops.SharedPrefix([([0, 2], 64)], 3, "cpu")
    assert not ops.attention_shared_pays(few, torch.bfloat16, 2, 64) and ops.attention_shared_pays(few, torch.float32, 2, 64)
    assert ops.attention_shared_pays(few, torch.bfloat16, 2, 80) and not ops.attention_shared_pays(ops.SharedPrefix([([0, 2], 3)], 3, "cpu"), torch.float32, 2, 64)
    assert not ops.attention_shared_pays(ops.SharedPrefix([(range(2049), 640)], 2049, "cpu"), torch.bfloat16, 2, 64)
