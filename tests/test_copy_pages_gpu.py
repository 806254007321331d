"""`ops.copy_pages` against plain indexing: sizes, types, strides, counts of moves, streams, graphs, refusals."""
import random

import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.cache import PAGE_TOKENS, KvNeed, SequenceCache, StateNeed

pytestmark = pytest.mark.gpu


def random_storage(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-100, 100, shape, device="cuda", generator=g).to(dtype)


def expected(storage, moves):
    """In the order of the moves; a page of four dimensions or more has rows."""
    want = storage.clone()
    for move in moves:
        rows = move[2] if len(move) > 2 else (storage.shape[-2] if storage.dim() >= 4 else 1)
        if storage.dim() >= 4:
            want[:, move[1], ..., :rows, :] = storage[:, move[0], ..., :rows, :]
        elif rows:
            want[:, move[1]] = storage[:, move[0]]
    return want


def draw_moves(pages, n, rows, seed, spread):
    rng = random.Random(seed)
    ids = rng.sample(range(pages), pages)
    targets, sources = ids[:n], ids[n:]
    return [(sources[i % spread % len(sources)], t, rng.randint(0, rows)) for i, t in enumerate(targets)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.int16])
@pytest.mark.parametrize("shape", [(3, 9, 2, 2, 64, 64), (1, 40, 2, 3, 64, 96), (2, 7, 1, 1, 64, 23), (4, 5, 2, 1, 64, 1), (2, 6, 5, 3), (2, 2, 7), (5, 8), (1, 3, 1, 1, 1, 8)])
def test_rows_of_pages(shape, dtype):
    storage = random_storage(shape, dtype)
    rows = shape[-2] if len(shape) >= 4 else 1
    for seed, spread in ((0, 1), (1, 1000)):   # one source for all, and a source each
        moves = draw_moves(shape[1], max(1, shape[1] // 2), rows, seed, spread)
        want = expected(storage, moves)
        ops.copy_pages(storage, moves)
        assert torch.equal(storage, want)


@pytest.mark.parametrize("n", [0, 1, 64, 65, 1024, 1025, 2100])
def test_counts_of_moves(n):
    storage = random_storage((2, 2 * n + 3, 1, 1, 4, 8), torch.bfloat16)
    moves = draw_moves(2 * n + 3, n, 4, n, 10 ** 6)
    want = expected(storage, moves)
    before = ops.kernels.launches
    ops.copy_pages(storage, moves)
    assert torch.equal(storage, want) and ops.kernels.launches - before == -(-n // 1024)


def test_pages_at_any_distance():
    base = random_storage((3, 20, 2, 2, 8, 16), torch.bfloat16)
    for view in (lambda t: t[1:], lambda t: t[:, 1:], lambda t: t[::2, ::3], lambda t: t.transpose(0, 1), lambda t: t[:, :, 1:2], lambda t: t[:, 3:4]):
        storage, other = base.clone(), base.clone()
        moves = [(0, 1, 3)] if view(storage).shape[1] > 1 else []
        if view(storage).shape[1] > 2:
            moves.append((0, 2, 8))
        view(other).copy_(expected(view(other), moves))
        ops.copy_pages(view(storage), moves)
        assert torch.equal(storage, other)
    odd = random_storage((1 + 4 * 6 * 10,), torch.bfloat16)[1:].view(1, 4, 1, 1, 6, 10)   # begins between 4-byte words
    want = expected(odd, [(3, 0, 5)])
    ops.copy_pages(odd, [(3, 0, 5)])
    assert torch.equal(odd, want)


def test_refusals():
    storage = random_storage((2, 6, 2, 2, 8, 16), torch.bfloat16)
    before = storage.clone()
    for bad in ([(0, 6)], [(0, 1, 9)], [(0, 1), (2, 1)], [(0, 1), (1, 2)]):
        with pytest.raises(ops.KernelError):
            ops.copy_pages(storage, bad)
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.copy_pages(storage.transpose(-1, -2), [(0, 1)])
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.copy_pages(storage[..., :8], [(0, 1)])
    with pytest.raises(ops.KernelError, match="overlap"):
        ops.copy_pages(storage[:, :1].expand(2, 6, 2, 2, 8, 16), [(0, 1)])
    with pytest.raises(ops.KernelError, match="entries and pages"):
        ops.copy_pages(storage.view(-1), [(0, 1)])
    assert torch.equal(storage, before)
    ops.copy_pages(storage[:0], [(0, 1)])
    ops.copy_pages(storage, [(0, 1, 0)])
    assert torch.equal(storage, before)


def test_on_another_stream_and_in_a_graph():
    storage = random_storage((4, 30, 2, 2, 64, 64), torch.bfloat16)
    moves = draw_moves(30, 12, 64, 5, 3)
    want = expected(storage, moves)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.copy_pages(storage, moves)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(storage, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(storage, moves)
    storage.copy_(random_storage(storage.shape, storage.dtype, 9))
    want = expected(storage, moves)
    graph.replay()
    assert torch.equal(storage, want)


def test_a_cache_on_the_gpu():
    needs = [KvNeed(2, 8), KvNeed(2, 8), KvNeed(1, 8, window=70), StateNeed((5,))]
    cache = SequenceCache(needs, 30 * PAGE_TOKENS, 5, 10 * PAGE_TOKENS, torch.bfloat16, "cuda")
    slot = cache.open()
    cache.reserve([(slot, 150)])
    for g in cache.kv_groups:
        g.storage.copy_(random_storage(g.storage.shape, torch.bfloat16, 1))
    cache.state_groups[0].storage[:, slot] = 7.0
    cache.advance(slot, 150)
    forks = cache.fork(slot, 3)
    cache.flush()

    def rows(g, s, n):
        first = g.first_needed(n)
        pages = g.table[s].long()
        at = torch.arange(first, n, device="cuda")
        return g.storage[:, pages[at // PAGE_TOKENS], :, :, at % PAGE_TOKENS]
    for g in cache.kv_groups:
        for f in forks:
            assert torch.equal(rows(g, f, 150), rows(g, slot, 150)) and int(g.table[f, 2]) != int(g.table[slot, 2])
            assert g.need.window or torch.equal(g.table[f, :2], g.table[slot, :2])
    assert (cache.state_groups[0].storage[:, forks] == 7.0).all()
    kept = [rows(g, forks[1], 150).clone() for g in cache.kv_groups]
    cache.close(slot)
    cache.close(forks[0])
    assert cache.compact() > 0
    assert all(torch.equal(rows(g, forks[1], 150), k) for g, k in zip(cache.kv_groups, kept))
    assert all(int(g.table.max()) < used for g, used in zip(cache.kv_groups, cache.pages_used()))
