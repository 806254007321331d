"""The cache that an engine makes for several continuations of a prompt holds all of them, whatever its groups keep."""
import random
from types import SimpleNamespace

import pytest
import torch

from qwenforge_b200 import ops
from qwenforge_b200.cache import BundleNeed, CacheFull, KvNeed, SequenceCache, StateNeed
from qwenforge_b200.engine.engine import StudentEngine
from tests.test_branches_cpu import plain_copy

NEEDS = {
    "full": [KvNeed(1, 4)],
    "window": [KvNeed(1, 4), KvNeed(1, 2, window=70)],
    "pooled": [BundleNeed((("kv", KvNeed(1, 4, window=20, pool=16)), ("blocks", KvNeed(1, 4, every=16)), ("conv", StateNeed((3,)))))],
    "pooled finely": [None, KvNeed(1, 4), BundleNeed((("in", BundleNeed((("blocks", KvNeed(1, 4, every=3)),))),))],
}


def engine_of(needs, most=None):
    engine = StudentEngine.__new__(StudentEngine)
    engine._max_cache_tokens, engine.cache, engine.cuda_graphs, engine.graph_decoder = most, None, False, None
    engine.model = SimpleNamespace(cache_needs=lambda: needs, new_cache=lambda tokens, seqs: SequenceCache(needs, tokens, seqs, 4096, torch.float32, "cpu"))
    return engine


def generate(cache, lengths, budgets, continuations):
    """The cache's side of one batch: prompts, forks behind them, room for every sequence's whole future, tokens one by one to the end."""
    slots = [cache.open() for _ in lengths]
    cache.reserve([(s, n + b - 1) for s, n, b in zip(slots, lengths, budgets)])
    for s, n in zip(slots, lengths):
        cache.advance(s, n)
    for s, n, b in list(zip(slots, lengths, budgets)):
        forks = cache.fork(s, continuations - 1)
        cache.reserve([(f, n + b - 1) for f in forks])
        slots += forks
    for s in slots:
        cache.close(s)


@pytest.mark.parametrize("kind", list(NEEDS))
def test_continuations_fit(kind, monkeypatch):
    monkeypatch.setattr(ops, "copy_pages", plain_copy)
    rng = random.Random(5)
    for _ in range(150):
        n, continuations = rng.randint(1, 3), rng.randint(1, 9)
        lengths = [rng.choice([1, 63, 64, 65, 191, 500, 1007, 1008, 1023, 1024, rng.randint(1, 1500)]) for _ in range(n)]
        budgets = [rng.randint(1, 200) for _ in lengths]
        engine = engine_of(NEEDS[kind])
        engine._ensure_cache(lengths, budgets, n, continuations)
        generate(engine.cache, lengths, budgets, continuations)


def test_what_does_not_fit_is_said_before_anything_runs():
    engine = engine_of(NEEDS["pooled"], most=1024 + 64)
    with pytest.raises(CacheFull, match="max_cache_tokens"):
        engine._ensure_cache([1023], [3], 1, 9)
    engine._ensure_cache([1023], [3], 1, 1)
    assert engine.cache.n_pages == 17
