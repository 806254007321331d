"""A cache's pages moved by the kernel: a sequence rewound into a page that others hold too, and compaction where something has to move."""
import pytest
import torch

from tests.helpers import SMALL_64, assert_logits_close, random_tokens
from tests.test_branches_engine_gpu import always_shared, model_of  # noqa: F401  (the fixture: shared reading whatever the size)

pytestmark = pytest.mark.gpu


def alone(model, *steps):
    """The last logits of a sequence of its own."""
    cache = model.new_cache(512, 1)
    slot = cache.open()
    for tokens in steps:
        logits = model.step(cache, [(slot, tokens)])
    return logits[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_branch_rewound_into_a_shared_page(dtype):
    model, _ = model_of(SMALL_64, dtype)
    cache = model.new_cache(2048, 4)
    slot, prompt, tail = cache.open(), random_tokens(1000, 150, 1), random_tokens(1000, 70, 2)
    model.step(cache, [(slot, prompt)])
    a, b = cache.fork(slot, 2)
    old = [group._held[a][1] for group in cache.kv_groups]
    assert all(group.pages.holders(page) == 3 for group, page in zip(cache.kv_groups, old))
    cache.rewind(a, 70)   # six rows of the second page, which all three hold
    for group, page in zip(cache.kv_groups, old):
        assert group._held[a][1] != page and group.pages.holders(group._held[a][1]) == 1 and group.pages.holders(page) == 2
        assert torch.equal(group.storage[:, group._held[a][1], :, :, :6], group.storage[:, page, :, :, :6])
    logits = model.step(cache, [(a, tail)])
    assert_logits_close(logits[0], alone(model, prompt[:70], tail), dtype)
    logits = model.step(cache, [(b, [3]), (a, [4]), (slot, [3])])
    want = alone(model, prompt, [3])
    assert_logits_close(logits[0], want, dtype)
    assert_logits_close(logits[2], want, dtype)
    assert_logits_close(logits[1], alone(model, prompt[:70], tail, [4]), dtype)
    model.raise_on_kernel_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compaction_behind_a_closed_sequence(dtype):
    model, _ = model_of(SMALL_64, dtype)
    cache = model.new_cache(2048, 6)
    prompts = [random_tokens(1000, n, n) for n in (90, 260, 200)]
    slots = [cache.open() for _ in prompts]
    model.step(cache, list(zip(slots, prompts)))
    fork = cache.fork(slots[2])[0]
    cache.close(slots[1])
    used = cache.pages_used()
    assert any(max(max(group._held[s].values()) for s in (slots[0], slots[2], fork)) >= n for group, n in zip(cache.kv_groups, used))
    assert cache.compact() > 0 and cache.pages_used() == used
    for group, n in zip(cache.kv_groups, used):
        assert all(page < n for s in (slots[0], slots[2], fork) for page in group._held[s].values())
    logits = model.step(cache, [(slots[0], [5]), (slots[2], [6]), (fork, [7])])
    for row, prompt, token in zip(logits, (prompts[0], prompts[2], prompts[2]), (5, 6, 7)):
        assert_logits_close(row, alone(model, prompt, [token]), dtype)
    assert cache.compact() == 0
    model.raise_on_kernel_error()
